"""The dense layer's operators in a run, as a serving step makes them: eager, streams, captured graphs."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H, G, D, HID, BS = 8, 2, 64, 320, 16


class Layer:
    def __init__(self, dsa, dev, seed=0):
        g = torch.Generator().manual_seed(seed)
        n = (H + 2 * G) * D
        self.dsa = dsa
        self.wqkv, self.sqkv = dsa.act_quant((torch.randn(n, HID, generator=g) / HID ** 0.5).to(dev))
        self.wo, self.so = dsa.act_quant((torch.randn(HID, H * D, generator=g) / (H * D) ** 0.5).to(dev))
        self.qw, self.kw = ((1 + torch.randn(D, generator=g) / 10).bfloat16().to(dev) for _ in range(2))
        ang = torch.arange(512).double().view(-1, 1) * 10000.0 ** (-torch.arange(0, D, 2).double() / D)
        self.cos, self.sin = ang.cos().float().to(dev), ang.sin().float().to(dev)
        self.kc = torch.zeros(64, BS, G, D, dtype=torch.bfloat16, device=dev)
        self.vc = torch.zeros_like(self.kc)

    def __call__(self, x, pos, slots, table, cu, kvl):
        dsa = self.dsa
        xq, xs = dsa.act_quant(x)
        qkv = dsa.quant_matmul(xq, self.wqkv, xs, self.sqkv)
        T = x.shape[0]
        q, k, v = (t.view(T, -1, D) for t in qkv.split([H * D, G * D, G * D], dim=1))
        qo = dsa.qk_norm_rope_paged(q, k, v, self.qw, self.kw, pos, self.cos, self.sin, self.kc, self.vc, slots)
        out, _ = dsa.paged_gqa_fwd(qo, self.kc, self.vc, table, actual_seq_lengths_query=cu, actual_seq_lengths_kv=kvl)
        oq, os = dsa.act_quant(out.view(T, H * D))
        return dsa.quant_matmul(oq, self.wo, os, self.so)


def _batch(dev, seqs, tables):
    """Positions, slots, table, prefix sums and lengths of seqs [(new, keys)]."""
    pos = torch.cat([torch.arange(n - s, n) for s, n in seqs])
    slots = torch.cat([torch.tensor([int(tables[b][j // BS]) * BS + j % BS for j in range(n - s, n)])
                       for b, (s, n) in enumerate(seqs)])
    i32 = lambda t: t.to(torch.int32).to(dev)
    return (i32(pos), i32(slots), i32(tables), i32(torch.tensor([s for s, _ in seqs]).cumsum(0)),
            i32(torch.tensor([n for _, n in seqs])))


def _tables(n, seed=1):
    return torch.randperm(64, generator=torch.Generator().manual_seed(seed))[:n * 8].view(n, 8)


def _tokens(dev, n, seed):
    return torch.randn(n, HID, generator=torch.Generator().manual_seed(seed)).bfloat16().to(dev)


def test_a_prompt_in_chunks_equals_a_prompt_at_once(dsa, dev):
    """The chunks' rows see the same keys: outputs agree to the order of the softmax's sums."""
    a, b = Layer(dsa, dev), Layer(dsa, dev)
    x = _tokens(dev, 100, 1)
    tab = _tables(1)
    whole = a(x, *_batch(dev, [(100, 100)], tab))
    parts, at = [], 0
    for n in (37, 1, 1, 40, 21):
        parts.append(b(x[at:at + n], *_batch(dev, [(n, at + n)], tab)))
        at += n
    got = torch.cat(parts)
    # The cache rows come from exact int32 sums and one order of operations per head: the same bits.
    assert torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)
    # Outputs: rounding orders differ in the attention (two half steps of bf16), then the int8 step of the second
    # quantiser and bf16 again; a step of int8 is 1/127 of a row's largest.
    scale = whole.float().abs().amax()
    assert (got.float() - whole.float()).abs().max() <= scale * (2 ** -6 + 2 / 127)


def test_batch_equals_single_sequences(dsa, dev):
    """A mixed batch gives what its sequences give alone, in the caches bit for bit."""
    tab = _tables(3)
    seqs = [(1, 65), (30, 90), (1, 128)]
    a, b = Layer(dsa, dev), Layer(dsa, dev)
    for layer in (a, b):
        layer.kc.copy_(torch.randn(layer.kc.shape, generator=torch.Generator().manual_seed(3)))
        layer.vc.copy_(torch.randn(layer.vc.shape, generator=torch.Generator().manual_seed(4)))
    x = _tokens(dev, 32, 2)
    whole = a(x, *_batch(dev, seqs, tab))
    at, parts = 0, []
    for i, (s, n) in enumerate(seqs):
        parts.append(b(x[at:at + s], *_batch(dev, [(s, n)], tab[i:i + 1])))
        at += s
    assert torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)
    scale = whole.float().abs().amax()
    assert (torch.cat(parts).float() - whole.float()).abs().max() <= scale * (2 ** -6 + 2 / 127)


def test_captured_step_replays(dsa, dev):
    """A decode step in a HIP graph, replayed on new inputs between eager work, against the eager step."""
    tab = _tables(4)
    seqs = [(1, 20), (1, 128), (1, 1), (1, 77)]
    a, b = Layer(dsa, dev), Layer(dsa, dev)
    x = _tokens(dev, 4, 0)
    args = _batch(dev, seqs, tab)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        a(x, *args)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = a(x, *args)
    for i in range(4):
        new = _tokens(dev, 4, 10 + i)
        x.copy_(new)
        nxt = _batch(dev, [(1, 1 + (n + 13 * i) % 128) for _, n in seqs], tab)
        for old, val in zip(args, nxt):
            old.copy_(val)
        a.kc.copy_(b.kc)
        a.vc.copy_(b.vc)
        graph.replay()
        torch.cuda.synchronize()
        want = b(new, *nxt)
        assert torch.equal(out, want)
        assert torch.equal(a.kc, b.kc) and torch.equal(a.vc, b.vc)
        torch.empty(1 << 20, device=dev).fill_(float("nan"))


def test_two_streams_at_once(dsa, dev):
    """Two layers on two streams, calls interleaved: each gives what it gives alone."""
    tab = _tables(2)
    seqs = [(40, 100), (1, 128)]
    want, layers = [], []
    for i in range(2):
        lone = Layer(dsa, dev, i)
        want.append(lone(_tokens(dev, 41, i), *_batch(dev, seqs, tab)))
        layers.append((Layer(dsa, dev, i), _tokens(dev, 41, i), _batch(dev, seqs, tab)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = [[], []]
    for _ in range(5):
        for i, (layer, x, args) in enumerate(layers):
            with torch.cuda.stream(streams[i]):
                outs[i].append(layer(x, *args))
    torch.cuda.synchronize()
    for i in range(2):
        for o in outs[i]:
            assert torch.equal(o, want[i])
