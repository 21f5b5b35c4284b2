"""A whole tree-drafted step, as a serving program runs it: plan, norms and keys into the cache, attention, acceptance, the
cache rows' order, pages back; eager, captured, on other streams, through torch.ops, from two threads."""
import random
import threading

import pytest
import torch

import tree_step_ref as R
from dense_layer_ref import assert_within

pytestmark = pytest.mark.gpu
V, H, G, D, BS, MB, LAYERS = 499, 16, 2, 64, 16, 20, 2


def next_token(token, position):
    """The model: what follows a token at a position."""
    return (token * 31 + position * 7 + 3) % V


class Server:
    """Sequences that decode over one pool of pages; every layer attends with vectors of (token, layer)."""

    def __init__(self, dsa, dev, B, T, seed, ops=False):
        self.dsa, self.dev, self.B, self.T, self.ops = dsa, dev, B, T, dsa.load_torch_ops() if ops else None
        g = torch.Generator().manual_seed(seed)
        make = lambda n: torch.randn((LAYERS, V, n, D), generator=g).to(torch.bfloat16).to(dev)
        self.eq, self.ek, self.ev = make(H), make(G), make(G)
        ang = torch.arange(MB * BS, dtype=torch.float64).view(-1, 1) * 10000.0 ** (-torch.arange(0, D, 2) / D)
        self.cos, self.sin = ang.cos().float().to(dev), ang.sin().float().to(dev)
        pages = B * MB
        self.kc = [torch.zeros(pages, BS, G, D, dtype=torch.bfloat16, device=dev) for _ in range(LAYERS)]
        self.vc = [torch.zeros_like(c) for c in self.kc]
        i32 = lambda *n: torch.full(n, -1, dtype=torch.int32, device=dev)
        self.table = i32(B, MB)
        self.free = torch.randperm(pages, generator=g).to(torch.int32).to(dev)
        self.count = torch.tensor([pages], dtype=torch.int32, device=dev)
        self.ctx = torch.zeros(B, dtype=torch.int32, device=dev)
        # A step's inputs.
        self.new, self.tokens, self.parents = i32(B), i32(T), i32(T)

    def step(self):
        d, o = self.dsa, self.ops
        cat = lambda x, layer: x[layer][self.tokens.clamp(min=0).long()]
        if o:
            cu, kv, pos, slots, missing, mask = o.paged_plan(self.new, self.ctx, self.table, self.free, self.count, BS, self.T,
                                                             self.parents, 64)
        else:
            cu, kv, pos, slots, missing, mask = d.paged_plan(self.new, self.ctx, self.table, self.free, self.count, BS, self.T,
                                                             parents=self.parents, max_nodes=64)
        outs = []
        for i in range(LAYERS):
            q, k, v = cat(self.eq, i), cat(self.ek, i), cat(self.ev, i)
            if o:
                q = o.qk_norm_rope_paged(q, k, v, None, None, pos, self.cos, self.sin, self.kc[i], self.vc[i], slots)
                outs += [q, *o.paged_tree_fwd(q, self.kc[i], self.vc[i], self.table, mask, kv, D ** -0.5, cu)]
            else:
                q = d.qk_norm_rope_paged(q, k, v, None, None, pos, self.cos, self.sin, self.kc[i], self.vc[i], slots)
                outs += [q, *d.paged_tree_fwd(q, self.kc[i], self.vc[i], self.table, mask, actual_seq_lengths_query=cu,
                                              actual_seq_lengths_kv=kv)]
        want = next_token(self.tokens.long(), pos.long()) % V
        scores = torch.zeros(self.T, V, dtype=torch.bfloat16, device=self.dev)
        scores.scatter_(1, want.view(-1, 1), 1.0)
        if o:
            accepted, path, chosen = o.tree_accept(scores, self.tokens, self.parents, cu, 64)
            o.paged_commit(self.kc + self.vc, self.table, self.ctx, path, accepted)
        else:
            accepted, path, chosen = d.tree_accept(scores, self.tokens, self.parents, actual_seq_lengths_query=cu, max_path=64)
            d.paged_commit(self.kc + self.vc, self.table, self.ctx, path, accepted)
        keep = self.ctx + accepted
        if o:
            o.paged_free(keep, self.table, self.free, self.count, BS)
        else:
            d.paged_free(keep, self.table, self.free, self.count, BS)
        self.ctx.copy_(keep)
        return (cu, kv, missing, mask, accepted, path, chosen) + tuple(outs)


def draft(rng, last, position, S):
    """A tree of S nodes behind the last token, some of whose branches the model agrees with."""
    par, tok, depth = [-1], [last], [0]
    for i in range(1, S):
        p = rng.randrange(max(0, i - 5), i)
        par.append(p)
        depth.append(depth[p] + 1)
        tok.append(next_token(tok[p], position + depth[p]) if rng.random() < 0.5 else rng.randrange(V))
    return par, tok


def load(srv, rng, texts):
    """The next step's trees into the server's inputs; returns their sizes."""
    sizes, par, tok = [], [], []
    for text in texts:
        at = len(text) - 1  # the last token is not in the cache yet
        S = rng.choice([0, 1, 3, 9, 20]) if at + 21 < MB * BS else 0
        sizes.append(S)
        p, t = draft(rng, text[-1], at, S) if S else ([], [])
        par, tok = par + p, tok + t
    pad = srv.T - len(par)
    for dst, src in ((srv.new, sizes), (srv.parents, par + [-1] * pad), (srv.tokens, tok + [-1] * pad)):
        dst.copy_(torch.tensor(src, dtype=torch.int32))
    return sizes


def follow(texts, sizes, accepted, chosen):
    """The tokens that a step yields; each must be what the model says."""
    for b, text in enumerate(texts):
        n = accepted[b]
        assert n == 0 if sizes[b] == 0 else n >= 1
        for t in chosen[b][:n]:
            assert t == next_token(text[-1], len(text) - 1)
            text.append(t)


def rotated(srv, layer, text):
    """Keys of a text's tokens, normed and rotated, from the operator without a cache."""
    t = torch.tensor(text, device=srv.dev)
    pos = torch.arange(len(text), device=srv.dev, dtype=torch.int32)
    return srv.dsa.qk_norm_rope(srv.eq[layer][t], srv.ek[layer][t], None, None, pos, srv.cos, srv.sin)[1]


def check_caches(srv, texts):
    """Every context's rows are those of its tokens, one after the other, as a program without trees would have left them."""
    table = srv.table.cpu()
    for b, text in enumerate(texts):
        n = len(text) - 1
        if n == 0:
            continue
        j = torch.arange(n)
        rows = (table[b].long()[j // BS] * BS + j % BS).to(srv.dev)
        t = torch.tensor(text[:-1], device=srv.dev)
        for i in range(LAYERS):
            assert torch.equal(srv.kc[i].view(-1, G, D)[rows], rotated(srv, i, text[:-1])), (b, i)
            assert torch.equal(srv.vc[i].view(-1, G, D)[rows], srv.ev[i][t]), (b, i)
    held = [-(-(len(t) - 1) // BS) for t in texts]
    assert [int((r >= 0).sum()) for r in table] == held
    pages = table[table >= 0].tolist() + srv.free[:int(srv.count)].tolist()
    assert sorted(pages) == list(range(srv.B * MB))


@pytest.mark.parametrize("ops", [False, True])
def test_decoding_yields_what_the_model_says(dsa, dev, ops):
    rng = random.Random(5)
    B, T = 6, 130
    srv = Server(dsa, dev, B, T, 1, ops)
    texts = [[rng.randrange(V)] for _ in range(B)]
    for step in range(25):
        sizes = load(srv, rng, texts)
        ctx = srv.ctx.tolist()
        before = [[c.cpu().clone() for c in srv.kc], [c.cpu().clone() for c in srv.vc]]
        r = srv.step()
        cu, kv, missing, mask, accepted, path, chosen = r[:7]
        assert not missing.any()
        follow(texts, sizes, accepted.tolist(), chosen.tolist())
        if step % 8 == 3:  # the attention of the whole trees, from the caches as they stood ahead of the commit
            parents = srv.parents.tolist()
            starts = [0] + cu.tolist()[:-1]
            for i in range(LAYERS):
                q, out, lse = r[7 + 3 * i:10 + 3 * i]
                kcs, vcs = before[0][i], before[1][i]
                tab = torch.full((B, MB), -1)
                # Rebuild the trees' rows: the keys by an operator call without a cache, in a pool of their own.
                pool_k = torch.zeros(B * MB, BS, G, D, dtype=torch.bfloat16)
                pool_v = torch.zeros_like(pool_k)
                for b in range(B):
                    tab[b] = torch.arange(b * MB, (b + 1) * MB)
                    S, t0 = sizes[b], starts[b]
                    if S == 0:
                        continue
                    tok = srv.tokens[t0:t0 + S].long()
                    chains = R.ancestors(parents[t0:t0 + S])
                    pos = torch.tensor([ctx[b] + len(x) - 1 for x in chains], dtype=torch.int32, device=dev)
                    k = dsa.qk_norm_rope(srv.eq[i][tok], srv.ek[i][tok], None, None, pos, srv.cos, srv.sin)[1].cpu()
                    n = ctx[b]
                    text = texts[b][:n]
                    if n:
                        pool_k.view(-1, G, D)[b * MB * BS:b * MB * BS + n] = rotated(srv, i, text).cpu()
                        pool_v.view(-1, G, D)[b * MB * BS:b * MB * BS + n] = srv.ev[i][torch.tensor(text, device=dev)].cpu()
                    pool_k.view(-1, G, D)[b * MB * BS + n:b * MB * BS + n + S] = k
                    pool_v.view(-1, G, D)[b * MB * BS + n:b * MB * BS + n + S] = srv.ev[i][tok].cpu()
                o, ot, l, lt = R.attention(q.cpu(), pool_k, pool_v, tab, mask.cpu(), starts, sizes, sizes, kv.tolist(), D ** -0.5)
                n = sum(sizes)
                assert_within(out[:n], o[:n], ot[:n], "out")
                assert_within(lse[:n], l[:n], lt[:n], "lse")
    check_caches(srv, texts)
    assert min(len(t) for t in texts) > 15


def test_captured_steps_replay_with_new_lengths(dsa, dev):
    """One graph, replayed with other trees, contexts and pages each time; eager work between the replays."""
    rng = random.Random(9)
    B, T = 5, 110
    eager, graphed = Server(dsa, dev, B, T, 2), Server(dsa, dev, B, T, 2)
    texts = [[rng.randrange(V)] for _ in range(B)]
    warm = torch.cuda.Stream(dev)
    warm.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(warm):
        graphed.new.zero_()
        graphed.step()
    torch.cuda.current_stream(dev).wait_stream(warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = graphed.step()
    for step in range(12):
        state = rng.getstate()
        sizes = load(eager, rng, texts)
        rng.setstate(state)
        load(graphed, rng, texts)
        want = eager.step()
        graph.replay()
        torch.cuda.synchronize()
        n = sum(sizes)
        for a, b in zip(outs[:7], want[:7]):
            assert torch.equal(a, b)
        for a, b in zip(outs[7:], want[7:]):
            assert torch.equal(a[:n], b[:n])
        for a, b in zip(graphed.kc + graphed.vc + [graphed.table, graphed.free, graphed.count, graphed.ctx],
                        eager.kc + eager.vc + [eager.table, eager.free, eager.count, eager.ctx]):
            assert torch.equal(a, b)
        follow(texts, sizes, want[4].tolist(), want[6].tolist())
    check_caches(graphed, texts)


def test_streams_and_threads(dsa, dev):
    """Two servers step at once, from a thread and on a stream each."""
    servers = [Server(dsa, dev, 4, 90, 3 + i) for i in range(2)]
    texts = [[[7 * b + i] for b in range(4)] for i in range(2)]
    torch.cuda.synchronize()
    failures = []

    def work(i):
        try:
            rng, stream = random.Random(i), torch.cuda.Stream(dev)
            with torch.cuda.stream(stream):
                for _ in range(10):
                    sizes = load(servers[i], rng, texts[i])
                    r = servers[i].step()
                    follow(texts[i], sizes, r[4].tolist(), r[6].tolist())
                check_caches(servers[i], texts[i])
            stream.synchronize()
        except BaseException as e:  # noqa: BLE001 - reported below
            failures.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, failures
