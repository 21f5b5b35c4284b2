"""Corners of the dense layer's operators on the GPU: wide integers, sinks, padding, other routes, threads, devices."""
import math
import threading

import pytest
import torch

import dense_layer_ref as ref
from test_paged_gqa_gpu import _check, _run, _setup, _want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("chunk", [1, 90])
def test_wide_table_entries_do_not_wrap(dsa, dev, chunk):
    """64-bit page numbers past 32 bits lie outside the pool; they do not come back as pages of it."""
    seqs = [(chunk, 150), (1, 70)]
    q, kc, vc, table = _setup(seqs, 8, 2, 64, 16, torch.bfloat16, seed=21)
    hidden, wide = table.clone(), table.long()
    for at, page in [((0, 1), 2**32), ((0, 3), -2**63), ((0, 4), 2**63 - 1), ((1, 0), 2**32 + int(table[1, 0])),
                     ((1, 2), 2**31), ((0, 6), -2**32 + 1)]:
        hidden[at], wide[at] = -1, page
    want = _run(dsa, dev, seqs, q, kc, vc, hidden)
    _check(want, _want(seqs, q, kc, vc, hidden))
    got = _run(dsa, dev, seqs, q, kc, vc, wide)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    got = dsa.load_torch_ops().paged_gqa_fwd(q.to(dev), kc.to(dev), vc.to(dev), wide.to(dev), i32([150, 70]), 64 ** -0.5,
                                             i32([chunk, chunk + 1]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("where", ["device", "host", "list"])
def test_wide_lengths_do_not_wrap(dsa, dev, where):
    """64-bit lengths past 32 bits are cut to what the table and q hold, as smaller ones past it are."""
    seqs = [(4, 64)]
    q, kc, vc, table = (t.to(dev) for t in _setup(seqs, 4, 1, 64, 16, torch.bfloat16, seed=22))
    whole = _run(dsa, dev, seqs, q, kc, vc, table)
    place = {"device": lambda x: torch.tensor(x, device=dev), "host": torch.tensor, "list": list}[where]
    ops = dsa.load_torch_ops()
    for cu, kl in [([2**32 + 2], [2**32 + 5]), ([2**63 - 1], [2**31])]:
        got = dsa.paged_gqa_fwd(q, kc, vc, table, actual_seq_lengths_query=place(cu), actual_seq_lengths_kv=place(kl))
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])
        if where == "device":
            got = ops.paged_gqa_fwd(q, kc, vc, table, place(kl), 64 ** -0.5, place(cu))
            assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])
    low = place([-2**63 + 5])
    out, lse = dsa.paged_gqa_fwd(q, kc, vc, table, actual_seq_lengths_query=low, actual_seq_lengths_kv=low)
    assert (out == 0).all() and torch.isinf(lse).all()


@pytest.mark.parametrize("dtype,big", [(torch.uint32, 2**32 - 3), (torch.uint64, 2**63 + 5), (torch.uint16, 2**16 - 1),
                                       (torch.uint8, 255)])
def test_unsigned_lengths(dsa, dev, dtype, big):
    """Lengths of unsigned types are cut as signed ones are."""
    seqs = [(4, 64)]
    q, kc, vc, table = (t.to(dev) for t in _setup(seqs, 4, 1, 64, 16, torch.bfloat16, seed=23))
    whole = _run(dsa, dev, seqs, q, kc, vc, table)
    n = torch.tensor([big], dtype=dtype)
    for place in (n, n.to(dev)):
        got = dsa.paged_gqa_fwd(q, kc, vc, table, actual_seq_lengths_query=place, actual_seq_lengths_kv=place)
        assert torch.equal(got[0], whole[0]) and torch.equal(got[1], whole[1])


# Batches in which whole sequences, single rows of a tile, or rows of a tile that several workgroups share see no key.
NOTHING = {"decode": [(1, 0), (1, 40), (1, 0)], "tokens before the keys": [(40, 20), (1, 5)], "shared": [(300, 280)],
           "none": [(90, 0)]}


@pytest.mark.parametrize("name", list(NOTHING))
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (16, 1, 128)])
def test_rows_that_see_nothing_keep_their_sink(dsa, dev, name, H, G, D):
    """lse is the sink however small or large its exponential is."""
    seqs = NOTHING[name]
    args = _setup(seqs, H, G, D, 16, torch.bfloat16, seed=24)
    sinks = torch.tensor([-200.0, -80.0, -1e4, torch.finfo(torch.float32).min, 0.0, 3.0, 100.0, 500.0]).repeat(H // 8)
    out, tol, lse, ltol = _want(seqs, *args, sinks=sinks)
    # Beside a large sink a row's keys have the factor 2^(m - sink) in fp32, which is 0 below 2^-126: the sum of at most n
    # weights of at most 1 times v, over a denominator of at least 1 (the sink's own), is then off by 2^-126 n |v|.
    tol = tol + 2.0 ** -126 * max(n for _, n in seqs) * args[2].double().abs().max()
    _check(_run(dsa, dev, seqs, *args, sinks=sinks), (out, tol, lse, ltol))


@pytest.mark.parametrize("name", list(NOTHING))
@pytest.mark.parametrize("H,G,D", [(8, 2, 64), (16, 1, 128)])
def test_sinks_that_are_not_finite(dsa, dev, name, H, G, D):
    """A sink of +infinity takes all the weight: out = 0, lse = +infinity.  One of -infinity takes none; NaN stays in
    its head's sums."""
    seqs = NOTHING[name]
    args = _setup(seqs, H, G, D, 16, torch.bfloat16, seed=25)
    free = _run(dsa, dev, seqs, *args)
    sinks = torch.full((H,), -math.inf)
    sinks[1], sinks[3], sinks[4] = math.inf, math.nan, 3e38
    out, lse = _run(dsa, dev, seqs, *args, sinks=sinks)
    assert (out[:, 1] == 0).all() and (lse[:, 1] == math.inf).all()
    assert torch.isnan(lse[:, 3]).all()
    assert (out[:, 4] == 0).all() and (lse[:, 4] == sinks[4].item()).all()
    rest = [h for h in range(H) if h not in (1, 3, 4)]
    assert torch.equal(out[:, rest], free[0][:, rest]) and torch.equal(lse[:, rest], free[1][:, rest])


def _us(f, n=5):
    f()
    times = []
    for _ in range(5):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(n):
            f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) / n * 1e3)
    return sorted(times)[2]


@pytest.mark.parametrize("S,lens,keys", [(300, [1, 0, 120], [2000, 900, 500]), (17, [1, 3, 17], [777, 3, 400]),
                                         (1100, [40, 1, 700], [40, 3000, 800])])
@pytest.mark.parametrize("win", [None, 50])
def test_padding_over_long_contexts(dsa, dev, S, lens, keys, win):
    """Tiles that hold padding only, beside sequences of many keys, with sinks."""
    B, H, G, D, bs = 3, 8, 2, 64, 16
    q, kc, vc, table = _setup([(S, n) for n in keys], H, G, D, bs, torch.bfloat16, seed=S)
    sinks = torch.randn(H, generator=torch.Generator().manual_seed(S))
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    out, lse = dsa.paged_gqa_fwd(q.view(B, S, H, D).to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                 actual_seq_lengths_query=i32(lens), actual_seq_lengths_kv=i32(keys), win_left=win,
                                 sinks=sinks.to(dev))
    want = ref.attention(q, kc, vc, table, [b * S for b in range(B)], [S] * B, lens, keys, D ** -0.5,
                         win=-1 if win is None else win, sinks=sinks)
    _check((out.view(B * S, H, D), lse.view(B * S, H)), want)
    for b in range(B):
        assert (out[b, lens[b]:] == 0).all()


@pytest.mark.parametrize("B,S", [(2, 1024), (8, 2048)])
def test_padding_reads_no_keys(dsa, dev, B, S):
    """A batch padded to S rows a sequence, one of them real, takes a fraction of the full batch's time (a share of
    the work of at most 1/32; a third allows for the launches and for workgroups that walk their keys alone)."""
    H, G, D, bs, n = 32, 2, 128, 64, 16384
    q = torch.randn(B, S, H, D, device=dev).bfloat16()
    kc, vc = (torch.randn(B * n // bs, bs, G, D, device=dev).bfloat16() for _ in range(2))
    table = torch.arange(B * n // bs, dtype=torch.int32, device=dev).view(B, -1)
    i32 = lambda x: torch.tensor([x] * B, dtype=torch.int32, device=dev)
    kl = i32(n)
    time = lambda ql: _us(lambda: dsa.paged_gqa_fwd(q, kc, vc, table, actual_seq_lengths_query=ql,
                                                    actual_seq_lengths_kv=kl))
    one, full = time(i32(1)), time(i32(S))
    assert one < full / 3, f"one token of {S}: {one:.0f} us, all: {full:.0f} us"


@pytest.mark.parametrize("route", ["native", "64-bit", "registered"])
@pytest.mark.parametrize("interleaved", [False, True])
def test_each_route_writes_the_cache_rows(dsa, dev, route, interleaved):
    """From caches of its own, each route writes every slot's key and value row and no other."""
    T, H, G, D, R, bs, nb = 21, 8, 2, 64, 32, 16, 5
    g = torch.Generator().manual_seed(31)
    q, k, v = (torch.randn(T, n, D, generator=g).bfloat16() for n in (H, G, G))
    qw, kw = torch.randn(D, generator=g), torch.randn(D, generator=g)
    ang = torch.arange(100).double().view(-1, 1) * 10000.0 ** (-torch.arange(0, R, 2).double() / R)
    cos, sin = ang.cos().float(), ang.sin().float()
    pos = torch.randint(0, 100, (T,), generator=g).to(torch.int32)
    slots = torch.randperm(nb * bs, generator=g)[:T].to(torch.int32)
    pos[1], slots[4], slots[5] = -1, -1, nb * bs
    kc0, vc0 = torch.randn(nb, bs, G, D, generator=g).bfloat16(), torch.randn(nb, bs, G, D, generator=g).bfloat16()
    kc, vc = kc0.clone().to(dev), vc0.clone().to(dev)
    a = [t.to(dev) for t in (q, k, v, qw, kw)]
    p, c, s, sl = (t.to(dev) for t in (pos, cos, sin, slots))
    if route == "native":
        qo = dsa.qk_norm_rope_paged(*a, p, c, s, kc, vc, sl, interleaved=interleaved)
    elif route == "64-bit":
        qo = dsa.qk_norm_rope_paged(*a, p.long(), c, s, kc, vc, sl.long(), interleaved=interleaved)
    else:
        qo = dsa.load_torch_ops().qk_norm_rope_paged(*a, p, c, s, kc, vc, sl, 1e-6, interleaved)
    u = ref.half_step(torch.bfloat16)
    within = lambda got, want, tol, what: ref.assert_within(got, want, tol + u * (want.abs() + tol), what)
    within(qo, *ref.norm_rope(q, qw, pos, cos, sin, interleaved=interleaved), "queries")
    wk, tol = ref.norm_rope(k, kw, pos, cos, sin, interleaved=interleaved)
    live = [t for t in range(T) if t not in (1, 4, 5)]
    at = slots[live].long()
    got_k, got_v = kc.cpu().view(-1, G, D), vc.cpu().view(-1, G, D)
    assert (got_k[at] != kc0.view(-1, G, D)[at]).flatten(1).any(1).all()
    within(got_k[at], wk[live], tol[live], "keys")
    assert torch.equal(got_v[at], v[live])
    rest = torch.ones(nb * bs, dtype=torch.bool)
    rest[at] = False
    assert torch.equal(got_k[rest], kc0.view(-1, G, D)[rest]) and torch.equal(got_v[rest], vc0.view(-1, G, D)[rest])


def test_caches_without_rows(dsa, dev):
    """Every slot lies outside a cache of no blocks: nothing is written, the queries come back."""
    g = torch.Generator().manual_seed(32)
    q = torch.randn(3, 2, 16, generator=g).bfloat16().to(dev)
    pos = torch.arange(3, dtype=torch.int32, device=dev)
    cos, sin = torch.rand(8, 8, generator=g).to(dev), torch.rand(8, 8, generator=g).to(dev)
    want, _ = dsa.qk_norm_rope(q, q, None, None, pos, cos, sin)
    kc, vc = (torch.empty(0, 16, 2, 16, dtype=torch.bfloat16, device=dev) for _ in range(2))
    for f in (dsa.qk_norm_rope_paged, dsa.load_torch_ops().qk_norm_rope_paged):
        assert torch.equal(f(q, q, q, None, None, pos, cos, sin, kc, vc, pos), want)


def _step(dsa, dev, seed):
    """A projection and an attention call of their own inputs."""
    g = torch.Generator().manual_seed(seed)
    x, w = (torch.randint(-127, 128, s, dtype=torch.int8, generator=g).to(dev) for s in ((40, 260), (300, 260)))
    xs, ws = torch.rand(40, generator=g).to(dev), torch.rand(300, generator=g).to(dev)
    seqs = [(1, 900), (33, 400 + seed), (1, 10)]
    args = [t.to(dev) for t in _setup(seqs, 16, 2, 128, 64, torch.bfloat16, seed=seed)]
    return lambda: (dsa.quant_matmul(x, w, xs, ws), *_run(dsa, dev, seqs, *args))


def test_calls_from_several_threads(dsa, dev):
    """Threads with streams of their own, calls at once: each gives what it gives alone."""
    steps = [_step(dsa, dev, i) for i in range(4)]
    want = [s() for s in steps]
    torch.cuda.synchronize()
    got, errors = [[] for _ in steps], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    got[i].append(steps[i]())
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # pragma: no cover - reported below
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(steps))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for i in range(len(steps)):
        assert len(got[i]) == 10
        for res in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(res, want[i]))


def test_another_device_than_the_current_one(dsa, dev):
    if torch.cuda.device_count() < 2:
        pytest.skip("one device here")
    want = _step(dsa, dev, 1)()
    with torch.cuda.device(0):
        got = _step(dsa, torch.device("cuda:1"), 1)()
    assert all(b.device.index == 1 and torch.equal(a.cpu(), b.cpu()) for a, b in zip(want, got))
