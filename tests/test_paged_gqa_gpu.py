"""Attention over a paged cache on the GPU: 64-bit results over batches, masks, pages, refusals."""
import math

import pytest
import torch

import dense_layer_ref as ref

pytestmark = pytest.mark.gpu


def _setup(seqs, H, G, D, bs, dtype, seed=0, scale=1.0, spare=2):
    """Packed queries and caches of seqs [(new, keys)], pages in random order, `spare` unused ones."""
    g = torch.Generator().manual_seed(seed)
    T = sum(s for s, _ in seqs)
    need = [-(-n // bs) for _, n in seqs]
    nb = sum(need) + spare
    q = (torch.randn(T, H, D, generator=g) * scale).to(dtype)
    kc, vc = torch.randn(nb, bs, G, D, generator=g).to(dtype), torch.randn(nb, bs, G, D, generator=g).to(dtype)
    order = torch.randperm(nb, generator=g).to(torch.int32)
    table = torch.full((len(seqs), max(max(need), 1)), nb - 1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return q, kc, vc, table


def _want(seqs, q, kc, vc, table, causal=True, win=-1, sinks=None, sm_scale=None):
    starts = [sum(s for s, _ in seqs[:b]) for b in range(len(seqs))]
    lens = [s for s, _ in seqs]
    return ref.attention(q, kc, vc, table, starts, lens, lens, [n for _, n in seqs],
                         q.shape[-1] ** -0.5 if sm_scale is None else sm_scale, causal, win, sinks)


def _run(dsa, dev, seqs, q, kc, vc, table, causal=True, win=None, sinks=None, sm_scale=None, **kw):
    cu = torch.tensor([s for s, _ in seqs]).cumsum(0).to(torch.int32)
    kl = torch.tensor([n for _, n in seqs], dtype=torch.int32)
    return dsa.paged_gqa_fwd(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), sm_scale,
                             actual_seq_lengths_query=cu.to(dev), actual_seq_lengths_kv=kl.to(dev), is_causal=causal,
                             win_left=win, sinks=None if sinks is None else sinks.to(dev), **kw)


def _check(got, want):
    out, lse = got
    o, tol, l, ltol = want
    ref.assert_within(lse, l, ltol, "lse")
    ref.assert_within(out, o, tol, "out")


BATCHES = {
    "token": [(1, 1)],
    "token of 33": [(1, 33)],
    "token, long": [(1, 5000)],
    "decode": [(1, 700), (1, 1), (1, 128), (1, 129), (1, 3000), (1, 31)],
    "decode, many": [(1, 1 + 37 * i) for i in range(40)],
    "chunk": [(70, 500)],
    "prompt": [(333, 333)],
    "mixed": [(1, 300), (130, 130), (1, 77), (17, 900), (64, 64), (1, 2049)],
    "none and few": [(0, 100), (3, 3), (0, 0), (5, 2), (1, 0), (2, 64)],
}


@pytest.mark.parametrize("name", list(BATCHES))
@pytest.mark.parametrize("H,G,D,bs,dtype", [(16, 1, 128, 64, torch.bfloat16), (8, 2, 64, 16, torch.float16),
                                            (5, 1, 128, 17, torch.float16), (6, 6, 64, 128, torch.bfloat16),
                                            (40, 2, 128, 7, torch.bfloat16), (64, 1, 64, 64, torch.bfloat16)])
def test_against_64_bits(dsa, dev, name, H, G, D, bs, dtype):
    seqs = BATCHES[name]
    args = _setup(seqs, H, G, D, bs, dtype, seed=len(name))
    _check(_run(dsa, dev, seqs, *args), _want(seqs, *args))


@pytest.mark.parametrize("name", ["token of 33", "decode", "mixed", "prompt", "none and few"])
@pytest.mark.parametrize("win", [0, 1, 31, 100, 10000])
def test_window_and_sinks(dsa, dev, name, win):
    seqs = BATCHES[name]
    args = _setup(seqs, 8, 2, 64, 32, torch.bfloat16, seed=win)
    sinks = torch.randn(8, generator=torch.Generator().manual_seed(win)) * 3
    _check(_run(dsa, dev, seqs, *args, win=win, sinks=sinks), _want(seqs, *args, win=win, sinks=sinks))
    _check(_run(dsa, dev, seqs, *args, win=win), _want(seqs, *args, win=win))


@pytest.mark.parametrize("name", ["decode", "mixed", "chunk"])
@pytest.mark.parametrize("win", [None, 200])
def test_not_causal(dsa, dev, name, win):
    seqs = BATCHES[name]
    args = _setup(seqs, 8, 2, 128, 64, torch.bfloat16, seed=4)
    _check(_run(dsa, dev, seqs, *args, causal=False, win=win), _want(seqs, *args, causal=False, win=-1 if win is None else win))


def test_long_prompt_of_few_heads(dsa, dev):
    """More than a workgroup's share of rows, a length that ends inside every tile."""
    seqs = [(1501, 2777), (1, 40), (600, 600)]
    args = _setup(seqs, 4, 2, 128, 48, torch.bfloat16, seed=8)
    _check(_run(dsa, dev, seqs, *args), _want(seqs, *args))


@pytest.mark.parametrize("H,G", [(32, 1), (8, 8)])
def test_many_rows(dsa, dev, H, G):
    """Enough tiles that each workgroup takes whole ones."""
    seqs = [(1200, 1200), (900, 1000), (1, 5)] + [(40, 64)] * 30
    args = _setup(seqs, H, G, 64, 64, torch.float16, seed=9)
    _check(_run(dsa, dev, seqs, *args), _want(seqs, *args))


@pytest.mark.parametrize("bs", [64, 20])
def test_a_tile_for_each_workgroup(dsa, dev, bs):
    """More tiles of rows than two rounds of workgroups, few sequences: no line to share."""
    seqs = [(1500, 1700), (1201, 1201)]
    args = _setup(seqs, 64, 1, 64, bs, torch.bfloat16, seed=bs)
    _check(_run(dsa, dev, seqs, *args, win=700), _want(seqs, *args, win=700))


def test_thousands_of_sequences(dsa, dev):
    """More slots than the line holds: decode tiles a workgroup each.  All sequences are alike but in their pages."""
    B, n, H, D, bs = 4300, 21, 4, 64, 16
    g = torch.Generator().manual_seed(1)
    q = torch.randn(B, 1, H, D, generator=g).bfloat16()
    kc, vc = torch.randn(2 * B, bs, 1, D, generator=g).bfloat16(), torch.randn(2 * B, bs, 1, D, generator=g).bfloat16()
    table = torch.randperm(2 * B, generator=g).to(torch.int32).view(B, 2)
    kl = torch.full((B,), n, dtype=torch.int32)
    out, lse = dsa.paged_gqa_fwd(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), actual_seq_lengths_kv=kl.to(dev))
    k, v = (c[table.long()].view(B, 2 * bs, D)[:, :n].double() for c in (kc, vc))
    s = torch.matmul(q.view(B, H, D).double(), k.transpose(1, 2)) * D ** -0.5
    w = torch.softmax(s, -1)
    u = ref.half_step(torch.bfloat16)
    # As in ref.attention: the weights' and the output's rounding, scores within (D + 4) half steps of their terms' sum.
    ds = (D + 4) * ref.F32 * torch.matmul(q.view(B, H, D).double().abs(), k.transpose(1, 2).abs()).max() * D ** -0.5
    want = torch.matmul(w, v)
    tol = (u + 2 * ds + (n + 64) * ref.F32 + 4e-7) * torch.matmul(w, v.abs()) + u * want.abs()
    ref.assert_within(out.view(B, H, D), want, tol, "out")
    l = torch.logsumexp(s, -1)
    ref.assert_within(lse.view(B, H), l, ds + (n + 64) * ref.F32 + 1e-6 + 4 * ref.F32 * l.abs(), "lse")


@pytest.mark.parametrize("scale", [8.0, 40.0])
def test_large_scores(dsa, dev, scale):
    """Rows that one key decides, with scores of hundreds either way."""
    seqs = [(1, 400), (50, 300)]
    args = _setup(seqs, 8, 2, 64, 16, torch.bfloat16, seed=3, scale=scale)
    _check(_run(dsa, dev, seqs, *args), _want(seqs, *args))


@pytest.mark.parametrize("seqs", [[(1, 70), (40, 100)], [(1, 1), (300, 333)], [(1, 20)] * 5])
@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_what_lies_behind_the_last_key(dsa, dev, seqs, what):
    """Rows of a page behind a sequence's keys, unused pages and other pools' rows hold anything."""
    q, kc, vc, table = _setup(seqs, 8, 2, 128, 64, torch.bfloat16, seed=6)
    want = _run(dsa, dev, seqs, q, kc, vc, table)
    live = torch.zeros(kc.shape[:2], dtype=torch.bool)
    for b, (_, n) in enumerate(seqs):
        for j in range(n):
            live[int(table[b, j // 64]), j % 64] = True
    kc, vc = kc.clone(), vc.clone()
    kc[~live], vc[~live] = what, what
    got = _run(dsa, dev, seqs, q, kc, vc, table)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("seqs,win", [([(50, 300)], None), ([(1, 300), (3, 77)], 64), ([(200, 200), (90, 333)], 100),
                                      ([(1, 20), (1, 500)], 10)])
@pytest.mark.parametrize("D,dtype", [(64, torch.bfloat16), (128, torch.float16)])
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_values_that_a_row_does_not_see(dsa, dev, seqs, win, D, dtype, what):
    """Infinities and NaN among a sequence's own keys reach the rows that see them, in their columns, and no others."""
    H, G, bs = 8, 2, 16
    q, kc, vc, table = _setup(seqs, H, G, D, bs, dtype, seed=12)
    clean, _ = _run(dsa, dev, seqs, q, kc, vc, table, win=win)
    kc2, vc2 = kc.clone(), vc.clone()
    bad_v, bad_k = [], []
    rows = []
    for b, (s, n) in enumerate(seqs):
        # A key before any row's window (if there is one), the first token's own, one in the middle, the last.
        for j, c in {(max(n - s - 12, 0), 3), (n - s, 17), (n - s // 2 - 1, 40), (n - 1, D - 1)}:
            vc2[table[b, j // bs], j % bs, j % G, c] = what
            bad_v.append((b, j, j % G, c))
        rows += [(b, n - s + i) for i in range(s)]
    got, _ = _run(dsa, dev, seqs, q, kc, vc2, table, win=win)
    sees = lambda row, b, j: row[0] == b and j <= row[1] and (win is None or j >= row[1] - win)
    want = clean.cpu().clone()
    hit = torch.zeros(want.shape, dtype=torch.bool)
    for b, j, g, c in bad_v:
        for t, row in enumerate(rows):
            if sees(row, b, j):
                hit[t, g * (H // G):(g + 1) * (H // G), c] = True
    got = got.cpu()
    assert torch.equal(got[~hit], want[~hit])
    assert not torch.isfinite(got[hit]).any()
    if math.isnan(what):  # a key: the whole row of a head that sees it
        for b, (s, n) in enumerate(seqs):
            j = n - s // 2 - 1
            kc2[table[b, j // bs], j % bs, 1, 5] = what
            bad_k.append((b, j))
        got, lse = (x.cpu() for x in _run(dsa, dev, seqs, q, kc2, vc, table, win=win))
        hit = torch.zeros(want.shape[:2], dtype=torch.bool)
        for b, j in bad_k:
            for t, row in enumerate(rows):
                if sees(row, b, j):
                    hit[t, H // G:] = True
        assert torch.equal(got[~hit], want[~hit]) and torch.isfinite(lse[~hit]).all()
        assert torch.isnan(got[hit]).all() and torch.isnan(lse[hit]).all()


@pytest.mark.parametrize("chunk", [20, 150])
@pytest.mark.parametrize("D", [64, 128])
def test_pages_outside_the_pool_hide_their_keys(dsa, dev, chunk, D):
    seqs = [(1, 300), (chunk, 200), (1, 64)]
    q, kc, vc, table = _setup(seqs, 8, 2, D, 32, torch.bfloat16, seed=7)
    table[0, 2], table[1, 0], table[1, 5], table[2, 0], table[2, 1] = -1, kc.shape[0], -1, -5, 2**31 - 1
    got = _run(dsa, dev, seqs, q, kc, vc, table)
    _check(got, _want(seqs, q, kc, vc, table))
    assert (got[0][-1] == 0).all() and torch.isinf(got[1][-1]).all()


@pytest.mark.parametrize("S,lens,keys", [(1, None, [9, 800, 1]), (1, [1, 0, 1], [9, 800, 0]), (37, None, [37, 60, 411]),
                                         (37, [37, 0, 20], [40, 5, 20]), (200, [200, 1, 63], [300, 900, 63])])
def test_padded_batches(dsa, dev, S, lens, keys):
    """[B, S, H, D] queries: the rows behind a sequence's tokens give zeros."""
    B, H, G, D, bs = 3, 8, 2, 128, 16
    real = [S] * B if lens is None else lens
    q, kc, vc, table = _setup([(S, n) for n in keys], H, G, D, bs, torch.bfloat16, seed=S)
    kl = torch.tensor(keys, dtype=torch.int32, device=dev)
    ql = None if lens is None else torch.tensor(lens, dtype=torch.int32, device=dev)
    out, lse = dsa.paged_gqa_fwd(q.view(B, S, H, D).to(dev), kc.to(dev), vc.to(dev), table.to(dev),
                                 actual_seq_lengths_query=ql, actual_seq_lengths_kv=kl)
    assert out.shape == (B, S, H, D) and lse.shape == (B, S, H)
    want = ref.attention(q, kc, vc, table, [b * S for b in range(B)], [S] * B, real, keys, D ** -0.5)
    _check((out.view(B * S, H, D), lse.view(B * S, H)), want)


def test_rows_behind_the_last_packed_sequence(dsa, dev):
    seqs = [(3, 50), (90, 90)]
    q, kc, vc, table = _setup(seqs + [(40, 0)], 8, 2, 64, 16, torch.bfloat16)
    out, lse = _run(dsa, dev, seqs, q, kc, vc, table[:2])
    assert (out[93:] == 0).all() and torch.isinf(lse[93:]).all()
    _check((out[:93], lse[:93]), _want(seqs, q[:93], kc, vc, table[:2]))


def test_lengths_of_other_types_and_places(dsa, dev):
    """Lists, host and 64-bit lengths take the Python route; the registered operator agrees too."""
    seqs = BATCHES["mixed"]
    q, kc, vc, table = _setup(seqs, 8, 2, 64, 16, torch.bfloat16)
    want = _run(dsa, dev, seqs, q, kc, vc, table)
    cu, kl = torch.tensor([s for s, _ in seqs]).cumsum(0), [n for _, n in seqs]
    a = [t.to(dev) for t in (q, kc, vc)]
    got = dsa.paged_gqa_fwd(*a, table.long().to(dev), actual_seq_lengths_query=cu, actual_seq_lengths_kv=kl)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = dsa.load_torch_ops().paged_gqa_fwd(*a, table.to(dev), torch.tensor(kl, device=dev), 64 ** -0.5, cu.to(dev))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_same_bits_each_time(dsa, dev):
    seqs = [(1, 9000), (33, 4000), (1, 10)]
    args = _setup(seqs, 16, 2, 128, 64, torch.bfloat16)
    a, b = _run(dsa, dev, seqs, *args), _run(dsa, dev, seqs, *args)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("win", [None, 500])
def test_long_chunks_are_repeated_to_the_bit(dsa, dev, D, win):
    """Whole and partly seen tiles in turn, a tile that ends inside a page, waves without rows in the last one."""
    seqs = [(1301, 2777), (1, 40), (270, 270)]
    args = _setup(seqs, 8, 2, D, 24, torch.bfloat16, seed=D)
    got = _run(dsa, dev, seqs, *args, win=win)
    _check(got, _want(seqs, *args, win=-1 if win is None else win))
    for _ in range(5):
        again = _run(dsa, dev, seqs, *args, win=win)
        assert torch.equal(got[0], again[0]) and torch.equal(got[1], again[1])


def test_lengths_past_the_table_are_cut(dsa, dev):
    """kv lengths above max_blocks * block_size and prefix sums above T are clamped, not followed."""
    seqs = [(4, 64)]
    q, kc, vc, table = _setup(seqs, 4, 1, 64, 16, torch.bfloat16)
    a = [t.to(dev) for t in (q, kc, vc, table)]
    big = torch.tensor([2**31 - 1], dtype=torch.int32, device=dev)
    out, lse = dsa.paged_gqa_fwd(*a, actual_seq_lengths_query=big, actual_seq_lengths_kv=big)
    want = _run(dsa, dev, seqs, q, kc, vc, table)
    assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    low = torch.tensor([-7], dtype=torch.int32, device=dev)
    out, lse = dsa.paged_gqa_fwd(*a, actual_seq_lengths_query=low, actual_seq_lengths_kv=low)
    assert (out == 0).all() and torch.isinf(lse).all()


def test_empty(dsa, dev):
    q, kc, vc, table = (t.to(dev) for t in _setup([(1, 5)], 4, 1, 64, 16, torch.bfloat16))
    z = torch.zeros(1, dtype=torch.int32, device=dev)
    out, lse = dsa.paged_gqa_fwd(q[:0], kc, vc, table, actual_seq_lengths_query=z, actual_seq_lengths_kv=z)
    assert out.shape == (0, 4, 64) and lse.shape == (0, 4)


def test_refusals(dsa, dev):
    q, kc, vc, table = (t.to(dev) for t in _setup([(2, 5)], 4, 2, 64, 16, torch.bfloat16))
    n = torch.tensor([2], dtype=torch.int32, device=dev)

    def call(q=q, kc=kc, vc=vc, table=table, sm_scale=None, **kw):
        return dsa.paged_gqa_fwd(q, kc, vc, table, sm_scale, **{**dict(actual_seq_lengths_query=n,
                                                                       actual_seq_lengths_kv=n), **kw})

    call()
    for match, kw in [("bfloat16", dict(q=q.float())), ("dtype", dict(vc=vc.half())),
                      ("64 or 128", dict(q=q[..., :32])), ("caches|k_cache", dict(kc=kc[..., :32])),
                      ("k_cache and v_cache", dict(vc=vc[:1])), ("multiple of kv_group", dict(q=q[:, :3])),
                      ("block_table", dict(table=table[0])), ("required", dict(actual_seq_lengths_kv=None)),
                      ("prefix sums", dict(actual_seq_lengths_query=None)),
                      ("batch", dict(q=torch.zeros(2, 1, 4, 64, dtype=torch.bfloat16, device=dev))),
                      ("B=1", dict(actual_seq_lengths_kv=torch.tensor([1, 2]))),
                      ("integers", dict(actual_seq_lengths_kv=torch.tensor([1.0]))),
                      ("win_left", dict(win_left=-1)), ("sm_scale", dict(sm_scale=0.0)),
                      ("sm_scale", dict(sm_scale=math.nan)), ("sinks", dict(sinks=torch.ones(3, device=dev))),
                      ("contiguous", dict(q=q.transpose(0, 1).contiguous().transpose(0, 1))),
                      ("HIP", dict(table=table.cpu()))]:
        with pytest.raises(ValueError, match=match):
            call(**kw)
