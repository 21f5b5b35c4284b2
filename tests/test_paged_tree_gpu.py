"""Attention of drafted trees over a paged cache against its formula in 64 bits."""
import math
import random

import pytest
import torch

import tree_step_ref as R
from dense_layer_ref import assert_within

pytestmark = pytest.mark.gpu


def ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


def build(dev, lens, H, G, D, bs, dtype, seed, W=None, hang=0.05, win=-1):
    """(nodes, context) of each sequence: queries, caches, table, masks of random trees, positions (on the CPU)."""
    g, rng = torch.Generator().manual_seed(seed), random.Random(seed)
    T = sum(s for s, _ in lens)
    mb = max(1, max(-(-(s + n) // bs) for s, n in lens))
    pages = list(range(len(lens) * mb + 2))
    rng.shuffle(pages)
    table = torch.tensor([[pages.pop() for _ in range(mb)] for _ in lens])
    shape = (len(lens) * mb + 2, bs, G, D)
    c = dict(q=torch.randn((T, H, D), generator=g).to(dtype), kc=torch.randn(shape, generator=g).to(dtype),
             vc=torch.randn(shape, generator=g).to(dtype), table=table, scale=D ** -0.5)
    chains = [R.ancestors(R.tree(rng, s, hang)) for s, _ in lens]
    W = W or max(1, max(-(-s // 64) for s, _ in lens))
    c["mask"] = torch.cat([R.mask_words(x, W, win) for x in chains])
    c["pos"] = torch.tensor([n + len(x) - 1 for (_, n), seq in zip(lens, chains) for x in seq])
    c["lens"] = [s for s, _ in lens]
    c["kv"] = [s + n for s, n in lens]
    return c


def run(dsa, dev, c, win=-1, sinks=None, what=""):
    lens = c["lens"]
    cu = torch.tensor(lens).cumsum(0)
    more = dict(positions=c["pos"].to(dev).int(), win_left=win) if win >= 0 else {}
    out, lse = dsa.paged_tree_fwd(c["q"].to(dev), c["kc"].to(dev), c["vc"].to(dev), c["table"].int().to(dev),
                                  c["mask"].to(dev), c["scale"], actual_seq_lengths_query=cu.int().to(dev),
                                  actual_seq_lengths_kv=ints(dev, c["kv"]), sinks=None if sinks is None else sinks.to(dev),
                                  **more)
    starts = [0] + cu.tolist()[:-1]
    kv = [min(max(n, 0), c["table"].shape[1] * c["kc"].shape[1]) for n in c["kv"]]
    o, ot, l, lt = R.attention(c["q"], c["kc"], c["vc"], c["table"], c["mask"], starts, lens, lens, kv, c["scale"], c["pos"],
                               win, sinks)
    assert_within(out, o, ot, "out " + what)
    assert_within(lse, l, lt, "lse " + what)
    return out, lse


SETS = {
    "one": [(1, 0)],
    "token": [(1, 130)],
    "small": [(8, 200)],
    "fresh": [(13, 0), (64, 0), (1, 0)],
    "mixed": [(1, 700), (24, 444), (7, 123), (0, 50), (127, 257), (61, 90), (5, 3001)],
    "edges": [(3, 61), (3, 62), (2, 63), (33, 31), (32, 32), (64, 64), (31, 97), (65, 127)],
    "batch": [(4, n) for n in range(100, 148)],
}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,H,G", [(128, 64, 4), (64, 8, 8), (128, 5, 1), (64, 64, 8), (128, 2, 2)])
@pytest.mark.parametrize("name", sorted(SETS))
def test_trees(dsa, dev, name, D, H, G, dtype):
    bs = {"one": 64, "token": 16, "edges": 16}.get(name, 64)
    run(dsa, dev, build(dev, SETS[name], H, G, D, bs, dtype, 1), what=name)


@pytest.mark.parametrize("win", [0, 1, 2, 40, 127, 5000])
@pytest.mark.parametrize("D,H,G", [(128, 32, 2), (64, 8, 2)])
@pytest.mark.parametrize("name", ["small", "mixed", "edges"])
def test_windows_and_sinks(dsa, dev, name, D, H, G, win):
    c = build(dev, SETS[name], H, G, D, 16, torch.bfloat16, 2, win=win)
    sinks = torch.randn(H, generator=torch.Generator().manual_seed(3)) * 3
    run(dsa, dev, c, win, sinks, name)


@pytest.mark.parametrize("bs", [1, 3, 7, 24, 200])
def test_odd_pages(dsa, dev, bs):
    for D, H, G, name in ((128, 16, 1, "mixed"), (64, 4, 2, "edges")):
        run(dsa, dev, build(dev, SETS[name], H, G, D, bs, torch.float16, 4), what=name)


@pytest.mark.parametrize("D,H,G", [(128, 16, 1), (64, 8, 4)])
def test_any_mask(dsa, dev, D, H, G):
    """Bits at random: rows without any, later nodes, nodes that the sequence does not have, words past the nodes."""
    for name in ("edges", "mixed", "fresh"):
        c = build(dev, SETS[name], H, G, D, 16, torch.bfloat16, 5, W=4)
        g = torch.Generator().manual_seed(6)
        c["mask"] = torch.randint(-2**63, 2**63 - 1, c["mask"].shape, generator=g, dtype=torch.int64)
        c["mask"][::5] = 0
        c["mask"][1::5] = -1
        run(dsa, dev, c, what=name)


def test_rows_that_see_nothing(dsa, dev):
    for sinks in (None, torch.tensor([0.5, -math.inf, math.inf, 3.0])):
        c = build(dev, [(9, 0), (70, 0), (2, 0)], 4, 2, 64, 16, torch.bfloat16, 7)
        c["mask"].zero_()
        out, lse = run(dsa, dev, c, sinks=sinks)
        assert not out.any()
        want = torch.full((4,), -math.inf) if sinks is None else sinks
        torch.testing.assert_close(lse.cpu(), want.expand_as(lse), atol=0, rtol=1e-6)


@pytest.mark.parametrize("n", [0, 1, 5, 9, 10**6])
def test_fewer_keys_than_nodes_and_more_than_the_table(dsa, dev, n):
    """Key counts that are no context and tree: the nodes' keys that there are."""
    for H, G, D in ((32, 2, 128), (4, 4, 64)):
        c = build(dev, [(9, 20), (40, 30)], H, G, D, 16, torch.bfloat16, 8)
        c["kv"] = [n, n]
        run(dsa, dev, c)


def test_nodes_past_the_mask(dsa, dev):
    """Trees of 100 nodes and masks of one word: the later nodes are seen by none, and see what their words say."""
    c = build(dev, [(100, 300), (80, 0)], 16, 4, 128, 64, torch.bfloat16, 9, W=1)
    run(dsa, dev, c)


@pytest.mark.parametrize("H,G,D", [(32, 2, 128), (2, 2, 64)])
def test_pages_outside_the_pool(dsa, dev, H, G, D):
    for bs in (16, 64, 5):
        c = build(dev, SETS["mixed"], H, G, D, bs, torch.bfloat16, 10)
        rng = random.Random(bs)
        flat = c["table"].view(-1)
        for i in range(0, flat.numel(), 3):
            flat[i] = rng.choice([-1, c["kc"].shape[0], 2**31 - 1, -2**31])
        run(dsa, dev, c, what=str(bs))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan, "max"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,G,D", [(32, 2, 128), (3, 3, 64), (64, 4, 64)])
def test_values_that_no_node_sees_do_not_reach_it(dsa, dev, bad, dtype, H, G, D):
    """Other branches' keys and values, keys ahead of a window, rows behind the last key."""
    value = torch.finfo(dtype).max if bad == "max" else bad
    lens = [(40, 200), (70, 33), (2, 500)]
    win = 100
    c = build(dev, lens, H, G, D, 16, dtype, 11, win=win)
    # Node 7 of each tree is seen by no other, and by itself no longer.
    for t0, (s, n), row in zip([0, 40, 110], lens, c["table"]):
        if s > 7:
            c["mask"][t0:t0 + s] &= ~torch.tensor([1 << 7] + [0] * (c["mask"].shape[1] - 1))
        dead = ([n + 7] if s > 7 else []) + list(range(0, max(0, n - win)))
        dead += list(range(n + s, -(-(n + s) // 16) * 16))
        for j in dead:
            at = int(row[j // 16]) * 16 + j % 16
            c["kc"].view(-1, G, D)[at] = value
            c["vc"].view(-1, G, D)[at] = value
    run(dsa, dev, c, win)


@pytest.mark.parametrize("H,G,D", [(32, 2, 128), (2, 2, 64)])
def test_values_that_are_not_finite_reach_their_rows_only(dsa, dev, H, G, D):
    """A node's value of infinity and NaN: in its descendants' rows and no other."""
    c = build(dev, [(40, 100)], H, G, D, 16, torch.bfloat16, 12, hang=0.0)
    for node, value in ((5, math.inf), (11, math.nan), (3, -math.inf)):
        at = int(c["table"][0, (100 + node) // 16]) * 16 + (100 + node) % 16
        c["vc"].view(-1, G, D)[at, :, node] = value
    cu = ints(dev, [40])
    out, _ = dsa.paged_tree_fwd(c["q"].to(dev), c["kc"].to(dev), c["vc"].to(dev), c["table"].int().to(dev), c["mask"].to(dev),
                                c["scale"], actual_seq_lengths_query=cu, actual_seq_lengths_kv=ints(dev, [140]))
    sees = ((c["mask"].view(-1, 1) >> torch.arange(40)) & 1).bool()
    bad = ~torch.isfinite(out.cpu().float())
    for node in (5, 11, 3):
        assert torch.equal(bad[:, 0, node], sees[:, node]), node
    other = [i for i in range(D) if i not in (5, 11, 3)]
    assert not bad[..., other].any()


@pytest.mark.parametrize("H,G,D", [(32, 2, 128), (3, 3, 64)])
@pytest.mark.parametrize("win", [-1, 9])
def test_padded_batches(dsa, dev, H, G, D, win):
    """[B, S, H, D] with lengths; rows behind them see nothing."""
    B, S, bs = 5, 70, 16
    lens, kv = [70, 1, 0, 33, 64], [300, 1, 40, 33, 500]
    c = build(dev, [(S, 440)] * B, H, G, D, bs, torch.bfloat16, 13)
    mask = c["mask"].view(B, S, -1)
    pos = torch.stack([torch.arange(n - L, n - L + S) for L, n in zip(lens, kv)])
    sinks = torch.randn(H, generator=torch.Generator().manual_seed(3))
    more = dict(positions=pos.to(dev), win_left=win) if win >= 0 else {}
    out, lse = dsa.paged_tree_fwd(c["q"].view(B, S, H, D).to(dev), c["kc"].to(dev), c["vc"].to(dev), c["table"].to(dev),
                                  mask.to(dev), actual_seq_lengths_query=ints(dev, lens),
                                  actual_seq_lengths_kv=ints(dev, kv), sinks=sinks.to(dev), **more)
    o, ot, l, lt = R.attention(c["q"], c["kc"], c["vc"], c["table"], c["mask"], [b * S for b in range(B)], [S] * B, lens, kv,
                               D ** -0.5, pos.view(-1), win, sinks)
    assert_within(out.view(-1, H, D), o, ot, "out")
    assert_within(lse.view(-1, H), l, lt, "lse")


def test_rows_behind_the_last_sequence(dsa, dev):
    c = build(dev, [(20, 300), (30, 77)], 32, 2, 128, 16, torch.bfloat16, 14)
    out, lse = dsa.paged_tree_fwd(c["q"].to(dev), c["kc"].to(dev), c["vc"].to(dev), c["table"].to(dev), c["mask"].to(dev),
                                  actual_seq_lengths_query=[20, 41], actual_seq_lengths_kv=[320, 98])
    assert not out[41:].any() and bool((lse[41:] == -math.inf).all()) and bool(torch.isfinite(lse[:41]).all())


@pytest.mark.parametrize("H,G,D", [(64, 4, 128), (8, 8, 64), (16, 2, 64)])
def test_a_chain_is_the_dense_attention(dsa, dev, H, G, D):
    """Masks of a chain say what the causal rule says, with a window too."""
    lens = [(1, 300), (33, 64), (100, 1000), (5, 0)]
    for win in (None, 50):
        c = build(dev, lens, H, G, D, 16, torch.bfloat16, 15)
        w = -1 if win is None else win
        mask = torch.cat([R.mask_words(R.ancestors(list(range(-1, s - 1))), 2, w) for s, _ in lens]).to(dev)
        pos = torch.cat([torch.arange(n, n + s) for s, n in lens]).to(dev)
        args = [c[k].to(dev) for k in ("q", "kc", "vc")] + [c["table"].int().to(dev)]
        cu, kv = torch.tensor(c["lens"]).cumsum(0), c["kv"]
        a = dsa.paged_tree_fwd(*args, mask, actual_seq_lengths_query=cu, actual_seq_lengths_kv=kv, win_left=win,
                               positions=pos if win else None)
        b = dsa.paged_gqa_fwd(*args, actual_seq_lengths_query=cu, actual_seq_lengths_kv=kv, win_left=win)
        # The same products and sums; units may be cut elsewhere: a rounding of the output and of the weights each.
        torch.testing.assert_close(a[0].float(), b[0].float(), atol=2 ** -8, rtol=2 ** -6)
        torch.testing.assert_close(a[1], b[1], atol=1e-4, rtol=1e-5)


def test_positions_outside_the_tree_count_as_the_nearest(dsa, dev):
    c = build(dev, [(30, 200), (70, 90)], 16, 2, 64, 16, torch.bfloat16, 16)
    g = torch.Generator().manual_seed(1)
    c["pos"] = torch.randint(-2**31, 2**31 - 1, (100,), generator=g)
    c["pos"][::7] = 2**31 - 1
    c["pos"][3::7] = -2**31
    for win in (0, 20, 150):
        run(dsa, dev, c, win)


def test_large_batch_of_tiles(dsa, dev):
    """More tiles than share a line: a workgroup each."""
    c = build(dev, [(61, 30 + i) for i in range(40)], 64, 16, 64, 16, torch.bfloat16, 17)
    run(dsa, dev, c)
    c = build(dev, [(1 + i % 3, 100 + i) for i in range(300)], 8, 8, 128, 16, torch.float16, 18)
    run(dsa, dev, c, 60, what="windows")


@pytest.mark.parametrize("B", [1024, 1025, 1100])
@pytest.mark.parametrize("padded", [False, True])
def test_many_sequences_in_tiles_of_256_rows(dsa, dev, B, padded):
    """Both sides of the lengths that a workgroup keeps a copy of, in the shared line's tiles of 256 rows; padded: some of
    the two rows of a sequence are padding."""
    rng = random.Random(B)
    H = 17 if padded else 16
    lens = [(rng.choice((0, 1, 2, 2)) if padded else rng.choice((2, 2, 2, 3)), rng.randint(0, 90)) for _ in range(B)]
    c = build(dev, lens, H, 1, 64, 16, torch.bfloat16, B)
    if not padded:
        run(dsa, dev, c)
        return
    cu = torch.tensor([0] + c["lens"]).cumsum(0).tolist()
    q, mask = torch.zeros(B, 2, H, 64, dtype=torch.bfloat16), torch.zeros(B, 2, 1, dtype=torch.int64)
    for b, (s, _) in enumerate(lens):
        q[b, :s], mask[b, :s] = c["q"][cu[b]:cu[b + 1]], c["mask"][cu[b]:cu[b + 1]]
    out, lse = dsa.paged_tree_fwd(q.to(dev), c["kc"].to(dev), c["vc"].to(dev), c["table"].int().to(dev), mask.to(dev),
                                  c["scale"], actual_seq_lengths_query=ints(dev, c["lens"]),
                                  actual_seq_lengths_kv=ints(dev, c["kv"]))
    o, ot, l, lt = R.attention(c["q"], c["kc"], c["vc"], c["table"], c["mask"], cu[:-1], c["lens"], c["lens"], c["kv"],
                               c["scale"])
    live = torch.tensor([i < s for s, _ in lens for i in range(2)])
    assert_within(out.cpu().reshape(2 * B, H, 64)[live], o, ot, "out")
    assert_within(lse.cpu().reshape(2 * B, H)[live], l, lt, "lse")
    assert not out.cpu().reshape(2 * B, H, 64)[~live].any() and bool(torch.isneginf(lse.cpu().reshape(2 * B, H)[~live]).all())
