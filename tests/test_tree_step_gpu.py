"""A tree-drafted step's operators on the GPU against their plain forms: plan, free, acceptance, cache rows."""
import random

import pytest
import torch

import tree_step_ref as R

pytestmark = pytest.mark.gpu
I32 = torch.int32


def ints(dev, x):
    return torch.tensor(x, dtype=I32, device=dev)


def make_lists(rng, ctx, bs, mb, spare, holes=0.0):
    """A table whose rows hold their contexts' pages (some left out), and a list of the other pages."""
    need = [min(-(-min(max(c, 0), 10**6) // bs), mb) for c in ctx]
    pages = list(range(sum(need) + spare))
    rng.shuffle(pages)
    table = [[-1] * mb for _ in ctx]
    for b, n in enumerate(need):
        for j in range(n):
            page = pages.pop()
            table[b][j] = -rng.randint(1, 9) if rng.random() < holes else page
    return table, pages


def check_plan(dsa, dev, new, ctx, table, free, count, bs, T, parents=None, max_nodes=0, win=-1):
    g_table, g_free, g_count = ints(dev, table), ints(dev, free), ints(dev, count)
    more = {} if parents is None else dict(parents=ints(dev, parents), max_nodes=max_nodes)
    if win >= 0:
        more["win_left"] = win
    got = dsa.paged_plan(ints(dev, new), ints(dev, ctx), g_table, g_free, g_count, bs, T, **more)
    want = R.plan(new, ctx, table, free, count, bs, T, parents, max_nodes, win)
    for name, g, w in zip(got._fields, got, want):
        if w is None or name == "tree_mask" and max_nodes == 0:
            assert g is None
        else:
            w = w if isinstance(w, torch.Tensor) else torch.tensor(w, dtype=I32)
            assert g.dtype == w.dtype and torch.equal(g.cpu(), w), name
    assert g_table.tolist() == table and g_count.tolist() == count and g_free.tolist() == free
    return got, g_table, g_free, g_count


@pytest.mark.parametrize("B,most,bs,mb", [(1, 1, 64, 4), (1, 200, 1, 300), (3, 9, 16, 8), (64, 61, 64, 40), (200, 7, 16, 30),
                                          (1500, 3, 128, 6), (17, 700, 16, 64)])
@pytest.mark.parametrize("tree", [False, True])
def test_plan(dsa, dev, B, most, bs, mb, tree):
    rng = random.Random(B * 1000 + most)
    new = [rng.randint(0, most) for _ in range(B)]
    ctx = [rng.randint(0, mb * bs - most) if mb * bs > most else 0 for _ in range(B)]
    table, free = make_lists(rng, ctx, bs, mb, sum(new) // bs + 2 * B)
    T = sum(new) + rng.randint(0, 5)
    parents = [p for s in new for p in R.tree(rng, s, 0.1)] + [0] * (T - sum(new)) if tree else None
    check_plan(dsa, dev, new, ctx, table, free + [-7, -7], [len(free)], bs, T, parents, max(new + [1]))


@pytest.mark.parametrize("win", [0, 1, 5, 1000])
@pytest.mark.parametrize("max_nodes", [1, 64, 65, 130])
def test_plan_masks_past_their_words_and_windows(dsa, dev, win, max_nodes):
    """Trees larger than their masks, deep chains, parents that are not before their children."""
    rng = random.Random(max_nodes)
    new = [130, 1, 0, 64, 65, 128]
    parents = list(range(-1, 129)) + [5] + R.tree(rng, 64) + [rng.randint(-3, 70) for _ in range(65)] + R.tree(rng, 128, 0.3)
    ctx = [0, 3, 4, 63, 64, 1000]
    table, free = make_lists(rng, ctx, 16, 80, 40)
    check_plan(dsa, dev, new, ctx, table, free, [len(free)], 16, sum(new), parents, max_nodes, win)


@pytest.mark.parametrize("win", [-1, 0, 63, 64, 500])
@pytest.mark.parametrize("new,max_nodes", [([0, 3, 60, 66, 1, 130, 500], 64), ([900, 70], 4096), ([7, 1017], 128),
                                           ([7, 1018], 0), ([200, 4500, 3, 700], 4096), ([77, 1500, 300], 200)])
def test_plan_long_runs(dsa, dev, new, max_nodes, win):
    """Rows whose parents are the rows before them, for whole sequences and parts, up to those that pass a workgroup's rows
    and the parents that it holds at once, beside branches and rows without parents."""
    rng = random.Random(sum(new) + win)
    parents = []
    for b, s in enumerate(new):
        for i in range(s):
            jump = b % 3 and rng.random() < 0.02
            parents.append(rng.randint(-1, i) if jump else i - 1)
    ctx = [rng.randint(0, 90) for _ in new]
    mb = (max(new) + 90) // 16 + 2
    table, free = make_lists(rng, ctx, 16, mb, sum(new) // 16 + 2 * len(new))
    check_plan(dsa, dev, new, ctx, table, free, [len(free)], 16, sum(new) + 2, parents + [0, 1], max_nodes, win)


@pytest.mark.parametrize("T", [1023, 1024, 1025, 2047, 2048, 2049])
@pytest.mark.parametrize("tree", [False, True])
def test_plan_on_both_sides_of_its_row_counts(dsa, dev, T, tree):
    rng = random.Random(T)
    new = [40] * (T // 40) + [T % 40]
    ctx = [rng.randint(0, 60) for _ in new]
    table, free = make_lists(rng, ctx, 16, 8, sum(new) // 16 + 2 * len(new))
    parents = [p for s in new for p in R.tree(rng, s, 0.05)] if tree else None
    check_plan(dsa, dev, new, ctx, table, free, [len(free)], 16, T, parents, 64)


@pytest.mark.parametrize("count", [0, 1, 5, -3, 10**9])
def test_plan_runs_out_of_pages_and_tables(dsa, dev, count):
    """Too few pages, contexts at and past the table's end, negative and huge lengths, holes in the context."""
    rng = random.Random(7)
    new = [5, 40, 0, -2, 3, 7, 2, 33]
    ctx = [10, 0, 5, 6, 62, 64, 2**31 - 1, -9]
    table, free = make_lists(rng, [min(c, 64) for c in ctx], 16, 4, 9, holes=0.2)
    check_plan(dsa, dev, new, ctx, table, free, [count], 16, 100)


@pytest.mark.parametrize("T", [0, 1, 30, 59])
def test_plan_cuts_lengths_at_its_rows(dsa, dev, T):
    rng = random.Random(3)
    new, ctx = [20, 0, 20, 2**31 - 1, 5], [1, 2, 3, 4, 5]
    table, free = make_lists(rng, ctx, 16, 8, 30)
    check_plan(dsa, dev, new, ctx, table, free, [len(free)], 16, T)
    table, free = make_lists(rng, ctx, 16, 8, 30)
    check_plan(dsa, dev, new, ctx, table, free, [len(free)], 16, T, [-1] * T, 70)


@pytest.mark.parametrize("B,T,bs,tree", [(5, 4096, 16, True), (5, 4097, 16, True), (3, 30000, 16, False),
                                         (2100, 9000, 64, True), (16384, 17000, 16, False)])
def test_plan_of_many_rows(dsa, dev, B, T, bs, tree):
    """Both sides of the number of rows that one workgroup writes, sums inside and outside the copy in LDS."""
    rng = random.Random(T)
    new = [T // B] * B
    new[B // 2] += T - sum(new) - 3
    ctx = [rng.randint(0, 40) for _ in range(B)]
    mb = (max(new) + 40) // bs + 2
    table, free = make_lists(rng, ctx, bs, mb, sum(new) // bs + 2 * B)
    parents = [p for s in new for p in [-1] + [rng.randrange(max(0, i - 9), i) for i in range(1, s)]] + [0] * 3 if tree else None
    check_plan(dsa, dev, new, ctx, table, free, [len(free)], bs, T, parents, 60)


@pytest.mark.parametrize("B", [1, 5, 16, 17, 64, 65, 300, 1500])
def test_free_undoes_a_plan_and_cuts_rows(dsa, dev, B):
    """Every lane group size; then whole requests and parts of them, with a list too short for all."""
    rng = random.Random(B)
    bs, mb = 16, 150 if B < 100 else 9
    new = [rng.randint(0, bs * mb // 3) for _ in range(B)]
    ctx = [rng.randint(0, bs * mb // 2) for _ in range(B)]
    table, free = make_lists(rng, ctx, bs, mb, sum(new) // bs + 2 * B)
    before = [list(r) for r in table], list(free)
    _, t, f, c = check_plan(dsa, dev, new, ctx, table, free, [len(free)], bs, sum(new))
    planned = t.clone()
    dsa.paged_free(ints(dev, ctx), t, f, c, bs)
    assert t.tolist() == before[0] and f.tolist() == before[1] and c.tolist() == [len(free)]
    held = int((planned >= 0).sum())
    for room in (held + 3, held // 2, 0):
        keep = [rng.choice([0, -5, 1, 2**31 - 1, rng.randint(0, bs * mb)]) for _ in range(B)]
        lists, count, table = [-3] * room, [min(2, room)], planned.tolist()
        t, f, c = planned.clone(), ints(dev, lists), ints(dev, count)
        dsa.paged_free(ints(dev, keep), t, f, c, bs)
        R.free(keep, table, lists, count, bs)
        assert t.tolist() == table and f.tolist() == lists and c.tolist() == count


@pytest.mark.parametrize("T", [300, 5000])
def test_plan_positions_without_masks(dsa, dev, T):
    """Trees whose masks are not made: their depths are."""
    rng = random.Random(T)
    new, ctx = [T - 60, 0, 50, 1], [30, 1, 2, 3]
    table, free = make_lists(rng, ctx, 16, T, T)
    parents = [p for s in new for p in R.tree(rng, s, 0.1)] + [3] * 9
    got = check_plan(dsa, dev, new, ctx, table, free, [len(free)], 16, T, parents, 0)[0]
    assert got.tree_mask is None
    table, free = make_lists(rng, ctx, 16, T, T)
    check_plan(dsa, dev, new, ctx, table, free, [len(free)], 16, T, [-1] * T, 0)


def test_plan_takes_other_integers_and_hosts(dsa, dev):
    rng = random.Random(2)
    new, ctx, par = [3, 0, 9], [7, 100, 30], [-1, 0, 0, -1, 0, 1, 2, 0, 0, 5, 5, 1]
    table, free = make_lists(rng, ctx, 16, 8, 9)
    want = R.plan(new, ctx, [list(r) for r in table], free, [len(free)], 16, 12, par, 9)
    for conv in (lambda x: torch.tensor(x, dtype=torch.int64, device=dev), lambda x: x, torch.tensor,
                 lambda x: torch.tensor(x, dtype=torch.int16, device=dev)):
        got = dsa.paged_plan(conv(new), conv(ctx), ints(dev, table), ints(dev, free), ints(dev, [len(free)]), 16, 12,
                             parents=conv(par), max_nodes=9)
        assert got.slots.tolist() == want[3] and torch.equal(got.tree_mask.cpu(), want[5])
    huge = dsa.paged_plan([2**40, 1], [2**40, -2**40], ints(dev, [[1], [2]]), ints(dev, free), ints(dev, [0]), 16, 4)
    assert huge.cu_seqlens.tolist() == [4, 4] and huge.kv_lens.tolist() == [2**30 + 4, 0] and huge.slots.tolist() == [-1] * 4


@pytest.mark.parametrize("change,msg", [(dict(block_table=torch.int64), "block_table changes"),
                                        (dict(free_blocks=torch.int64), "free_blocks changes"),
                                        (dict(free_count=torch.int64), "free_count changes"), (dict(block_size=0), "block_size"),
                                        (dict(num_tokens=-1), "num_tokens"), (dict(num_tokens=2**30), "num_tokens"),
                                        (dict(max_nodes=-1), "max_nodes"), (dict(max_nodes=4097), "max_nodes"),
                                        (dict(win_left=-1), "win_left"), (dict(parents=None, win_left=3), "win_left"),
                                        (dict(new_lens=[1, 2]), "new_lens must"), (dict(context_lens=[1.0] * 3), "context_lens"),
                                        (dict(parents=[0] * 3), "parents must")])
def test_plan_refusals(dsa, dev, change, msg):
    kw = dict(new_lens=ints(dev, [1, 2, 1]), context_lens=ints(dev, [0, 0, 0]), block_table=ints(dev, [[-1] * 2] * 3),
              free_blocks=ints(dev, [0, 1, 2, 3]), free_count=ints(dev, [4]), block_size=16, num_tokens=4,
              parents=ints(dev, [0] * 4), max_nodes=4)
    for k, v in change.items():
        kw[k] = kw[k].to(v) if isinstance(v, torch.dtype) else v
    with pytest.raises(ValueError, match=msg):
        dsa.paged_plan(**kw)
    wide = ints(dev, [[-1] * 4] * 3)[:, ::2]
    with pytest.raises(ValueError, match="contiguous"):
        dsa.paged_free(ints(dev, [0] * 3), wide, ints(dev, [0]), ints(dev, [0]), 16)


# ------------------------------------------------------------------------------- acceptance


def trees(rng, lens, V, agree):
    """Parents, drafted tokens and choices of sequences, a child's token the choice with probability `agree`."""
    parents, tokens, choices = [], [], []
    for s in lens:
        par = R.tree(rng, s, 0.05)
        cho = [rng.randrange(V) for _ in range(s)]
        tok = [cho[p] if p >= 0 and rng.random() < agree else rng.randrange(V) for p in par]
        parents, tokens, choices = parents + par, tokens + tok, choices + cho
    return parents, tokens, choices


def check_accept(dsa, dev, scores, lens, parents, tokens, P, plain=None):
    cu = torch.tensor(lens).cumsum(0).tolist()
    got = dsa.tree_accept(scores, ints(dev, tokens), ints(dev, parents), actual_seq_lengths_query=ints(dev, cu), max_path=P)
    want = R.accept(plain if plain is not None else scores.cpu(), tokens, parents, cu, P)
    for name, g, w in zip(("accepted", "path", "chosen"), got, want):
        assert g.dtype == I32 and torch.equal(g.cpu(), w), name
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 7, 8, 63, 1000, 8192, 8193, 20011])
@pytest.mark.parametrize("rows", ["few", "many"])
def test_accept(dsa, dev, dtype, V, rows):
    """Both ways over the scores: all rows in a first launch, and those on the path only."""
    rng = random.Random(V)
    lens = [5, 1, 0, 61, 8] if rows == "few" else [5, 1, 0, 61, 8] + [40] * (1 + (64 << 20) // (40 * V * 2))
    if sum(lens) > 60000:  # short rows: any number of them is few bytes, and 65536 is past a grid's rows
        lens = [5, 1, 0, 61, 8] + [4000] * 17
    parents, tokens, choices = trees(rng, lens, V, 0.6)
    g = torch.Generator(device=dev).manual_seed(V)
    x = torch.randn(sum(lens), V, generator=g, device=dev).to(dtype)
    for t, c in enumerate(choices):  # the choice on top, but for rows left to their own
        choices[t] = c if t % 5 else -1
    at = ints(dev, choices).long()
    keep = at >= 0
    x[torch.nonzero(keep).view(-1), at[keep]] = 9.0
    check_accept(dsa, dev, x, lens, parents, tokens, 9)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("V", [5, 4099])
@pytest.mark.parametrize("many", [False, True])
def test_accept_equal_scores_infinities_and_nan(dsa, dev, dtype, V, many):
    """Equal largest scores, both zeros, infinities, NaN of both signs, rows that hold nothing else, all negative rows."""
    inf, nan = float("inf"), float("nan")
    g = torch.Generator().manual_seed(V)
    x = torch.randint(-3, 4, (12, V), generator=g).float()
    x[1] = -inf
    x[2] = nan
    x[3, 1:] = nan
    x[4] = -5.0
    x[4, 3] = -0.0
    x[4, 4] = 0.0
    x[5, 2], x[5, 4] = inf, inf
    x[6], x[6, V - 1] = -inf, torch.finfo(dtype).min
    x[7, 0] = -nan
    x[8] = 1.0
    x[9], x[9, V - 1] = nan, -inf
    x[10] = torch.finfo(dtype).min
    x = x.to(dtype)
    if many:
        x = torch.cat([x, torch.zeros(1 + (40 << 20) // V, V, dtype=dtype)])
    T = x.shape[0]
    assert T <= 65535 or V == 5
    lens = [1] * 12 + ([T - 12] if many else [])
    check_accept(dsa, dev, x.to(dev), lens, [-1] * T, [0] * T, 1)
    # A choice of none matches no token, -1 among them either.
    check_accept(dsa, dev, x.to(dev), [12] + lens[12:], list(range(-1, 11)) + [-1] * (T - 12), [-1] * T, 12)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,wide,offset", [(1000, 1003, 0), (1000, 1001, 3), (33, 40, 1), (20000, 20001, 7)])
def test_accept_rows_that_lie_apart(dsa, dev, dtype, V, wide, offset):
    rng = random.Random(V)
    lens = [9, 30]
    parents, tokens, choices = trees(rng, lens, V, 0.7)
    x = torch.full((sum(lens), wide + offset), 50.0, device=dev, dtype=dtype)  # larger values beside the rows
    x[:, offset:offset + V] = torch.randn(sum(lens), V, generator=torch.Generator(device=dev).manual_seed(1), device=dev)
    x = x[:, offset:offset + V]
    x[torch.arange(sum(lens)), choices] = 9.0
    check_accept(dsa, dev, x, lens, parents, tokens, 30)
    check_accept(dsa, dev, x.t().contiguous().t(), lens, parents, tokens, 30)


@pytest.mark.parametrize("P", [1, 2, 7, 2500])
def test_accept_given_choices(dsa, dev, P):
    """Trees of more nodes than a workgroup has threads; integers of other widths; long paths cut."""
    rng = random.Random(P)
    lens = [2000, 0, 1, 300, 257, 1025]
    parents, tokens, choices = trees(rng, lens, 3, 0.5)
    parents[:2000], tokens[:2000], choices[:2000] = range(-1, 1999), [1] * 2000, [1] * 2000
    check_accept(dsa, dev, ints(dev, choices), lens, parents, tokens, P, plain=choices)
    cu = torch.tensor(lens).cumsum(0)
    wide = lambda x: torch.tensor(x, dtype=torch.int64, device=dev)
    got = dsa.tree_accept(wide(choices), wide(tokens), wide(parents), actual_seq_lengths_query=cu, max_path=P)
    assert torch.equal(got[1].cpu(), R.accept(choices, tokens, parents, cu.tolist(), P)[1])
    # Past 31 bits nothing matches, equal or not.
    far = dsa.tree_accept(wide([2**31, 5]), wide([0, 2**31]), wide([-1, 0]), actual_seq_lengths_query=wide([2]), max_path=2)
    assert far[0].tolist() == [1] and far[2].tolist() == [[-1, -1]]


def test_accept_sums_that_are_not_sums(dsa, dev):
    """Sums that fall, or pass the rows, stay within them; empty calls."""
    x = torch.zeros(6, 10, device=dev)
    for cu in ([9, 20], [4, 2], [-3, 6], [2**31 - 1, -2**31]):
        a, p, c = dsa.tree_accept(x, ints(dev, [0] * 6), ints(dev, [-1, 0, 1, 2, 3, 4]), actual_seq_lengths_query=ints(dev, cu),
                                  max_path=8)
        assert int(a.max()) <= 6 and int(p.max()) <= 5
    a, p, c = dsa.tree_accept(x[:0], ints(dev, []), ints(dev, []), actual_seq_lengths_query=ints(dev, [0, 0]), max_path=3)
    assert a.tolist() == [0, 0] and p.tolist() == [[-1] * 3] * 2 and c.tolist() == [[-1] * 3] * 2


# ------------------------------------------------------------------------------- the cache rows' order


def some_path(rng, S, n):
    return sorted(rng.sample(range(S), min(n, S)))


@pytest.mark.parametrize("shape,dtype", [((), torch.float32), ((4, 128), torch.bfloat16), ((1, 576), torch.float16), ((2, 64), torch.float32),
                                         ((1, 128), torch.float8_e4m3fn), ((1,), torch.float32), ((3, 6), torch.int16),
                                         ((5000,), torch.uint8), ((1, 4), torch.uint8)])
@pytest.mark.parametrize("bs", [1, 16, 64])
def test_commit(dsa, dev, shape, dtype, bs):
    rng = random.Random(bs)
    B, S = 5, 40
    mb = -(-(100 + S) // bs)
    nb = B * mb + 2
    ctx = [rng.randint(0, 100) for _ in range(B)]
    pages = list(range(nb))
    rng.shuffle(pages)
    table = [[pages.pop() for _ in range(mb)] for _ in range(B)]
    table[1][(ctx[1] + 2) // bs] = -1  # rows without a page stay
    table[2][-1] = nb
    path = [some_path(rng, S, rng.randint(1, 30)) for _ in range(B)]
    accepted = [len(p) for p in path]
    accepted[3] = 2
    path = [p + [-1] * (31 - len(p)) for p in path]
    path[4] = [0, 0, 5, 4, 9, 1, 9] + [-1] * 24  # not a path: places below their own move nothing
    accepted[4] = 99
    g = torch.Generator().manual_seed(bs)
    caches = [torch.randint(0, 256, (nb, bs) + shape, generator=g).to(torch.uint8).to(dtype) if dtype != torch.float8_e4m3fn
              else torch.randn((nb, bs) + shape, generator=g).to(dtype) for _ in range(3)]
    got = [c.to(dev) for c in caches]
    raw = [c.view(nb, bs, -1).view(torch.uint8) for c in caches]
    R.commit(raw, table, ctx, path, accepted)
    dsa.paged_commit(got, ints(dev, table), ints(dev, ctx), ints(dev, path), ints(dev, accepted))
    for a, b in zip(got, raw):
        assert torch.equal(a.view(nb, bs, -1).view(torch.uint8).cpu(), b)


@pytest.mark.parametrize("n", [1, 7, 128, 129, 300])
def test_commit_many_caches_of_different_rows(dsa, dev, n):
    """Caches past one launch's, rows of several widths side by side, paths past a wave's lanes."""
    rng = random.Random(n)
    B, bs, mb, S = 3, 16, 16, 150
    pages = list(range(B * mb))
    rng.shuffle(pages)
    table = [[pages.pop() for _ in range(mb)] for _ in range(B)]
    ctx, path = [0, 77, 100], [some_path(rng, S, 130), some_path(rng, S, 65), some_path(rng, S, 3)]
    accepted = [len(p) for p in path]
    path = [p + [-1] * (130 - len(p)) for p in path]
    g = torch.Generator().manual_seed(n)
    caches = [torch.randn((B * mb, bs, [4, 1, 516, 260, 3][i % 5]), generator=g) for i in range(n)]
    got = [c.to(dev) for c in caches]
    R.commit(caches, table, ctx, path, accepted)
    dsa.paged_commit(tuple(got), ints(dev, table), ints(dev, ctx), ints(dev, path), ints(dev, accepted))
    for a, b in zip(got, caches):
        assert torch.equal(a.cpu(), b)


def test_commit_caches_off_16_bytes_and_refusals(dsa, dev):
    flat = torch.randn(1 + 4 * 16 * 8, device=dev)
    c = flat[1:].view(4, 16, 8)  # contiguous, 4 bytes off
    want = [c.cpu().clone()]
    args = [[1, 3]], [3], [[0, 2, 5]], [3]
    R.commit(want, *args)
    dsa.paged_commit(c, *(ints(dev, x) for x in args))
    assert torch.equal(c.cpu(), want[0])
    t, ctx, p, a = (ints(dev, x) for x in args)
    with pytest.raises(dsa.DSAError, match="overlap"):
        dsa.paged_commit([c, c], t, ctx, p, a)
    with pytest.raises(dsa.DSAError, match="multiples of 4"):
        dsa.paged_commit(torch.zeros(4, 16, 3, dtype=torch.uint8, device=dev), t, ctx, p, a)
    with pytest.raises(ValueError, match="alike"):
        dsa.paged_commit([c, torch.zeros(5, 16, 8, device=dev)], t, ctx, p, a)
    with pytest.raises(ValueError, match="contiguous"):
        dsa.paged_commit(torch.zeros(4, 16, 8, 2, device=dev)[..., 0], t, ctx, p, a)
    with pytest.raises(ValueError, match="path"):
        dsa.paged_commit(c, t, ctx, p.float(), a)
    with pytest.raises(ValueError, match="accepted"):
        dsa.paged_commit(c, t, ctx, p, ints(dev, [1, 2]))
    dsa.paged_commit(c, t.long(), [3], p.long(), a.long())  # moved again: the rows now there
    R.commit(want, *args)
    assert torch.equal(c.cpu(), want[0])


@pytest.mark.parametrize("ops", [False, True])
@pytest.mark.parametrize("dtype", [torch.int64, torch.uint32, torch.uint64])
def test_accept_numbers_past_31_bits_match_nothing(dsa, dev, dtype, ops):
    """Two of them are not alike, nor is either the largest of 31 bits."""
    top, far = 2**31 - 1, 2**32 - 5
    wide = lambda x: torch.tensor(x, dtype=torch.int64, device=dev).to(dtype)
    args = (wide([top, far, far, 7, 2**31 + 1]), wide([0, far, top, 2**31, 7]), ints(dev, [-1, 0, 0, 2, 3]))
    if ops:
        accepted, path, chosen = dsa.load_torch_ops().tree_accept(*args, ints(dev, [5]), 4)
    else:
        accepted, path, chosen = dsa.tree_accept(*args, actual_seq_lengths_query=ints(dev, [5]), max_path=4)
    assert accepted.tolist() == [2] and path.tolist() == [[0, 2, -1, -1]] and chosen.tolist() == [[top, -1, -1, -1]]


@pytest.mark.parametrize("T", [2048, 2049])
def test_plan_keeps_no_large_masks_beside_its_other_parts(dsa, dev, T):
    """64 words a row: masks of 1 MB, and of more, which are an allocation of their own."""
    table, free = [[-1] * (T // 64 + 1)], list(range(T // 64 + 1))
    got, *_ = check_plan(dsa, dev, [T], [0], table, free, [len(free)], 64, T, [(i - 1) // 2 if i else -1 for i in range(T)], 4096)
    parts = [x.untyped_storage().data_ptr() for x in got]
    assert len(set(parts[:5])) == 1 and (parts[5] == parts[0]) == (T == 2048)
    assert all(x.data_ptr() % 16 == 0 and x.is_contiguous() for x in got)
