"""A tree-drafted step's operators where offsets pass 31 and 32 bits, and at their largest sizes."""
import random

import pytest
import torch

import tree_step_ref as R
from dense_layer_ref import assert_within

pytestmark = pytest.mark.gpu


def ints(dev, x):
    return torch.tensor(x, dtype=torch.int32, device=dev)


@pytest.mark.parametrize("bs", [64, 24])
def test_attention_pages_past_32_bits(dsa, dev, bs):
    """Pages at both ends of pools of more than 2^32 bytes and 2^31 elements."""
    H, G, D = 32, 2, 128
    nb = (2**31 + 2**28) // (bs * G * D)
    g = torch.Generator(device=dev).manual_seed(1)
    pool = lambda: torch.zeros(nb, bs, G, D, dtype=torch.bfloat16, device=dev)
    kc, vc = pool(), pool()
    lens, ctx = [40, 1, 7], [300, 100, 33]
    rng = random.Random(bs)
    mb = 15
    pages = rng.sample(range(nb - 40, nb), 30) + rng.sample(range(40), 15)
    rng.shuffle(pages)
    table = torch.tensor(pages).view(3, mb)
    for p in pages:
        kc[p].normal_(generator=g)
        vc[p].normal_(generator=g)
    T = sum(lens)
    q = torch.randn(T, H, D, generator=g, device=dev).to(torch.bfloat16)
    mask = torch.cat([R.mask_words(R.ancestors(R.tree(rng, s)), 1) for s in lens])
    cu, kv = torch.tensor(lens).cumsum(0), [a + b for a, b in zip(lens, ctx)]
    out, lse = dsa.paged_tree_fwd(q, kc, vc, table.int().to(dev), mask.to(dev), actual_seq_lengths_query=cu.int().to(dev),
                                  actual_seq_lengths_kv=ints(dev, kv))
    small = {p: i for i, p in enumerate(pages)}
    at = torch.tensor(pages, device=dev)
    o, ot, l, lt = R.attention(q.cpu(), kc[at].cpu(), vc[at].cpu(), torch.tensor([[small[int(p)] for p in r] for r in table]),
                               mask, [0] + cu.tolist()[:-1], lens, lens, kv, D ** -0.5)
    assert_within(out, o, ot, "out")
    assert_within(lse, l, lt, "lse")


def test_commit_rows_past_32_bits(dsa, dev):
    nb, bs, width = 70000, 64, 512  # 4.6 GB of bf16
    c = torch.zeros(nb, bs, width, dtype=torch.bfloat16, device=dev)
    table, ctx, path, accepted = [[nb - 1, 3, nb - 2], [5, nb - 7, 9]], [60, 100], [[0, 9, 20, 70], [0, 3, 5, 40]], [4, 4]
    g = torch.Generator(device=dev).manual_seed(1)
    pages = [p for r in table for p in r]
    for p in pages:
        c[p].normal_(generator=g)
    at = torch.tensor(pages, device=dev)
    want = [c[at].cpu()]
    R.commit(want, [[0, 1, 2], [3, 4, 5]], ctx, path, accepted)
    dsa.paged_commit(c, ints(dev, table), ints(dev, ctx), ints(dev, path), ints(dev, accepted))
    assert torch.equal(c[at].cpu(), want[0])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_accept_scores_past_32_bits(dsa, dev, dtype):
    """Scores of more than 2^32 bytes and 2^31 elements; the last sequences lie behind both."""
    T, V = 17000, 131071
    x = torch.zeros(T, V, dtype=dtype, device=dev)
    lens = [T - 40, 20, 20]
    rng = random.Random(1)
    parents = [-1] * (T - 40) + R.tree(rng, 20) + R.tree(rng, 20)
    tokens = [0] * (T - 40) + [rng.randrange(V) for _ in range(40)]
    plain = [0] * T
    for t in range(T - 40, T):
        first = T - 40 if t < T - 20 else T - 20
        child = next((i for i in range(t + 1 - first, 20) if parents[first + i] == t - first), None)
        plain[t] = tokens[first + child] if child is not None else V - 1
        x[t, plain[t]] = 1.0
    cu = torch.tensor(lens).cumsum(0).tolist()
    got = dsa.tree_accept(x, ints(dev, tokens), ints(dev, parents), actual_seq_lengths_query=ints(dev, cu), max_path=20)
    for g, w in zip(got, R.accept(plain, tokens, parents, cu, 20)):
        assert torch.equal(g.cpu(), w)


def test_masks_past_32_bits_and_a_million_rows(dsa, dev):
    """A plan of 2^20 rows in sequences of up to 4096 nodes: 64 words a row, half a GB of masks, walks of 4096 steps."""
    T, W = 1 << 20, 64
    new = [4096] * 200 + [1] * 8 + [3] * 40
    new.append(T - sum(new) - 5)
    B = len(new)
    parents = torch.full((T,), -1, dtype=torch.int32)
    at = 0
    for b, s in enumerate(new):
        s = min(s, T - at)
        i = torch.arange(s, dtype=torch.int32)
        parents[at:at + s] = i - 1 if b % 50 == 0 else (i - 1) // 2  # chains among binary trees
        parents[at] = -1
        at += s
    mb = max(new) // 128 + 2
    table = torch.full((B, mb), -1, dtype=torch.int32, device=dev)
    free = torch.arange(T // 128 + B * 2, dtype=torch.int32, device=dev)
    count = torch.tensor([free.numel()], dtype=torch.int32, device=dev)
    p = dsa.paged_plan(ints(dev, new), ints(dev, [0] * B), table, free, count, 128, T, parents=parents.to(dev), max_nodes=4096)
    assert p.cu_seqlens.tolist() == torch.tensor(new).cumsum(0).tolist() and not p.missing.any()
    cu = [0] + p.cu_seqlens.tolist()
    for b in (0, 1, 50, 199, 210):
        s = new[b]
        chains = R.ancestors(parents[cu[b]:cu[b] + s].tolist()) if b else None
        for i in sorted({0, 1, s // 2, s - 1} & set(range(s))):
            row = p.tree_mask[cu[b] + i].cpu()
            chain = chains[i] if chains else list(range(i, -1, -1))
            assert torch.equal(row, R.mask_words([chain], W)[0]), (b, i)
            assert int(p.positions[cu[b] + i]) == len(chain) - 1
    assert bool((p.slots[-5:] == -1).all()) and not p.tree_mask[-5:].any()
    used = p.slots[:T - 5].long()
    assert int(used.min()) >= 0 and used.unique().numel() == T - 5


def test_large_masks_in_the_attention(dsa, dev):
    """4096 nodes of one sequence, 64 words a row."""
    S, H, G, D, bs = 4096, 4, 2, 64, 64
    g = torch.Generator().manual_seed(2)
    rng = random.Random(2)
    nb = (S + 100) // bs + 1
    q, kc, vc = (torch.randn(s, generator=g).to(torch.bfloat16) for s in ((S, H, D), (nb, bs, G, D), (nb, bs, G, D)))
    parents = [-1] + [rng.randrange(max(0, i - 300), i) for i in range(1, S)]
    mask = R.mask_words(R.ancestors(parents), 64)
    table = torch.randperm(nb, generator=g).view(1, nb)
    out, lse = dsa.paged_tree_fwd(q.to(dev), kc.to(dev), vc.to(dev), table.to(dev), mask.to(dev),
                                  actual_seq_lengths_query=[S], actual_seq_lengths_kv=[S + 77])
    o, ot, l, lt = R.attention(q, kc, vc, table, mask, [0], [S], [S], [S + 77], D ** -0.5)
    assert_within(out, o, ot, "out")
    assert_within(lse, l, lt, "lse")
