"""The dense layer's operators where offsets pass 31 and 32 bits, checked at samples."""
import pytest
import torch

import dense_layer_ref as ref

pytestmark = pytest.mark.gpu


def test_caches_past_4_gib(dsa, dev):
    """Pages and slots at the far end of pools of 4.3 GB each: decode, chunk, and the rows written there."""
    G, D, bs, H = 1, 128, 64, 16
    nb = 264000
    assert nb * bs * G * D * 2 > 2**32
    kc, vc = (torch.zeros(nb, bs, G, D, dtype=torch.bfloat16, device=dev) for _ in range(2))
    g = torch.Generator().manual_seed(1)
    seqs = [(1, 130), (200, 300)]
    pages = [[nb - 1, nb - 7, nb - 3], [nb - 20 + i for i in range(5)]]
    for row in pages:
        for p in row:
            kc[p] = torch.randn(bs, G, D, generator=g).bfloat16().to(dev)
            vc[p] = torch.randn(bs, G, D, generator=g).bfloat16().to(dev)
    # A copy of the pages in use, numbered from 0, for the 64-bit result.
    flat = [p for row in pages for p in row]
    small_k, small_v = kc[flat].cpu(), vc[flat].cpu()
    table = torch.zeros(2, 5, dtype=torch.int32)
    small = torch.zeros(2, 5, dtype=torch.int32)
    table[0, :3], table[1] = torch.tensor(pages[0]), torch.tensor(pages[1])
    small[0, :3], small[1] = torch.arange(3), torch.arange(3, 8)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    for sel in ([0], [0, 1]):  # few rows a sequence, many rows a sequence
        part = [seqs[i] for i in sel]
        T = sum(s for s, _ in part)
        q = torch.randn(T, H, D, generator=g).bfloat16()
        cu = torch.tensor([s for s, _ in part]).cumsum(0).to(torch.int32).to(dev)
        out, lse = dsa.paged_gqa_fwd(q.to(dev), kc, vc, table[sel].to(dev), actual_seq_lengths_query=cu,
                                     actual_seq_lengths_kv=i32([n for _, n in part]))
        starts = [sum(s for s, _ in part[:b]) for b in range(len(part))]
        lens = [s for s, _ in part]
        o, tol, l, ltol = ref.attention(q, small_k, small_v, small[sel], starts, lens, lens, [n for _, n in part],
                                        D ** -0.5)
        ref.assert_within(out, o, tol, "out")
        ref.assert_within(lse, l, ltol, "lse")
    k, v = torch.randn(2, G, D, generator=g).bfloat16(), torch.randn(2, G, D, generator=g).bfloat16()
    cos, sin = torch.ones(4, D // 2), torch.zeros(4, D // 2)
    pos = torch.tensor([1, 2], dtype=torch.int32)
    slots = torch.tensor([nb * bs - 1, nb * bs - 2], dtype=torch.int32)
    dsa.qk_norm_rope_paged(k.to(dev), k.to(dev), v.to(dev), None, None, pos.to(dev), cos.to(dev), sin.to(dev), kc, vc,
                           slots.to(dev))
    want, tol = ref.norm_rope(k, None, pos, cos, sin)
    got = kc[-1, [-1, -2]]
    ref.assert_within(got, want, tol + ref.half_step(torch.bfloat16) * (want.abs() + tol))
    assert torch.equal(vc[-1, [-1, -2]].cpu(), v)


def test_norms_past_2_31_elements(dsa, dev):
    T, H, G, D = 280000, 62, 2, 128
    assert T * H * D > 2**31
    q = torch.full((T, H, D), 2.0, dtype=torch.bfloat16, device=dev)
    q[:, :, ::2] = -1.0
    k = q[:, :G]  # strided view
    cos, sin = torch.ones(1, D // 2, device=dev), torch.zeros(1, D // 2, device=dev)
    pos = torch.zeros(T, dtype=torch.int32, device=dev)
    qo, ko = dsa.qk_norm_rope(q, k, None, None, pos, cos, sin)
    del q
    at = torch.tensor([0, 1, T // 2, T - 1], device=dev)
    row = torch.tensor([-1.0, 2.0], dtype=torch.float64).repeat(D // 2) / (2.5 + 1e-6) ** 0.5
    tol = row.abs() * (ref.half_step(torch.bfloat16) + (D / 2 + 8) * ref.F32)
    for x in (qo, ko):
        ref.assert_within(x[at], row.expand(4, x.shape[1], D), tol.expand(4, x.shape[1], D))


@pytest.mark.parametrize("M,N,K", [(70000, 31000, 16), (16500, 33, 131071), (8, 16500, 131071)])
def test_products_past_2_31(dsa, dev, M, N, K):
    """More than 2^31 outputs, bytes of x, bytes of w."""
    assert max(M * N, M * K, N * K) > 2**31
    g = torch.Generator(device=dev).manual_seed(K)
    x = torch.randint(-127, 128, (M, K), dtype=torch.int8, device=dev, generator=g)
    w = torch.randint(-127, 128, (N, K), dtype=torch.int8, device=dev, generator=g)
    xs, ws = torch.rand(M, device=dev, generator=g), torch.rand(N, device=dev, generator=g)
    out = dsa.quant_matmul(x, w, xs, ws)
    mi = torch.tensor([0, M // 3, M - 2, M - 1], device=dev)
    ni = torch.tensor([0, N // 2, N - 2, N - 1], device=dev)
    want, tol = ref.quant_matmul(x[mi].cpu(), w[ni].cpu(), xs[mi].cpu(), ws[ni].cpu())
    got = out[mi][:, ni]
    ref.assert_within(got, want, tol + ref.half_step(torch.bfloat16) * (want.abs() + tol))
