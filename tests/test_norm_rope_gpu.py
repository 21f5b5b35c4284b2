"""Head norms with rotation on the GPU: 64-bit results, views, caches, padding, refusals."""
import math

import pytest
import torch

import dense_layer_ref as ref

pytestmark = pytest.mark.gpu


def _tables(P, R):
    ang = torch.arange(P, dtype=torch.float64).view(-1, 1) * (10000.0 ** (-torch.arange(0, R, 2).double() / max(R, 1)))
    return ang.cos().float(), ang.sin().float()


def _within(got, want, tol):
    u = ref.half_step(got.dtype)
    ref.assert_within(got, want, tol + u * (want.abs() + tol) + (2.0 ** -25 if got.dtype == torch.float16 else 0))


CASES = [(1, 1, 1, 8, 0), (1, 64, 4, 128, 128), (5, 8, 2, 64, 32), (3, 3, 3, 96, 48), (7, 24, 8, 64, 64), (2, 16, 1, 256, 64),
         (9, 2, 1, 512, 512), (33, 5, 5, 128, 16), (130, 10, 2, 200, 160), (4, 1, 1, 72, 16), (3, 2, 2, 24, 16)]


@pytest.mark.parametrize("T,H,G,D,R", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_against_64_bits(dsa, dev, T, H, G, D, R, interleaved, dtype):
    g = torch.Generator().manual_seed(T + H + D + R)
    q, k = (torch.randn(T, H, D, generator=g) * 3).to(dtype), torch.randn(T, G, D, generator=g).to(dtype)
    qw, kw = (1 + torch.randn(D, generator=g) / 10).to(dtype), torch.randn(D, generator=g).to(dtype)
    P = 5000
    cos, sin = _tables(P, R)
    pos = torch.randint(0, P, (T,), generator=g).to(torch.int32)
    a = [t.to(dev) for t in (q, k, qw, kw, pos, cos, sin)]
    qo, ko = dsa.qk_norm_rope(*a, interleaved=interleaved)
    _within(qo, *ref.norm_rope(q, qw, pos, cos, sin, interleaved=interleaved))
    _within(ko, *ref.norm_rope(k, kw, pos, cos, sin, interleaved=interleaved))
    if dtype == torch.bfloat16:
        ops = dsa.load_torch_ops()
        q2, k2 = ops.qk_norm_rope(*a, 1e-6, interleaved)
        assert torch.equal(q2, qo) and torch.equal(k2, ko)


@pytest.mark.parametrize("kind", ["none", "fp32", "q only"])
def test_weights(dsa, dev, kind):
    g = torch.Generator().manual_seed(1)
    T, H, G, D, R = 6, 4, 2, 128, 64
    q, k = torch.randn(T, H, D, generator=g).half(), torch.randn(T, G, D, generator=g).half()
    qw = None if kind == "none" else torch.randn(D, generator=g)
    kw = torch.randn(D, generator=g) if kind == "fp32" else None
    cos, sin = _tables(64, R)
    pos = torch.arange(T)
    up = lambda t: None if t is None else t.to(dev)
    qo, ko = dsa.qk_norm_rope(up(q), up(k), up(qw), up(kw), up(pos), up(cos), up(sin), eps=1e-3)
    _within(qo, *ref.norm_rope(q, qw, pos, cos, sin, eps=1e-3))
    _within(ko, *ref.norm_rope(k, kw, pos, cos, sin, eps=1e-3))


@pytest.mark.parametrize("T,H,G,D,R", [(1, 8, 2, 128, 128), (21, 8, 2, 64, 32), (70, 12, 3, 96, 96)])
@pytest.mark.parametrize("interleaved", [False, True])
def test_paged(dsa, dev, T, H, G, D, R, interleaved):
    """Views of one projection in, keys and values to their cache rows; every other row is left as it was."""
    g = torch.Generator().manual_seed(T)
    bs, nb = 16, 9
    qkv = torch.randn(T, (H + 2 * G) * D + 8, generator=g).bfloat16().to(dev)
    q = qkv[:, :H * D].view(T, H, D)
    k = qkv[:, H * D:(H + G) * D].view(T, G, D)
    v = qkv[:, (H + G) * D:(H + 2 * G) * D].view(T, G, D)
    qw, kw = torch.randn(D, generator=g).bfloat16().to(dev), torch.randn(D, generator=g).bfloat16().to(dev)
    cos, sin = (t.to(dev) for t in _tables(100, R))
    pos = torch.randint(0, 100, (T,), generator=g).to(torch.int32)
    slots = torch.randperm(nb * bs, generator=g)[:T].to(torch.int32)
    if T > 4:
        pos[1], pos[2], slots[3], slots[4] = -1, 100, -1, nb * bs  # padding, and tokens without a row
    kc0 = torch.randn(nb, bs, G, D, generator=g).bfloat16()
    vc0 = torch.randn(nb, bs, G, D, generator=g).bfloat16()
    kc, vc = kc0.to(dev), vc0.to(dev)
    qo = dsa.qk_norm_rope_paged(q, k, v, qw, kw, pos.to(dev), cos, sin, kc, vc, slots.to(dev),
                                interleaved=interleaved)
    q2, ko = dsa.qk_norm_rope(q, k, qw, kw, pos.to(dev), cos, sin, interleaved=interleaved)
    assert torch.equal(qo, q2)
    want_k, want_v = kc0.view(-1, G, D), vc0.view(-1, G, D)
    for t in range(T):
        s = int(slots[t])
        if 0 <= s < nb * bs and 0 <= int(pos[t]) < 100:
            want_k[s], want_v[s] = ko[t].cpu(), v[t].cpu()
    assert torch.equal(kc.cpu().view(-1, G, D), want_k) and torch.equal(vc.cpu().view(-1, G, D), want_v)
    _within(qo, *ref.norm_rope(q.cpu(), qw.cpu(), pos, cos.cpu(), sin.cpu(), interleaved=interleaved))
    if T > 4:
        assert (qo[1:3] == 0).all()
    # The registered operator writes the same caches; int64 positions and slots take the Python route.
    ops = dsa.load_torch_ops()
    for call in (lambda a, b: ops.qk_norm_rope_paged(q, k, v, qw, kw, pos.to(dev), cos, sin, a, b, slots.to(dev), 1e-6,
                                                     interleaved),
                 lambda a, b: dsa.qk_norm_rope_paged(q, k, v, qw, kw, pos.long().to(dev), cos, sin, a, b,
                                                     slots.long().to(dev), interleaved=interleaved)):
        a, b = kc0.to(dev), vc0.to(dev)
        kc3, vc3 = kc.clone(), vc.clone()
        a.copy_(kc3), b.copy_(vc3)
        assert torch.equal(call(a, b), qo)
        assert torch.equal(a, kc) and torch.equal(b, vc)


@pytest.mark.parametrize("interleaved", [False, True])
def test_many_tokens(dsa, dev, interleaved):
    """Enough rows that a group takes several heads of a token; 29 rows a token, in sets that do not end with it."""
    T, H, G, D, R, bs = 9101, 23, 3, 64, 48, 128
    g = torch.Generator().manual_seed(11)
    q, k, v = (torch.randn(T, n, D, generator=g).bfloat16() for n in (H, G, G))
    qw, kw = torch.randn(D, generator=g), torch.randn(D, generator=g)
    cos, sin = _tables(T, R)
    pos = torch.randperm(T, generator=g).to(torch.int32)
    nb = T // bs + 2
    slots = torch.randperm(nb * bs, generator=g)[:T].to(torch.int32)
    kc, vc = torch.zeros(nb, bs, G, D, dtype=torch.bfloat16, device=dev), torch.zeros(nb, bs, G, D, dtype=torch.bfloat16,
                                                                                     device=dev)
    up = lambda t: t.to(dev)
    qo = dsa.qk_norm_rope_paged(up(q), up(k), up(v), up(qw), up(kw), up(pos), up(cos), up(sin), kc, vc, up(slots),
                                interleaved=interleaved)
    _within(qo, *ref.norm_rope(q, qw, pos, cos, sin, interleaved=interleaved))
    at = slots.long()
    kv, vv = kc.cpu().view(-1, G, D), vc.cpu().view(-1, G, D)
    _within(kv[at], *ref.norm_rope(k, kw, pos, cos, sin, interleaved=interleaved))
    assert torch.equal(vv[at], v)
    rest = torch.ones(nb * bs, dtype=torch.bool)
    rest[at] = False
    assert (kv[rest] == 0).all() and (vv[rest] == 0).all()


def test_wide_slots_do_not_wrap(dsa, dev):
    """64-bit slots and positions past 32 bits mark padding, they do not come back as small ones."""
    q = torch.ones(2, 1, 16, dtype=torch.bfloat16, device=dev)
    cos, sin = (t.to(dev) for t in _tables(8, 16))
    kc = torch.zeros(1, 8, 1, 16, dtype=torch.bfloat16, device=dev)
    vc = torch.zeros_like(kc)
    pos = torch.tensor([1, 2**32 + 1], device=dev)
    slots = torch.tensor([2**32 + 3, 2], device=dev)
    for f in (dsa.qk_norm_rope_paged, dsa.load_torch_ops().qk_norm_rope_paged):
        qo = f(q, q, q, None, None, pos, cos, sin, kc, vc, slots)
        assert (kc == 0).all() and (vc == 0).all()
        assert (qo[1] == 0).all() and (qo[0] != 0).any()


def test_values_out_of_the_ordinary(dsa, dev):
    """A row of zeros, a large and a tiny one; a NaN and an infinity stay in their heads."""
    D, R = 64, 64
    x = torch.zeros(4, 3, D, dtype=torch.bfloat16)
    g = torch.Generator().manual_seed(2)
    x[1] = (torch.randn(3, D, generator=g) * 1e15).bfloat16()
    x[2] = (torch.randn(3, D, generator=g) * 1e-20).bfloat16()
    x[3] = torch.randn(3, D, generator=g).bfloat16()
    bad = x.clone()
    bad[3, 1, 5], bad[3, 2, 7] = math.nan, math.inf
    cos, sin = _tables(8, R)
    pos = torch.arange(4).to(torch.int32)
    up = lambda t: t.to(dev)
    qo, _ = dsa.qk_norm_rope(up(x), up(x), None, None, up(pos), up(cos), up(sin))
    want, tol = ref.norm_rope(x, None, pos, cos, sin)
    # Squares of 1e-20 vanish beside eps in either precision.
    _within(qo, want, tol + 1e-30)
    qb, _ = dsa.qk_norm_rope(up(bad), up(bad), None, None, up(pos), up(cos), up(sin))
    assert torch.equal(qb[:3], qo[:3]) and torch.equal(qb[3, 0], qo[3, 0])
    assert torch.isnan(qb[3, 1]).all()


def test_refusals(dsa, dev):
    q = torch.zeros(4, 2, 64, dtype=torch.bfloat16, device=dev)
    cos, sin = (t.to(dev) for t in _tables(8, 64))
    pos = torch.zeros(4, dtype=torch.int32, device=dev)
    call = lambda q=q, k=q, qw=None, kw=None, pos=pos, cos=cos, sin=sin, **kw_: dsa.qk_norm_rope(q, k, qw, kw, pos, cos,
                                                                                                sin, **kw_)
    call()
    with pytest.raises(ValueError, match="bfloat16"):
        call(q=q.float())
    with pytest.raises(ValueError, match="dtype"):
        call(k=q.half())
    with pytest.raises(ValueError, match="k must be"):
        call(k=q[:3])
    with pytest.raises(ValueError, match="contiguous"):
        call(q=q.transpose(0, 1).contiguous().transpose(0, 1))
    with pytest.raises(ValueError, match="16 bytes"):
        call(q=torch.zeros(4, 132, dtype=torch.bfloat16, device=dev)[:, 4:].view(4, 2, 64))
    with pytest.raises(ValueError, match="q_weight"):
        call(qw=torch.ones(63, device=dev))
    with pytest.raises(ValueError, match="one dtype"):
        call(qw=torch.ones(64, device=dev), kw=torch.ones(64, dtype=torch.bfloat16, device=dev))
    with pytest.raises(ValueError, match="positions"):
        call(pos=pos[:3])
    with pytest.raises(ValueError, match="multiple of 16"):
        call(cos=cos[:, :4].contiguous(), sin=sin[:, :4].contiguous())
    with pytest.raises(ValueError, match="float32"):
        call(cos=cos.double(), sin=sin.double())
    with pytest.raises(ValueError, match="eps"):
        call(eps=-1.0)
    kc = torch.zeros(2, 8, 2, 64, dtype=torch.bfloat16, device=dev)
    paged = lambda kc=kc, vc=kc.clone(), slots=pos, v=q: dsa.qk_norm_rope_paged(q, q, v, None, None, pos, cos, sin, kc,
                                                                               vc, slots)
    with pytest.raises(ValueError, match="k_cache"):
        paged(kc=kc[..., :32].contiguous())
    with pytest.raises(ValueError, match="v_cache"):
        paged(vc=kc[:1])
    with pytest.raises(ValueError, match="slots"):
        paged(slots=pos[:2])
    with pytest.raises(ValueError, match="v has"):
        paged(v=q[:, :1])
    with pytest.raises(ValueError, match="required"):
        paged(v=None)
    with pytest.raises(ValueError, match="caches of their own"):
        paged(vc=kc)
