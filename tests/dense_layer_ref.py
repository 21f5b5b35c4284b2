"""The dense layer's operators in 64 bits, and what their kernels' roundings may add up to."""
import math

import torch


def half_step(dtype):
    """Largest relative error of one rounding to dtype."""
    return torch.finfo(dtype).eps / 2


F32 = half_step(torch.float32)


def quant_matmul(x, w, xs, ws, bias=None):
    """(result, tolerance before the output's rounding): x [M, K], w [N, K] int8."""
    y = (x.double() @ w.double().t()) * xs.double().view(-1, 1) * ws.double().view(1, -1)
    # The exact int32 sum is rounded once to fp32, scaled twice, and the bias is added: a half step each.
    tol = 3.01 * F32 * y.abs()
    if bias is not None:
        y = y + bias.double()
        tol = tol + F32 * (y.abs() + tol)
    return y, tol


def norm_rope(x, w, positions, cos, sin, eps=1e-6, interleaved=False):
    """(result, tolerance before the output's rounding): x [T, n, D]; zeros where a position is outside the table."""
    T, n, D = x.shape
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * w.double()
    P, half = cos.shape
    ok = (positions >= 0) & (positions < P)
    p = positions.long().clamp(0, max(P - 1, 0))
    out, mag = y.clone(), y.abs()
    if half and P:
        c, s = cos.double()[p].view(T, 1, half), sin.double()[p].view(T, 1, half)
        ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
        ib = ia + 1 if interleaved else ia + half
        a, b = y[..., ia], y[..., ib]
        out[..., ia], out[..., ib] = a * c - b * s, b * c + a * s
        mag[..., ia] = mag[..., ib] = (a * c).abs() + (b * s).abs() + (b * c).abs() + (a * s).abs()
    out[~ok] = 0
    # The sum of D squares: at most D half steps (under the root a half each, and its own and the division's), the
    # two products of the norm, the rotation's product and sum.
    return out, (D / 2 + 8) * F32 * mag


def attention(q, kc, vc, table, starts, spans, lens, kv_lens, scale, causal=True, win=-1, sinks=None):
    """(out, out tolerance, lse, lse tolerance), the roundings of a 16-bit kernel counted; one head at a time.

    Sequence b's rows are starts[b] .. + spans[b]; the first lens[b] hold tokens."""
    T, H, D = q.shape
    nb, bs, G, _ = kc.shape
    u = half_step(q.dtype)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    ltol = torch.zeros(T, H, dtype=torch.float64)
    if sinks is not None:
        # A row that sees nothing: its sink, to base 2 and back, is two products with rounded constants, four half
        # steps (log2(e) and ln(2) as fp32 numbers, and each product).
        lse[:] = sinks.double().view(1, -1)
        ltol[:] = 4.01 * F32 * lse.abs()
    kf, vf = kc.reshape(-1, G, D), vc.reshape(-1, G, D)
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0  # half a step of the smallest fp16 values
    for b, (t0, span, L, n) in enumerate(zip(starts, spans, lens, kv_lens)):
        if L == 0 or n == 0:
            continue
        j = torch.arange(n)
        page = table[b].long()[j // bs]
        there = (page >= 0) & (page < nb)
        rows = torch.where(there, page, 0) * bs + j % bs
        p = n - L + torch.arange(L).view(-1, 1)
        see = there.view(1, -1).expand(L, n)
        if causal:
            see = see & (j <= p)
        if win >= 0:
            see = see & (j >= p - win)
        for h in range(H):
            g = h // (H // G)
            k, v = kf[rows, g].double(), vf[rows, g].double()
            v = torch.where(there.view(-1, 1), v, 0)
            k = torch.where(there.view(-1, 1), k, 0)
            qq = q[t0:t0 + L, h].double()
            s = torch.where(see, qq @ k.t() * scale, -math.inf)
            l = torch.logsumexp(s, 1)
            # fp32 sums of D exact products, the scale and base-2 factor: error of a score.
            ds = (D + 4) * F32 * (qq.abs() @ k.abs().t()).max() * scale
            if sinks is not None:
                l = torch.logaddexp(l, sinks[h].double())
            w = torch.where(see, torch.exp(s - torch.where(torch.isinf(l), 0.0, l).view(-1, 1)), 0)
            o, mag = w @ v, w @ v.abs()
            top = torch.where(torch.isinf(s), -math.inf, s).amax(1)
            # l, less the row's largest score, is at least 0 but for a sink: the weights' rounding to 16 bits, below
            # fp16's normal range an absolute one against the sum of them; exponentials and sums in fp32.
            share = torch.exp(torch.where(torch.isinf(top), 0.0, top - l)).view(-1, 1)
            rel = u + 2 * ds + (n + 64) * F32 + 4e-7
            out[t0:t0 + L, h] = o
            tol[t0:t0 + L, h] = rel * mag + tiny * n * share * v.abs().amax() + u * o.abs() + tiny
            lse[t0:t0 + L, h] = l
            ltol[t0:t0 + L, h] = ds + (n + 64) * F32 + 1e-6 + 4 * F32 * torch.where(torch.isinf(l), 0.0, l.abs())
    return out, tol, lse, ltol


def assert_within(got, want, tol, what=""):
    got, want = got.double().cpu(), want.cpu()
    same = got == want  # infinities
    bad = ~(same | ((got - want).abs() <= tol.cpu()))
    if bad.any():
        i = tuple(torch.nonzero(bad)[0].tolist())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; first at {i}: {got[i]} for {want[i]}, "
                             f"tolerance {tol.cpu()[i] if tol.dim() else tol}")
