"""Measured calls of the dense attention layer around the sparse path, through the public entry points.

The layer is a serving step: an 8-bit projection of the quantised activations (``quant_matmul``),
the per-head norms of queries and keys with their position rotation, keys and values going to the
paged cache (``qk_norm_rope``, ``qk_norm_rope_paged``), and the attention of the new tokens over
that cache (``paged_gqa_fwd``).  ``own`` false: ``run`` computes the operators in elementary torch
operations in 32 bits; ``own`` true: it calls the package.  ``exact`` is the definition in 64 bits.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # One token's fused QKV projection (64 query and 2 x 4 key/value heads of 128): the weights' bytes.
        dict(name="qmm_token", kind="qmm", M=1, N=9216, K=7168, dtype="bf16", bias=False),
        # The output projection of a decode batch of 64 sequences.
        dict(name="qmm_batch", kind="qmm", M=64, N=7168, K=8192, dtype="bf16", bias=False),
        # A ragged chunk through a layer of odd sizes, with a bias, kept in 32 bits.
        dict(name="qmm_odd", kind="qmm", M=1021, N=2113, K=4099, dtype="fp32", bias=True),
        # The QKV projection of a whole 16K-token prompt.
        dict(name="qmm_prefill", kind="qmm", M=16384, N=9216, K=7168, dtype="bf16", bias=False),
        # A decode batch: 24 tokens at far positions, keys and values to their cache rows.
        dict(name="rope_decode", kind="rope", T=24, H=64, G=4, D=128, R=128, dtype="bf16", pairs="half", paged=True),
        # A chunk of a 64-wide model that rotates half of each head, neighbours paired; no cache.
        dict(name="rope_chunk", kind="rope", T=1021, H=24, G=8, D=64, R=32, dtype="fp16", pairs="next", paged=False),
        # A 32K-token prompt.
        dict(name="rope_prefill", kind="rope", T=32768, H=64, G=4, D=128, R=128, dtype="bf16", pairs="half", paged=True),
        # The smallest attention call: one new token of one sequence.
        dict(name="attn_token", kind="attn", lens="1:4097", H=64, G=4, D=128, block=64, win=-1, sinks=False,
             dtype="bf16"),
        # A decode batch: 64 sequences of 8K tokens.
        dict(name="attn_decode", kind="attn", lens="64x1:8192", H=64, G=4, D=128, block=64, win=-1, sinks=False,
             dtype="bf16"),
        # A serving step's mixed batch: chunks beside single tokens, window of 1024 keys, sinks, odd lengths.
        dict(name="attn_mixed", kind="attn", lens="511:7001 1:44444 1:123 257:257 1:9001 37:30001", H=64, G=8, D=64,
             block=128, win=1023, sinks=True, dtype="fp16"),
        # A 512-token chunk at the end of a 64K-token context.
        dict(name="attn_chunk", kind="attn", lens="512:65536", H=64, G=8, D=128, block=64, win=-1, sinks=False,
             dtype="bf16"),
        # A whole 16K-token prompt: the largest call.
        dict(name="attn_prefill", kind="attn", lens="16384:16384", H=64, G=4, D=128, block=128, win=-1, sinks=False,
             dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _lens(case):
    """(new tokens, keys) of each sequence, from "count x new:keys" words."""
    out = []
    for word in case["lens"].split():
        times, _, pair = word.rpartition("x")
        out += [tuple(int(n) for n in pair.split(":"))] * int(times or 1)
    return out


def _draw_lens(rng):
    """One chunk of a long context, whole prompts, a decode batch, or a decode batch with chunks in it."""
    shape = rng.choice(["chunk", "prompt", "decode", "mixed"])
    if shape == "prompt":
        s = _log_int(rng, 100, 12000)
        pairs = [(s, s)] * (1 if s > 3000 else rng.randint(1, 4))
    elif shape == "chunk":
        s = _log_int(rng, 2, 2000)
        pairs = [(s, s + _log_int(rng, 100, 60000 if s < 1000 else 20000))]
    else:
        pairs = [(1, _log_int(rng, 1, 20000)) for _ in range(_log_int(rng, 1, 64))]
        if shape == "mixed":
            for _ in range(rng.randint(1, 3)):
                s = _log_int(rng, 2, 1000)
                pairs.insert(rng.randint(0, len(pairs)), (s, s + _log_int(rng, 1, 30000)))
    return " ".join("%d:%d" % p for p in pairs)


def draw(rng):
    kind = rng.choice(["qmm", "qmm", "rope", "attn", "attn"])
    dt = rng.choice(["bf16", "bf16", "fp16"])
    if kind == "qmm":
        N, K = _log_int(rng, 256, 18000), _log_int(rng, 256, 18000)
        if rng.random() < 0.7:  # most layers' sizes are multiples of 64
            N, K = 64 * max(1, N // 64), 64 * max(1, K // 64)
        top = min(16384, 1082331758592 // (N * K))
        return dict(kind="qmm", M=_log_int(rng, 1, top), N=N, K=K, dtype=rng.choice([dt, dt, "fp32"]),
                    bias=rng.random() < 0.3)
    if kind == "rope":
        D = rng.choice([64, 128, 128, 256])
        G = rng.choice([1, 2, 4, 8])
        H = G * rng.choice([1, 4, 8, 16])
        return dict(kind="rope", T=_log_int(rng, 1, min(32768, 301989888 // ((H + 2 * G) * D))), H=H, G=G, D=D,
                    R=rng.choice([D, D, D // 2, 32]), dtype=dt, pairs=rng.choice(["half", "next"]),
                    paged=rng.random() < 0.6)
    G, D = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    H = G * rng.choice([m for m in (1, 4, 5, 8, 16) if G * m <= 64])
    return dict(kind="attn", lens=_draw_lens(rng), H=H, G=G, D=D, block=rng.choice([16, 64, 128]),
                win=rng.choice([-1, -1, -1, 127, 1023]), sinks=rng.random() < 0.3, dtype=dt)


# ------------------------------------------------------------------------------- inputs


def _gen(seed):
    dev = torch.device("cuda")
    return dev, torch.Generator(device=dev).manual_seed(seed)


def _normal(g, dev, shape, dtype, scale=1.0):
    return torch.randn(shape, generator=g, device=dev, dtype=dtype).mul_(scale)


def _int8_rows(g, dev, rows, n):
    """Rows as the row quantiser leaves them: normal values whose largest is near 127, and their scales."""
    x = torch.randn((rows, n), generator=g, device=dev)
    s = x.abs().amax(dim=1, keepdim=True).clamp_(min=1e-4).div_(127.0)
    return x.div_(s).round_().clamp_(-127, 127).to(torch.int8), s


def _tables(P, R, dev):
    """Cosines and sines of positions 0 .. P-1 at R/2 frequencies: angles in 64 bits, stored in 32."""
    freq = 10000.0 ** (-torch.arange(0, R, 2, device=dev, dtype=torch.float64) / R)
    ang = torch.arange(P, device=dev, dtype=torch.float64).view(-1, 1) * freq
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    dev, g = _gen(seed)
    c = dict(case)
    dt = _DT[c["dtype"]]
    st = {"case": c}
    if own:
        from __graft_entry__ import load_package

        st["pkg"] = load_package()
        st["pkg"].load_library()
    if c["kind"] == "qmm":
        st["x"], st["xs"] = _int8_rows(g, dev, c["M"], c["K"])
        st["w"], st["ws"] = _int8_rows(g, dev, c["N"], c["K"])
        st["ws"].mul_(c["K"] ** -0.5)
        st["bias"] = _normal(g, dev, (c["N"],), torch.float32) if c["bias"] else None
    elif c["kind"] == "rope":
        T, H, G, D = c["T"], c["H"], c["G"], c["D"]
        # The projection's output holds a token's queries, keys and values side by side.
        st["qkv"] = _normal(g, dev, (T, (H + 2 * G) * D), dt, 2.0)
        st["qw"] = (1 + _normal(g, dev, (D,), torch.float32, 0.1)).to(dt)
        st["kw"] = (1 + _normal(g, dev, (D,), torch.float32, 0.1)).to(dt)
        P = 65536
        st["cos"], st["sin"] = _tables(P, c["R"], dev)
        # Decode tokens sit anywhere; a chunk's are consecutive.
        if T <= 64:
            st["pos"] = torch.randint(0, P, (T,), generator=g, device=dev).to(torch.int32)
        else:
            st["pos"] = torch.arange(P - T, P, device=dev, dtype=torch.int32)
        if c["paged"]:
            bs = 64
            nb = -(-T // bs) + 3
            st["kc"] = _normal(g, dev, (nb, bs, G, D), dt)
            st["vc"] = _normal(g, dev, (nb, bs, G, D), dt)
            # Pages in random order; within a page tokens are consecutive.
            table = torch.randperm(nb, generator=g, device=dev)
            t = torch.arange(T, device=dev)
            st["slots"] = (table[t // bs] * bs + t % bs).to(torch.int32)
    else:
        lens, G, H, D, bs = _lens(c), c["G"], c["H"], c["D"], c["block"]
        T, B = sum(s for s, _ in lens), len(lens)
        nb = [-(-n // bs) for _, n in lens]
        total = sum(nb) + 1
        st["q"] = _normal(g, dev, (T, H, D), dt)
        st["kc"] = _normal(g, dev, (total, bs, G, D), dt)
        st["vc"] = _normal(g, dev, (total, bs, G, D), dt)
        order = torch.randperm(total, generator=g, device=dev).to(torch.int32)
        st["table"] = torch.zeros((B, max(nb)), dtype=torch.int32, device=dev)
        at = 0
        for b, n in enumerate(nb):
            st["table"][b, :n] = order[at:at + n]
            at += n
        st["cu"] = torch.tensor([s for s, _ in lens], device=dev).cumsum(0).to(torch.int32)
        st["kvl"] = torch.tensor([n for _, n in lens], device=dev).to(torch.int32)
        st["sinks"] = _normal(g, dev, (H,), torch.float32) if c["sinks"] else None
    return st


# ------------------------------------------------------------------------------- one pass


def _split(st):
    """Queries, keys and values of the projection's output: views of it."""
    c = st["case"]
    H, G, D, x = c["H"], c["G"], c["D"], st["qkv"]
    return (x[:, :H * D].view(-1, H, D), x[:, H * D:(H + G) * D].view(-1, G, D), x[:, (H + G) * D:].view(-1, G, D))


def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    pkg, c = st["pkg"], st["case"]
    if c["kind"] == "qmm":
        return pkg.quant_matmul(st["x"], st["w"], st["xs"], st["ws"], st["bias"], dtype=_DT[c["dtype"]])
    if c["kind"] == "rope":
        q, k, v = _split(st)
        if not c["paged"]:
            return pkg.qk_norm_rope(q, k, st["qw"], st["kw"], st["pos"], st["cos"], st["sin"],
                                    interleaved=c["pairs"] == "next")
        qo = pkg.qk_norm_rope_paged(q, k, v, st["qw"], st["kw"], st["pos"], st["cos"], st["sin"], st["kc"], st["vc"],
                                    st["slots"], interleaved=c["pairs"] == "next")
        return qo, st["kc"], st["vc"]
    return pkg.paged_gqa_fwd(st["q"], st["kc"], st["vc"], st["table"], actual_seq_lengths_query=st["cu"],
                             actual_seq_lengths_kv=st["kvl"], win_left=c["win"] if c["win"] >= 0 else None,
                             sinks=st["sinks"])


def _norm_rope(x, w, cos, sin, pairs, eps=1e-6):
    """Norm of each head of x [T, heads, D], its first 2 * cos.shape[1] elements rotated."""
    x = x.float()
    y = x * torch.rsqrt((x * x).mean(dim=-1, keepdim=True) + eps) * w.float()
    R = 2 * cos.shape[1]
    a, b = (y[..., :R // 2], y[..., R // 2:R]) if pairs == "half" else (y[..., 0:R:2], y[..., 1:R:2])
    c, s = cos.unsqueeze(1), sin.unsqueeze(1)
    ra, rb = a * c - b * s, b * c + a * s
    rot = torch.cat((ra, rb), dim=-1) if pairs == "half" else torch.stack((ra, rb), dim=-1).flatten(-2)
    return torch.cat((rot, y[..., R:]), dim=-1)


def _run_plain(st):
    c = st["case"]
    dt = _DT[c["dtype"]]
    if c["kind"] == "qmm":
        y = torch.mm(st["x"].float(), st["w"].float().t())
        y.mul_(st["xs"]).mul_(st["ws"].view(1, -1))
        if st["bias"] is not None:
            y.add_(st["bias"])
        return y.to(dt)
    if c["kind"] == "rope":
        q, k, v = _split(st)
        p = st["pos"].long()
        cos, sin = st["cos"][p], st["sin"][p]
        qo = _norm_rope(q, st["qw"], cos, sin, c["pairs"]).to(dt)
        ko = _norm_rope(k, st["kw"], cos, sin, c["pairs"]).to(dt)
        if not c["paged"]:
            return qo, ko
        at = st["slots"].long()
        st["kc"].view(-1, c["G"], c["D"])[at] = ko
        st["vc"].view(-1, c["G"], c["D"])[at] = v
        return qo, st["kc"], st["vc"]
    return _attend_plain(st, dt)


def _attend_plain(st, dt):
    c = st["case"]
    H, G, D, bs, win = c["H"], c["G"], c["D"], c["block"], c["win"]
    dev = st["q"].device
    out = torch.empty(st["q"].shape, dtype=dt, device=dev)
    lse = torch.empty(st["q"].shape[:2], dtype=torch.float32, device=dev)
    t0 = 0
    for b, (S, n) in enumerate(_lens(c)):
        rows = st["table"][b, :-(-n // bs)].long()
        k = st["kc"][rows].view(-1, G, D)[:n].float().permute(1, 2, 0).contiguous()
        v = st["vc"][rows].view(-1, G, D)[:n].float().permute(1, 0, 2).contiguous()
        step = max(1, (1 << 28) // (H * n))
        for s in range(0, S, step):
            m = min(step, S - s)
            q = st["q"][t0 + s:t0 + s + m].float().view(m, G, H // G, D).permute(1, 0, 2, 3).reshape(G, -1, D)
            x = torch.bmm(q, k).mul_(D ** -0.5).view(G, m, H // G, n)
            pos = torch.arange(n - S + s, n - S + s + m, device=dev).view(m, 1)
            col = torch.arange(n, device=dev).view(1, n)
            hide = col > pos
            if win >= 0:
                hide |= col < pos - win
            x.masked_fill_(hide.view(1, m, 1, n), -math.inf)
            top = x.amax(dim=-1, keepdim=True)
            if st["sinks"] is not None:
                sink = st["sinks"].view(G, 1, H // G, 1)
                top = torch.maximum(top, sink)
            e = x.sub_(top).exp_()
            total = e.sum(dim=-1, keepdim=True)
            if st["sinks"] is not None:
                total = total + torch.exp(sink - top)
            o = torch.bmm(e.view(G, -1, n), v).view(G, m, H // G, D).div_(total)
            out[t0 + s:t0 + s + m] = o.permute(1, 0, 2, 3).reshape(m, H, D).to(dt)
            lse[t0 + s:t0 + s + m] = (top + torch.log(total)).squeeze(-1).permute(1, 0, 2).reshape(m, H)
        t0 += S
    return out, lse


# ------------------------------------------------------------------------------- what a pass cannot do without


def _keys(S, n, win):
    """(query, key) pairs of S causal rows that end at n keys, and the keys any of them sees."""
    pairs = 0
    for p in range(n - S, n):
        pairs += min(p, win) + 1 if win >= 0 else p + 1
    return pairs, n if win < 0 else min(n, S + win)


def work(case):
    c = case
    sz = _SIZE[c["dtype"]]
    if c["kind"] == "qmm":
        M, N, K = c["M"], c["N"], c["K"]
        return {"bytes": M * K + N * K + 4 * (M + N) + (4 * N if c["bias"] else 0) + M * N * sz, "flops": 2 * M * N * K}
    if c["kind"] == "rope":
        heads = c["H"] + (2 if c["paged"] else 1) * c["G"]
        return {"bytes": c["T"] * (2 * heads * c["D"] * sz + 4 * c["R"] + (8 if c["paged"] else 4)), "flops": 0}
    seen = [_keys(s, n, c["win"]) for s, n in _lens(c)]
    T = sum(s for s, _ in _lens(c))
    return {"bytes": T * c["H"] * (2 * c["D"] * sz + 4) + sum(n for _, n in seen) * 2 * c["G"] * c["D"] * sz,
            "flops": 4 * c["H"] * c["D"] * sum(p for p, _ in seen)}


# ------------------------------------------------------------------------------- 64-bit results


def _exact_rope(x, w, cos, sin, pairs):
    x = x.double()
    y = x / (x.pow(2).mean(dim=-1, keepdim=True) + 1e-6).sqrt() * w.double()
    half = cos.shape[1]
    out = y.clone()
    for i in range(half):
        ia, ib = (i, half + i) if pairs == "half" else (2 * i, 2 * i + 1)
        c, s = cos[:, i].double().view(-1, 1), sin[:, i].double().view(-1, 1)
        out[..., ia] = y[..., ia] * c - y[..., ib] * s
        out[..., ib] = y[..., ia] * s + y[..., ib] * c
    return out


def _exact_attn(st):
    """One head at a time: softmax(q k^T / sqrt(D)) v over the keys a row sees, a sink's mass beside it."""
    c = st["case"]
    H, G, D, bs, win = c["H"], c["G"], c["D"], c["block"], c["win"]
    dev = st["q"].device
    out = torch.empty(st["q"].shape, dtype=torch.float64, device=dev)
    lse = torch.empty(st["q"].shape[:2], dtype=torch.float64, device=dev)
    first = 0
    for b, (S, n) in enumerate(_lens(c)):
        i = torch.arange(n, device=dev)
        row = st["table"][b].long()[i // bs] * bs + i % bs
        for h in range(H):
            g = h // (H // G)
            kt = st["kc"].view(-1, G, D)[row, g].double().t().contiguous()
            v = st["vc"].view(-1, G, D)[row, g].double()
            for a in range(0, S, 4096):
                z = min(S, a + 4096)
                w = (st["q"][first + a:first + z, h].double() @ kt) / math.sqrt(D)
                at = n - S + torch.arange(a, z, device=dev).view(-1, 1)
                see = i <= at
                if win >= 0:
                    see = see & (i >= at - win)
                w = torch.where(see, w, -math.inf)
                l = torch.logsumexp(w, dim=1)
                if st["sinks"] is not None:
                    l = torch.logaddexp(l, st["sinks"][h].double())
                out[first + a:first + z, h] = torch.exp(w - l.view(-1, 1)) @ v
                lse[first + a:first + z, h] = l
        first += S
    return out, lse


def exact(case, seed):
    st = prepare(case, seed)
    c = st["case"]
    if c["kind"] == "qmm":
        y = st["x"].double() @ st["w"].double().t().contiguous()
        y = y * st["xs"].double() * st["ws"].double().view(1, -1)
        return y if st["bias"] is None else y + st["bias"].double()
    if c["kind"] == "rope":
        q, k, v = _split(st)
        p = st["pos"].long()
        cos, sin = st["cos"][p], st["sin"][p]
        qo, ko = _exact_rope(q, st["qw"], cos, sin, c["pairs"]), _exact_rope(k, st["kw"], cos, sin, c["pairs"])
        if not c["paged"]:
            return qo, ko
        kc, vc = st["kc"].double(), st["vc"].double()
        for cache, rows in ((kc, ko), (vc, v.double())):
            cache.view(-1, c["G"], c["D"]).index_copy_(0, st["slots"].long(), rows)
        return qo, kc, vc
    return _exact_attn(st)
