"""A tree-drafted decoding step's operators, plainly: page plan, attention in 64 bits with what its kernels' roundings may
add up to, acceptance and the cache rows' order."""
import math

import torch

from dense_layer_ref import F32, half_step

TOP = 2**30  # lengths count up to this


def tree(rng, S, hang=0.0):
    """Parents of S nodes, each behind its own; a share of them hangs nowhere."""
    return [-1 if i == 0 or rng.random() < hang else rng.randrange(max(0, i - 6), i) for i in range(S)]


def ancestors(parents):
    """For each node itself and its ancestors, itself first; parents that are not before their child are none."""
    out = []
    for i, p in enumerate(parents):
        out.append([i] + (out[p] if 0 <= p < i else []))
    return out


def mask_words(chains, W, win=-1):
    rows = []
    for chain in chains:
        words = [0] * W
        for a in chain[:win + 1] if win >= 0 else chain:
            if a < 64 * W:
                words[a // 64] |= 1 << (a % 64)
        rows.append([w - 2**64 if w >= 2**63 else w for w in words])
    return torch.tensor(rows, dtype=torch.int64).reshape(len(chains), W)


def plan(new, ctx, table, free, count, bs, T, parents=None, max_nodes=0, win=-1):
    """(cu, kv, positions, slots, missing, mask or None); table (a list of rows) and count (a list of one) change."""
    cap = lambda x: min(max(x, 0), TOP)
    mb, n = len(table[0]), min(max(count[0], 0), len(free))
    cu, kv, pos, slots, missing, masks, t = [], [], [], [], [], [], 0
    W = -(-max_nodes // 64)
    for b, (S, at) in enumerate(zip(new, ctx)):
        S, at = min(cap(S), T - t), cap(at)
        short = 0
        for j in range(at // bs, (at + S - 1) // bs + 1 if S else 0):
            if j >= mb:
                short += 1
            elif table[b][j] < 0:
                if n > 0:
                    n -= 1
                    table[b][j] = free[n]
                else:
                    short += 1
        chains = ancestors(parents[t:t + S]) if parents is not None else None
        if parents is not None:
            masks.append(mask_words(chains, W, win))
        for i in range(S):
            j = (at + i) // bs
            page = table[b][j] if j < mb else -1
            slot = page * bs + (at + i) % bs
            slots.append(slot if page >= 0 and slot < 2**31 else -1)
            pos.append(at + (len(chains[i]) - 1 if chains is not None else i))
        t += S
        cu.append(t)
        kv.append(at + S)
        missing.append(short)
    count[0] = n
    pad = T - t
    if parents is not None:
        masks.append(torch.zeros(pad, W, dtype=torch.int64))
    return (cu, kv, pos + [-1] * pad, slots + [-1] * pad, missing, torch.cat(masks) if masks else None)


def free(keep, table, free_list, count, bs):
    """Changes table, free_list and count (lists)."""
    n, room, back = min(max(count[0], 0), len(free_list)), len(free_list), []
    for b, k in enumerate(keep):
        k = min(max(k, 0), TOP)
        for j in range(-(-k // bs), len(table[b])):
            if table[b][j] < 0:
                break
            back.append((b, j))
    for i, (b, j) in enumerate(back):
        to = n + len(back) - 1 - i
        if to < room:
            free_list[to] = table[b][j]
            table[b][j] = -1
    count[0] = min(n + len(back), room)


def accept(scores, tokens, parents, cu, P):
    """(accepted, path, chosen): scores a [T, V] tensor, or a list of choices."""
    out, t = [], 0
    for end in cu:
        path, chosen, at = [], [], 0
        while end > t and at >= 0 and len(path) < P:
            if isinstance(scores, torch.Tensor):
                x = scores[t + at].double()
                x = torch.where(torch.isnan(x), -math.inf, x)
                want = -1 if x.max() == -math.inf else int(torch.nonzero(x == x.max())[0])
            else:
                want = scores[t + at]
            path.append(at)
            chosen.append(want)
            at = next((i for i in range(at + 1, end - t) if parents[t + i] == at and tokens[t + i] == want and want >= 0), -1)
        out.append((len(path), path + [-1] * (P - len(path)), chosen + [-1] * (P - len(chosen))))
        t = end
    return tuple(torch.tensor([o[k] for o in out], dtype=torch.int32) for k in range(3))


def commit(caches, table, ctx, path, accepted):
    """Rows of the caches (CPU tensors), one after the other, in place."""
    nb, bs = caches[0].shape[:2]

    def row(b, j):
        page = table[b][j // bs] if j // bs < len(table[b]) else -1
        return page * bs + j % bs if 0 <= page < nb else -1

    for b, n in enumerate(accepted):
        for k in range(min(max(n, 0), len(path[b]))):
            if path[b][k] <= k:
                continue
            src, to = row(b, ctx[b] + path[b][k]), row(b, ctx[b] + k)
            if src >= 0 and to >= 0:
                for c in caches:
                    flat = c.view(nb * bs, -1)
                    flat[to] = flat[src].clone()


def attention(q, kc, vc, table, mask, starts, spans, lens, kv_lens, scale, positions=None, win=-1, sinks=None):
    """(out, out tolerance, lse, lse tolerance) of nodes: sequence b's rows are starts[b] .. + spans[b], the first lens[b]
    of them nodes.  The tolerances count a 16-bit kernel's roundings, as the dense attention's do."""
    T, H, D = q.shape
    nb, bs, G, _ = kc.shape
    u = half_step(q.dtype)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    ltol = torch.zeros(T, H, dtype=torch.float64)
    if sinks is not None:
        lse[:] = sinks.double().view(1, -1)
        ltol[:] = 4.01 * F32 * lse.abs()
    kf, vf = kc.reshape(-1, G, D), vc.reshape(-1, G, D)
    tiny = 2.0 ** -25 if q.dtype == torch.float16 else 0.0
    W = mask.shape[-1]
    for b, (t0, span, L, n) in enumerate(zip(starts, spans, lens, kv_lens)):
        if L == 0 or n == 0:
            continue
        first = n - L
        j = torch.arange(n)
        page = table[b].long()[j // bs]
        there = (page >= 0) & (page < nb)
        rows = torch.where(there, page, 0) * bs + j % bs
        node = j - first
        known = (node >= 0) & (node < 64 * W)
        at = torch.where(known, node, 0)
        see = ((mask[t0:t0 + L][:, at // 64] >> (at % 64)) & 1).bool() & known
        old = j < first
        if win >= 0:
            p = positions[t0:t0 + L].long().clamp(first, n - 1).view(-1, 1)
            see = see | (old & (j >= p.clamp(min=0) - win))
        else:
            see = see | old
        see = see & there
        for h in range(H):
            g = h // (H // G)
            k, v = kf[rows, g].double(), vf[rows, g].double()
            # What no row sees must not matter, whatever it is.
            dead = ~(there & see.any(0))
            v = torch.where(dead.view(-1, 1), 0, v)
            k = torch.where(dead.view(-1, 1), 0, k)
            qq = q[t0:t0 + L, h].double()
            s = torch.where(see, qq @ k.t() * scale, -math.inf)
            l = torch.logsumexp(s, 1)
            ds = (D + 4) * F32 * (qq.abs() @ k.abs().t()).max() * scale
            if sinks is not None:
                l = torch.logaddexp(l, sinks[h].double())
            w = torch.where(see, torch.exp(s - torch.where(torch.isinf(l), 0.0, l).view(-1, 1)), 0)
            o, mag = w @ v, w @ v.abs()
            top = torch.where(torch.isinf(s), -math.inf, s).amax(1)
            share = torch.exp(torch.where(torch.isinf(top), 0.0, top - l)).view(-1, 1)
            rel = u + 2 * ds + (n + 64) * F32 + 4e-7
            out[t0:t0 + L, h] = o
            tol[t0:t0 + L, h] = rel * mag + tiny * n * share * v.abs().amax() + u * o.abs() + tiny
            lse[t0:t0 + L, h] = l
            ltol[t0:t0 + L, h] = ds + (n + 64) * F32 + 1e-6 + 4 * F32 * torch.where(torch.isinf(l), 0.0, l.abs())
    return out, tol, lse, ltol
