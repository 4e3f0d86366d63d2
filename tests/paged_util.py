"""Plain 64-bit forms of the paged-step operators, for their GPU tests."""
import math

import numpy as np

HALF = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative


def torch_dtype(dt):
    import torch
    return {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dt]


def batch_plain(cached, added, free, head, table, page, tokens):
    """The step's bookkeeping, one request after the other."""
    table = table.copy()
    head = min(max(head, 0), len(free))
    seq, start, pos, slot, last, waits, admitted = [], [0], [], [], [], False, 0
    for r, (c, n) in enumerate(zip(cached, added)):
        c, n = max(int(c), 0), max(int(n), 0)
        first, end = -(-c // page), -(-(c + n) // page)
        waits = (waits or len(pos) + n > tokens or head + end - first > len(free) or end > table.shape[1]
                 or c + n > 2 ** 31 - 1)
        if waits:
            n = 0
        else:
            admitted += 1
            table[r, first:end] = free[head:head + end - first]
            head += end - first
        for p in range(c, c + n):
            pg = int(table[r, p // page])
            pos.append(p)
            s = pg * page + p % page
            slot.append(s if pg >= 0 and s < 2 ** 31 else -1)
        seq.append(c + n)
        start.append(len(pos))
        last.append(max(0, len(pos) - 1))
    pad = tokens - len(pos)
    return dict(seq_lens=seq, query_start=start, positions=pos + [0] * pad, slots=slot + [-1] * pad, last_rows=last,
                free_head_out=[head], admitted=[admitted], block_table=table)


def scatter_plain(qkv, nq, nkv, hd, cos, sin, qk_norm, q_norm, k_norm, norm_v, eps, add_one):
    """float64 q [T,Nq,Hd], k, v [T,Nkv,Hd] of qkv (torch)."""
    import torch
    x = qkv.double().reshape(-1, nq + 2 * nkv, hd)
    q, k, v = x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:]

    def norm(y, w):
        y = y / (y.square().mean(-1, keepdim=True) + float(np.float32(eps))).sqrt()
        return y if w is None else y * (w.double() + (1.0 if add_one else 0.0))

    def rope(y):
        a, b = y[..., :hd // 2], y[..., hd // 2:]
        c, s = cos.double()[:, None], sin.double()[:, None]
        return torch.cat([a * c - b * s, b * c + a * s], -1)

    if qk_norm:
        q, k = norm(q, q_norm), norm(k, k_norm)
    if norm_v:
        v = norm(v, None)
    if cos is not None:
        q, k = rope(q), rope(k)
    return q, k, v


def attention_plain(q, k_pages, v_pages, table, seq_lens, query_start, scale, kind, window, sinks):
    """(float64 out, sum_j p_j |v_j|, which rows belong to a request); numpy lengths, torch tensors. Only visible
    keys enter, so what the others hold does not matter."""
    import torch
    T, nq, hd = q.shape
    _, nkv, page, _ = k_pages.shape
    g = nq // nkv
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    mag = torch.zeros_like(out)
    owned = torch.zeros(T, dtype=torch.bool, device=q.device)
    for r, length in enumerate(seq_lens):
        t0, t1 = int(query_start[r]), int(query_start[r + 1])
        owned[t0:t1] = True
        if length == 0 or t1 == t0:
            continue
        j = torch.arange(length, device=q.device)
        rows = table[r].long()[j // page]
        k = k_pages[rows, :, j % page].double()  # [len, Nkv, Hd]
        v = v_pages[rows, :, j % page].double()
        pos = torch.arange(length - (t1 - t0), length, device=q.device)[:, None]
        seen = torch.ones(t1 - t0, length, dtype=torch.bool, device=q.device) if kind == 2 else j <= pos
        if kind == 1:
            seen = seen & ((pos - j < window) | (j < sinks))
        clean = ~seen.any(0)
        k[clean] = 0
        v[clean] = 0
        for h in range(nq):
            s = q[t0:t1, h].double() @ k[:, h // g].T * scale
            s = torch.where(seen, s, torch.full_like(s, -math.inf))
            m = s.amax(1, keepdim=True)
            p = torch.exp(s - torch.where(m.isinf(), torch.zeros_like(m), m))
            p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
            vv = v[:, h // g]
            if not torch.isfinite(vv).all():  # a row sums over the keys that it sees
                for i in range(t1 - t0):
                    out[t0 + i, h] = p[i, seen[i]] @ vv[seen[i]]
                    mag[t0 + i, h] = p[i, seen[i]] @ vv[seen[i]].abs()
                continue
            out[t0:t1, h] = p @ vv
            mag[t0:t1, h] = p @ vv.abs()
    return out, mag, owned


def attention_tolerance(out, mag, q, k_pages, scale, dt, hd):
    """Element bound. With h half a step of the type: the store rounds by h |o|; P in the type rounds each weight by
    h, and their sum by as much again: 2 h sum p|v|; a score is an fp32 dot of hd products, off by at most
    hd 2^-24 scale |q||k|, its exponential and the running rescaling by a few 2^-22, both entering numerator and
    denominator: twice that times sum p|v|."""
    import torch
    h = HALF[dt]
    kk = k_pages.float()
    kmax = torch.where(torch.isfinite(kk), kk, torch.zeros_like(kk)).norm(dim=-1).max().item()
    qmax = q.float().norm(dim=-1).max().item()
    ds = hd * 2.0 ** -24 * scale * kmax * qmax + 2.0 ** -19
    hp = 0.0 if dt == "f32" else 2 * h
    return h * out.abs() + (hp + 2 * ds) * mag + 1e-30


def sample_plain(x, u, t=1.0, k=0, p=1.0, m=0.0):
    """One row's token; x float64."""
    x = np.where(np.isnan(x), -np.inf, x)
    order = np.lexsort((np.arange(x.size), -x))
    top = x[order[0]]
    if top == -np.inf:
        return -1
    if not t > 0:
        return int(order[0])
    t = float(np.float32(t))
    if k > 0:
        order = order[:k]

    def weight(i):
        with np.errstate(invalid="ignore", over="ignore"):
            return np.where(x[i] == top, 1.0, np.where(x[i] == -np.inf, 0.0, np.exp((x[i] - top) / t)))
    if p < 1:
        c = np.cumsum(weight(order))
        n = int(np.searchsorted(c, float(np.float32(p)) * c[-1], side="left")) + 1
        order = order[:max(n, 1)]
    if m > 0:
        order = order[weight(order) >= min(float(np.float32(m)), 1.0)]
    order = np.sort(order)
    c = np.cumsum(weight(order))
    return int(order[min(np.searchsorted(c, float(np.float32(u)) * c[-1], side="right"), order.size - 1)])
