"""Plain fp64 forms of the token mixers (attention over the INT8 cache, drafted trees, gated delta rule) for the
tests, written from the definitions: every (query, position) pair is looked at on its own."""
from __future__ import annotations

import math

import torch

PIN = 4096


def ring_cell(j: int, cap: int) -> int:
    if cap <= 2 * PIN or j < PIN:
        return j % cap if cap <= 2 * PIN else j
    return PIN + (j - PIN) % (cap - PIN)


def in_ring(j: int, end: int, cap: int) -> bool:
    if cap <= 2 * PIN:
        return j >= end - cap
    return j < PIN or j >= max(PIN, end - (cap - PIN))


def seen(p, end, max_ctx, window, sinks, cap):
    """Positions that a query at p sees (cap None: the full-context mirror)."""
    hi = min(p + 1, end, max_ctx)
    js = set(range(max(0, p - window + 1), hi)) | set(range(0, min(sinks, hi)))
    return sorted(j for j in js if cap is None or in_ring(j, end, cap))


def rows64(codes, scales, hd, head):
    """fp64 rows [cells, hd] of one kv head."""
    c = codes[:, head * hd:(head + 1) * hd].double().unflatten(1, (-1, 64))
    s = scales.view(torch.float16)[:, head * hd // 64:(head + 1) * hd // 64].double()
    return (c * s.unsqueeze(-1)).flatten(1)


def attention(q, cells, kvh, hd, scale, rows, drafts=None, draft_rows=None):
    """rows[t]: the cells that query t sees; draft_rows[t]: the drafts. Returns out, lse and, per output element,
    mag = sum_j p_j |v_j| and (per row) dot = max_j scale * sum_d |q_d k_d|, which the bounds are made of."""
    T, qh, _ = q.shape
    dev = q.device
    out = torch.zeros(T, qh, hd, dtype=torch.float64, device=dev)
    mag, lse = torch.zeros_like(out), torch.full((T, qh), -math.inf, dtype=torch.float64, device=dev)
    dot = torch.zeros(T, qh, dtype=torch.float64, device=dev)
    for h in range(kvh):
        k, v = rows64(cells[0], cells[1], hd, h), rows64(cells[2], cells[3], hd, h)
        if drafts is not None:
            dk, dv = rows64(drafts[0], drafts[1], hd, h), rows64(drafts[2], drafts[3], hd, h)
        for t in range(T):
            at = torch.tensor(rows[t], dtype=torch.long, device=dev)
            kk, vv = k[at], v[at]
            if drafts is not None:
                at = torch.tensor(draft_rows[t], dtype=torch.long, device=dev)
                kk, vv = torch.cat([kk, dk[at]]), torch.cat([vv, dv[at]])
            if kk.shape[0] == 0:
                continue
            g = slice(h * qh // kvh, (h + 1) * qh // kvh)
            x = scale * (q[t, g].double() @ kk.T)
            dot[t, g] = scale * (q[t, g].double().abs() @ kk.abs().T).amax(1)
            p = torch.softmax(x, 1)
            lse[t, g] = torch.logsumexp(x, 1)
            out[t, g], mag[t, g] = p @ vv, p @ vv.abs()
    return out, lse, mag, dot


def delta_rule(q, k, v, g, beta, state, scale, l2_eps=None):
    """Token by token. state [heads, v, k] or None."""
    T, kh, d = q.shape
    vh = v.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    if l2_eps is not None:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + l2_eps)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + l2_eps)
    q, k = (x.repeat_interleave(vh // kh, 1) for x in (q, k))
    s = torch.zeros(vh, d, d, dtype=torch.float64, device=q.device) if state is None else state.double().clone()
    o, snaps = torch.zeros_like(v), []
    for t in range(T):
        s = s * torch.exp(g[t].double())[:, None, None]
        e = beta[t].double()[:, None] * (v[t] - torch.einsum("hvk,hk->hv", s, k[t]))
        s = s + e[:, :, None] * k[t][:, None, :]
        o[t] = scale * torch.einsum("hvk,hk->hv", s, q[t])
        snaps.append(s)
    return o, s, snaps
