"""The token mixers of a hybrid layer as measured cases: attention over the INT8 KV cache (sliding window and
pinned first tokens), attention for a tree of drafted tokens over the same cache, and the gated delta rule.

`run` computes a case in its plain form (elementary torch operations, fp32) or, where `own` is true, through the
framework's entry points. `exact` computes the same from the definition in fp64.
"""
import math
import os
import sys

import torch

own = False

GROUP = 64   # elements per cache scale
SINK_PIN = 4096  # ring cells pinned to the first positions when ring_cap > 2 * SINK_PIN
CHUNK = 64   # tokens per chunk of the plain delta rule


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _library():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "wzy-flash-serve_b200")
    if path not in sys.path:
        sys.path.insert(0, path)
    import wzyb200

    return wzyb200


def _attn(name, T, qh, kvh, hd, base, window, sinks, source, cap, dtype, gated_q=False):
    return {"name": name, "op": "attn", "T": T, "qh": qh, "kvh": kvh, "hd": hd, "base": base, "window": window,
            "sinks": sinks, "source": source, "cap": cap, "dtype": dtype, "gated_q": gated_q}


def _tree(name, N, qh, kvh, hd, base, window, sinks, source, cap, dtype):
    return {"name": name, "op": "tree", "T": N, "qh": qh, "kvh": kvh, "hd": hd, "base": base, "window": window,
            "sinks": sinks, "source": source, "cap": cap, "dtype": dtype, "gated_q": False}


def _gdn(name, T, kh, vh, hd, dtype, packed, l2, snaps):
    return {"name": name, "op": "gdn", "T": T, "kh": kh, "vh": vh, "hd": hd, "dtype": dtype, "packed": packed,
            "l2": l2, "snaps": snaps}


def listed():
    return [
        # one decoded token of the fp16 configuration's layer in a short chat, ring not yet full
        _attn("attn_decode_ring_5k_f16", 1, 16, 2, 256, 5000, 4096, 64, "ring", 8192, "f16"),
        # a verify window of 8 tokens of the reference model's layer (fp32, q interleaved with its gate), 32K ring
        _attn("attn_verify8_ring_32k_f32", 8, 24, 2, 256, 200003, 28000, 4096, "ring", 32768, "f32", True),
        # one decoded token that sees a whole 256K context through the full-context mirror
        _attn("attn_decode_full_256k_f16", 1, 16, 2, 256, 262142, 262144, 0, "full", 8192, "f16"),
        # a prefill chunk of a long document, sliding window over the ring
        _attn("attn_prefill4096_ring_f16", 4096, 16, 2, 256, 61440, 8192, 128, "ring", 32768, "f16"),
        # an odd-sized first chunk of a prompt, narrow window, fp32
        _attn("attn_prefill1021_full_f32", 1021, 8, 2, 128, 0, 509, 4, "full", 512, "f32"),
        # a few drafted tokens early in a chat: the shortest tree
        _tree("tree_7_ring_600_f16", 7, 12, 4, 64, 600, 8192, 0, "ring", 8192, "f16"),
        # a wide tree of drafts over the 32K ring
        _tree("tree_26_ring_32k_f16", 26, 16, 2, 256, 30001, 28000, 1024, "ring", 32768, "f16"),
        # a full tree over a 128K context in fp32
        _tree("tree_64_full_128k_f32", 64, 24, 2, 256, 131072, 262144, 0, "full", 8192, "f32"),
        # one decoded token's recurrence
        _gdn("gdn_decode_1_f16", 1, 16, 32, 128, "f16", True, True, False),
        # a verify window with the state after every token kept for the rollback
        _gdn("gdn_verify8_snaps_f32", 8, 16, 48, 128, "f32", True, True, True),
        # an odd-sized prompt in fp32
        _gdn("gdn_prefill_2049_f32", 2049, 16, 48, 128, "f32", False, True, False),
        # a long document's prefill
        _gdn("gdn_prefill_32768_f16", 32768, 16, 32, 128, "f16", True, True, False),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attn", "attn", "tree", "gdn", "gdn"])
    dtype = rng.choice(["f16", "f32"])
    if op == "gdn":
        kh, vh = rng.choice([(16, 32), (16, 48), (4, 4), (2, 6), (8, 24)])
        T = _log_int(rng, 1, 32768 * 32 // max(32, vh))
        return _gdn("", T, kh, vh, rng.choice([64, 128, 128]), dtype, rng.random() < 0.5, rng.random() < 0.7,
                    T <= 16 and rng.random() < 0.5)
    qh, kvh, hd = rng.choice([(16, 2, 256), (24, 2, 256), (8, 2, 128), (32, 8, 128), (12, 4, 64), (6, 1, 64)])
    source = rng.choice(["ring", "full"])
    cap = rng.choice([16384, 32768]) if source == "ring" else 512
    if op == "tree":
        T = _log_int(rng, 1, 64)
        base = _log_int(rng, 1, 131072)
    else:
        T = _log_int(rng, 1, 4096)
        base = _log_int(rng, 1, 262144 - T) - 1
    sinks = rng.choice([0, _log_int(rng, 1, 4096)])
    window = _log_int(rng, 16, 262144)
    # the largest listed prefill's work, and a window that the ring still holds for the first query
    window = min(window, max(16, 4096 * 8192 // T))
    if source == "ring":
        window = min(window, cap - SINK_PIN - T)
    make = _tree if op == "tree" else _attn
    c = make("", T, qh, kvh, hd, base, window, sinks, source, cap, dtype)
    c["gated_q"] = op == "attn" and rng.random() < 0.3
    return c


def _max_ctx(case):
    return case["base"] + case["T"] + 77


def _ring_cells(pos, cap):
    if cap <= 2 * SINK_PIN:
        return pos % cap
    return torch.where(pos < SINK_PIN, pos, SINK_PIN + (pos - SINK_PIN).clamp(min=0) % (cap - SINK_PIN))


def _resident(pos, end, cap):
    if cap <= 2 * SINK_PIN:
        return pos >= end - cap
    return (pos < SINK_PIN) | (pos >= max(SINK_PIN, end - (cap - SINK_PIN)))


def _cells(cells, kvh, hd, gen, dev):
    """`cells` cache cells of normed keys and of values ~N(0,1), quantised per 64-element group: codes and fp16 scales."""
    out = []
    for _ in range(2):
        x = torch.randn(cells, kvh * hd // GROUP, GROUP, generator=gen, device=dev)
        s = (x.abs().amax(-1) / 127).half()
        q = torch.round(x / s.float().unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
        out += [q.reshape(cells, kvh * hd), s]
    return out


def _prepare_attn(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    T, qh, kvh, hd, base, cap = (case[k] for k in ("T", "qh", "kvh", "hd", "base", "cap"))
    tree = case["op"] == "tree"
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32
    end = base if tree else base + T
    # what earlier appends left: positions [0, end) in the mirror, their resident part in the ring; cells that
    # nothing was appended to hold codes and NaN scales
    s = {"case": case}
    if case["source"] == "ring":
        pos = torch.arange(end, device=dev)
        pos = pos[_resident(pos, end, cap)]
        cell = _ring_cells(pos, cap)
        cache = []
        for i, x in enumerate(_cells(pos.numel(), kvh, hd, gen, dev)):
            full = torch.full((cap, x.shape[1]), 3 if i % 2 == 0 else float("nan"), dtype=x.dtype, device=dev)
            full[cell] = x
            cache.append(full)
    else:
        cache = _cells(_max_ctx(case), kvh, hd, gen, dev)
        for i in (1, 3):
            cache[i][end:] = float("nan")
    s["kq"], s["ks"], s["vq"], s["vs"] = cache
    wide = 2 * hd if case["gated_q"] else hd
    s["q"] = (1.5 * torch.randn(T, qh, wide, generator=gen, device=dev)).to(dt)[:, :, :hd]
    s["out"] = torch.empty(T, qh, hd, dtype=dt, device=dev)
    s["lse"] = torch.empty(T, qh, dtype=torch.float32, device=dev)
    s["base"] = torch.tensor([base], dtype=torch.int32, device=dev)
    if tree:
        s["dkq"], s["dks"], s["dvq"], s["dvs"] = _cells(T, kvh, hd, gen, dev)
        # a drafter's tree: each node hangs below an earlier one, or below the last committed token
        u = torch.rand(T, generator=gen, device=dev).tolist()
        sees = torch.zeros(T, T, dtype=torch.bool)
        depth = [0] * T
        for i in range(T):
            p = int(u[i] * (i + 1)) - 1
            if p >= 0:
                sees[i] = sees[p]
                depth[i] = depth[p] + 1
            sees[i, i] = True
        words = (T + 31) // 32
        bits = torch.zeros(T, words * 32, dtype=torch.int64)
        bits[:, :T] = sees
        packed = (bits.reshape(T, words, 32) << torch.arange(32)).sum(-1)
        s["mask"] = torch.where(packed >= 2**31, packed - 2**32, packed).to(torch.int32).to(dev)
        s["depth"] = torch.tensor(depth, dtype=torch.int32, device=dev)
    if own:
        wz = _library()
        blank = [torch.zeros(cap, x.shape[1], dtype=x.dtype, device=dev) for x in cache]
        if case["source"] == "ring":
            s["cache"] = wz.kv_cache(*cache, cap, _max_ctx(case))
        else:
            s["cache"] = wz.kv_cache(*blank, cap, _max_ctx(case), *cache)
        s["blank"] = blank
        if tree:
            s["drafts"] = wz.kv_cache(s["dkq"], s["dks"], s["dvq"], s["dvs"], T, T)
        s["ws"] = torch.empty(max(16, wz.kv_attn_workspace_bytes(T, qh, kvh, hd)), dtype=torch.uint8, device=dev)
    return s


def _prepare_gdn(case, seed):
    dev = _device()
    gen = torch.Generator(device=dev).manual_seed(seed)
    T, kh, vh, hd = (case[k] for k in ("T", "kh", "vh", "hd"))
    dt = torch.float16 if case["dtype"] == "f16" else torch.float32

    def conv_out(*shape):  # the causal conv's SiLU output
        x = torch.randn(*shape, generator=gen, device=dev)
        return x * torch.sigmoid(x)

    x = conv_out(T, (2 * kh + vh) * hd)
    if not case["l2"]:  # normed before the call
        qk = x[:, : 2 * kh * hd].reshape(T, 2 * kh, hd)
        qk /= qk.square().sum(-1, keepdim=True).sqrt() + 1e-6
    x = x.to(dt)
    q, k, v = x[:, : kh * hd], x[:, kh * hd : 2 * kh * hd], x[:, 2 * kh * hd :]
    if not case["packed"]:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    s = {"case": case, "q": q.unflatten(1, (kh, hd)), "k": k.unflatten(1, (kh, hd)), "v": v.unflatten(1, (vh, hd))}
    a = 1 + 15 * torch.rand(vh, generator=gen, device=dev)
    dt0 = 1e-3 * 100 ** torch.rand(vh, generator=gen, device=dev)
    s["g"] = -a * dt0 * torch.exp(0.5 * torch.randn(T, vh, generator=gen, device=dev))
    s["beta"] = torch.sigmoid(torch.randn(T, vh, generator=gen, device=dev))
    s["state"] = 0.2 * torch.randn(vh, hd, hd, generator=gen, device=dev)
    s["o"] = torch.empty(T, vh, hd, dtype=dt, device=dev)
    s["state_out"] = torch.empty_like(s["state"])
    s["snaps"] = torch.empty(T, vh, hd, hd, device=dev) if case["snaps"] else None
    if own:
        wz = _library()
        s["ws"] = torch.empty(max(16, wz.gdn_delta_rule_workspace_bytes(T, kh, vh, hd)), dtype=torch.uint8, device=dev)
    return s


def prepare(case, seed):
    return _prepare_gdn(case, seed) if case["op"] == "gdn" else _prepare_attn(case, seed)


def _seen_positions(case, dev):
    """The cache positions that some query of the case may see, ascending."""
    T, base = case["T"], case["base"]
    end = base if case["op"] == "tree" else base + T
    lo = max(0, min(end, base - case["window"] + 1))
    pos = torch.arange(lo, end, device=dev)
    if case["sinks"] and lo:
        pos = torch.cat([torch.arange(min(case["sinks"], lo), device=dev), pos])
    if case["source"] == "ring":
        pos = pos[_resident(pos, end, case["cap"])]
    return pos


def _plain_attn(s):
    case = s["case"]
    T, qh, kvh, hd = (case[k] for k in ("T", "qh", "kvh", "hd"))
    dev = s["q"].device
    pos = _seen_positions(case, dev)
    cell = _ring_cells(pos, case["cap"]) if case["source"] == "ring" else pos
    tree = case["op"] == "tree"

    def rows(codes, scales, drafts, draft_scales):
        c, sc = codes[cell], scales[cell]
        if tree:
            c, sc = torch.cat([c, drafts]), torch.cat([sc, draft_scales])
        x = c.float().unflatten(1, (-1, GROUP)) * sc.float().unsqueeze(-1)
        return x.reshape(-1, kvh, hd).transpose(0, 1)

    k = rows(s["kq"], s["ks"], s.get("dkq"), s.get("dks"))
    v = rows(s["vq"], s["vs"], s.get("dvq"), s.get("dvs"))
    at = case["base"] + (s["depth"].long() if tree else torch.arange(T, device=dev))
    sees = (pos <= at[:, None]) & ((pos < case["sinks"]) | (pos > at[:, None] - case["window"]))
    if tree:
        j = torch.arange(T, device=dev)
        sees = torch.cat([sees, (s["mask"][:, j // 32] >> (j % 32)) & 1 == 1], 1)
    per = qh // kvh
    q = s["q"].float().reshape(T, kvh, per, hd).permute(1, 2, 0, 3).reshape(kvh, per * T, hd)
    x = (q @ k.transpose(1, 2)) * (1 / math.sqrt(hd))
    x = x.reshape(kvh, per, T, -1).masked_fill(~sees, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = (p.reshape(kvh, per * T, -1) @ v).reshape(kvh, per, T, hd) / total
    lse = (top + torch.log(total)).squeeze(-1)
    return {"out": o.permute(2, 0, 1, 3).reshape(T, qh, hd).to(s["q"].dtype),
            "lse": lse.permute(2, 0, 1).reshape(T, qh)}


def _plain_gdn(s):
    case = s["case"]
    T, kh, vh, hd = (case[k] for k in ("T", "kh", "vh", "hd"))
    q, k, v = (s[n].float() for n in ("q", "k", "v"))
    if case["l2"]:
        q = q * torch.rsqrt(q.square().sum(-1, keepdim=True) + 1e-6)
        k = k * torch.rsqrt(k.square().sum(-1, keepdim=True) + 1e-6)
    q = q * (1 / math.sqrt(hd))
    n = 1 if case["snaps"] else min(T, CHUNK)  # tokens per chunk; a kept state ends a chunk
    pad = -T % n

    def chunks(x):  # [T, heads, ...] -> [heads, chunks, n, ...]
        x = torch.cat([x, x.new_zeros(pad, *x.shape[1:])]) if pad else x
        return x.unflatten(0, (-1, n)).movedim(2, 0)

    q, k = (chunks(x.repeat_interleave(vh // kh, 1)) for x in (q, k))
    v, g, beta = chunks(v), chunks(s["g"]), chunks(s["beta"])
    g = g.cumsum(-1)
    low = torch.ones(n, n, dtype=torch.bool, device=q.device).tril()
    decay = torch.exp((g.unsqueeze(-1) - g.unsqueeze(-2)).masked_fill(~low, -math.inf))
    a = (k @ k.transpose(-1, -2)) * decay * beta.unsqueeze(-1)
    a = a.tril(-1)
    inv = torch.eye(n, device=q.device).expand_as(a).clone()
    for i in range(1, n):  # forward substitution of (I + a)^-1
        inv[..., i, :i] = -(a[..., i, None, :i] @ inv[..., :i, :i]).squeeze(-2)
    grown = torch.exp(g).unsqueeze(-1)
    u = inv @ (v * beta.unsqueeze(-1))
    w = inv @ (k * beta.unsqueeze(-1) * grown)
    p = (q @ k.transpose(-1, -2)) * decay
    q = q * grown
    k = k * torch.exp(g[..., -1:] - g).unsqueeze(-1)
    last = torch.exp(g[..., -1])[..., None, None]
    state = s["state"].transpose(1, 2)  # [heads, k, v]
    outs, states = [], []
    for c in range(q.shape[1]):
        new = u[:, c] - w[:, c] @ state
        outs.append(q[:, c] @ state + p[:, c] @ new)
        state = state * last[:, c] + k[:, c].transpose(1, 2) @ new
        states.append(state)
    o = torch.cat(outs, 1)[:, :T].transpose(0, 1)
    r = {"o": o.to(s["v"].dtype), "state": state.transpose(1, 2).contiguous()}
    if case["snaps"]:
        r["snaps"] = torch.stack(states).transpose(2, 3).contiguous()
    return r


def run(state):
    case = state["case"]
    if not own:
        return _plain_gdn(state) if case["op"] == "gdn" else _plain_attn(state)
    wz = _library()
    s = state
    if case["op"] == "gdn":
        wz.gdn_delta_rule(s["q"], s["k"], s["v"], s["g"], s["beta"], s["o"], s["state_out"], state_in=s["state"],
                          state_snaps=s["snaps"], qk_l2norm=case["l2"], l2_eps=1e-6, workspace=s["ws"])
        r = {"o": s["o"], "state": s["state_out"]}
        if case["snaps"]:
            r["snaps"] = s["snaps"]
        return r
    source = wz.KV_RING if case["source"] == "ring" else wz.KV_FULL
    more = dict(window=case["window"], sinks=case["sinks"], source=source, d_base_pos=s["base"], lse=s["lse"],
                workspace=s["ws"])
    if case["op"] == "tree":
        wz.kv_tree_attn(s["q"], s["out"], s["cache"], s["drafts"], s["mask"], case["kvh"], depth=s["depth"], **more)
    else:
        wz.kv_attn(s["q"], s["out"], s["cache"], case["kvh"], **more)
    return {"out": s["out"], "lse": s["lse"]}


def work(case):
    T, size = case["T"], 2 if case["dtype"] == "f16" else 4
    if case["op"] == "gdn":
        kh, vh, hd = case["kh"], case["vh"], case["hd"]
        states = 2 + (T if case["snaps"] else 0)
        return {"bytes": size * T * (2 * kh + 2 * vh) * hd + 8 * T * vh + 4 * states * vh * hd * hd,
                "flops": 6 * T * vh * hd * hd}
    qh, kvh, hd, base = case["qh"], case["kvh"], case["hd"], case["base"]
    cpu = torch.device("cpu")
    pos = _seen_positions(case, cpu)
    tree = case["op"] == "tree"
    at = torch.arange(base, base + T)  # a tree's depths differ with the seed: their window is counted from base
    if tree:
        at = torch.full((T,), base)
    hi = torch.searchsorted(pos, at, right=True)
    first = torch.searchsorted(pos, at - case["window"], right=True)
    sunk = torch.searchsorted(pos, torch.minimum(torch.full_like(at, case["sinks"]), at - case["window"] + 1))
    pairs = int((hi - first + sunk.clamp(min=0)).sum())
    cells = pos.numel()
    if tree:
        cells += T
        pairs += T * max(1, T.bit_length())
    return {"bytes": 2 * size * T * qh * hd + 4 * T * qh + cells * kvh * 2 * (hd + 2 * hd // GROUP),
            "flops": 4 * hd * qh * pairs}


# ---- the definitions in fp64 ---------------------------------------------------------------------


def _exact_attn(case, s):
    T, qh, kvh, hd, base = (case[k] for k in ("T", "qh", "kvh", "hd", "base"))
    dev = s["q"].device
    tree = case["op"] == "tree"
    end = base if tree else base + T
    cap = case["cap"]
    at = [base + (int(d) if tree else t) for t, d in enumerate(s["depth"].tolist() if tree else range(T))]
    where = torch.tensor(at, device=dev)
    # every position that the cache holds, by brute force over all of them
    j = torch.arange(end, device=dev)
    if case["source"] == "ring":
        if cap <= 8192:
            j = j[j >= end - cap]
            cell = torch.remainder(j, cap)
        else:
            j = j[(j < 4096) | (j >= end - cap + 4096)]
            cell = torch.where(j < 4096, j, 4096 + torch.remainder(j - 4096, cap - 4096))
    else:
        cell = j
    near = (j < case["sinks"]) | (j > min(at) - case["window"])
    j, cell = j[near], cell[near]
    out = torch.empty(T, qh, hd, dtype=torch.float64, device=dev)
    lse = torch.empty(T, qh, dtype=torch.float64, device=dev)
    if tree:
        words = s["mask"].long() & 0xFFFFFFFF
        bits = torch.stack([(words[:, n // 32] >> (n % 32)) & 1 for n in range(T)], 1).bool()
    for h in range(kvh):
        cols, groups = slice(h * hd, (h + 1) * hd), slice(h * hd // 64, (h + 1) * hd // 64)

        def take(codes, scales, at_cells):
            x = codes[at_cells][:, cols].double()
            return x * scales[at_cells][:, groups].double().repeat_interleave(64, 1)

        k, v = take(s["kq"], s["ks"], cell), take(s["vq"], s["vs"], cell)
        if tree:
            n = torch.arange(T, device=dev)
            k = torch.cat([k, take(s["dkq"], s["dks"], n)])
            v = torch.cat([v, take(s["dvq"], s["dvs"], n)])
        for g in range(h * (qh // kvh), (h + 1) * (qh // kvh)):
            for t0 in range(0, T, 1024):
                rows = where[t0 : t0 + 1024, None]
                ok = (j <= rows) & ((j < case["sinks"]) | (rows - j < case["window"]))
                if tree:
                    ok = torch.cat([ok, bits[t0 : t0 + 1024]], 1)
                x = s["q"][t0 : t0 + 1024, g].double() @ k.T / math.sqrt(hd)
                x = torch.where(ok, x, torch.full_like(x, -math.inf))
                z = torch.logsumexp(x, 1)
                lse[t0 : t0 + 1024, g] = z
                out[t0 : t0 + 1024, g] = torch.exp(x - z[:, None]) @ v
    return {"out": out, "lse": lse}


def _exact_gdn(case, s):
    T, kh, vh, hd = (case[k] for k in ("T", "kh", "vh", "hd"))
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    if case["l2"]:
        q = q / torch.sqrt((q * q).sum(-1, keepdim=True) + 1e-6)
        k = k / torch.sqrt((k * k).sum(-1, keepdim=True) + 1e-6)
    head = torch.arange(vh, device=q.device) // (vh // kh)
    q, k = q[:, head] / math.sqrt(hd), k[:, head]
    keep, beta = torch.exp(s["g"].double()), s["beta"].double()
    m = s["state"].double().clone()  # [heads, v, k]
    o = torch.empty(T, vh, hd, 1, dtype=torch.float64, device=q.device)
    snaps = []
    keep, beta, v, kc, kr, qc = (keep[..., None, None], beta[..., None, None], v[..., None], k[..., None],
                                 k[..., None, :], q[..., None])
    for t in range(T):
        m *= keep[t]
        m += (beta[t] * (v[t] - m @ kc[t])) @ kr[t]
        torch.matmul(m, qc[t], out=o[t])
        if case["snaps"]:
            snaps.append(m.clone())
    r = {"o": o.squeeze(-1), "state": m}
    if case["snaps"]:
        r["snaps"] = torch.stack(snaps)
    return r


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_gdn(case, s) if case["op"] == "gdn" else _exact_attn(case, s)
