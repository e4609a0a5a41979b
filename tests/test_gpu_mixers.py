"""GPU tests of the token mixers against plain fp64 forms: attention over the INT8 KV cache (window and sinks,
ring and mirror), attention for a tree of drafts, and the gated delta rule.

Bounds. Attention: the weights p * vs are rounded to fp16 (fp16 calls; 2^-11 of each, so 2^-11 sum p|v|) or kept
to 22 bits (fp32 calls), the output is rounded to its type, and a score's fp32 sum of up to 256 products is off
by at most 2^-17 of sum |q k| (256 additions at 2^-24, cut off instead of rounded), which moves each weight, and
the result by twice that in sum p|v|; the base-2 exponential and the sums of weights stay within 2^-20.
Delta rule: |k| <= 1, beta <= 1 and decays <= 1 make a step's map of norm <= 1, so the error is at most the sum of
the steps' roundings: 2^-22 of the state's largest magnitude per step (four roundings at 2^-24) and a fixed part for
the norms and for products split into two fp16 parts (22 bits) over 64-token chunks."""
from __future__ import annotations

import math

import pytest
import torch

import mixers_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def quantised(cells, kvd, r, spread=1.0):
    x = spread * torch.randn(cells, kvd // 64, 64, generator=r, device=DEV)
    s = (x.abs().amax(-1) / 127).half()
    q = torch.round(x / s.float().unsqueeze(-1)).clamp(-127, 127).to(torch.int8)
    return [q.reshape(cells, kvd), s.view(torch.int16)]


def make_cache(wz, end, cap, max_ctx, kvd, r, full, junk=float("nan")):
    """Rows of positions 0..end-1 and a cache that holds them; cells without a row hold `junk` scales."""
    n = max(0, min(end, max_ctx))
    rows = quantised(max(n, 1), kvd, r) + quantised(max(n, 1), kvd, r, 2.0)
    plane = []
    for i, x in enumerate(rows):
        def blank(cells):
            y = torch.full((cells, x.shape[1]), 5, dtype=x.dtype, device=DEV)
            if i % 2:
                y.view(torch.float16).fill_(junk)
            return y
        if full:
            y = blank(max(1, max_ctx))
            y[:n] = x[:n]
        else:
            y = blank(cap)
            js = [j for j in range(n) if ref.in_ring(j, end, cap)]
            if js:
                y[torch.tensor([ref.ring_cell(j, cap) for j in js], device=DEV)] = x[torch.tensor(js, device=DEV)]
        plane.append(y)
    if full:
        tiny = [torch.zeros(16, x.shape[1], dtype=x.dtype, device=DEV) for x in plane]
        desc = wz.kv_cache(*tiny, 16, max_ctx, *plane)
        desc.keep = tiny
    else:
        desc = wz.kv_cache(*plane, cap, max_ctx)
    return rows, plane, desc


def check_attention(q, got, lse, want):
    o, wl, mag, dot = want
    score = dot * 2.0**-17 + 2.0**-20
    unit = 2.0**-11 if q.dtype == torch.float16 else 2.0**-21
    bound = mag * (2 * unit + 2 * score.unsqueeze(-1)) + (2.0**-24 if q.dtype == torch.float16 else 0)
    assert torch.isfinite(got).all()
    err = (got.double() - o).abs()
    assert (err <= bound).all(), float((err - bound).max())
    if lse is not None:
        empty = torch.isinf(wl)
        assert torch.equal(torch.isneginf(lse), empty)
        le = (lse.double() - wl).abs()[~empty]
        assert (le <= (score * math.sqrt(2) + wl.abs() * 2.0**-22)[~empty]).all()
        assert (got[empty] == 0).all()


def workspace(wz, T, qh, kvh, hd):
    return torch.empty(max(16, wz.kv_attn_workspace_bytes(T, qh, kvh, hd)), dtype=torch.uint8, device=DEV)


def run_attn(wz, dtype, T, qh, kvh, hd, base, window, sinks, source, cap, max_ctx, seed=0, gated=False, junk=float("nan"),
             with_lse=True, spread=1.5):
    r = gen(seed)
    end = base + T
    full = source == "full"
    rows, plane, desc = make_cache(wz, end, cap, max_ctx, kvh * hd, r, full, junk)
    wide = 2 * hd if gated else hd
    q = (spread * torch.randn(T, qh, wide, generator=r, device=DEV)).to(dtype)[:, :, :hd]
    out = torch.full((T, qh, hd + (8 if gated else 0)), 7.0, dtype=dtype, device=DEV)[:, :, :hd]
    lse = torch.zeros(T, qh, device=DEV) if with_lse else None
    ws = workspace(wz, T, qh, kvh, hd)
    ws.view(torch.uint8).fill_(255)
    d_base = torch.tensor([base - 3], dtype=torch.int32, device=DEV)
    wz.kv_attn(q, out, desc, kvh, window, sinks, source=wz.KV_FULL if full else wz.KV_RING, d_base_pos=d_base,
               pos_offset=3, lse=lse, workspace=ws)
    see = [ref.seen(base + t, end, max_ctx, window, sinks, None if full else cap) for t in range(T)]
    want = ref.attention(q, rows, kvh, hd, hd**-0.5, see)
    check_attention(q, out, lse, want)
    return out


DTYPES = [torch.float16, torch.float32]
HEADS = [(16, 2, 256), (24, 2, 256), (8, 2, 128), (6, 1, 64), (3, 3, 64)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("qh,kvh,hd", HEADS)
@pytest.mark.parametrize("T,base,window,sinks", [(1, 0, 100, 0), (1, 777, 300, 5), (2, 63, 64, 1), (9, 500, 40, 17),
                                                 (33, 0, 7, 0), (70, 131, 65, 64)])
def test_attn_small(wz, dtype, qh, kvh, hd, T, base, window, sinks):
    run_attn(wz, dtype, T, qh, kvh, hd, base, window, sinks, "full", 16, base + T + 3)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 5, 130])
@pytest.mark.parametrize("base,cap,window,sinks", [
    (50, 300, 90, 10),      # ring not yet full
    (999, 200, 70, 0),      # wrapped many times
    (999, 200, 190, 60),    # sinks have left a small ring, and the first queries' window partly too
    (4090, 8200, 40, 4),    # window across the end of the pinned cells
    (9000, 8200, 64, 4200),  # sinks reach past the pinned cells
    (20000, 8200, 3000, 5),  # sliding part wrapped
    (12290, 8192, 5000, 3),  # the largest ring without pinned cells
])
def test_attn_ring(wz, dtype, T, base, cap, window, sinks):
    run_attn(wz, dtype, T, 4, 2, 64, base, window, sinks, "ring", cap, 1 << 20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 3, 40])
def test_attn_rows_that_see_nothing(wz, dtype, T):
    out = run_attn(wz, dtype, T, 4, 2, 128, 10, 0, 0, "full", 16, 100)
    assert (out == 0).all()
    run_attn(wz, dtype, T, 4, 2, 128, 10, 0, 3, "full", 16, 100)  # the sinks alone
    run_attn(wz, dtype, T, 4, 2, 128, -2, 5, 1, "full", 16, 100)  # positions before the first see nothing
    run_attn(wz, dtype, T, 4, 2, 128, 90, 2, 0, "full", 16, 91)   # positions past max_ctx were not appended
    run_attn(wz, dtype, T, 4, 2, 128, 10, 4, 0, "full", 16, 0)    # an empty cache


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("junk", [float("inf"), float("-inf"), float("nan"), 65504.0])
@pytest.mark.parametrize("T", [1, 20])
def test_attn_unseen_cells_do_not_matter(wz, dtype, junk, T):
    run_attn(wz, dtype, T, 8, 1, 256, 40, 30, 2, "ring", 96, 1 << 20, junk=junk)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attn_infinite_and_huge_cells(wz, dtype):
    """A cell with an infinite or NaN scale spoils the rows that see it and no others, and a value 2^20 times the
    others', seen by the later rows only, leaves the earlier rows' results as they are without it."""
    T, hd = 40, 64
    r = gen(3)
    rows, plane, desc = make_cache(wz, T, 16, T, hd, r, True)
    q = torch.randn(T, 4, hd, generator=r, device=DEV).to(dtype)
    outs = []
    for bad in (1.0, float("inf"), float("nan"), 60000.0):
        plane[3].view(torch.float16)[25, 0] = bad
        out = torch.zeros(T, 4, hd, dtype=dtype, device=DEV)
        wz.kv_attn(q, out, desc, 1, 100, source=wz.KV_FULL, workspace=workspace(wz, T, 4, 1, hd))
        outs.append(out)
    for o in outs[1:3]:
        assert torch.equal(o[:25], outs[0][:25])
        assert not torch.isfinite(o[25:]).any(-1).any()
    err = (outs[3][:25].double() - outs[0][:25].double()).abs().max()
    assert err <= 2.0**-9 if dtype == torch.float16 else 2.0**-18


@pytest.mark.parametrize("dtype", DTYPES)
def test_attn_query_magnitudes(wz, dtype):
    """Scores far apart (softmax close to one-hot) and tiny queries."""
    run_attn(wz, dtype, 9, 4, 2, 128, 200, 150, 4, "full", 16, 300, spread=30.0)
    run_attn(wz, dtype, 9, 4, 2, 128, 200, 150, 4, "full", 16, 300, spread=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 8, 17])
def test_attn_strides_and_no_lse(wz, dtype, T):
    run_attn(wz, dtype, T, 24, 2, 256, 1500, 1200, 8, "ring", 2048, 1 << 20, gated=True, with_lse=False)


def test_attn_split_keys_agree_with_one_row_tile(wz):
    """A long context is split over many CTAs for one token; the same token inside a long chunk is not."""
    r = gen(5)
    T, qh, kvh, hd = 700, 8, 1, 128
    _, _, desc = make_cache(wz, T, 16, T, kvh * hd, r, True)
    q = torch.randn(T, qh, hd, generator=r, device=DEV)
    out, one = torch.zeros(T, qh, hd, device=DEV), torch.zeros(1, qh, hd, device=DEV)
    wz.kv_attn(q, out, desc, kvh, T, source=wz.KV_FULL, workspace=workspace(wz, T, qh, kvh, hd))
    wz.kv_attn(q[-1:], one, desc, kvh, T, source=wz.KV_FULL, pos_offset=T - 1, workspace=workspace(wz, 1, qh, kvh, hd))
    assert (out[-1:] - one).abs().max() <= 2.0**-16


def test_attn_offsets_past_32_bits(wz):
    """Cells whose byte offset passes 2^32."""
    hd, kvh, n = 256, 8, 2_200_000
    kvd = hd * kvh
    r = gen(8)
    plane = [torch.zeros(n, kvd, dtype=torch.int8, device=DEV), torch.zeros(n, kvd // 64, dtype=torch.int16, device=DEV)]
    plane = plane + [plane[0], plane[1]]  # k and v share their planes
    tail = quantised(64, kvd, r)
    plane[0][-64:], plane[1][-64:] = tail[0], tail[1]
    tiny = [torch.zeros(16, x.shape[1], dtype=x.dtype, device=DEV) for x in plane]
    desc = wz.kv_cache(*tiny, 16, n, *plane)
    for T in (1, 30):
        q = torch.randn(T, kvh, hd, generator=r, device=DEV)
        out, lse = torch.zeros(T, kvh, hd, device=DEV), torch.zeros(T, kvh, device=DEV)
        wz.kv_attn(q, out, desc, kvh, 33, source=wz.KV_FULL, pos_offset=n - T, lse=lse, workspace=workspace(wz, T, kvh, kvh, hd))
        see = [[64 - T + t - 32 + i for i in range(33)] for t in range(T)]
        check_attention(q, out, lse, ref.attention(q, tail + tail, kvh, hd, hd**-0.5, see))


def make_tree(n, r):
    u = torch.rand(n, generator=r, device=DEV).tolist()
    sees, depth = [], []
    for i in range(n):
        p = int(u[i] * (i + 1)) - 1
        sees.append(([] if p < 0 else sees[p]) + [i])
        depth.append(0 if p < 0 else depth[p] + 1)
    return sees, depth


def mask_words(sees, n):
    m = torch.zeros(n, (n + 31) // 32, dtype=torch.int64)
    for i, js in enumerate(sees):
        for j in js:
            m[i, j // 32] |= 1 << (j % 32)
    return torch.where(m >= 2**31, m - 2**32, m).to(torch.int32).to(DEV)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [1, 2, 7, 33, 70])
@pytest.mark.parametrize("qh,kvh,hd,base,window,sinks,source,cap", [
    (16, 2, 256, 300, 64, 4, "full", 16), (8, 2, 128, 0, 64, 4, "full", 16), (6, 1, 64, 1000, 120, 0, "ring", 256),
    (12, 4, 64, 9000, 2000, 4100, "ring", 8200), (24, 2, 256, 50, 3, 0, "ring", 128)])
def test_tree(wz, dtype, n, qh, kvh, hd, base, window, sinks, source, cap):
    r = gen(n + base)
    full = source == "full"
    rows, plane, desc = make_cache(wz, base, cap, 1 << 14, kvh * hd, r, full)
    drafts = quantised(n, kvh * hd, r) + quantised(n, kvh * hd, r, 2.0)
    sees, depth = make_tree(n, r)
    q = (1.5 * torch.randn(n, qh, hd, generator=r, device=DEV)).to(dtype)
    out, lse = torch.empty_like(q), torch.zeros(n, qh, device=DEV)
    wz.kv_tree_attn(q, out, desc, wz.kv_cache(*drafts, n, n), mask_words(sees, n), kvh, window,
                    torch.tensor(depth, dtype=torch.int32, device=DEV), sinks=sinks, source=wz.KV_FULL if full else wz.KV_RING,
                    pos_offset=base, lse=lse, workspace=workspace(wz, n, qh, kvh, hd))
    see = [ref.seen(base + d, base, 1 << 14, window, sinks, None if full else cap) for d in depth]
    check_attention(q, out, lse, ref.attention(q, rows, kvh, hd, hd**-0.5, see, drafts, sees))


@pytest.mark.parametrize("dtype", DTYPES)
def test_tree_node_without_ancestors_or_cache(wz, dtype):
    """Nodes whose mask row is empty over an empty cache see nothing, drafts they do not see may hold NaN."""
    n, hd = 40, 128
    r = gen(1)
    drafts = quantised(n, hd, r) + quantised(n, hd, r)
    drafts[1].view(torch.float16)[7] = float("nan")
    drafts[3].view(torch.float16)[7] = float("inf")
    sees = [[] if i % 3 == 0 else [j for j in range(n) if j != 7 and (i + j) % 2] for i in range(n)]
    _, _, desc = make_cache(wz, 0, 16, 64, hd, r, False)
    q = torch.randn(n, 4, hd, generator=r, device=DEV).to(dtype)
    out, lse = torch.ones_like(q), torch.zeros(n, 4, device=DEV)
    wz.kv_tree_attn(q, out, desc, wz.kv_cache(*drafts, n, n), mask_words(sees, n), 1, 64,
                    torch.zeros(n, dtype=torch.int32, device=DEV), lse=lse, workspace=workspace(wz, n, 4, 1, hd))
    clean = [x.clone() for x in drafts]
    clean[1][7], clean[3][7] = 0, 0
    want = ref.attention(q, clean, 1, hd, hd**-0.5, [[]] * n, clean, sees)
    check_attention(q, out, lse, want)


def test_chain_of_drafts_is_a_chunk(wz):
    """A tree that is one chain gives what the same tokens give once they are appended to the cache."""
    n, base, qh, kvh, hd = 8, 200, 8, 2, 128
    kvd = kvh * hd
    r = gen(2)
    k, v = (torch.randn(base + n, kvd, generator=r, device=DEV) for _ in range(2))

    def planes(cells):
        return [torch.zeros(cells, w, dtype=t, device=DEV) for _ in range(2) for w, t in ((kvd, torch.int8), (kvd // 64, torch.int16))]

    ring, drafts = planes(512), planes(n)
    cache, dcache = wz.kv_cache(*ring, 512, 4096), wz.kv_cache(*drafts, n, n)
    wz.kv_append_int8_f32(k[:base], v[:base], base, kvh, hd, cache)
    wz.kv_append_int8_f32(k[base:], v[base:], n, kvh, hd, dcache)
    q = torch.randn(n, qh, hd, generator=r, device=DEV)
    tree, chunk = torch.zeros_like(q), torch.zeros_like(q)
    ws = workspace(wz, n, qh, kvh, hd)
    wz.kv_tree_attn(q, tree, cache, dcache, mask_words([list(range(i + 1)) for i in range(n)], n), kvh, 150,
                    torch.arange(n, dtype=torch.int32, device=DEV), sinks=3, pos_offset=base, workspace=ws)
    wz.kv_append_int8_f32(k[base:], v[base:], n, kvh, hd, cache, pos_offset=base)
    wz.kv_attn(q, chunk, cache, kvh, 150, sinks=3, pos_offset=base, workspace=ws)
    assert (tree - chunk).abs().max() <= 2.0**-18


def test_attn_on_a_side_stream_and_in_a_graph(wz):
    r = gen(4)
    T, qh, kvh, hd = 2, 16, 2, 256
    _, _, desc = make_cache(wz, 2000, 16, 2100, kvh * hd, r, True)
    q = torch.randn(T, qh, hd, generator=r, device=DEV)
    want, got = torch.zeros_like(q), torch.zeros_like(q)
    base = torch.tensor([1500], dtype=torch.int32, device=DEV)
    ws = workspace(wz, T, qh, kvh, hd)
    kw = dict(source=wz.KV_FULL, d_base_pos=base, workspace=ws)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        wz.kv_attn(q, got, desc, kvh, 4000, **kw)
    for pos in (1500, 10, 1990):  # the length is read on the device
        base.fill_(pos)
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            wz.kv_attn(q, want, desc, kvh, 4000, **kw)
        torch.cuda.synchronize()
        assert torch.equal(got, want)


# ---- the gated delta rule ------------------------------------------------------------------------


def gdn_inputs(T, kh, vh, hd, dtype, r, packed, l2, decay=0.1):
    x = torch.randn(T, (2 * kh + vh) * hd, generator=r, device=DEV)
    x = x * torch.sigmoid(x)
    if not l2:
        y = x[:, :2 * kh * hd].reshape(T, 2 * kh, hd)
        y /= y.norm(dim=-1, keepdim=True) * 1.01
    x = x.to(dtype)
    q, k, v = x[:, :kh * hd], x[:, kh * hd:2 * kh * hd], x[:, 2 * kh * hd:]
    if not packed:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    g = -decay * torch.exp(torch.randn(T, vh, generator=r, device=DEV))
    beta = torch.sigmoid(torch.randn(T, vh, generator=r, device=DEV))
    s0 = 0.3 * torch.randn(vh, hd, hd, generator=r, device=DEV)
    return q.unflatten(1, (kh, hd)), k.unflatten(1, (kh, hd)), v.unflatten(1, (vh, hd)), g, beta, s0


def gdn_workspace(wz, T, kh, vh, hd):
    ws = torch.empty(max(16, wz.gdn_delta_rule_workspace_bytes(T, kh, vh, hd)), dtype=torch.uint8, device=DEV)
    ws.fill_(255)
    return ws


def check_gdn(dtype, T, o, s, want_o, want_s, big, scale):
    tol = big * ((T + 64) * 2.0**-22)
    assert (s.double() - want_s).abs().max() <= tol
    err = (o.double() - want_o).abs()
    unit = 2.0**-10 if dtype == torch.float16 else 0.0  # o, and the weights of a chunk's own tokens, in fp16
    assert (err <= unit * want_o.abs().clamp(min=unit * big * scale) + 11.4 * scale * tol + (2.0**-11 * big * scale if unit else 0)).all(), float(err.max())


def run_gdn(wz, dtype, T, kh, vh, hd, packed=False, l2=True, zero_state=False, in_place=False, snaps=False, seed=0, **kw):
    r = gen(seed + T)
    q, k, v, g, beta, s0 = gdn_inputs(T, kh, vh, hd, dtype, r, packed, l2, **kw)
    scale = hd**-0.5
    st = None if zero_state else s0
    want_o, want_s, want_snaps = ref.delta_rule(q, k, v, g, beta, st, scale, 1e-6 if l2 else None)
    big = max(float(x.abs().max()) for x in want_snaps + [s0.double()]) + float(v.abs().max())
    o = torch.full((T, vh, hd), 9.0, dtype=dtype, device=DEV)
    out = s0.clone() if in_place else torch.full_like(s0, 9.0)
    sn = torch.full((T, vh, hd, hd), 9.0, device=DEV) if snaps else None
    wz.gdn_delta_rule(q, k, v, g, beta, o, out, state_in=out if in_place else st, state_snaps=sn, qk_l2norm=l2,
                      workspace=gdn_workspace(wz, T, kh, vh, hd))
    check_gdn(dtype, T, o, out, want_o, want_s, big, scale)
    if snaps:
        for t in range(T):
            assert (sn[t].double() - want_snaps[t]).abs().max() <= big * ((T + 64) * 2.0**-22)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 8, 15, 16, 17, 63, 64, 65, 127, 128, 129, 200, 333])
def test_gdn_lengths(wz, dtype, hd, T):
    run_gdn(wz, dtype, T, 2, 4, hd, packed=T % 2 == 1)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("kh,vh", [(1, 1), (16, 32), (16, 48), (3, 3), (2, 10)])
@pytest.mark.parametrize("T", [1, 100])
def test_gdn_heads(wz, dtype, kh, vh, T):
    run_gdn(wz, dtype, T, kh, vh, 128, packed=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 5, 150])
def test_gdn_states(wz, dtype, T):
    run_gdn(wz, dtype, T, 2, 4, 128, zero_state=True)
    run_gdn(wz, dtype, T, 2, 4, 128, in_place=True)
    run_gdn(wz, dtype, T, 2, 4, 128, l2=False)
    run_gdn(wz, dtype, T, 2, 4, 64, snaps=True)
    run_gdn(wz, dtype, T, 2, 4, 128, snaps=True, in_place=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [3, 130, 200])
@pytest.mark.parametrize("decay", [0.0, 1e-4, 3.0, 60.0])
def test_gdn_decays(wz, dtype, T, decay):
    run_gdn(wz, dtype, T, 2, 4, 128, decay=decay)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [6, 140])
def test_gdn_reset_and_degenerate_tokens(wz, dtype, T):
    """g = -inf forgets the state, beta = 0 leaves it, zero keys and queries are no division by zero."""
    r = gen(9)
    q, k, v, g, beta, s0 = gdn_inputs(T, 2, 4, 128, dtype, r, False, True)
    g[T // 2, 1] = -math.inf
    g[T // 2 + 1, 2] = -200.0
    g[1] = 0.0
    beta[T // 3] = 0.0
    k[2], q[T - 2] = 0, 0
    v[T // 2, 0] = 0
    o, out = torch.zeros_like(v), torch.zeros_like(s0)
    want_o, want_s, snaps = ref.delta_rule(q, k, v, g, beta, s0, 128**-0.5, 1e-6)
    wz.gdn_delta_rule(q, k, v, g, beta, o, out, state_in=s0, workspace=gdn_workspace(wz, T, 2, 4, 128))
    big = max(float(x.abs().max()) for x in snaps + [s0.double()]) + float(v.abs().max())
    check_gdn(dtype, T, o, out, want_o, want_s, big, 128**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size", [2.0**-12, 2.0**12])
def test_gdn_value_magnitudes(wz, dtype, size):
    """The rule is linear in (v, state): scaled inputs give scaled results, at any size that the types hold."""
    T = 200
    r = gen(10)
    q, k, v, g, beta, s0 = gdn_inputs(T, 2, 4, 128, torch.float32, r, False, True)
    q, k = q.to(dtype), k.to(dtype)
    v = (v * size).to(dtype)
    s0 = s0 * size
    o, out = torch.zeros_like(v), torch.zeros_like(s0)
    want_o, want_s, snaps = ref.delta_rule(q, k, v, g, beta, s0, 128**-0.5, 1e-6)
    wz.gdn_delta_rule(q, k, v, g, beta, o, out, state_in=s0, workspace=gdn_workspace(wz, T, 2, 4, 128))
    big = max(float(x.abs().max()) for x in snaps + [s0.double()]) + float(v.abs().max())
    if dtype == torch.float16 and size < 1:  # outputs near fp16's subnormals
        assert (o.double() - want_o).abs().max() <= 2.0**-24 + 2.0**-10 * float(want_o.abs().max())
        assert (out.double() - want_s).abs().max() <= big * ((T + 64) * 2.0**-22)
    else:
        check_gdn(dtype, T, o, out, want_o, want_s, big, 128**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gdn_correlated_keys(wz, dtype):
    """Keys that hardly change make the chunk's triangular system far from diagonal."""
    T = 192
    r = gen(11)
    q, k, v, g, beta, s0 = gdn_inputs(T, 2, 4, 128, torch.float32, r, False, True, decay=1e-3)
    k = (k[:1] + 0.05 * k).to(dtype)
    q, v = q.to(dtype), v.to(dtype)
    beta = 0.9 + 0.1 * beta
    o, out = torch.zeros_like(v), torch.zeros_like(s0)
    want_o, want_s, snaps = ref.delta_rule(q, k, v, g, beta, s0, 128**-0.5, 1e-6)
    wz.gdn_delta_rule(q, k, v, g, beta, o, out, state_in=s0, workspace=gdn_workspace(wz, T, 2, 4, 128))
    big = max(float(x.abs().max()) for x in snaps + [s0.double()]) + float(v.abs().max())
    check_gdn(dtype, T, o, out, want_o, want_s, big, 128**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gdn_in_two_calls_and_no_tokens(wz, dtype):
    T, cut = 300, 131
    r = gen(12)
    q, k, v, g, beta, s0 = gdn_inputs(T, 2, 4, 128, dtype, r, True, True)
    ws = gdn_workspace(wz, T, 2, 4, 128)
    o, s = torch.zeros(T, 4, 128, dtype=dtype, device=DEV), torch.zeros_like(s0)
    wz.gdn_delta_rule(q, k, v, g, beta, o, s, state_in=s0, workspace=ws)
    o2, s2 = torch.zeros_like(o), torch.zeros_like(s0)
    wz.gdn_delta_rule(q[:0], k[:0], v[:0], g[:0], beta[:0], o2[:0], s2, state_in=s0, workspace=ws)
    assert torch.equal(s2, s0)
    for a, b in ((0, cut), (cut, T)):
        wz.gdn_delta_rule(q[a:b], k[a:b], v[a:b], g[a:b], beta[a:b], o2[a:b], s2, state_in=s2, workspace=ws)
    big = float(s.abs().max() + v.abs().max())
    assert (s - s2).abs().max() <= big * (T + 64) * 2.0**-21
    assert (o.float() - o2.float()).abs().max() <= big * (2.0**-9 if dtype == torch.float16 else 2.0**-12)


# ---- both mixers together ------------------------------------------------------------------------


def test_example_chunks_and_tokens_agree_with_one_chunk(wz):
    """The example's prompt in chunks and its tokens one by one give what one long chunk gives: attention to the
    rounding of k's appended codes and the fp16 outputs, the delta rule to its own bounds."""
    import example_mixers as ex

    # attention outputs are means of values of size 1 with weights off by 2^-11 and rounded to fp16: 2^-9 of the largest
    kw = dict(ring=9000, max_ctx=16384, window=300, sinks=8)
    ya, yb, tree, attn, gdn = ex.run(prompt=640, chunk=160, decoded=5, **kw)
    za, zb, *_ = ex.run(prompt=645, chunk=645, decoded=0, **kw)
    assert (ya.float() - za.float()).abs().max() <= 2.0**-9 * za.float().abs().max()
    assert (yb.float() - zb.float()).abs().max() <= 2.0**-8 * zb.float().abs().max()
    assert int(attn.pos) == 647 and torch.isfinite(tree).all()
    assert wz.read_faults() == 0


@pytest.mark.parametrize("dtype", DTYPES)
def test_attn_long_context_sums_do_not_drift(wz, dtype):
    """Values that all add up: a chunk that one CTA walks 100,000 keys for (no split) stays within the usual bound."""
    n, T, qh, kvh, hd = 100_000, 1200, 32, 2, 64
    r = gen(20)
    x = torch.randn(n, kvh, 64, generator=r, device=DEV)
    planes = []
    for y in (x, 3 + torch.randn(n, kvh, 64, generator=r, device=DEV)):
        s = (y.abs().amax(-1) / 127).half()
        planes += [torch.round(y / s.float().unsqueeze(-1)).clamp(-127, 127).to(torch.int8).reshape(n, kvh * hd), s.view(torch.int16)]
    tiny = [torch.zeros(16, p.shape[1], dtype=p.dtype, device=DEV) for p in planes]
    q = torch.randn(T, qh, hd, generator=r, device=DEV).to(dtype)
    out, lse = torch.empty_like(q), torch.zeros(T, qh, device=DEV)
    assert wz.kv_attn_workspace_bytes(T, qh, kvh, hd) == 0  # not split
    wz.kv_attn(q, out, wz.kv_cache(*tiny, 16, n, *planes), kvh, n, source=wz.KV_FULL, pos_offset=n - T, lse=lse)
    at = [0, 7, T - 1]
    want = ref.attention(q[at], planes, kvh, hd, hd**-0.5, [list(range(n - T + t + 1)) for t in at])
    check_attention(q[at], out[at], lse[at], want)


# ---- sizes of the factors of the delta rule ------------------------------------------------------


def gdn_call(wz, q, k, v, g, beta, s0, **kw):
    T, kh, hd = q.shape
    vh = v.shape[1]
    o, out = torch.full_like(v, 9.0, memory_format=torch.contiguous_format), torch.full((vh, hd, hd), 9.0, device=DEV)
    wz.gdn_delta_rule(q, k, v, g, beta, o, out, state_in=s0, workspace=gdn_workspace(wz, T, kh, vh, hd), **kw)
    return o, out


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T", [50, 200])
@pytest.mark.parametrize("by", ["scale", "q"])
@pytest.mark.parametrize("down", [12, 20])
def test_gdn_outputs_follow_small_queries_and_scales(wz, dtype, hd, T, by, down):
    """o is linear in scale * q. A power of two there moves exponents only, so the outputs' bits stay the same (where they
    are normal numbers) whatever the size, and hold the bounds of the recurrence at that size."""
    r = gen(13)
    q, k, v, g, beta, s0 = gdn_inputs(T, 2, 4, hd, torch.float32, r, False, False)
    # q's elements are multiples of 2^-4, so that 2^-20 of them is exact in fp16 as well
    q, k, v = (torch.round(16 * q) / 16).to(dtype), k.to(dtype), (512 * v).to(dtype)
    s0 = 512 * s0
    scale, f = hd**-0.5, 2.0**-down
    assert torch.equal((q * f).to(dtype).double(), q.double() * f)
    o1, s1 = gdn_call(wz, q, k, v, g, beta, s0, scale=scale, qk_l2norm=False)
    o2, s2 = gdn_call(wz, q * f if by == "q" else q, k, v, g, beta, s0, scale=scale * (f if by == "scale" else 1), qk_l2norm=False)
    want_o, want_s, snaps = ref.delta_rule(q, k, v, g, beta, s0, scale * f, None)
    big = max(float(x.abs().max()) for x in snaps + [s0.double()]) + float(v.abs().max())
    tol = big * ((T + 64) * 2.0**-22)
    assert torch.equal(s1, s2) and (s2.double() - want_s).abs().max() <= tol
    unit = 2.0**-10 if dtype == torch.float16 else 0.0
    bound = unit * want_o.abs() + scale * f * (float(q.double().abs().sum(-1).max()) * tol + 2 * unit * big) + (2.0**-25 if unit else 0.0)
    assert ((o2.double() - want_o).abs() <= bound).all()
    # where the smaller output is a normal number before its rounding (2^-14 itself may have been rounded up to)
    normal = o1.double().abs() * f > (2.0**-14 if dtype == torch.float16 else 2.0**-126)
    assert normal.any() or (dtype == torch.float16 and down == 20)
    assert torch.equal(o2.double()[normal], (o1.double() * f)[normal])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [50, 200])
@pytest.mark.parametrize("down", [12, 30])
def test_gdn_small_betas(wz, dtype, T, down):
    """From an empty state every step adds beta (v - S k) k^T: with small betas throughout, a state of their size, whose
    error is bounded by its own magnitude and that of beta v (two roundings at 2^-22 of either per step)."""
    r = gen(14)
    q, k, v, g, beta, _ = gdn_inputs(T, 2, 4, 128, dtype, r, False, True)
    beta = beta * 2.0**-down
    want_o, want_s, snaps = ref.delta_rule(q, k, v, g, beta, None, 128**-0.5, 1e-6)
    big = max(float(x.abs().max()) for x in snaps) + float((beta.double().unsqueeze(-1) * v.double()).abs().max())
    _, s = gdn_call(wz, q, k, v, g, beta, None)
    assert (s.double() - want_s).abs().max() <= big * (T + 64) * 2.0**-22


# ---- uneven queries and keys ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("T", [1, 7, 40])
@pytest.mark.parametrize("up", [0, 6, 12])
def test_attn_uneven_groups(wz, dtype, hd, T, up):
    """A query whose first group is 2^up times the others, over keys whose first group is 2^-up of theirs: all groups have
    their share of the score, so none may lose bits beside the largest. 1, 7 and 40 tokens of 4 heads: both kernels."""
    r = gen(21)
    n = 300
    rows, plane, desc = make_cache(wz, n, 16, n, hd, r, True)
    for x in (rows[1], plane[1]):
        x.view(torch.float16)[:, 0] *= 2.0**-up
    q = torch.randn(T, 4, hd, generator=r, device=DEV)
    q[:, :, :64] *= 2.0**up
    q = q.to(dtype)
    out, lse = torch.zeros_like(q), torch.zeros(T, 4, device=DEV)
    wz.kv_attn(q, out, desc, 1, n, source=wz.KV_FULL, pos_offset=n - T, lse=lse, workspace=workspace(wz, T, 4, 1, hd))
    see = [list(range(n - T + t + 1)) for t in range(T)]
    check_attention(q, out, lse, ref.attention(q, rows, 1, hd, hd**-0.5, see))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [1, 20, 40])
@pytest.mark.parametrize("base", [2**30 - 21, 2**31 - 21, 2**31 + 5, 2**40])
@pytest.mark.parametrize("window,sinks,seen", [(2**62, 0, 40), (7, 3, 3), (0, 2**40, 40), (9, 0, 0)])
def test_attn_positions_past_31_bits(wz, dtype, T, base, window, sinks, seen):
    """Queries that stand far past a short cache's end see its cells by the same rule."""
    r = gen(22)
    hd, n = 64, 40
    rows, plane, desc = make_cache(wz, n, 16, n, hd, r, True)
    q = torch.randn(T, 8, hd, generator=r, device=DEV).to(dtype)
    out, lse = torch.ones_like(q), torch.zeros(T, 8, device=DEV)
    wz.kv_attn(q, out, desc, 1, window, sinks, source=wz.KV_FULL, pos_offset=base, lse=lse, workspace=workspace(wz, T, 8, 1, hd))
    check_attention(q, out, lse, ref.attention(q, rows, 1, hd, hd**-0.5, [list(range(seen))] * T))


@pytest.mark.parametrize("dtype", DTYPES)
def test_attn_no_tokens(wz, dtype):
    """Empty tensors through the bindings."""
    _, _, desc = make_cache(wz, 10, 16, 100, 64, gen(23), False)
    q = torch.empty(0, 4, 64, dtype=dtype, device=DEV)
    wz.kv_attn(q, torch.empty_like(q), desc, 1, 16, lse=torch.empty(0, 4, device=DEV))
    wz.kv_tree_attn(q, torch.empty_like(q), desc, desc, torch.empty(0, 0, dtype=torch.int32, device=DEV), 1, 16,
                    torch.empty(0, dtype=torch.int32, device=DEV))


# ---- rows beside cells that they do not see, scales ----------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [8, 40])  # both kernels
@pytest.mark.parametrize("bad", [float("inf"), float("nan"), 60000.0])
def test_attn_earlier_rows_keep_their_bits(wz, dtype, T, bad):
    """A cell that only the later rows see, with an infinite, a NaN or a 2^20-fold value scale: the earlier rows' weights are
    scaled by what they see alone, so their bits stay; the later rows are spoiled, or right for the huge cell."""
    n, hd, at = 40, 64, 36
    r = gen(24)
    rows, plane, desc = make_cache(wz, n, 16, n, hd, r, True)
    q = torch.randn(T, 4, hd, generator=r, device=DEV).to(dtype)
    base, ws = n - T, workspace(wz, T, 4, 1, hd)
    outs = []
    for scale in (1.0, bad):
        rows[3].view(torch.float16)[at, 0] = plane[3].view(torch.float16)[at, 0] = scale
        out, lse = torch.zeros_like(q), torch.zeros(T, 4, device=DEV)
        wz.kv_attn(q, out, desc, 1, 100, source=wz.KV_FULL, pos_offset=base, lse=lse, workspace=ws)
        outs.append((out, lse))
    early = at - base
    assert torch.equal(outs[0][0][:early], outs[1][0][:early]) and torch.equal(outs[0][1][:early], outs[1][1][:early])
    if math.isfinite(bad):
        see = [list(range(base + t + 1)) for t in range(T)]
        if dtype == torch.float16:  # means of values up to 60000 * 127 pass fp16's range
            assert torch.isinf(outs[1][0][early:]).any() or outs[1][0][early:].abs().max() > 1000
        else:
            check_attention(q, *outs[1], ref.attention(q, rows, 1, hd, hd**-0.5, see))
    else:
        assert not torch.isfinite(outs[1][0][early:]).any(-1).any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [2, 40])
@pytest.mark.parametrize("scale", [0.0, 1e-4, 0.3, -0.2])
def test_attn_scale(wz, dtype, T, scale):
    r = gen(25)
    n, hd = 150, 128
    rows, _, desc = make_cache(wz, n, 16, n, 2 * hd, r, True)
    q = torch.randn(T, 8, hd, generator=r, device=DEV).to(dtype)
    out, lse = torch.zeros_like(q), torch.zeros(T, 8, device=DEV)
    wz.kv_attn(q, out, desc, 2, n, scale=scale, source=wz.KV_FULL, pos_offset=n - T, lse=lse, workspace=workspace(wz, T, 8, 2, hd))
    o, wl, mag, _ = ref.attention(q, rows, 2, hd, scale, [list(range(n - T + t + 1)) for t in range(T)])
    dot = torch.zeros_like(wl)  # the largest sum of |scale q k|, which a negative scale's maximum is not
    for h in range(2):
        k = ref.rows64(rows[0], rows[1], hd, h).abs()
        dot[:, 4 * h:4 * h + 4] = abs(scale) * (q[:, 4 * h:4 * h + 4].double().abs() @ k.T).amax(-1)
    check_attention(q, out, lse, (o, wl, mag, dot))


# ---- the delta rule over many chunks and segments ------------------------------------------------


def delta_rule_long(q, k, v, g, beta, state, scale):
    """ref.delta_rule without keeping every state; also, per token, the largest |state| and the sum of the earlier steps'
    shares in an error at it: a step's map shrinks an error by its decay at least."""
    T, kh, d = q.shape
    vh = v.shape[1]
    q, k, v, beta, keep = q.double(), k.double(), v.double(), beta.double(), torch.exp(g.double())
    q, k = (x / torch.sqrt((x * x).sum(-1, keepdim=True) + 1e-6) for x in (q, k))
    q, k = (x.repeat_interleave(vh // kh, 1) for x in (q, k))
    s, o, size = state.double().clone(), torch.zeros_like(v), torch.zeros(T, dtype=torch.float64, device=v.device)
    eff, most = torch.zeros(vh, dtype=torch.float64, device=v.device), torch.zeros(vh, dtype=torch.float64, device=v.device)
    for t in range(T):
        s *= keep[t][:, None, None]
        e = beta[t][:, None] * (v[t] - (s @ k[t].unsqueeze(-1)).squeeze(-1))
        s += e[:, :, None] * k[t][:, None, :]
        o[t] = scale * (s @ q[t].unsqueeze(-1)).squeeze(-1)
        size[t] = s.abs().max()
        eff = eff * keep[t] + 1
        most = torch.maximum(most, eff)
    return o, s, size, float(most.max())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,kh,vh,hd", [(1100, 2, 4, 128), (2111, 2, 4, 64), (6037, 16, 32, 128), (3100, 16, 48, 128)])
def test_gdn_many_chunks_and_segments(wz, dtype, T, kh, vh, hd):
    """More than 16 chunks (the columns' exponents are set anew), and lengths that take two segments of the workspace in one
    type or in both, the last one ragged; state in place, a workspace of the exact size with a guard behind it."""
    r = gen(30 + T)
    q, k, v, g, beta, s0 = gdn_inputs(T, kh, vh, hd, dtype, r, True, True)
    want_o, want_s, size, eff = delta_rule_long(q, k, v, g, beta, s0, hd**-0.5)
    need = wz.gdn_delta_rule_workspace_bytes(T, kh, vh, hd)
    ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    ws[:need] = 255
    o, state = torch.full((T + 1, vh, hd), 9.0, dtype=dtype, device=DEV), s0.clone()
    wz.gdn_delta_rule(q, k, v, g, beta, o[:T], state, state_in=state, workspace=ws[:need])
    assert (ws[need:] == 0xA5).all() and (o[T] == 9).all()
    big = float(max(size.max(), s0.abs().max()) + v.abs().max())
    # check_gdn's bound with the steps that count under the decays in the place of all T
    check_gdn(dtype, min(T, math.ceil(eff)), o[:T], state, want_o, want_s, big, hd**-0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [2111, 3200])
def test_gdn_falling_magnitudes(wz, dtype, T):
    """Values and states that shrink by 2^20 over the call: the columns' exponents follow them down every 16 chunks, so an
    error is bounded by the magnitudes of the last 17 chunks, not by the call's largest."""
    r = gen(31)
    q, k, v, g, beta, s0 = gdn_inputs(T, 2, 4, 128, torch.float32, r, False, True)
    fall = 2.0 ** (10 - 20 * torch.arange(T, device=DEV) / T)
    q, k, v, s0 = q.to(dtype), k.to(dtype), (v * fall[:, None, None]).to(dtype), s0 * 2.0**10
    want_o, want_s, size, eff = delta_rule_long(q, k, v, g, beta, s0, 128**-0.5)
    o, state = torch.zeros_like(v), torch.zeros_like(s0)
    wz.gdn_delta_rule(q, k, v, g, beta, o, state, state_in=s0, workspace=gdn_workspace(wz, T, 2, 4, 128))
    late = slice(T - 17 * 64, T)
    big = float(size[late].max() + v[late].abs().max())
    assert (state.double() - want_s).abs().max() <= big * (math.ceil(eff) + 64) * 2.0**-22


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T", [60, 150])  # token by token, chunked
@pytest.mark.parametrize("l2", [True, False])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("what", ["q", "k", "v", "g", "beta"])
def test_gdn_infinities_and_nan_reach_no_earlier_token(wz, dtype, T, l2, bad, what):
    """A q spoils its own token's outputs, a v its column from its token on, a k, g or beta its head from there on; all
    other outputs and states keep their bits."""
    if what == "g" and bad == -math.inf:
        pytest.skip("a reset")
    r = gen(26)
    x = gdn_inputs(T, 2, 4, 128, dtype, r, False, l2)
    names, at = ["q", "k", "v", "g", "beta", "s0"], T - 55
    assert 0 < at % 64 < 63
    clean = gdn_call(wz, *x, qk_l2norm=l2)
    y = [t.clone() for t in x]
    y[names.index(what)][(at, 1) if what in ("g", "beta") else (at, 1, 33)] = bad
    o, s = gdn_call(wz, *y, qk_l2norm=l2)
    spoiled_o, spoiled_s = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(s, dtype=torch.bool)
    if what == "q":
        spoiled_o[at, 2:] = True
    elif what == "v":
        spoiled_o[at:, 1, 33] = spoiled_s[1, 33] = True
    else:
        heads = slice(2, 4) if what == "k" else slice(1, 2)  # two value heads share a key head
        spoiled_o[at:, heads] = spoiled_s[heads] = True
    assert torch.equal(o[~spoiled_o], clean[0][~spoiled_o]) and torch.equal(s[~spoiled_s], clean[1][~spoiled_s])
    assert not torch.isfinite(o[spoiled_o]).any() and not torch.isfinite(s[spoiled_s]).any()


@pytest.mark.parametrize("T", [2, 40])
@pytest.mark.parametrize("size", [2.0**-140, 2.0**-60, 2.0**60, 2.0**119, 2.0**122])
def test_attn_query_sizes_over_fp32s_range(wz, T, size):
    """Scores far below 1 weigh all cells alike, scores far above 1 take the largest alone; nothing overflows on the way as
    long as the scores themselves are fp32 numbers (they reach 8 times the query's largest element here, at most)."""
    r = gen(27)
    n, hd = 64, 64
    rows, _, desc = make_cache(wz, n, 16, n, hd, r, True)
    q = torch.randn(T, 4, hd, generator=r, device=DEV) * size
    out, lse = torch.zeros_like(q), torch.zeros(T, 4, device=DEV)
    wz.kv_attn(q, out, desc, 1, n, source=wz.KV_FULL, pos_offset=n - T, lse=lse, workspace=workspace(wz, T, 4, 1, hd))
    o, wl, mag, _ = ref.attention(q, rows, 1, hd, hd**-0.5, [list(range(n - T + t + 1)) for t in range(T)])
    assert torch.isfinite(out).all() and torch.isfinite(lse).all()
    assert ((lse.double() - wl).abs() <= wl.abs() * 2.0**-16 + 2.0**-18).all()
    if size < 1:
        assert ((out.double() - o).abs() <= mag * 2.0**-19).all()
    else:  # one cell's value, unless two scores are as close as their own error
        v = ref.rows64(rows[2], rows[3], hd, 0)
        assert ((out.double().unsqueeze(2) - v).abs().amax(-1).amin(-1) <= 2.0**-20 * v.abs().max()).all()


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("T", [90, 400])
def test_gdn_fp16_outputs_are_rounded_once(wz, hd, T):
    """An fp16 call computes as the fp32 call on the same numbers does and rounds its outputs at the end. The two calls'
    results before that are within 2^-18 of each other (relative to the output's size, 22-bit parts and their sums), so a
    share of 2 * 2^-18 / 2^-11 of the roundings may fall the other way, and those by one step."""
    r = gen(28)
    q, k, v, g, beta, s0 = gdn_inputs(T, 2, 4, hd, torch.float16, r, False, True)
    o16, s16 = gdn_call(wz, q, k, v, g, beta, s0)
    o32, s32 = gdn_call(wz, q.float(), k.float(), v.float(), g, beta, s0)
    off = o16 != o32.half()
    assert off.double().mean() <= 2.0**-6
    assert ((o16.float() - o32).abs() <= 2.0**-10 * o32.abs() + 2.0**-24).all()
