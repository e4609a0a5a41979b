// kv_attn.cu -- attention over the INT8 KV cache that kv_append.cu writes: a sliding window plus a few first
// tokens that stay visible, for a chunk of new tokens (one to thousands) or for a tree of drafted tokens.
//
// Per query row (token t, query head) with its kv head's cells j:
//   x_j = scale * sum_g ks[j,g] * (q_g . kc[j,g])      g: 64-element groups, kc: int8 codes, ks: fp16 scales
//   o_g = sum_j softmax(x)_j vs[j,g] vc[j,g],          lse = ln sum_j exp(x_j)
// Codes are integers up to 127, exact in fp16, so the tensor cores multiply the codes themselves and the
// scales stay fp32: on the K side they multiply the per-group partial products, on the V side the softmax
// weights (one scaled copy of the weights per group). Products accumulate in fp32, statistics are fp32.
// The one rounding to fewer bits for fp16 calls is the scaled weight p * vs to fp16 (relative 2^-12 each,
// the size of the output's own rounding); fp32 calls split q and p * vs into two fp16 parts (22 bits).
//
// Weights entering the tensor cores are p * vs * 2^(7 - E) with a running E per row (from the largest finite
// scale among the cells that the row sees, as the running maximum of its scores), so they sit in fp16's
// upper range whatever the scales' size, and a row's result does not depend on cells it does not see. A
// row's running maximum moves only when a score passes it by 2^8: its weights stay below 2^15 either way.
// The second part of an fp32 call's weight enters 2^11 times as large and its products come back by 2^-11,
// so that it is not cut off at fp16's smallest number.
#include "launch.hpp"
#include "common.cuh"

namespace wzyb {

constexpr int kAttnMaxRanges = 5;

struct KvAttnArgs {
    const void* q;
    int64_t q_head, q_row;  // elements between heads / tokens
    void* out;
    int64_t o_head, o_row;
    float* lse;
    wzyb_kv_cache c;       // the committed tokens
    wzyb_kv_cache d;       // drafts: node i at ring cell i (tree calls)
    const uint32_t* mask;  // [T, mask_words] (tree calls)
    const int32_t* depth;
    int mask_words;
    int tree;
    int from_full;
    int T, G, kv_heads;  // G: query heads per kv head
    const int32_t* d_base_pos;
    int64_t pos_offset;
    int64_t window, sinks;
    float scale_log2;  // scale * log2(e)
    uint64_t ring_div, ring_recip;
    int splits;
    float* part_o;   // [splits, T * q_heads, HD]
    float2* part_ml;  // [splits, T * q_heads]: running maximum (log2 units) and sum
};

// The visible cells of a row tile as up to five ranges of positions (pinned part and recent part of the
// ring, each cut by the sinks and by the window; then the drafts), cut into tiles of kN keys that never
// cross a range. Built by one thread, read by all.
struct KeyPlan {
    int lo[kAttnMaxRanges], hi[kAttnMaxRanges];
    int first[kAttnMaxRanges + 1];  // first tile of each range
    int ranges;
    int draft;  // index of the draft range, or -1
    int row_hi_min, row_lo_max;  // over the tile's rows: every row sees (lo_max, hi_min]
    int sinks;
};

__device__ __forceinline__ int clamp_i32(int64_t x, int lo) {
    return (int)(x < lo ? lo : (x > 0x7FFFFFFF ? 0x7FFFFFFF : x));
}

// A row sees positions j with j <= hi and (j < sinks or j > lo).
struct RowSpan {
    int hi, lo;
};
__device__ __forceinline__ RowSpan row_span(const KvAttnArgs& a, int64_t base, int t) {
    const int64_t p = base + (a.tree ? (int64_t)__ldg(a.depth + t) : t);
    RowSpan r;
    r.hi = clamp_i32(p, -1);
    r.lo = clamp_i32(p - a.window, -1);
    return r;
}

template <int kN>
__device__ __forceinline__ void plan_push(KeyPlan& k, int64_t lo, int64_t hi) {
    if (lo >= hi) return;
    const int n = k.ranges++;
    k.lo[n] = (int)lo;
    k.hi[n] = (int)hi;
    k.first[n + 1] = k.first[n] + (int)((hi - lo + kN - 1) / kN);
}

// Tokens [t0, t1) of the call. Run by one warp, whose lanes share the rows; lane 0 writes.
template <int kN>
__device__ __forceinline__ void build_plan(const KvAttnArgs& a, KeyPlan& k, int64_t base, int t0, int t1, int lane) {
    int hi_min = 0x7FFFFFFF, hi_max = -1, lo_min = 0x7FFFFFFF, lo_max = -1;
    for (int t = t0 + lane; t < t1; t += 32) {
        const RowSpan r = row_span(a, base, t);
        hi_min = min(hi_min, r.hi);
        hi_max = max(hi_max, r.hi);
        lo_min = min(lo_min, r.lo);
        lo_max = max(lo_max, r.lo);
    }
    hi_min = __reduce_min_sync(0xffffffffu, hi_min);
    hi_max = __reduce_max_sync(0xffffffffu, hi_max);
    lo_min = __reduce_min_sync(0xffffffffu, lo_min);
    lo_max = __reduce_max_sync(0xffffffffu, lo_max);
    if (lane != 0) return;
    const int64_t end = base + (a.tree ? 0 : a.T);  // one past the last appended position
    const int64_t sinks = a.sinks < 0x7FFFFFFF ? a.sinks : 0x7FFFFFFF;
    k.ranges = 0;
    k.first[0] = 0;
    k.draft = -1;
    k.row_hi_min = hi_min;
    k.row_lo_max = lo_max;
    k.sinks = (int)sinks;
    int64_t stop = (int64_t)hi_max + 1 < end ? (int64_t)hi_max + 1 : end;
    stop = stop < a.c.max_ctx ? stop : a.c.max_ctx;
    const int64_t near = (int64_t)lo_min + 1;  // first position inside some row's window
    const int64_t cap = a.c.ring_cap;
    const bool pinned = !a.from_full && cap > 2 * kKvSinkPin;
    int64_t from[2] = {0, 0}, to[2] = {pinned ? kKvSinkPin : 0, stop};
    if (pinned)
        from[1] = end - (cap - kKvSinkPin) > kKvSinkPin ? end - (cap - kKvSinkPin) : kKvSinkPin;
    else if (!a.from_full)
        from[1] = end - cap > 0 ? end - cap : 0;
    for (int s = 0; s < 2; ++s) {
        const int64_t b = to[s] < stop ? to[s] : stop, lo = from[s];
        const int64_t sink_end = sinks < b ? sinks : b, win = near > lo ? near : lo;
        if (sink_end >= win) {  // the two parts touch
            plan_push<kN>(k, lo, b);
        } else {
            plan_push<kN>(k, lo, sink_end);
            plan_push<kN>(k, win, b);
        }
    }
    if (a.tree) {
        k.draft = k.ranges;
        plan_push<kN>(k, 0, a.T);
    }
}

// Tile `i` of the plan: its range, first position and key count.
struct KeyTile {
    int pos, count;
    bool draft;
};
template <int kN>
__device__ __forceinline__ KeyTile key_tile(const KeyPlan& k, int i) {
    int r = 0;
#pragma unroll
    for (int n = 1; n < kAttnMaxRanges; ++n)
        if (n < k.ranges && i >= k.first[n]) r = n;
    KeyTile t;
    t.pos = k.lo[r] + (i - k.first[r]) * kN;
    t.count = min(kN, k.hi[r] - t.pos);
    t.draft = r == k.draft;
    return t;
}

// Every row of the row tile sees the whole key tile.
template <int kN>
__device__ __forceinline__ bool tile_unmasked(const KeyPlan& k, const KeyTile& t) {
    const int last = t.pos + t.count - 1;
    return !t.draft && t.count == kN && last <= k.row_hi_min && (last < k.sinks || t.pos > k.row_lo_max);
}

__device__ __forceinline__ int64_t cell_of(const KvAttnArgs& a, bool draft, int pos) {
    return draft || a.from_full ? pos : kv_ring_cell(pos, a.c.ring_cap, a.ring_div, a.ring_recip);
}

// The planes of one kv head: codes of cell c at kq + c * kvd, scales at ks + c * spc.
struct Planes {
    const int8_t* kq;
    const int8_t* vq;
    const uint16_t* ks;
    const uint16_t* vs;
};
template <int HD>
__device__ __forceinline__ Planes planes_of(const KvAttnArgs& a, bool draft, int head) {
    const wzyb_kv_cache& c = draft ? a.d : a.c;
    const bool full = !draft && a.from_full;
    Planes p;
    p.kq = (full ? c.full_k_q : c.ring_k_q) + head * HD;
    p.vq = (full ? c.full_v_q : c.ring_v_q) + head * HD;
    p.ks = (full ? c.full_k_s : c.ring_k_s) + head * (HD / 64);
    p.vs = (full ? c.full_v_s : c.ring_v_s) + head * (HD / 64);
    return p;
}

// HD / 64 consecutive fp16 scales (aligned to their own size) as fp32.
template <int NG>
__device__ __forceinline__ void load_scales(const uint16_t* p, float (&s)[NG]) {
    if constexpr (NG == 4) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u.x));
        const float2 y = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
        s[0] = x.x;
        s[1] = x.y;
        s[2] = y.x;
        s[3] = y.y;
    } else if constexpr (NG == 2) {
        const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(p));
        const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&u));
        s[0] = x.x;
        s[1] = x.y;
    } else {
        s[0] = __half2float(__ushort_as_half(__ldg(p)));
    }
}

// Two int8 codes as fp16, exactly: with the sign bit flipped (u = c + 128) the byte under the high byte
// 0x64 is the fp16 number 1024 + u, and 1024 + u - 1152 = c. `sel` picks the bytes of flipped word w.
__device__ __forceinline__ uint32_t codes_f16(uint32_t w, uint32_t sel) {
    const uint32_t u = __byte_perm(w, 0x64646464u, sel);
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
constexpr uint32_t kSelLo = 0x4140u, kSelHi = 0x4342u;  // bytes 0, 1 and bytes 2, 3

// fp16 pair and, for fp32 calls, 2^11 times what it leaves of the pair
constexpr float kLoUp = 2048.f;
__device__ __forceinline__ void split_f16(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = pack_f16((x - f.x) * kLoUp, (y - f.y) * kLoUp);
}

// Exponent e with x < 2^e <= 2x for a positive finite scale, -1000 for 0, infinities and NaN: the running
// scale exponent E is the maximum over the visible keys' scales.
__device__ __forceinline__ int scale_exp(float x) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t e = b >> 23;  // scales are >= 0; a set sign bit lands outside [1, 254]
    return e >= 1 && e <= 254 ? (int)e - 126 : -1000;
}
__device__ __forceinline__ float exp2_int(int e) {  // 2^e, 0 below the normal range
    return e < -126 ? 0.f : __int_as_float((e + 127) << 23);
}

// Query rows of a tile to shared memory as fp16 (kSplit: two parts of x * 2^-e, e from the row's largest
// magnitude, so every fp32 row uses fp16's range). One warp per row in turn. qs[row * ld + col]; the
// factor that turns a raw dot into log2 units goes to row_scale.
template <typename T, int HD, bool kSplit>
__device__ __forceinline__ void stage_rows(const KvAttnArgs& a, int head, int row0, int rows, int ntile, __half* qs,
                                           __half* ql, int ld, float* row_scale, int warp, int nwarps, int lane) {
    for (int r = warp; r < ntile; r += nwarps) {
        constexpr int kE = HD / 32;  // consecutive elements per lane
        float x[kE];
        const int row = row0 + r;
        if (row < rows) {
            const int t = row / a.G, g = row - t * a.G;
            const T* p = static_cast<const T*>(a.q) + t * a.q_row + (int64_t)(head * a.G + g) * a.q_head + lane * kE;
#pragma unroll
            for (int i = 0; i < kE; ++i) x[i] = (float)p[i];
        } else {
#pragma unroll
            for (int i = 0; i < kE; ++i) x[i] = 0.f;
        }
        float f = a.scale_log2;
        if constexpr (kSplit) {
            float am = 0.f;
#pragma unroll
            for (int i = 0; i < kE; ++i) am = fmaxf(am, fabsf(x[i]));
            am = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(am)));
            int e = scale_exp(am);
            if (e < -100 || e > 120) e = 0;
            const float down = exp2_int(-e);
            f *= exp2_int(e);
#pragma unroll
            for (int i = 0; i < kE; ++i) x[i] *= down;
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) {
            const __half h = __float2half_rn(x[i]);
            qs[r * ld + lane * kE + i] = h;
            if constexpr (kSplit) ql[r * ld + lane * kE + i] = __float2half_rn(x[i] - __half2float(h));
        }
        if (lane == 0) row_scale[r] = f;
    }
}

// A row's result: o / l with one split, otherwise the unnormalised part with its (m, l).
template <typename T>
__device__ __forceinline__ void store_out2(T* p, float x, float y);
template <>
__device__ __forceinline__ void store_out2<__half>(__half* p, float x, float y) {
    *reinterpret_cast<__half2*>(p) = __floats2half2_rn(x, y);
}
template <>
__device__ __forceinline__ void store_out2<float>(float* p, float x, float y) {
    *reinterpret_cast<float2*>(p) = make_float2(x, y);
}

// ----------------------------------------------------------------------------------------------------
// Few query rows per kv head (decode): a CTA takes 8 rows and a share of the key tiles, its warps take
// 16-key tiles in turn. The products are transposed, x^T = K q^T and o^T = V^T p^T, so the keys (and the
// output's dimensions) fill the MMA's 16 rows and the 8 query rows its 8 columns: nothing is padded for a
// group of 8 query heads. A lane's part of K and V comes straight from global memory in the order in which
// the MMA takes it (any order of the contracted dimension is right as long as both operands have the same):
// 16 bytes of K per row and group, 8 bytes of V per key and group. Weights pass from the accumulator layout
// of the first product to the operand layout of the second by an 8x8 register transpose.
// ----------------------------------------------------------------------------------------------------
template <typename T, int HD>
__global__ void __launch_bounds__(128) kv_attn_few_kernel(const KvAttnArgs a) {
    pdl_begin();
    constexpr bool kSplit = sizeof(T) == 4;
    constexpr int NG = HD / 64, kN = 16, kWarps = 4, kLd = HD + 8;
    __shared__ KeyPlan plan;
    __shared__ __align__(16) __half qs[8 * kLd];
    __shared__ __align__(16) __half ql[kSplit ? 8 * kLd : 8];
    __shared__ float row_scale[8];
    __shared__ float sm[kWarps][8], sl[kWarps][8];
    __shared__ __align__(16) float so[kWarps][8][HD + 4];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int split = blockIdx.x, row0 = blockIdx.y * 8, head = blockIdx.z;
    const int rows = a.T * a.G;
    const int64_t base = (a.d_base_pos ? (int64_t)__ldg(a.d_base_pos) : 0) + a.pos_offset;
    const int t_first = row0 / a.G, t_last = (min(row0 + 8, rows) - 1) / a.G;
    if (warp == 0) build_plan<kN>(a, plan, base, t_first, t_last + 1, lane);
    stage_rows<T, HD, kSplit>(a, head, row0, rows, 8, qs, ql, kLd, row_scale, warp, kWarps, lane);
    __syncthreads();

    const int ntiles = plan.first[plan.ranges];
    const int tb = (int)((int64_t)ntiles * split / a.splits), te = (int)((int64_t)ntiles * (split + 1) / a.splits);
    const int kvd = a.kv_heads * HD, spc = a.kv_heads * NG;

    // rows 2*t4 and 2*t4 + 1 of the tile
    int rt[2];
    RowSpan span[2];
    float rs[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        rt[i] = min(row0 + 2 * t4 + i, rows - 1) / a.G;
        span[i] = row_span(a, base, rt[i]);
        rs[i] = row_scale[2 * t4 + i];
    }

    float o[NG][4][4];
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[i][j][c] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int E[2] = {-1000, -1000};

    for (int it = tb + warp; it < te; it += kWarps) {
        const KeyTile kt = key_tile<kN>(plan, it);
        const Planes pl = planes_of<HD>(a, kt.draft, head);
        // lanes 0..15 find the tile's cells; a key past the tile's end takes the first one's cell (its
        // scales count as 0 and its scores as -inf)
        const int mine = lane & 15;
        const int my_cell = (int)cell_of(a, kt.draft, kt.pos + (mine < kt.count ? mine : 0));
        int kcell[2], vcell[4];
#pragma unroll
        for (int i = 0; i < 2; ++i) kcell[i] = __shfl_sync(0xffffffffu, my_cell, g + 8 * i);
#pragma unroll
        for (int i = 0; i < 4; ++i) vcell[i] = __shfl_sync(0xffffffffu, my_cell, 2 * t4 + (i & 1) + (i >> 1) * 8);
        uint4 kr[2][NG];
        uint2 vr[4][NG];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < NG; ++n)
                kr[i][n] = __ldg(reinterpret_cast<const uint4*>(pl.kq + (int64_t)kcell[i] * kvd + n * 64 + t4 * 16));
        float ks[2][NG], vs[2][NG];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            load_scales<NG>(pl.ks + (int64_t)kcell[i] * spc, ks[i]);
            load_scales<NG>(pl.vs + (int64_t)kcell[i] * spc, vs[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int n = 0; n < NG; ++n)
                vr[i][n] = __ldg(reinterpret_cast<const uint2*>(pl.vq + (int64_t)vcell[i] * kvd + n * 64 + g * 8));

        // scores of keys g and g + 8 for rows 2*t4, 2*t4 + 1: s[0], s[1] and s[2], s[3]
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            const uint32_t w0[4] = {kr[0][n].x, kr[0][n].y, kr[0][n].z, kr[0][n].w};
            const uint32_t w1[4] = {kr[1][n].x, kr[1][n].y, kr[1][n].z, kr[1][n].w};
            const uint4 q0 = *reinterpret_cast<const uint4*>(qs + g * kLd + n * 64 + t4 * 16);
            const uint4 q1 = *reinterpret_cast<const uint4*>(qs + g * kLd + n * 64 + t4 * 16 + 8);
            const uint32_t qb[8] = {q0.x, q0.y, q0.z, q0.w, q1.x, q1.y, q1.z, q1.w};
            uint32_t qc[8];
            if constexpr (kSplit) {
                const uint4 r0 = *reinterpret_cast<const uint4*>(ql + g * kLd + n * 64 + t4 * 16);
                const uint4 r1 = *reinterpret_cast<const uint4*>(ql + g * kLd + n * 64 + t4 * 16 + 8);
                qc[0] = r0.x, qc[1] = r0.y, qc[2] = r0.z, qc[3] = r0.w;
                qc[4] = r1.x, qc[5] = r1.y, qc[6] = r1.z, qc[7] = r1.w;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t x0 = w0[j] ^ 0x80808080u, x1 = w1[j] ^ 0x80808080u;
                const uint32_t fa[4] = {codes_f16(x0, kSelLo), codes_f16(x1, kSelLo), codes_f16(x0, kSelHi),
                                        codes_f16(x1, kSelHi)};
                mma_f16(acc, fa, qb[2 * j], qb[2 * j + 1]);
                if constexpr (kSplit) mma_f16(acc, fa, qc[2 * j], qc[2 * j + 1]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) s[c] = fmaf(acc[c], ks[c >> 1][n], s[c]);
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) s[c] *= rs[c & 1];
        int ek[2] = {-1000, -1000}, e[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < NG; ++n) ek[i] = max(ek[i], scale_exp(vs[i][n]));
        if (tile_unmasked<kN>(plan, kt)) {  // warp-uniform
            e[0] = e[1] = max(ek[0], ek[1]);
        } else {
            e[0] = e[1] = -1000;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = g + (c >> 1) * 8, pos = kt.pos + key;
                bool see = key < kt.count;
                if (kt.draft) {
                    if (see) see = (__ldg(a.mask + (int64_t)rt[c & 1] * a.mask_words + (pos >> 5)) >> (pos & 31)) & 1u;
                } else {
                    see = see && pos <= span[c & 1].hi && (pos < plan.sinks || pos > span[c & 1].lo);
                }
                if (see)
                    e[c & 1] = max(e[c & 1], ek[c >> 1]);
                else
                    s[c] = -INFINITY;
            }
        }
        float top[2] = {fmaxf(s[0], s[2]), fmaxf(s[1], s[3])};
        if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f || e[0] > E[0] || e[1] > E[1])) {
            float alpha[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) {
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], x));
                    e[i] = max(e[i], __shfl_xor_sync(0xffffffffu, e[i], x));
                }
                alpha[i] = 1.f;
                if (top[i] > m[i] + 8.f || e[i] > E[i]) {
                    top[i] = fmaxf(top[i], m[i]);
                    e[i] = max(e[i], E[i]);
                    alpha[i] = ex2_approx(m[i] - (top[i] == -INFINITY ? 0.f : top[i]));
                    l[i] *= alpha[i];
                    alpha[i] *= exp2_int(E[i] - e[i]);
                    m[i] = top[i];
                    E[i] = e[i];
                }
            }
#pragma unroll
            for (int i = 0; i < NG; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[i][j][c] *= alpha[c & 1];
        }
        const float mr[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
        float p[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            p[c] = ex2_approx(s[c] - mr[c & 1]);
            l[c & 1] += p[c];
        }
        float up[2];  // largest scale to [2^6, 2^7)
#pragma unroll
        for (int i = 0; i < 2; ++i) up[i] = E[i] <= -1000 ? 0.f : exp2_int(7 - E[i]);
        uint32_t vx[4][2];
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            // masked places: a weight of 0 stays 0 whatever the cell's scale (infinite or NaN) is
            float w[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) w[c] = p[c] == 0.f ? 0.f : p[c] * (vs[c >> 1][n] * up[c & 1]);
            uint32_t b0, b1, c0 = 0, c1 = 0;
            if constexpr (kSplit) {
                split_f16(w[0], w[1], b0, c0);
                split_f16(w[2], w[3], b1, c1);
                c0 = transpose8(c0);
                c1 = transpose8(c1);
            } else {
                b0 = pack_f16(w[0], w[1]);
                b1 = pack_f16(w[2], w[3]);
            }
            b0 = transpose8(b0);
            b1 = transpose8(b1);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                vx[i][0] = vr[i][n].x ^ 0x80808080u;
                vx[i][1] = vr[i][n].y ^ 0x80808080u;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {  // dimensions n*64 + 8*g + 2*j (row g) and + 1 (row g + 8)
                const uint32_t sel = (j & 1) ? 0x7362u : 0x5140u;
                const uint32_t near = __byte_perm(vx[0][j >> 1], vx[1][j >> 1], sel);
                const uint32_t far = __byte_perm(vx[2][j >> 1], vx[3][j >> 1], sel);
                const uint32_t fa[4] = {codes_f16(near, kSelLo), codes_f16(near, kSelHi), codes_f16(far, kSelLo),
                                        codes_f16(far, kSelHi)};
                if constexpr (kSplit) {
                    float acc[4] = {0.f, 0.f, 0.f, 0.f};
                    mma_f16(acc, fa, c0, c1);
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[c] *= 1.f / kLoUp;
                    mma_f16(acc, fa, b0, b1);
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[n][j][c] += acc[c];
                } else {
                    mma_f16(o[n][j], fa, b0, b1);
                }
            }
        }
    }

    // join the warps' parts in order
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    if (g == 0) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            sm[warp][2 * t4 + i] = m[i];
            sl[warp][2 * t4 + i] = l[i];
        }
    }
    float back[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) back[i] = E[i] <= -1000 ? 0.f : exp2_int(E[i] - 7);
#pragma unroll
    for (int n = 0; n < NG; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c)
                so[warp][2 * t4 + (c & 1)][n * 64 + 8 * g + 2 * j + (c >> 1)] = o[n][j][c] * back[c & 1];
    __syncthreads();
    for (int r = warp; r < 8; r += kWarps) {
        const int row = row0 + r;
        if (row >= rows) break;
        float top = -INFINITY, sum = 0.f, f[kWarps];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, sm[w][r]);
        const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            f[w] = ex2_approx(sm[w][r] - ref);
            sum += sl[w][r] * f[w];
        }
        const int t = row / a.G, hq = head * a.G + (row - t * a.G);
        const int64_t orow = (int64_t)t * a.G * a.kv_heads + hq;
        float norm = 1.f;
        if (a.splits == 1) {
            norm = sum == 0.f ? 0.f : 1.f / sum;
            if (lane == 0 && a.lse != nullptr) a.lse[orow] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
        } else if (lane == 0) {
            a.part_ml[(int64_t)split * rows * a.kv_heads + orow] = make_float2(top, sum);
        }
#pragma unroll
        for (int c = 0; c < HD / 64; ++c) {
            float2 x = make_float2(0.f, 0.f);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                const float2 y = *reinterpret_cast<const float2*>(&so[w][r][c * 64 + 2 * lane]);
                if (f[w] != 0.f) {
                    x.x = fmaf(y.x, f[w], x.x);
                    x.y = fmaf(y.y, f[w], x.y);
                }
            }
            if (a.splits == 1) {
                if (sum == 0.f) x = make_float2(0.f, 0.f);
                store_out2(static_cast<T*>(a.out) + t * a.o_row + hq * a.o_head + c * 64 + 2 * lane, x.x * norm, x.y * norm);
            } else {
                *reinterpret_cast<float2*>(a.part_o + ((int64_t)split * rows * a.kv_heads + orow) * HD + c * 64 + 2 * lane) = x;
            }
        }
    }
}

// ----------------------------------------------------------------------------------------------------
// Many query rows per kv head (prefill, large trees): a CTA takes 16 rows per warp and walks its share of
// 64-key tiles. The tile's codes come by cp.async as bytes while the tile before is worked through, are
// widened once to fp16 in shared memory and used by every warp. Rows lead (x = q K^T, o = p V), so the
// weights go from the first product's accumulators to the second's operand within each lane.
// ----------------------------------------------------------------------------------------------------
template <typename T, int HD, int kWarps>
struct TileSmem {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kRows = 16 * kWarps, kLd = HD + 8, kN = 64, NG = HD / 64;
    __half qs[kRows * kLd];
    __half ql[kSplit ? kRows * kLd : 8];
    __half kf[kN * kLd];
    __half vf[kN * kLd];
    int8_t raw[2][kN * HD];
    float ks[kN][NG], vs[kN][NG];
    float row_scale[kRows];
    KeyPlan plan;
    int e_key[kN], e_max[kWarps];
};

template <typename T, int HD, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 1) kv_attn_tile_kernel(const KvAttnArgs a) {
    pdl_begin();
    using S = TileSmem<T, HD, kWarps>;
    constexpr bool kSplit = S::kSplit;
    constexpr int NG = S::NG, kN = S::kN, kLd = S::kLd, kThreads = kWarps * 32;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    S& sm = *reinterpret_cast<S*>(smem_raw);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int split = blockIdx.x, row0 = blockIdx.y * S::kRows, head = blockIdx.z;
    const int rows = a.T * a.G;
    const int64_t base = (a.d_base_pos ? (int64_t)__ldg(a.d_base_pos) : 0) + a.pos_offset;
    if (warp == 0)
        build_plan<kN>(a, sm.plan, base, row0 / a.G, (min(row0 + S::kRows, rows) - 1) / a.G + 1, lane);
    stage_rows<T, HD, kSplit>(a, head, row0, rows, S::kRows, sm.qs, sm.ql, kLd, sm.row_scale, warp, kWarps, lane);
    __syncthreads();
    const KeyPlan& plan = sm.plan;
    const int ntiles = plan.first[plan.ranges];
    const int tb = (int)((int64_t)ntiles * split / a.splits), te = (int)((int64_t)ntiles * (split + 1) / a.splits);
    const int kvd = a.kv_heads * HD, spc = a.kv_heads * NG;

    int rt[2];
    RowSpan span[2];
    float rs[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        rt[i] = min(row0 + warp * 16 + g + 8 * i, rows - 1) / a.G;
        span[i] = row_span(a, base, rt[i]);
        rs[i] = sm.row_scale[warp * 16 + g + 8 * i];
    }

    // bytes of tile `it` into sm.raw; keys past the tile's end are not fetched (their bytes are whatever
    // the buffer held: finite codes, whose scales count as 0)
    auto fetch = [&](int it) {
        const KeyTile kt = key_tile<kN>(plan, it);
        const Planes pl = planes_of<HD>(a, kt.draft, head);
        constexpr int kChunks = HD / 16;
#pragma unroll 4
        for (int i = tid; i < kN * kChunks; i += kThreads) {
            const int key = i / kChunks, c = (i % kChunks) * 16;
            if (key >= kt.count) continue;
            const int64_t at = cell_of(a, kt.draft, kt.pos + key) * kvd + c;
            cp_async16(&sm.raw[0][key * HD + c], pl.kq + at);
            cp_async16(&sm.raw[1][key * HD + c], pl.vq + at);
        }
        cp_async_commit();
    };
    // scales of one key per thread
    float nks[NG], nvs[NG];
    auto fetch_scales = [&](int it) {
#pragma unroll
        for (int n = 0; n < NG; ++n) nks[n] = nvs[n] = 0.f;
        if (tid < kN) {
            const KeyTile kt = key_tile<kN>(plan, it);
            if (tid < kt.count) {
                const Planes pl = planes_of<HD>(a, kt.draft, head);
                const int64_t at = cell_of(a, kt.draft, kt.pos + tid) * spc;
                load_scales<NG>(pl.ks + at, nks);
                load_scales<NG>(pl.vs + at, nvs);
            }
        }
    };

    float o[HD / 8][4];
#pragma unroll
    for (int i = 0; i < HD / 8; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[i][c] = 0.f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int E[2] = {-1000, -1000};
    for (int i = tid; i < (int)sizeof(sm.raw) / 16; i += kThreads) reinterpret_cast<uint4*>(sm.raw)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();

    if (tb < te) {
        fetch(tb);
        fetch_scales(tb);
    }
    for (int it = tb; it < te; ++it) {
        cp_async_wait<0>();
        int e = -1000;
        if (tid < kN) {
#pragma unroll
            for (int n = 0; n < NG; ++n) {
                sm.ks[tid][n] = nks[n];
                sm.vs[tid][n] = nvs[n];
                e = max(e, scale_exp(nvs[n]));
            }
            sm.e_key[tid] = e;
        }
        e = __reduce_max_sync(0xffffffffu, e);
        if (lane == 0) sm.e_max[warp] = e;
        __syncthreads();
        for (int i = tid; i < kN * HD / 16; i += kThreads) {
            const int key = i / (HD / 16), c = (i % (HD / 16)) * 16;
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                const uint4 w = *reinterpret_cast<const uint4*>(&sm.raw[b][key * HD + c]);
                const uint32_t x[4] = {w.x ^ 0x80808080u, w.y ^ 0x80808080u, w.z ^ 0x80808080u, w.w ^ 0x80808080u};
                uint4* const d = reinterpret_cast<uint4*>((b ? sm.vf : sm.kf) + key * kLd + c);
                d[0] = make_uint4(codes_f16(x[0], kSelLo), codes_f16(x[0], kSelHi), codes_f16(x[1], kSelLo),
                                  codes_f16(x[1], kSelHi));
                d[1] = make_uint4(codes_f16(x[2], kSelLo), codes_f16(x[2], kSelHi), codes_f16(x[3], kSelLo),
                                  codes_f16(x[3], kSelHi));
            }
        }
#pragma unroll
        for (int w = 0; w < kWarps; ++w) e = max(e, sm.e_max[w]);
        __syncthreads();
        const KeyTile kt = key_tile<kN>(plan, it);
        if (it + 1 < te) {
            fetch(it + 1);
            fetch_scales(it + 1);
        }

        float s[kN / 8][4];
#pragma unroll
        for (int i = 0; i < kN / 8; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) s[i][c] = 0.f;
        const int qrow = warp * 16 + (lane & 15), qcol = (lane >> 4) * 8;
        const int krow = (lane & 7) + ((lane >> 4) << 3), kcol = ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            float acc[kN / 8][4];
#pragma unroll
            for (int i = 0; i < kN / 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
                uint32_t fa[4], fl[4];
                ldmatrix_x4(fa, sm.qs + qrow * kLd + n * 64 + kk * 16 + qcol);
                if constexpr (kSplit) ldmatrix_x4(fl, sm.ql + qrow * kLd + n * 64 + kk * 16 + qcol);
#pragma unroll
                for (int i = 0; i < kN / 16; ++i) {
                    uint32_t fb[4];
                    ldmatrix_x4(fb, sm.kf + (i * 16 + krow) * kLd + n * 64 + kk * 16 + kcol);
                    mma_f16(acc[2 * i], fa, fb[0], fb[1]);
                    mma_f16(acc[2 * i + 1], fa, fb[2], fb[3]);
                    if constexpr (kSplit) {
                        mma_f16(acc[2 * i], fl, fb[0], fb[1]);
                        mma_f16(acc[2 * i + 1], fl, fb[2], fb[3]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kN / 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) s[i][c] = fmaf(acc[i][c], sm.ks[i * 8 + 2 * t4 + (c & 1)][n], s[i][c]);
        }
        float top[2] = {-INFINITY, -INFINITY};
        int er[2] = {e, e};
        if (tile_unmasked<kN>(plan, kt)) {  // CTA-uniform
#pragma unroll
            for (int i = 0; i < kN / 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s[i][c] *= rs[c >> 1];
                    top[c >> 1] = fmaxf(top[c >> 1], s[i][c]);
                }
        } else {
            er[0] = er[1] = -1000;
#pragma unroll
            for (int i = 0; i < kN / 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    s[i][c] *= rs[c >> 1];
                    const int key = i * 8 + 2 * t4 + (c & 1), pos = kt.pos + key;
                    bool see = key < kt.count;
                    if (kt.draft) {
                        if (see) see = (__ldg(a.mask + (int64_t)rt[c >> 1] * a.mask_words + (pos >> 5)) >> (pos & 31)) & 1u;
                    } else {
                        see = see && pos <= span[c >> 1].hi && (pos < plan.sinks || pos > span[c >> 1].lo);
                    }
                    if (see)
                        er[c >> 1] = max(er[c >> 1], sm.e_key[key]);
                    else
                        s[i][c] = -INFINITY;
                    top[c >> 1] = fmaxf(top[c >> 1], s[i][c]);
                }
        }
        if (__any_sync(0xffffffffu, top[0] > m[0] + 8.f || top[1] > m[1] + 8.f || er[0] > E[0] || er[1] > E[1])) {
            float alpha[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) {
                    top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], x));
                    er[i] = max(er[i], __shfl_xor_sync(0xffffffffu, er[i], x));
                }
                alpha[i] = 1.f;
                if (top[i] > m[i] + 8.f || er[i] > E[i]) {
                    top[i] = fmaxf(top[i], m[i]);
                    er[i] = max(er[i], E[i]);
                    alpha[i] = ex2_approx(m[i] - (top[i] == -INFINITY ? 0.f : top[i]));
                    l[i] *= alpha[i];
                    alpha[i] *= exp2_int(E[i] - er[i]);
                    m[i] = top[i];
                    E[i] = er[i];
                }
            }
#pragma unroll
            for (int i = 0; i < HD / 8; ++i)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[i][c] *= alpha[c >> 1];
        }
        const float mr[2] = {m[0] == -INFINITY ? 0.f : m[0], m[1] == -INFINITY ? 0.f : m[1]};
#pragma unroll
        for (int i = 0; i < kN / 8; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                s[i][c] = ex2_approx(s[i][c] - mr[c >> 1]);
                l[c >> 1] += s[i][c];
            }
        float up[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) up[i] = E[i] <= -1000 ? 0.f : exp2_int(7 - E[i]);
        const int vrow = (lane & 7) + ((lane >> 3) & 1) * 8, vcol = (lane >> 4) * 8;
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            // the tile's products of one group, added to o afterwards: the tensor cores cut each sum off
            // towards zero, which over thousands of tiles would be a drift of the running sums
            float acc[8][4];
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[j][c] = 0.f;
#pragma unroll
            for (int part = kSplit ? 1 : 0; part >= 0; --part) {  // fp32 calls: the second parts first
#pragma unroll
                for (int kk = 0; kk < kN / 16; ++kk) {
                    uint32_t fa[4];
#pragma unroll
                    for (int b = 0; b < 2; ++b) {  // keys kk*16 + b*8 + 2*t4, + 1
                        const float v0 = sm.vs[kk * 16 + b * 8 + 2 * t4][n], v1 = sm.vs[kk * 16 + b * 8 + 2 * t4 + 1][n];
                        const float (&p)[4] = s[2 * kk + b];
                        // masked places: a weight of 0 stays 0 whatever the cell's scale (infinite or NaN) is
                        const float w[4] = {p[0] == 0.f ? 0.f : p[0] * (v0 * up[0]), p[1] == 0.f ? 0.f : p[1] * (v1 * up[0]),
                                            p[2] == 0.f ? 0.f : p[2] * (v0 * up[1]), p[3] == 0.f ? 0.f : p[3] * (v1 * up[1])};
                        if (part == 1) {
                            uint32_t hi;
                            split_f16(w[0], w[1], hi, fa[2 * b]);
                            split_f16(w[2], w[3], hi, fa[2 * b + 1]);
                        } else {
                            fa[2 * b] = pack_f16(w[0], w[1]);
                            fa[2 * b + 1] = pack_f16(w[2], w[3]);
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t fb[4];
                        ldmatrix_x4_t(fb, sm.vf + (kk * 16 + vrow) * kLd + n * 64 + j * 16 + vcol);
                        mma_f16(acc[2 * j], fa, fb[0], fb[1]);
                        mma_f16(acc[2 * j + 1], fa, fb[2], fb[3]);
                    }
                }
                if (part == 1) {
#pragma unroll
                    for (int j = 0; j < 8; ++j)
#pragma unroll
                        for (int c = 0; c < 4; ++c) acc[j][c] *= 1.f / kLoUp;
                }
            }
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) o[n * 8 + j][c] += acc[j][c];
        }
        __syncthreads();  // kf, vf and the scales are free
    }

#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float back = E[i] <= -1000 ? 0.f : exp2_int(E[i] - 7);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
        l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
        const int row = row0 + warp * 16 + g + 8 * i;
        if (row >= rows) continue;
        const int t = row / a.G, hq = head * a.G + (row - t * a.G);
        const int64_t orow = (int64_t)t * a.G * a.kv_heads + hq;
        if (a.splits == 1) {
            const float norm = l[i] == 0.f ? 0.f : back / l[i];
            if (t4 == 0 && a.lse != nullptr) a.lse[orow] = l[i] == 0.f ? -INFINITY : (m[i] + log2f(l[i])) * 0.6931471805599453f;
            T* const p = static_cast<T*>(a.out) + t * a.o_row + hq * a.o_head + 2 * t4;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n) store_out2(p + n * 8, o[n][2 * i] * norm, o[n][2 * i + 1] * norm);
        } else {
            const int64_t at = (int64_t)split * rows * a.kv_heads + orow;
            if (t4 == 0) a.part_ml[at] = make_float2(m[i], l[i]);
            float* const p = a.part_o + at * HD + 2 * t4;
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
                *reinterpret_cast<float2*>(p + n * 8) = make_float2(o[n][2 * i] * back, o[n][2 * i + 1] * back);
        }
    }
}

// Joins the splits' parts of one row per CTA, in split order: HD / 4 lanes of 4 elements, the other threads
// take every kPar-th split; their sums meet in shared memory.
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv_attn_join_kernel(const KvAttnArgs a) {
    pdl_begin();
    constexpr int kLanes = HD / 4, kPar = 256 / kLanes;
    __shared__ float w[1024];
    __shared__ __align__(16) float4 part[kPar][kLanes];
    __shared__ float red[2];
    const int tid = threadIdx.x;
    const int qh = a.G * a.kv_heads;
    const int64_t row = blockIdx.x, nrows = (int64_t)a.T * qh;
    if (tid < 32) {
        float top = -INFINITY, sum = 0.f;
        for (int s = tid; s < a.splits; s += 32) top = fmaxf(top, a.part_ml[s * nrows + row].x);
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        const float ref = top == -INFINITY ? 0.f : top;
        for (int s = tid; s < a.splits; s += 32) {
            const float2 ml = a.part_ml[s * nrows + row];
            const float f = ex2_approx(ml.x - ref);
            w[s] = f;
            sum += ml.y * f;
        }
        sum = group_sum<32>(sum);
        if (tid == 0) {
            red[0] = top;
            red[1] = sum;
        }
    }
    __syncthreads();
    const float top = red[0], sum = red[1];
    const int c = tid % kLanes, s0 = tid / kLanes;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int s = s0; s < a.splits; s += kPar) {
        const float f = w[s];
        if (f == 0.f) continue;
        const float4 y = *reinterpret_cast<const float4*>(a.part_o + (s * nrows + row) * HD + 4 * c);
        x.x = fmaf(y.x, f, x.x);
        x.y = fmaf(y.y, f, x.y);
        x.z = fmaf(y.z, f, x.z);
        x.w = fmaf(y.w, f, x.w);
    }
    part[s0][c] = x;
    __syncthreads();
    if (s0 != 0) return;
#pragma unroll
    for (int i = 1; i < kPar; ++i) {
        const float4 y = part[i][c];
        x.x += y.x;
        x.y += y.y;
        x.z += y.z;
        x.w += y.w;
    }
    const float norm = sum == 0.f ? 0.f : 1.f / sum;
    const int t = (int)(row / qh), hq = (int)(row % qh);
    T* const p = static_cast<T*>(a.out) + t * a.o_row + hq * a.o_head + 4 * c;
    store_out2(p, x.x * norm, x.y * norm);
    store_out2(p + 2, x.z * norm, x.w * norm);
    if (tid == 0 && a.lse != nullptr) a.lse[row] = sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// Which kernel a call takes and how far the keys may be split, from the sizes alone (the key count is only
// known on the device). The workspace function and the launcher share it.
constexpr int kAttnCtas = 296;  // two CTAs per SM
struct AttnShape {
    bool few;
    int tile_rows, row_tiles, max_splits;
};
static AttnShape attn_shape(int64_t T, int q_heads, int kv_heads, bool f32) {
    AttnShape s;
    const int64_t rows = T * (q_heads / kv_heads);
    s.few = rows <= 16;
    s.tile_rows = s.few ? 8 : (f32 || rows <= 64 ? 64 : 128);
    s.row_tiles = (int)((rows + s.tile_rows - 1) / s.tile_rows);
    const int64_t ctas = (int64_t)s.row_tiles * kv_heads;
    s.max_splits = (int)(ctas >= (s.few ? kAttnCtas : kAttnCtas / 2) ? 1 : (s.few ? kAttnCtas : kAttnCtas / 2) / ctas);
    return s;
}

template <typename T, int HD>
static int launch_attn(KvAttnArgs& a, const AttnShape& s, cudaStream_t stream) {
    const dim3 grid(a.splits, s.row_tiles, a.kv_heads);
    int rc = WZYB_OK;
    if (s.few) {
        launch_k(kv_attn_few_kernel<T, HD>, grid, 128, 0, stream, a);
    } else if (s.tile_rows == 64) {
        const auto kern = kv_attn_tile_kernel<T, HD, 4>;
        rc = ensure_smem((const void*)kern, (int)sizeof(TileSmem<T, HD, 4>));
        if (rc != WZYB_OK) return rc;
        launch_k(kern, grid, 128, sizeof(TileSmem<T, HD, 4>), stream, a);
    } else if constexpr (sizeof(T) == 2) {
        const auto kern = kv_attn_tile_kernel<T, HD, 8>;
        rc = ensure_smem((const void*)kern, (int)sizeof(TileSmem<T, HD, 8>));
        if (rc != WZYB_OK) return rc;
        launch_k(kern, grid, 256, sizeof(TileSmem<T, HD, 8>), stream, a);
    }
    if (a.splits > 1) launch_k(kv_attn_join_kernel<T, HD>, a.T * a.G * a.kv_heads, 256, 0, stream, a);
    return launch_status();
}

static bool planes_aligned(const wzyb_kv_cache& c, bool full) {
    return full ? aligned16(c.full_k_q) && aligned16(c.full_v_q) && aligned16(c.full_k_s) && aligned16(c.full_v_s)
                : aligned16(c.ring_k_q) && aligned16(c.ring_v_q) && aligned16(c.ring_k_s) && aligned16(c.ring_v_s);
}

template <typename T>
static int attn_entry(const wzyb_kv_attn_args* p, const wzyb_kv_cache* drafts, const uint32_t* mask,
                      const int32_t* depth, bool tree, int64_t T_, cudaStream_t stream) {
    if (p == nullptr || p->cache == nullptr) return WZYB_ERR_NULL;
    const wzyb_kv_attn_args& x = *p;
    const wzyb_kv_cache& c = *x.cache;
    if (x.source != WZYB_KV_RING && x.source != WZYB_KV_FULL) return WZYB_ERR_VALUE;
    const bool full = x.source == WZYB_KV_FULL;
    if (!x.q || !x.out) return WZYB_ERR_NULL;
    if (full ? !(c.full_k_q && c.full_k_s && c.full_v_q && c.full_v_s)
             : !(c.ring_k_q && c.ring_k_s && c.ring_v_q && c.ring_v_s))
        return WZYB_ERR_NULL;
    if (tree && (!drafts || !mask || !depth || !drafts->ring_k_q || !drafts->ring_k_s || !drafts->ring_v_q ||
                 !drafts->ring_v_s))
        return WZYB_ERR_NULL;
    constexpr int64_t kMaxPos = 0x7FFFFFFF;
    if (T_ < 0 || T_ > (1 << 22) || x.kv_heads < 1 || x.kv_heads > 64 || x.q_heads < 1 || x.q_heads > 256 ||
        x.q_heads % x.kv_heads != 0 || (x.head_dim != 64 && x.head_dim != 128 && x.head_dim != 256) ||
        x.window < 0 || x.sinks < 0 || c.max_ctx < 0 || c.max_ctx > kMaxPos ||
        (!full && (c.ring_cap < 1 || c.ring_cap > kMaxPos)))
        return WZYB_ERR_SHAPE;
    if (tree && (T_ > WZYB_TREE_MAX_NODES || drafts->ring_cap < T_)) return WZYB_ERR_SHAPE;
    if (x.q_head_stride < 0 || x.q_row_stride < 0 || (x.q_heads > 1 && x.out_head_stride < x.head_dim) ||
        (T_ > 1 && x.out_row_stride < (x.q_heads - 1) * x.out_head_stride + x.head_dim))
        return WZYB_ERR_SHAPE;
    constexpr int64_t kB = sizeof(T);
    if (!aligned16(x.q) || !aligned16(x.out) || ((x.q_head_stride * kB) % 16) != 0 || ((x.q_row_stride * kB) % 16) != 0 ||
        ((x.out_head_stride * kB) % 16) != 0 || ((x.out_row_stride * kB) % 16) != 0 || !planes_aligned(c, full) ||
        (tree && !planes_aligned(*drafts, false)) || ((uintptr_t)x.lse & 3) != 0 || ((uintptr_t)mask & 3) != 0 ||
        ((uintptr_t)depth & 3) != 0)
        return WZYB_ERR_ALIGN;
    if (T_ == 0) return WZYB_OK;
    const AttnShape s = attn_shape(T_, x.q_heads, x.kv_heads, sizeof(T) == 4);
    if (s.max_splits > 1) {
        if (!x.workspace) return WZYB_ERR_NULL;
        if (!aligned16(x.workspace)) return WZYB_ERR_ALIGN;
        if (x.workspace_bytes < wzyb_kv_attn_workspace(T_, x.q_heads, x.kv_heads, x.head_dim)) return WZYB_ERR_SHAPE;
    }
    DeviceInfo di;
    const int rc = device_info(&di);
    if (rc != WZYB_OK) return rc;
    KvAttnArgs a = {};
    a.q = x.q;
    a.q_head = x.q_head_stride;
    a.q_row = x.q_row_stride;
    a.out = x.out;
    a.o_head = x.out_head_stride;
    a.o_row = x.out_row_stride;
    a.lse = x.lse;
    a.c = c;
    if (tree) a.d = *drafts;
    a.mask = mask;
    a.depth = depth;
    a.mask_words = (int)((T_ + 31) / 32);
    a.tree = tree;
    a.from_full = full;
    a.T = (int)T_;
    a.G = x.q_heads / x.kv_heads;
    a.kv_heads = x.kv_heads;
    a.d_base_pos = x.d_base_pos;
    a.pos_offset = x.pos_offset;
    a.window = x.window < (int64_t(1) << 40) ? x.window : (int64_t(1) << 40);
    a.sinks = x.sinks;
    a.scale_log2 = x.scale * kLog2e;
    a.ring_div = full ? 1 : (uint64_t)(c.ring_cap <= 2 * kKvSinkPin ? c.ring_cap : c.ring_cap - kKvSinkPin);
    a.ring_recip = ~0ull / a.ring_div;
    // the most keys that a row tile can see, known here; a split takes at least two key tiles of each warp
    int64_t keys = (x.sinks < kMaxPos ? x.sinks : kMaxPos) + (a.window < kMaxPos ? a.window : kMaxPos) + T_;
    const int64_t held = full || c.ring_cap > c.max_ctx ? c.max_ctx : c.ring_cap;
    keys = (keys < held ? keys : held) + (tree ? T_ : 0);
    const int64_t most = keys / (s.few ? 128 : 128) + 1;
    a.splits = (int)(most < s.max_splits ? most : s.max_splits);
    if (a.splits > 1) {
        const int64_t rows = T_ * x.q_heads;
        a.part_ml = static_cast<float2*>(x.workspace);
        a.part_o = reinterpret_cast<float*>(a.part_ml + (((int64_t)a.splits * rows + 1) & ~int64_t(1)));
    }
    switch (x.head_dim) {
        case 64: return launch_attn<T, 64>(a, s, stream);
        case 128: return launch_attn<T, 128>(a, s, stream);
        default: return launch_attn<T, 256>(a, s, stream);
    }
}

}  // namespace wzyb

extern "C" {

int64_t wzyb_kv_attn_workspace(int64_t T, int q_heads, int kv_heads, int head_dim) {
    if (T < 1 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0 || head_dim < 1) return 0;
    int64_t most = 0;
    for (int f32 = 0; f32 < 2; ++f32) {
        const int64_t n = wzyb::attn_shape(T, q_heads, kv_heads, f32 != 0).max_splits;
        const int64_t bytes = n > 1 ? n * T * q_heads * (head_dim * 4 + 8) + 16 : 0;
        most = bytes > most ? bytes : most;
    }
    return most;
}
int wzyb_kv_attn_f16(const wzyb_kv_attn_args* a, int64_t T, wzyb_stream_t stream) {
    return wzyb::attn_entry<__half>(a, nullptr, nullptr, nullptr, false, T, (cudaStream_t)stream);
}
int wzyb_kv_attn_f32(const wzyb_kv_attn_args* a, int64_t T, wzyb_stream_t stream) {
    return wzyb::attn_entry<float>(a, nullptr, nullptr, nullptr, false, T, (cudaStream_t)stream);
}
int wzyb_kv_tree_attn_f16(const wzyb_kv_attn_args* a, const wzyb_kv_cache* drafts, const uint32_t* mask,
                          const int32_t* depth, int64_t nodes, wzyb_stream_t stream) {
    return wzyb::attn_entry<__half>(a, drafts, mask, depth, true, nodes, (cudaStream_t)stream);
}
int wzyb_kv_tree_attn_f32(const wzyb_kv_attn_args* a, const wzyb_kv_cache* drafts, const uint32_t* mask,
                          const int32_t* depth, int64_t nodes, wzyb_stream_t stream) {
    return wzyb::attn_entry<float>(a, drafts, mask, depth, true, nodes, (cudaStream_t)stream);
}

}  // extern "C"
