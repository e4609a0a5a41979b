// kv_attn.cu -- attention over the INT8 KV cache that kv_append.cu writes: a sliding window plus a few first
// tokens that stay visible, for a chunk of new tokens (one to thousands) or for a tree of drafted tokens.
//
// Per query row (token t, query head) with its kv head's cells j:
//   x_j = scale * sum_g ks[j,g] * (q_g . kc[j,g])      g: 64-element groups, kc: int8 codes, ks: fp16 scales
//   o_g = sum_j softmax(x)_j vs[j,g] vc[j,g],          lse = ln sum_j exp(x_j)
// Codes are integers up to 127, exact in fp16, so the tensor cores multiply the codes themselves and the
// scales stay fp32: on the K side they multiply the per-group partial products, on the V side the softmax
// weights (one scaled copy of the weights per group). Products accumulate in fp32, statistics are fp32.
// The one rounding to fewer bits for fp16 calls is the scaled weight p * vs to fp16 (2^-12 of each at most, the size
// of the output's own rounding; error against 64 bits 2.9e-4 where the output's rounding alone gives 2.1e-4): a
// second part, as fp32 calls have it, would double p V and the weights' work, 1100 of a tile's 4200 cycles. fp32 calls
// split q and p * vs into two fp16 parts (22 bits).
//
// Weights entering the tensor cores are p * vs * 2^(7 - E) with a running E per row (from the largest finite
// scale among the cells that the row sees, as the running maximum of its scores), so they sit in fp16's
// upper range whatever the scales' size, and a row's result does not depend on cells it does not see. A
// row's running maximum moves only when a score passes it by 2^8: its weights stay below 2^15 either way.
// The second part of an fp32 call's weight or query element enters 2^11 times as large and its products come back by
// 2^-11, so that it is not cut off at fp16's smallest number.
#include <type_traits>

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
    int ring_step;  // ring_div, or the largest int where cells do not wrap
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

// Positions and cells are ints. No cell lies at this one or past it, so a query's own position may be cut to it, and
// sums with a tile's size stay in range.
constexpr int kMaxPos = 0x40000000;
__device__ __forceinline__ int clamp_pos(int64_t x) { return (int)(x < -1 ? -1 : (x > kMaxPos ? kMaxPos : x)); }

// A row sees positions j with j <= hi and (j < sinks or j > lo).
struct RowSpan {
    int hi, lo;
};
__device__ __forceinline__ RowSpan row_span(const KvAttnArgs& a, int64_t base, int t) {
    const int64_t p = base + (a.tree ? (int64_t)__ldg(a.depth + t) : t);
    RowSpan r;
    r.hi = clamp_pos(p);
    r.lo = clamp_pos(p - a.window);
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

// HD / 64 consecutive fp16 scales (aligned to their own size)
template <int NG>
__device__ __forceinline__ void load_scale_bits(const uint16_t* p, uint16_t (&s)[NG]) {
    if constexpr (NG == 4) {
        const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
        s[0] = (uint16_t)u.x;
        s[1] = (uint16_t)(u.x >> 16);
        s[2] = (uint16_t)u.y;
        s[3] = (uint16_t)(u.y >> 16);
    } else if constexpr (NG == 2) {
        const uint32_t u = __ldg(reinterpret_cast<const uint32_t*>(p));
        s[0] = (uint16_t)u;
        s[1] = (uint16_t)(u >> 16);
    } else {
        s[0] = __ldg(p);
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
    hi = *reinterpret_cast<const uint32_t*>(&h);
    // 2^11 (x - h), exact: the difference and both products by powers of two are
    const float2 r = ffma2(__half22float2(h), splat2(-kLoUp), fmul2(make_float2(x, y), splat2(kLoUp)));
    lo = pack_f16(r.x, r.y);
}

// Exponent e with x < 2^e <= 2x for a positive finite scale, -1000 for 0, infinities and NaN: the running
// scale exponent E is the maximum over the visible keys' scales.
__device__ __forceinline__ int scale_exp(float x) {
    const uint32_t b = __float_as_uint(x);
    const uint32_t e = b >> 23;  // scales are >= 0; a set sign bit lands outside [1, 254]
    return e >= 1 && e <= 254 ? (int)e - 126 : -1000;
}
// The exponent by which a query row is scaled down, from its largest magnitude's: rows whose scores are 0 either way, and
// infinite or NaN ones (-1000), as they are; 2^-e stays a normal number.
__device__ __forceinline__ int row_exp(int e) { return e < -100 ? 0 : (e > 126 ? 126 : e); }
__device__ __forceinline__ float exp2_int(int e) {  // 2^e, 0 below the normal range
    return e < -126 ? 0.f : __int_as_float((e + 127) << 23);
}

// Query rows of a tile to shared memory as fp16 (kSplit: two parts of x * 2^-e, e from the row's largest
// magnitude, so every fp32 row uses fp16's range; the second part 2^11 times as large, so that elements far below
// the largest, which meet groups with large scales, keep their bits). One warp per row in turn. qs[row * ld + col]; the
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
            e = row_exp(e);
            const float down = exp2_int(-e);
            f *= exp2_int(e);
#pragma unroll
            for (int i = 0; i < kE; ++i) x[i] *= down;
        }
#pragma unroll
        for (int i = 0; i < kE; ++i) {
            const __half h = __float2half_rn(x[i]);
            qs[r * ld + lane * kE + i] = h;
            if constexpr (kSplit) ql[r * ld + lane * kE + i] = __float2half_rn((x[i] - __half2float(h)) * kLoUp);
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
// Bound: the cells' bytes once (528 per key and kv head of 256) on long contexts, launch latency on short ones. 1 fp16
// token, 16/2 heads of 256: 262,144 keys in 65 us, 4.2 TB/s, held by issue slots and load latency at 8 warps per SM
// (225 registers, two tiles' codes in flight; 785 warp instructions per tile); 5120 keys in a call of 10.8 us.
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

    // K of the next tile is on its way while the current one is worked through (its registers are free once the
    // scores are there); V of the current one while its scores are computed.
    KeyTile kt = {};
    int my_cell = 0, range_end = 0, range_hi = 0, cell_limit = 0;  // the current range's end in tiles and positions
    Planes pl = {};
    uint4 kr[2][NG];
    uint16_t ksb[2][NG];
    auto load_k = [&](int it) {
        // Inside a range the next tile's cells are kWarps * kN further on (one step back where the ring wraps: a tile
        // holds no more keys than the ring). Lanes 0..15 have a key each; one past the tile's end has the first
        // one's cell (its scales count as 0 and its scores as -inf).
        const int mine = lane & 15;
        if (it < range_end && kt.count == kN && a.ring_step >= kWarps * kN) {
            kt.pos += kWarps * kN;
            kt.count = min(kN, range_hi - kt.pos);
            my_cell += kWarps * kN;
            if (my_cell >= cell_limit) my_cell -= a.ring_step;
            if (kt.count < kN) my_cell = __shfl_sync(0xffffffffu, my_cell, mine < kt.count ? mine : 0);
        } else {
            int r = 0;
#pragma unroll
            for (int n = 1; n < kAttnMaxRanges; ++n)
                if (n < plan.ranges && it >= plan.first[n]) r = n;
            kt = key_tile<kN>(plan, it);
            range_end = plan.first[r + 1];
            range_hi = plan.hi[r];
            pl = planes_of<HD>(a, kt.draft, head);
            cell_limit = kt.draft || a.from_full ? 0x7FFFFFFF : (int)a.c.ring_cap;
            my_cell = (int)cell_of(a, kt.draft, kt.pos + (mine < kt.count ? mine : 0));
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int cell = __shfl_sync(0xffffffffu, my_cell, g + 8 * i);
#pragma unroll
            for (int n = 0; n < NG; ++n)
                kr[i][n] = __ldg(reinterpret_cast<const uint4*>(pl.kq + (int64_t)cell * kvd + n * 64 + t4 * 16));
            load_scale_bits<NG>(pl.ks + (int64_t)cell * spc, ksb[i]);
        }
        // the tile's V rows, which are loaded a turn later, to L2 (a 128-byte line per lane)
        if (HD > 128 || lane < 16) prefetch_l2(pl.vq + (int64_t)my_cell * kvd + (lane >> 4) * 128);
    };
    if (tb + warp < te) load_k(tb + warp);
    for (int it = tb + warp; it < te; it += kWarps) {
        const KeyTile now = kt;
        uint2 vr[4][NG];
        uint16_t vsb[2][NG];
        float ks[2][NG], vs[2][NG];
        {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int cell = __shfl_sync(0xffffffffu, my_cell, 2 * t4 + (i & 1) + (i >> 1) * 8);
#pragma unroll
                for (int n = 0; n < NG; ++n)
                    vr[i][n] = __ldg(reinterpret_cast<const uint2*>(pl.vq + (int64_t)cell * kvd + n * 64 + g * 8));
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
                load_scale_bits<NG>(pl.vs + (int64_t)__shfl_sync(0xffffffffu, my_cell, g + 8 * i) * spc, vsb[i]);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < NG; ++n) ks[i][n] = __half2float(__ushort_as_half(ksb[i][n]));

        // scores of keys g and g + 8 for rows 2*t4, 2*t4 + 1: s[0], s[1] and s[2], s[3]
        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int n = 0; n < NG; ++n) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
            [[maybe_unused]] float low[4] = {0.f, 0.f, 0.f, 0.f};
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
                if constexpr (kSplit) mma_f16(low, fa, qc[2 * j], qc[2 * j + 1]);
            }
            if constexpr (kSplit) {
#pragma unroll
                for (int c = 0; c < 4; ++c) acc[c] = fmaf(low[c], 1.f / kLoUp, acc[c]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) s[c] = fmaf(acc[c], ks[c >> 1][n], s[c]);
        }
        if (it + kWarps < te) load_k(it + kWarps);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int n = 0; n < NG; ++n) vs[i][n] = __half2float(__ushort_as_half(vsb[i][n]));
#pragma unroll
        for (int c = 0; c < 4; ++c) s[c] *= rs[c & 1];
        int ek[2], e[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            uint32_t top_bits = 0;  // finite fp16 scales order like their bits
#pragma unroll
            for (int n = 0; n < NG; ++n) top_bits = max(top_bits, (uint32_t)vsb[i][n]);
            ek[i] = scale_exp(__half2float(__ushort_as_half((uint16_t)top_bits)));
            if (top_bits >= 0x7C00u) {  // an infinity or NaN among them
                ek[i] = -1000;
#pragma unroll
                for (int n = 0; n < NG; ++n) ek[i] = max(ek[i], scale_exp(vs[i][n]));
            }
        }
        if (tile_unmasked<kN>(plan, now)) {  // warp-uniform
            e[0] = e[1] = max(ek[0], ek[1]);
        } else {
            e[0] = e[1] = -1000;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int key = g + (c >> 1) * 8, pos = now.pos + key;
                bool see = key < now.count;
                if (now.draft) {
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
// Many query rows per kv head (prefill, verify windows, trees): a CTA takes 128 rows and walks its share of
// 64-key tiles on the 5th-generation tensor cores. Tensor memory (512 columns, one row per lane): columns
// 0..255 hold a tile's scores, 64 per 64-element group (the groups' scales differ per key, so each group's
// products have their own accumulator), and then, in the same columns, the weights: per group the fp16 copy of
// p * vs (and for fp32 calls its second part); columns 256..511 hold the tile's p V.
//   softmax warps (8 or 16): a row is 2 or 4 lanes, each with a share of the tile's keys:
//               scores from tensor memory, running maximum, exponentials, weights back to tensor memory
//   cell warps (4): the tile's codes from global memory (K a tile ahead, V a product ahead, in registers), widened to fp16 into
//               128-byte rows of shared memory with the 128-byte swizzle. Keys and values have the same layout:
//               K is read with the dimension contracted (K-major), V with the keys contracted (MN-major)
//   one warp    issues the MMAs: S_g = Q_g K_g^T, then o_g = P_g V_g with P_g from tensor memory
// o is summed in tensor memory (and scaled there when a row's maximum moves), or with kReg every tile's p V is
// taken from there onto fp32 registers (up to 128 a lane, so with 8 softmax warps). The tensor cores cut their sums off
// towards zero, up to 2^-23 per 16 keys (measured: 1.7e-3 of a value-biased o over 262,144 keys, 2e-4 over 32,768;
// in registers 2e-4, the output's rounding, at any length). So fp32 calls, and fp16 calls in which a CTA may walk more
// than kAttnDriftKeys, sum in registers; shorter fp16 calls in tensor memory, which is faster.
// 64 keys per tile: the four groups' scores and the tile's p V then fill tensor memory, so a tile's products and its
// softmax take turns, and that sum bounds the kernel. Measured with 16/2 heads of 256: 4096 fp16 tokens with a window
// of 8192 in 1440 us, a tile 4200 cycles (scores 1000, softmax and weights 2700, p V 500); 64 fp32 nodes of 24/2 heads
// over 131,072 cells in 738 us, a tile 5900 cycles (scores 2000, softmax with split weights 3500), kReg.
// Every wait is bounded. A role whose wait gives up ends its loop; the others, which wait for it, run out beside it.
// ----------------------------------------------------------------------------------------------------
// Issued by one elected lane of a converged warp: the warp-uniform operands stay in uniform registers (inside an
// `if (lane == 0)` each MMA cost about 130 cycles of moving them there, 4 times its own time).
__device__ __forceinline__ void tc_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add)
        : "memory");
}
// d = a * b + d * 2^-11
__device__ __forceinline__ void tc_mma_ss_down11(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, 1, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%4, %4, %4, %4}, p, 11;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(0)
        : "memory");
}
__device__ __forceinline__ void tc_mma_ts_down11(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, 1, 0;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%4, %4, %4, %4}, p, 11;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(0)
        : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile(
        "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar))
        : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 16 columns of this warp's 32 lanes
__device__ __forceinline__ void tc_ld16(float* r, uint32_t at) {
    uint32_t* u = reinterpret_cast<uint32_t*>(r);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
          "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(at));
}
__device__ __forceinline__ void tc_st(uint32_t at, const uint32_t (&u)[4]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3])
                 : "memory");
}
__device__ __forceinline__ void tc_st(uint32_t at, const uint32_t (&u)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(at), "r"(u[0]), "r"(u[1]),
                 "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7])
                 : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t at, const float (&r)[16]) {
    const uint32_t* u = reinterpret_cast<const uint32_t*>(r);
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at),
        "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]),
        "r"(u[10]), "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15])
        : "memory");
}
// Operand descriptor of rows of 128 bytes with the 128-byte swizzle, 8-row blocks 1024 bytes apart (both as the
// rows of a K-major operand and as the contracted index of an MN-major one of 64 columns).
__device__ __forceinline__ uint64_t tc_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr & 0x3FFFF) >> 4) | (uint64_t)(1024 >> 4) << 16 | (uint64_t)(1024 >> 4) << 32 |
           (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// fp16 x fp16 -> fp32, M = 128, N = 64
constexpr uint32_t kTcIdesc = (1u << 4) | ((64u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kTcIdescBMn = kTcIdesc | (1u << 16);  // B is MN-major

// by a whole warp, which goes on together
__device__ __forceinline__ bool tc_wait_warp(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, mbar_wait_asleep(bar, parity));
}

// the n lowest bits (none for n <= 0, all for n >= 32)
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u); }

// One arrival per warp, after all its lanes' work (32 arrivals on one word are taken one after the other).
__device__ __forceinline__ void warp_arrive(uint64_t* bar, int lane) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

constexpr int kTileMasked = 1, kTileDraft = 2, kTileBad = 4;  // bad: a value scale is infinite or NaN

template <typename T, int HD, bool kReg>
struct TcSmem {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kRows = 128, kN = 64, NG = HD / 64;
    static constexpr int kSW = kReg ? 8 : 16, kParts = kSW / 4;  // softmax warps; lanes per row
    static constexpr int kThreads = (kSW + 8) * 32;
    static constexpr int kPairs = (NG + 1) / 2;  // groups are handed on two at a time
    // [group][row][64 dims], 128-byte rows, swizzled
    __half q[kSplit ? 2 : 1][NG][kRows * 64];
    __half k[NG][kN * 64];
    __half v[NG][kN * 64];
    float ks[2][NG][kN], vs[2][NG][kN];
    float row_up[kSplit ? kRows : 4];
    float x_max[2][kParts][kRows];  // [tile parity][part][row]
    int x_exp[2][kParts][kRows];
    int e_key[2][kN], e_max[2][2];
    int4 tile[2];  // position, keys, kTile* flags
    int bad[2][2];
    // one warp's 32 rows of kOutCols columns on their way out; for HD = 256 they take the operands' place
    static constexpr int kOutCols = HD / kParts < 32 ? HD / kParts : 32, kOutLd = kOutCols + 4, kOutWarp = 32 * kOutLd;
    float out[HD == 256 ? 4 : kSW * kOutWarp];
    uint64_t k_full, v_full, s_full[kPairs], p_full[kPairs], x_full[4], o_full, done;
    KeyPlan plan;
    uint32_t tmem;
};

// Element offset of query row `row` of a kv head, -1 past the last one.
__device__ __forceinline__ int64_t q_offset(const KvAttnArgs& a, int head, int row, int rows) {
    if (row >= rows) return -1;
    const int t = row / a.G;
    return t * a.q_row + (int64_t)(head * a.G + (row - t * a.G)) * a.q_head;
}

template <typename T, int HD, bool kReg>
__global__ void __launch_bounds__(TcSmem<T, HD, kReg>::kThreads, 1) kv_attn_tile_kernel(const KvAttnArgs a) {
    pdl_begin();
    using S = TcSmem<T, HD, kReg>;
    constexpr bool kSplit = S::kSplit;
    static_assert(kReg || !kSplit, "fp32 sums stay in registers");
    constexpr int NG = S::NG, kN = S::kN, kSW = S::kSW, kParts = S::kParts, kPairs = S::kPairs, kKeys = kN / kParts, kDims = HD / kParts;
    extern __shared__ __align__(1024) uint8_t attn_smem[];
    S& sm = *reinterpret_cast<S*>(attn_smem);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int split = blockIdx.y, row0 = (gridDim.x - 1 - blockIdx.x) * S::kRows, head = blockIdx.z;
    const int rows = a.T * a.G;
    const int64_t base = (a.d_base_pos ? (int64_t)__ldg(a.d_base_pos) : 0) + a.pos_offset;

    if (warp == kSW + 4) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sm.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    } else if (warp == kSW + 5) {
        build_plan<kN>(a, sm.plan, base, row0 / a.G, (min(row0 + S::kRows, rows) - 1) / a.G + 1, lane);
    } else if (warp == kSW + 6 && lane == 0) {
        mbar_init(&sm.k_full, 4);
        mbar_init(&sm.v_full, 4);
        for (int i = 0; i < kPairs; ++i) {
            mbar_init(&sm.s_full[i], i == 0 ? 2 : 1);  // the first also hands the cell warps' scales on
            mbar_init(&sm.p_full[i], kSW);
        }
        for (int i = 0; i < 4; ++i) mbar_init(&sm.x_full[i], kParts);
        mbar_init(&sm.o_full, 1);
        mbar_init(&sm.done, 1);
        fence_mbar_init();
    }
    if (warp < kSW) {
        // Query rows to shared memory, a lane 8 elements, several rows of a warp in flight. fp32
        // rows enter as two fp16 parts of x * 2^-e, e from the row's largest magnitude, so they use fp16's range; the
        // second part 2^11 times as large.
        constexpr int kL = HD / 8, kPer = 32 / kL, kRowsQ = S::kRows / kSW, kMineQ = kRowsQ / kPer;  // lanes per row, rows
        constexpr int kMostQ = kSplit ? 4 : 8, kBatch = kMineQ < kMostQ ? kMineQ : kMostQ;          // at a time, ...
        const int col = (lane % kL) * 8, g = col / 64, c16 = (col % 64) / 8;
        // lane i finds the warp's row i (one division per warp: straight code that runs once costs its fetch)
        const int64_t mine_at = q_offset(a, head, row0 + warp * kRowsQ + lane % kRowsQ, rows);
#pragma unroll 1
        for (int r0 = warp * kRowsQ; r0 < (warp + 1) * kRowsQ; r0 += kPer * kBatch) {
            uint4 raw[kBatch][sizeof(T) / 2];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int64_t at = __shfl_sync(0xffffffffu, mine_at, r0 - warp * kRowsQ + b * kPer + lane / kL);
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                    raw[b][i] = at < 0 ? make_uint4(0, 0, 0, 0)
                                       : __ldg(reinterpret_cast<const uint4*>(static_cast<const T*>(a.q) + at + col) + i);
            }
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                const int r = r0 + b * kPer + lane / kL;
                const int at = r * 128 + ((c16 ^ (r & 7)) << 4);
                if constexpr (!kSplit) {
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(sm.q[0][g]) + at) = raw[b][0];
                } else {
                    float x[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = reinterpret_cast<const float*>(&raw[b][0])[i];
                    float am = 0.f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) am = fmaxf(am, fabsf(x[i]));
#pragma unroll
                    for (int o = kL / 2; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
                    int e = scale_exp(am);
                    e = row_exp(e);
                    const float down = exp2_int(-e);
                    uint32_t h[4], l[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) split_f16(x[2 * i] * down, x[2 * i + 1] * down, h[i], l[i]);
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(sm.q[0][g]) + at) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4*>(reinterpret_cast<uint8_t*>(sm.q[kSplit][g]) + at) = make_uint4(l[0], l[1], l[2], l[3]);
                    if (col == 0) sm.row_up[r] = exp2_int(e);
                }
            }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const KeyPlan& plan = sm.plan;
    const int ntiles = plan.first[plan.ranges];
    const int tb = (int)((int64_t)ntiles * split / a.splits), te = (int)((int64_t)ntiles * (split + 1) / a.splits);
    // all 512 columns were asked for, so they start at 0; the constant keeps the MMAs' operands immediate
    constexpr uint32_t tmem = 0;

    // registers: launched with 128 (512 threads) or 80 (768 threads) each; 256 x 208 + 128 x 64 + 128 x 32
    // and 512 x 96 + 128 x 64 + 128 x 32 are the same totals
    if (warp < kSW) {
        if constexpr (kReg)
            asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        else
            asm volatile("setmaxnreg.inc.sync.aligned.u32 96;");
        const int part = warp >> 2, r = (warp & 3) * 32 + lane, row = row0 + r, key0 = part * kKeys;
        const uint32_t mine = tmem + ((uint32_t)(warp & 3) << 21);  // this warp's 32 lanes
        const uint32_t o_at = mine + 256 + part * kDims;
        const int t = min(row, rows - 1) / a.G;
        const RowSpan span = row_span(a, base, t);
        const float up = kSplit ? sm.row_up[r] : 1.f;
        float o[kReg ? kDims : 1];
        if constexpr (kReg) {
#pragma unroll
            for (int i = 0; i < kDims; ++i) o[i] = 0.f;
        }
        float m = -INFINITY, l = 0.f, alpha = 1.f;
        int E = -1000;
        auto unit = [](int e) { return e <= -1000 ? 7 : e; };  // while only scales of 0 have been seen
        bool ok = true;
        // sums in registers: the previous tile's p V onto o
        auto drain = [&](uint32_t parity) {
            ok = tc_wait_warp(&sm.o_full, parity);
            if (!ok) return;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < kDims; c += 32) {
                float x[32];
                tc_ld16(x, o_at + c);
                tc_ld16(x + 16, o_at + c + 16);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 32; i += 2) {
                    const float2 y = ffma2(make_float2(o[c + i], o[c + i + 1]), splat2(alpha), make_float2(x[i], x[i + 1]));
                    o[c + i] = y.x;
                    o[c + i + 1] = y.y;
                }
            }
        };
        for (int it = tb; it < te; ++it) {
            const int n = it - tb, b = n & 1;
            if constexpr (kReg) {
                if (n > 0) {
                    drain(b ^ 1);
                    if (!ok) break;
                }
            }
            float s[kKeys];
#pragma unroll
            for (int i = 0; i < kKeys; ++i) s[i] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                if (g % 2 == 0) {
                    ok = ok && tc_wait_warp(&sm.s_full[g / 2], b);
                    if (!ok) break;
                    tc_fence_after();
                }
#pragma unroll
                for (int c = 0; c < kKeys; c += 16) {
                    float x[16];
                    tc_ld16(x, mine + g * 64 + key0 + c);
                    tc_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&sm.ks[b][g][key0 + c + i]);
                        const float2 y0 = ffma2(make_float2(x[i], x[i + 1]), make_float2(f.x, f.y), make_float2(s[c + i], s[c + i + 1]));
                        const float2 y1 = ffma2(make_float2(x[i + 2], x[i + 3]), make_float2(f.z, f.w), make_float2(s[c + i + 2], s[c + i + 3]));
                        s[c + i] = y0.x;
                        s[c + i + 1] = y0.y;
                        s[c + i + 2] = y1.x;
                        s[c + i + 3] = y1.y;
                    }
                }
            }
            if (!ok) break;
            float top = -INFINITY;
            const int4 tile = sm.tile[b];
            int e = max(sm.e_max[b][0], sm.e_max[b][1]);
            if (tile.z & kTileMasked) {  // CTA-uniform
                uint32_t see = 0;
                if (tile.z & kTileDraft) {
                    const int wd = (tile.x + key0) >> 5;
                    see = wd < a.mask_words ? __ldg(a.mask + (int64_t)t * a.mask_words + wd) >> (key0 & 31) : 0u;
                    see &= low_bits(tile.y - key0);
                } else {
                    const int p0 = tile.x + key0;
                    see = (low_bits(span.hi + 1 - p0) & ~low_bits(span.lo + 1 - p0)) | low_bits(min(plan.sinks, span.hi + 1) - p0);
                    see &= low_bits(tile.y - key0);
                }
                e = -1000;
#pragma unroll
                for (int i = 0; i < kKeys; ++i) {
                    if (see >> i & 1u)
                        e = max(e, sm.e_key[b][key0 + i]);
                    else
                        s[i] = -INFINITY;
                }
                sm.x_exp[b][part][r] = e;
            }
#pragma unroll
            for (int i = 0; i < kKeys; ++i) top = fmaxf(top, s[i]);
            sm.x_max[b][part][r] = top * up;
            // the warps of these 32 rows; also: their scores have been read, so weights may take their columns (a
            // warp's weights lie where another one's scores were, so the fences order the two warps' accesses)
            tc_fence_before();
            warp_arrive(&sm.x_full[warp & 3], lane);
            ok = tc_wait_warp(&sm.x_full[warp & 3], b);
            if (!ok) break;
            tc_fence_after();
            top = sm.x_max[b][0][r];
#pragma unroll
            for (int i = 1; i < kParts; ++i) top = fmaxf(top, sm.x_max[b][i][r]);
            if (tile.z & kTileMasked) {
#pragma unroll
                for (int i = 0; i < kParts; ++i) e = max(e, sm.x_exp[b][i][r]);
            }
            alpha = 1.f;
            if (top > m + 8.f || e > E) {
                top = fmaxf(top, m);
                e = max(e, E);
                alpha = ex2_approx(m - (top == -INFINITY ? 0.f : top)) * exp2_int(unit(E) - unit(e));
                l *= alpha;
                m = top;
                E = e;
            }
            if constexpr (!kReg) {
                if (n > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    ok = tc_wait_warp(&sm.o_full, b ^ 1);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < kDims; c += 16) {
                        float x[16];
                        tc_ld16(x, o_at + c);
                        tc_wait_ld();
#pragma unroll
                        for (int i = 0; i < 16; ++i) x[i] *= alpha;
                        tc_st16(o_at + c, x);
                    }
                }
            }
            // p * 2^(7 - E), so that p * vs has the weights' size; l sums these
            const float shift = (m == -INFINITY ? 0.f : m) - (float)(7 - unit(E));
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int i = 0; i < kKeys; i += 2) {
                float2 y = make_float2(s[i], s[i + 1]);
                y = kSplit ? ffma2(y, splat2(up), splat2(-shift)) : fadd2(y, splat2(-shift));
                s[i] = ex2_approx(y.x);
                s[i + 1] = ex2_approx(y.y);
                sum = fadd2(sum, make_float2(s[i], s[i + 1]));
            }
            l += sum.x + sum.y;
            // A weight of 0 (a place that the row does not see) stays 0 whatever the cell's scale is: that takes
            // a comparison per weight, which only tiles with an infinite or NaN scale pay for.
            auto weights = [&](int g, auto bad) {
                constexpr int kPiece = kSplit ? 8 : 16;
#pragma unroll
                for (int c = 0; c < kKeys; c += kPiece) {
                    uint32_t hi[kPiece / 2];
                    [[maybe_unused]] uint32_t lo[kPiece / 2];
#pragma unroll
                    for (int i = 0; i < kPiece; i += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(&sm.vs[b][g][key0 + c + i]);
                        float2 w0 = fmul2(make_float2(s[c + i], s[c + i + 1]), make_float2(f.x, f.y));
                        float2 w1 = fmul2(make_float2(s[c + i + 2], s[c + i + 3]), make_float2(f.z, f.w));
                        if constexpr (decltype(bad)::value) {
                            w0 = make_float2(s[c + i] == 0.f ? 0.f : w0.x, s[c + i + 1] == 0.f ? 0.f : w0.y);
                            w1 = make_float2(s[c + i + 2] == 0.f ? 0.f : w1.x, s[c + i + 3] == 0.f ? 0.f : w1.y);
                        }
                        if constexpr (kSplit) {
                            split_f16(w0.x, w0.y, hi[i / 2], lo[i / 2]);
                            split_f16(w1.x, w1.y, hi[i / 2 + 1], lo[i / 2 + 1]);
                        } else {
                            hi[i / 2] = pack_f16(w0.x, w0.y);
                            hi[i / 2 + 1] = pack_f16(w1.x, w1.y);
                        }
                    }
                    tc_st(mine + g * 64 + (key0 + c) / 2, hi);
                    if constexpr (kSplit) tc_st(mine + g * 64 + 32 + (key0 + c) / 2, lo);
                }
                if (g % 2 == 1 || g == NG - 1) {
                    tc_wait_st();
                    tc_fence_before();
                    warp_arrive(&sm.p_full[g / 2], lane);
                }
            };
            if (sm.bad[b][0] | sm.bad[b][1]) {
#pragma unroll 1
                for (int g = 0; g < NG; ++g) weights(g, std::true_type{});
            } else {
#pragma unroll
                for (int g = 0; g < NG; ++g) weights(g, std::false_type{});
            }
        }
        if (te > tb && ok) {
            if constexpr (kReg) {
                drain((te - tb - 1) & 1);
            } else {
                ok = tc_wait_warp(&sm.o_full, (te - tb - 1) & 1);
                tc_fence_after();
            }
        }
        // the row's sum over its lanes, then its o
        sm.x_max[0][part][r] = l;
        warp_arrive(&sm.x_full[warp & 3], lane);
        ok = ok && tc_wait_warp(&sm.x_full[warp & 3], (te - tb) & 1);
        if (ok) {
            l = sm.x_max[0][0][r];
#pragma unroll
            for (int i = 1; i < kParts; ++i) l += sm.x_max[0][i][r];
            const int gq = row - t * a.G, hq = head * a.G + gq;
            const int64_t orow = (int64_t)t * a.G * a.kv_heads + hq, at = (int64_t)split * rows * a.kv_heads + orow;
            const float back = exp2_int(unit(E) - 7);  // of l and of o
            const float norm = a.splits > 1 ? back : (l == 0.f ? 0.f : 1.f / l);
            if (row < rows && part == 0) {
                if (a.splits > 1)
                    a.part_ml[at] = make_float2(m, l * back);
                else if (a.lse != nullptr)
                    a.lse[orow] = l == 0.f ? -INFINITY : (m + (float)(unit(E) - 7) + log2f(l)) * 0.6931471805599453f;
            }
            // Through shared memory, so that a row's columns leave as whole 128-byte lines (a lane's own row, 16
            // bytes at a time, took 5 us for 128 rows of 256).
            constexpr int kCols = S::kOutCols, kLd = S::kOutLd, kQuads = kCols / 4, kRowsAt = 32 / kQuads;
            static_assert(HD < 256 || kSW * S::kOutWarp * 4 <= (int)(sizeof(sm.q) + sizeof(sm.k) + sizeof(sm.v)), "the operands' place");
            float* const slab = (HD == 256 ? reinterpret_cast<float*>(&sm.q) : sm.out) + warp * S::kOutWarp;
            // element offset of this lane's row in the output or the parts, -1 past the last row
            const int64_t my_at = row >= rows ? -1 : (a.splits > 1 ? at * HD : t * a.o_row + hq * a.o_head) + part * kDims;
#pragma unroll
            for (int c = 0; c < kDims; c += kCols) {
#pragma unroll
                for (int i = 0; i < kCols; i += 16) {
                    float x[16];
                    if constexpr (kReg) {
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = o[c + i + j] * norm;
                    } else {
#pragma unroll
                        for (int j = 0; j < 16; ++j) x[j] = 0.f;
                        if (te > tb) {
                            tc_ld16(x, o_at + c + i);
                            tc_wait_ld();
#pragma unroll
                            for (int j = 0; j < 16; ++j) x[j] = l == 0.f ? 0.f : x[j] * norm;
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 16; j += 4)
                        *reinterpret_cast<float4*>(slab + lane * kLd + i + j) = make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
                }
                __syncwarp();
                const int cq = (lane % kQuads) * 4;
#pragma unroll 1
                for (int i = lane / kQuads; i < 32; i += kRowsAt) {
                    const float4 y = *reinterpret_cast<const float4*>(slab + i * kLd + cq);
                    const int64_t to = __shfl_sync(0xffffffffu, my_at, i) + c + cq;
                    if (to < c + cq) continue;
                    if (a.splits > 1) {
                        *reinterpret_cast<float4*>(a.part_o + to) = y;
                    } else {
                        store_out2(static_cast<T*>(a.out) + to, y.x, y.y);
                        store_out2(static_cast<T*>(a.out) + to + 2, y.z, y.w);
                    }
                }
                __syncwarp();
            }
        }
    } else if (warp < kSW + 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
        const int u = tid - kSW * 32;
        constexpr int kCh = HD / 16, kMine = kN * kCh / 128, kStep = 128 / kCh;  // 16-byte pieces of a row; rows per thread
        // lanes of odd groups take the neighbouring key, whose swizzle differs in the lowest bit: 8 lanes that store
        // together use 8 different banks
        const int c = u % kCh, first = (u / kCh) ^ (c / 4 & 1);
        const int kvd = a.kv_heads * HD, spc = a.kv_heads * NG;
        uint4 raw[kMine];  // one tile's K or V pieces: 64 for both would not fit beside the rest
        uint16_t sc[NG];  // K scales of key u (u < 64) or V scales of key u - 64, converted when they are used
        // the tile being loaded: its cells are consecutive, but for one step back by `div` where the ring wraps (a
        // tile holds no more keys than the ring)
        KeyTile kt;
        int cell0 = 0;
        const int div = (int)a.ring_div;
        auto find = [&](int it) {
            kt = key_tile<kN>(plan, it);
            cell0 = (int)cell_of(a, kt.draft, kt.pos);
        };
        auto cell = [&](int key) {
            const int x = cell0 + key;
            return !kt.draft && !a.from_full && x >= (int)a.c.ring_cap ? x - div : x;
        };
        // the tile's 16-byte pieces into registers; keys past its end get zero codes (and zero scales)
        auto load = [&](bool value) {
            const int8_t* const src = (kt.draft ? (value ? a.d.ring_v_q : a.d.ring_k_q)
                                                : (a.from_full ? (value ? a.c.full_v_q : a.c.full_k_q) : (value ? a.c.ring_v_q : a.c.ring_k_q))) +
                                      head * HD + c * 16;
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int key = first + i * kStep;
                raw[i] = key < kt.count ? __ldg(reinterpret_cast<const uint4*>(src + (int64_t)cell(key) * kvd)) : make_uint4(0, 0, 0, 0);
            }
        };
        auto load_sc = [&]() {
            const int key = u & 63;
            const bool value = u >= 64;
            const uint16_t* const src = (kt.draft ? (value ? a.d.ring_v_s : a.d.ring_k_s)
                                                  : (a.from_full ? (value ? a.c.full_v_s : a.c.full_k_s) : (value ? a.c.ring_v_s : a.c.ring_k_s))) +
                                        head * NG;
#pragma unroll
            for (int g = 0; g < NG; ++g) sc[g] = 0;
            if (key < kt.count) load_scale_bits<NG>(src + (int64_t)cell(key) * spc, sc);
        };
        auto widen = [&](__half (&dst)[NG][kN * 64]) {
            uint8_t* const d = reinterpret_cast<uint8_t*>(dst[c / 4]);
#pragma unroll
            for (int i = 0; i < kMine; ++i) {
                const int key = first + i * kStep, c16 = (c % 4) * 2;
                const uint32_t w[4] = {raw[i].x ^ 0x80808080u, raw[i].y ^ 0x80808080u, raw[i].z ^ 0x80808080u, raw[i].w ^ 0x80808080u};
                *reinterpret_cast<uint4*>(d + key * 128 + ((c16 ^ (key & 7)) << 4)) =
                    make_uint4(codes_f16(w[0], kSelLo), codes_f16(w[0], kSelHi), codes_f16(w[1], kSelLo), codes_f16(w[1], kSelHi));
                *reinterpret_cast<uint4*>(d + key * 128 + (((c16 + 1) ^ (key & 7)) << 4)) =
                    make_uint4(codes_f16(w[2], kSelLo), codes_f16(w[2], kSelHi), codes_f16(w[3], kSelLo), codes_f16(w[3], kSelHi));
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        };
        bool ok = true;
        if (tb < te) {
            find(tb);
            load_sc();
            load(false);
        }
        for (int it = tb; it < te; ++it) {
            const int n = it - tb, b = n & 1;
            if (n > 0) ok = tc_wait_warp(&sm.s_full[kPairs - 1], b ^ 1);  // K's memory is free
            if (!ok) break;
            int e = -1000;
            bool bad = false;
            const float f = u < 64 ? a.scale_log2 : 1.f;  // scores in log2 units
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float x = __half2float(__ushort_as_half(sc[g]));
                (u < 64 ? sm.ks : sm.vs)[b][g][u & 63] = x * f;
                e = max(e, scale_exp(x));
                bad = bad || !(fabsf(x) <= 65504.f);
            }
            if (u >= 64) {
                sm.e_key[b][u - 64] = e;
                e = __reduce_max_sync(0xffffffffu, e);
                if (lane == 0) sm.e_max[b][(u - 64) >> 5] = e;
                bad = __any_sync(0xffffffffu, bad);
                if (lane == 0) sm.bad[b][(u - 64) >> 5] = bad ? kTileBad : 0;
            }
            if (u == 0)
                sm.tile[b] = make_int4(kt.pos, kt.count, (tile_unmasked<kN>(plan, kt) ? 0 : kTileMasked) | (kt.draft ? kTileDraft : 0), 0);
            widen(sm.k);
            warp_arrive(&sm.k_full, lane);
            load(true);
            if (n > 0) ok = tc_wait_warp(&sm.o_full, b ^ 1);  // V's memory is free
            if (!ok) break;
            widen(sm.v);
            warp_arrive(&sm.v_full, lane);
            if (it + 1 < te) {
                find(it + 1);
                load_sc();
                load(false);
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 32;");
        if (warp == kSW + 4 && tb < te) {  // the whole warp, converged; one lane issues
            const uint64_t qd = tc_desc(smem_u32(sm.q[0][0])), ql = tc_desc(smem_u32(sm.q[kSplit ? 1 : 0][0]));
            const uint64_t kd = tc_desc(smem_u32(sm.k[0])), vd = tc_desc(smem_u32(sm.v[0]));
            constexpr uint64_t kQG = S::kRows * 128 >> 4, kKG = kN * 128 >> 4;  // a group's bytes in descriptor units
            bool ok = true;
            for (int n = 0; n < te - tb && ok; ++n) {
                const int b = n & 1;
                ok = tc_wait_warp(&sm.k_full, b);
                if (n > 0) ok = ok && tc_wait_warp(&sm.o_full, b ^ 1);  // the weights' columns are free
                if (!ok) break;
                if (lane == 0) mbar_arrive(&sm.s_full[0]);
                tc_fence_after();
#pragma unroll 1
                for (int g = 0; g < NG; ++g) {
                    if constexpr (kSplit) {  // the second parts first: they come back by 2^-11 as the first ones are added
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            tc_mma_ss(tmem + g * 64, ql + g * kQG + x * 2, kd + g * kKG + x * 2, kTcIdesc, x > 0);
                        tc_mma_ss_down11(tmem + g * 64, qd + g * kQG, kd + g * kKG, kTcIdesc);
                    } else {
                        tc_mma_ss(tmem + g * 64, qd + g * kQG, kd + g * kKG, kTcIdesc, 0);
                    }
#pragma unroll
                    for (int x = 1; x < 4; ++x)
                        tc_mma_ss(tmem + g * 64, qd + g * kQG + x * 2, kd + g * kKG + x * 2, kTcIdesc, 1);
                    if (g % 2 == 1 || g == NG - 1) tc_commit(&sm.s_full[g / 2]);
                }
                ok = tc_wait_warp(&sm.v_full, b);
#pragma unroll 1
                for (int g = 0; g < NG; ++g) {
                    if (g % 2 == 0) {
                        ok = ok && tc_wait_warp(&sm.p_full[g / 2], b);
                        if (!ok) break;
                        tc_fence_after();
                    }
                    const uint32_t d = tmem + 256 + g * 64, p = tmem + g * 64;
                    if constexpr (kSplit) {
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            tc_mma_ts(d, p + 32 + x * 8, vd + g * kKG + x * (2048 >> 4), kTcIdescBMn, x > 0);
                        tc_mma_ts_down11(d, p, vd + g * kKG, kTcIdescBMn);
                    } else {
                        tc_mma_ts(d, p, vd + g * kKG, kTcIdescBMn, !kReg && n > 0);
                    }
#pragma unroll
                    for (int x = 1; x < 4; ++x) tc_mma_ts(d, p + x * 8, vd + g * kKG + x * (2048 >> 4), kTcIdescBMn, 1);
                }
                if (!ok) break;
                tc_commit(&sm.o_full);
            }
            // nothing of this CTA's is in flight when its memory goes
            tc_commit(&sm.done);
            mbar_wait_until(&sm.done, 0, globaltimer_ns() + kWaitLimitNs);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kSW + 4) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
}

// Joins the splits' parts: the sums weighted by 2^(m - largest m), always in split order.
template <typename T, int HD, int N>
__device__ __forceinline__ void join_store(const KvAttnArgs& a, int64_t row, int col, const float (&x)[N], float norm) {
    const int qh = a.G * a.kv_heads, t = (int)(row / qh), hq = (int)(row - (int64_t)t * qh);
    T* const p = static_cast<T*>(a.out) + t * a.o_row + hq * a.o_head + col;
#pragma unroll
    for (int i = 0; i < N; i += 2) store_out2(p + i, x[i] * norm, x[i + 1] * norm);
}
__device__ __forceinline__ float join_lse(float top, float sum) {
    return sum == 0.f ? -INFINITY : (top + log2f(sum)) * 0.6931471805599453f;
}

// Both joins read the parts once, mostly from L2, and are bound by latency: one row's loads go out together.
// Few splits (at most kJoinFew): a warp per row, all its parts in flight. 8168 rows of 128 with 2 splits: 6.6 us cold
// (a CTA per row took 32).
constexpr int kJoinFew = 8;
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv_attn_join_rows_kernel(const KvAttnArgs a) {
    pdl_begin();
    constexpr int kV = HD / 32;  // consecutive elements per lane
    const int lane = threadIdx.x & 31;
    const int64_t nrows = (int64_t)a.T * a.G * a.kv_heads, row = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= nrows) return;
    float2 ml[kJoinFew];
    float y[kJoinFew][kV];
#pragma unroll
    for (int s = 0; s < kJoinFew; ++s) {
        ml[s] = make_float2(-INFINITY, 0.f);
        if (s < a.splits) {
            ml[s] = __ldg(a.part_ml + s * nrows + row);
            const float* const p = a.part_o + (s * nrows + row) * HD + lane * kV;
            if constexpr (kV == 2) {
                const float2 u = __ldg(reinterpret_cast<const float2*>(p));
                y[s][0] = u.x;
                y[s][1] = u.y;
            } else {
#pragma unroll
                for (int i = 0; i < kV; i += 4) {
                    const float4 u = __ldg(reinterpret_cast<const float4*>(p + i));
                    y[s][i] = u.x;
                    y[s][i + 1] = u.y;
                    y[s][i + 2] = u.z;
                    y[s][i + 3] = u.w;
                }
            }
        }
    }
    float top = -INFINITY, sum = 0.f, x[kV] = {};
#pragma unroll
    for (int s = 0; s < kJoinFew; ++s) top = fmaxf(top, ml[s].x);
    const float ref = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int s = 0; s < kJoinFew; ++s) {
        const float f = ex2_approx(ml[s].x - ref);
        if (s < a.splits && f != 0.f) {
            sum = fmaf(ml[s].y, f, sum);
#pragma unroll
            for (int i = 0; i < kV; ++i) x[i] = fmaf(y[s][i], f, x[i]);
        }
    }
    join_store<T, HD, kV>(a, row, lane * kV, x, sum == 0.f ? 0.f : 1.f / sum);
    if (lane == 0 && a.lse != nullptr) a.lse[row] = join_lse(top, sum);
}

// Many splits of few rows (decode): a CTA per row and 64 columns; 16 threads take each column quad, every 16th
// split each, and meet in shared memory. 16 rows of 256 with 148 splits: 8.8 us cold (a CTA per whole row 11.4).
template <typename T, int HD>
__global__ void __launch_bounds__(256) kv_attn_join_kernel(const KvAttnArgs a) {
    pdl_begin();
    constexpr int kMost = 320;  // splits, two per thread at most
    __shared__ float w[kMost], red[2][8];
    __shared__ __align__(16) float4 part[16][17];
    const int tid = threadIdx.x, lane = tid & 31, c = tid & 15, s0 = tid >> 4;
    const int64_t row = blockIdx.x, nrows = (int64_t)a.T * a.G * a.kv_heads;
    const float* const p = a.part_o + row * HD + blockIdx.y * 64 + c * 4;
    float2 ml[2];
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int s = tid + 256 * i;
        ml[i] = s < a.splits ? __ldg(a.part_ml + s * nrows + row) : make_float2(-INFINITY, 0.f);
        top = fmaxf(top, ml[i].x);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) red[0][tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, red[0][i]);
    const float ref = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float f = ex2_approx(ml[i].x - ref);
        if (tid + 256 * i < a.splits) w[tid + 256 * i] = f;
        sum = fmaf(ml[i].y, f, sum);
    }
    sum = group_sum<32>(sum);
    if (lane == 0) red[1][tid >> 5] = sum;
    __syncthreads();
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += red[1][i];
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 10
    for (int s = s0; s < a.splits; s += 16) {
        const float f = w[s];
        const float4 y = __ldg(reinterpret_cast<const float4*>(p + s * nrows * HD));
        if (f != 0.f) {
            x.x = fmaf(y.x, f, x.x);
            x.y = fmaf(y.y, f, x.y);
            x.z = fmaf(y.z, f, x.z);
            x.w = fmaf(y.w, f, x.w);
        }
    }
    part[s0][c] = x;
    __syncthreads();
    if (tid < 16) {
        float z[4] = {};
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float4 y = part[i][tid];
            z[0] += y.x;
            z[1] += y.y;
            z[2] += y.z;
            z[3] += y.w;
        }
        join_store<T, HD, 4>(a, row, blockIdx.y * 64 + tid * 4, z, sum == 0.f ? 0.f : 1.f / sum);
        if (tid == 0 && blockIdx.y == 0 && a.lse != nullptr) a.lse[row] = join_lse(top, sum);
    }
}

// Which kernel a call takes and how far its keys may be split, from the sizes alone (how many keys there are is only
// known on the device; `keys` is the most there can be). us per call, few-row kernel / tile kernel:
//   rows per kv head    24          32          48         64          96
//   2x256 fp16   2K     10 / 15     10 / 15     12 / 16    12 / 16     15 / 23 (fp32)
//               28K     24 / 29     28 / 29     39 / 29    48 / 30     84 / 43 (fp32)
//              131K     83 / 106   105 / 106   152 / 108  198 / 108   359 / 152 (fp32)
//   2x128 fp16 131K     62 / 65     79 / 68;   8x128 fp16 28K  46 / 59,  75 / 59
// so few rows are up to 32 of head_dim 256 and up to 24 of the others, and up to 96 where no more than 6144 keys
// can be seen (the lines through these figures cross at 6200 to 8800).
constexpr int kAttnSms = 148;  // two CTAs per SM for few rows, one for many
constexpr int64_t kAttnFewKeys = 6144, kAttnFewKeysRows = 96;
struct AttnShape {
    bool few;
    int tile_rows, row_tiles, max_splits;
};
static AttnShape attn_shape(int64_t T, int q_heads, int kv_heads, int head_dim, int64_t keys) {
    AttnShape s;
    const int64_t rows = T * (q_heads / kv_heads);
    s.few = rows <= (head_dim == 256 ? 32 : 24) || (rows <= kAttnFewKeysRows && keys <= kAttnFewKeys);
    s.tile_rows = s.few ? 8 : 128;
    s.row_tiles = (int)((rows + s.tile_rows - 1) / s.tile_rows);
    const int64_t ctas = (int64_t)s.row_tiles * kv_heads, most = s.few ? 2 * kAttnSms : kAttnSms;
    s.max_splits = (int)(ctas >= most ? 1 : most / ctas);
    return s;
}

// Keys that one CTA may add up in tensor memory: a drift of 2^-23 * 16384 / 16, half an fp16 rounding.
constexpr int64_t kAttnDriftKeys = 16384;
template <typename T, int HD, bool kReg>
static int launch_tiles(const KvAttnArgs& a, dim3 grid, cudaStream_t stream) {
    using S = TcSmem<T, HD, kReg>;
    const auto kern = kv_attn_tile_kernel<T, HD, kReg>;
    const int rc = ensure_smem((const void*)kern, (int)sizeof(S));
    if (rc == WZYB_OK) launch_k(kern, grid, S::kThreads, sizeof(S), stream, a);
    return rc;
}
template <typename T, int HD>
static int launch_attn(KvAttnArgs& a, const AttnShape& s, int64_t keys, cudaStream_t stream) {
    int rc = WZYB_OK;
    if (s.few) {
        launch_k(kv_attn_few_kernel<T, HD>, dim3(a.splits, s.row_tiles, a.kv_heads), 128, 0, stream, a);
    } else {
        const dim3 grid(s.row_tiles, a.splits, a.kv_heads);
        if (sizeof(T) == 2 && keys / a.splits <= kAttnDriftKeys) {
            if constexpr (sizeof(T) == 2) rc = launch_tiles<T, HD, false>(a, grid, stream);
        } else {
            rc = launch_tiles<T, HD, true>(a, grid, stream);
        }
        if (rc != WZYB_OK) return rc;
    }
    const int out_rows = a.T * a.G * a.kv_heads;
    if (a.splits > kJoinFew)
        launch_k(kv_attn_join_kernel<T, HD>, dim3(out_rows, HD / 64), 256, 0, stream, a);
    else if (a.splits > 1)
        launch_k(kv_attn_join_rows_kernel<T, HD>, (out_rows + 7) / 8, 256, 0, stream, a);
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
    if (T_ != 0 && (!x.q || !x.out)) return WZYB_ERR_NULL;
    if (full ? !(c.full_k_q && c.full_k_s && c.full_v_q && c.full_v_s)
             : !(c.ring_k_q && c.ring_k_s && c.ring_v_q && c.ring_v_s))
        return WZYB_ERR_NULL;
    if (tree && (!drafts || (T_ != 0 && (!mask || !depth || !drafts->ring_k_q || !drafts->ring_k_s || !drafts->ring_v_q ||
                                         !drafts->ring_v_s))))
        return WZYB_ERR_NULL;
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
        ((uintptr_t)depth & 3) != 0 || ((uintptr_t)x.d_base_pos & 3) != 0)
        return WZYB_ERR_ALIGN;
    if (T_ == 0) return WZYB_OK;
    // the most keys that a row tile can see, as far as the host knows
    const int64_t window = x.window < kMaxPos ? x.window : kMaxPos, sinks = x.sinks < kMaxPos ? x.sinks : kMaxPos;
    const int64_t held = full || c.ring_cap > c.max_ctx ? c.max_ctx : c.ring_cap, span = sinks + window + T_;
    const int64_t keys = (span < held ? span : held) + (tree ? T_ : 0);
    const AttnShape s = attn_shape(T_, x.q_heads, x.kv_heads, x.head_dim, keys);
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
    a.window = x.window < (int64_t(1) << 62) ? x.window : (int64_t(1) << 62);  // p - window stays in range
    a.sinks = x.sinks;
    a.scale_log2 = x.scale * kLog2e;
    a.ring_div = full ? 1 : (uint64_t)(c.ring_cap <= 2 * kKvSinkPin ? c.ring_cap : c.ring_cap - kKvSinkPin);
    a.ring_recip = ~0ull / a.ring_div;
    a.ring_step = full ? 0x7FFFFFFF : (int)a.ring_div;
    // a split takes two key tiles of each warp (few rows) or of the CTA at least
    const int64_t most = keys / 128 + 1;
    a.splits = (int)(most < s.max_splits ? most : s.max_splits);
    if (a.splits > 1) {
        const int64_t rows = T_ * x.q_heads;
        a.part_ml = static_cast<float2*>(x.workspace);
        a.part_o = reinterpret_cast<float*>(a.part_ml + (((int64_t)a.splits * rows + 1) & ~int64_t(1)));
    }
    switch (x.head_dim) {
        case 64: return launch_attn<T, 64>(a, s, keys, stream);
        case 128: return launch_attn<T, 128>(a, s, keys, stream);
        default: return launch_attn<T, 256>(a, s, keys, stream);
    }
}

}  // namespace wzyb

extern "C" {

int64_t wzyb_kv_attn_workspace(int64_t T, int q_heads, int kv_heads, int head_dim) {
    if (T < 1 || kv_heads < 1 || q_heads < 1 || q_heads % kv_heads != 0 || head_dim < 1) return 0;
    int64_t n = 1;  // either kernel may be taken, by what the call's window is
    for (const int64_t keys : {int64_t(0), int64_t(1) << 30}) {
        const int64_t m = wzyb::attn_shape(T, q_heads, kv_heads, head_dim, keys).max_splits;
        n = m > n ? m : n;
    }
    return n > 1 ? n * T * q_heads * (head_dim * 4 + 8) + 16 : 0;
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
