// gdn_delta.cu -- the gated delta rule (GDN), the recurrence whose output the GDN gated norm takes.
//
// Per value head, with the state S as [v, k] (column j of the value dimension is one k-vector S_j):
//   S_j <- e^(g_t) S_j;   d_j = beta_t (v_t[j] - S_j . k_t);   S_j += d_j k_t;   o_t[j] = scale S_j . q_t
// Value columns never mix, so every kernel here gives each column to one owner for the whole sequence.
#include "launch.hpp"
#include "common.cuh"

namespace wzyb {

struct GdnDeltaArgs {
    const void* q;  // [T, k_heads, HD]
    const void* k;
    const void* v;  // [T, v_heads, HD]
    int64_t q_row, k_row, v_row, o_row;  // elements between tokens
    const float* g;     // [T, v_heads]
    const float* beta;  // [T, v_heads]
    const float* state_in;  // [v_heads, HD, HD] or NULL
    float* state_out;
    float* snaps;  // [T, v_heads, HD, HD] or NULL
    void* o;       // [T, v_heads, HD]
    int64_t T;
    int k_heads, v_heads;
    float scale;
    int l2norm;
    float l2_eps;
};

// The recurrence token by token. 8 lanes own a column (HD / 8 of its elements each, in registers for
// the whole call), a warp 4 columns, a CTA of 8 warps 32 columns of one head. Both dots of a token are
// taken on the old state, S . k and S . q, so one reduction (three xor shuffles) serves both:
//   o = scale (e^g S.q + d k.q),  with k.q once per token.
// q, k, v of a block of tokens are converted, normed and staged in shared memory by the whole CTA while
// the previous block is worked through. fp32 throughout (expf and FMA), whatever the inputs' type.
// Bound: the state's bytes for few tokens (1 fp16 token of 32 heads of 128: 4.4 us, the call 10.1 with its host time;
// 8 fp32 tokens of 48 heads with every state written, 32 MB: call 10.5 us), for many the chain of dot, reduction and
// update, 0.31 us per token. 8 lanes per column keep that chain at three shuffles and the state at 16 registers.
template <typename T, int HD>
__global__ void __launch_bounds__(256) gdn_recurrent_kernel(const GdnDeltaArgs a) {
    pdl_begin();
    constexpr int kTok = 16;          // tokens per staged block: 8 elements of q and of k per staging thread
    constexpr int kLanes = HD / 8;    // staging lanes per token
    constexpr int kE = HD / 32;       // float4 of the state per lane
    __shared__ __align__(16) float sk[2][kTok][HD];
    __shared__ __align__(16) float sq[2][kTok][HD];
    __shared__ float sv[2][kTok][32];
    __shared__ float sdec[2][kTok], sbeta[2][kTok], skq[2][kTok];
    __shared__ float so[2][kTok][33];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x / (HD / 32), c0 = (blockIdx.x % (HD / 32)) * 32;
    const int hk = h / (a.v_heads / a.k_heads);
    const int col = c0 + warp * 4 + (lane >> 3), l8 = lane & 7;

    float2 s[2 * kE];  // elements 4*l8 + 32*i .. +3 of this column
    const int64_t sbase = ((int64_t)h * HD + col) * HD + 4 * l8;
    if (a.state_in != nullptr) {
#pragma unroll
        for (int i = 0; i < kE; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(a.state_in + sbase + 32 * i);
            s[2 * i] = make_float2(x.x, x.y);
            s[2 * i + 1] = make_float2(x.z, x.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2 * kE; ++i) s[i] = make_float2(0.f, 0.f);
    }

    const T* const gq = static_cast<const T*>(a.q) + hk * HD;
    const T* const gk = static_cast<const T*>(a.k) + hk * HD;
    const T* const gv = static_cast<const T*>(a.v) + h * HD + c0;
    T* const go = static_cast<T*>(a.o) + h * HD + c0;
    const int st = tid / kLanes, sl = (tid % kLanes) * 8;  // staged token and first element of this thread
    constexpr int kVPer = kTok * 32 / 256;                 // staged v elements per thread

    float fq[8], fk[8], fv[kVPer], fg = 0.f, fb = 0.f;
    auto fetch = [&](int64_t t0) {
        const int64_t t = t0 + st;
        if (st < kTok && t < a.T) {
            Vec8<T>::load_ro(gq + t * a.q_row + sl, fq);
            Vec8<T>::load_ro(gk + t * a.k_row + sl, fk);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) fq[i] = fk[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < kVPer; ++i) {
            const int64_t tv = t0 + warp + 8 * i;
            fv[i] = tv < a.T ? (float)gv[tv * a.v_row + lane] : 0.f;
        }
        if (tid < kTok && t0 + tid < a.T) {
            fg = a.g[(t0 + tid) * a.v_heads + h];
            fb = a.beta[(t0 + tid) * a.v_heads + h];
        }
    };
    auto stage = [&](int b) {
        float qq = 0.f, kk = 0.f, kq = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            qq = fmaf(fq[i], fq[i], qq);
            kk = fmaf(fk[i], fk[i], kk);
            kq = fmaf(fk[i], fq[i], kq);
        }
        qq = group_sum<kLanes>(qq);
        kk = group_sum<kLanes>(kk);
        kq = group_sum<kLanes>(kq);
        const float rq = (a.l2norm ? rsqrtf(qq + a.l2_eps) : 1.f) * a.scale;
        const float rk = a.l2norm ? rsqrtf(kk + a.l2_eps) : 1.f;
        if (st < kTok) {
            float4* const dq = reinterpret_cast<float4*>(&sq[b][st][sl]);
            float4* const dk = reinterpret_cast<float4*>(&sk[b][st][sl]);
            dq[0] = make_float4(fq[0] * rq, fq[1] * rq, fq[2] * rq, fq[3] * rq);
            dq[1] = make_float4(fq[4] * rq, fq[5] * rq, fq[6] * rq, fq[7] * rq);
            dk[0] = make_float4(fk[0] * rk, fk[1] * rk, fk[2] * rk, fk[3] * rk);
            dk[1] = make_float4(fk[4] * rk, fk[5] * rk, fk[6] * rk, fk[7] * rk);
            if (sl == 0) skq[b][st] = kq * rq * rk;
        }
#pragma unroll
        for (int i = 0; i < kVPer; ++i) sv[b][warp + 8 * i][lane] = fv[i];
        if (tid < kTok) {
            sdec[b][tid] = expf(fg);
            sbeta[b][tid] = fb;
        }
    };

    fetch(0);
    stage(0);
    int b = 0;
    for (int64_t t0 = 0; t0 < a.T; t0 += kTok, b ^= 1) {
        __syncthreads();  // block b is staged, and the outputs of the block before are all in shared memory
        if (t0 > 0) {
#pragma unroll
            for (int i = 0; i < kVPer; ++i) {
                const int64_t t = t0 - kTok + warp + 8 * i;
                go[t * a.o_row + lane] = (T)so[b ^ 1][warp + 8 * i][lane];
            }
        }
        const bool more = t0 + kTok < a.T;
        if (more) fetch(t0 + kTok);
        const int n = (int)(a.T - t0 < kTok ? a.T - t0 : kTok);
        for (int t = 0; t < n; ++t) {
            float2 k2[2 * kE], q2[2 * kE];
#pragma unroll
            for (int i = 0; i < kE; ++i) {
                const float4 x = *reinterpret_cast<const float4*>(&sk[b][t][4 * l8 + 32 * i]);
                const float4 y = *reinterpret_cast<const float4*>(&sq[b][t][4 * l8 + 32 * i]);
                k2[2 * i] = make_float2(x.x, x.y);
                k2[2 * i + 1] = make_float2(x.z, x.w);
                q2[2 * i] = make_float2(y.x, y.y);
                q2[2 * i + 1] = make_float2(y.z, y.w);
            }
            float2 dk2 = fmul2(s[0], k2[0]), dq2 = fmul2(s[0], q2[0]);
#pragma unroll
            for (int i = 1; i < 2 * kE; ++i) {
                dk2 = ffma2(s[i], k2[i], dk2);
                dq2 = ffma2(s[i], q2[i], dq2);
            }
            float sk_dot = dk2.x + dk2.y, sq_dot = dq2.x + dq2.y;
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) {
                sk_dot += __shfl_xor_sync(0xffffffffu, sk_dot, o);
                sq_dot += __shfl_xor_sync(0xffffffffu, sq_dot, o);
            }
            const float dec = sdec[b][t];
            const float d = sbeta[b][t] * (sv[b][t][warp * 4 + (lane >> 3)] - dec * sk_dot);
            const float2 d2 = splat2(d), dec2 = splat2(dec);
#pragma unroll
            for (int i = 0; i < 2 * kE; ++i) s[i] = ffma2(k2[i], d2, fmul2(s[i], dec2));
            if (l8 == 0) so[b][t][warp * 4 + (lane >> 3)] = fmaf(d, skq[b][t], dec * sq_dot);
            if (a.snaps != nullptr) {
                float* const p = a.snaps + (t0 + t) * (int64_t)a.v_heads * HD * HD + sbase;
#pragma unroll
                for (int i = 0; i < kE; ++i)
                    __stcs(reinterpret_cast<float4*>(p + 32 * i),
                           make_float4(s[2 * i].x, s[2 * i].y, s[2 * i + 1].x, s[2 * i + 1].y));
            }
        }
        if (more) stage(b ^ 1);
    }
    __syncthreads();
    const int64_t tl = (a.T - 1) / kTok * kTok;  // the last block's outputs
#pragma unroll
    for (int i = 0; i < kVPer; ++i) {
        const int64_t t = tl + warp + 8 * i;
        if (t < a.T) go[t * a.o_row + lane] = (T)so[b ^ 1][warp + 8 * i][lane];
    }
#pragma unroll
    for (int i = 0; i < kE; ++i)
        *reinterpret_cast<float4*>(a.state_out + sbase + 32 * i) =
            make_float4(s[2 * i].x, s[2 * i].y, s[2 * i + 1].x, s[2 * i + 1].y);
}

// ----------------------------------------------------------------------------------------------------
// The chunked form, for many tokens. With G the running sum of g inside a chunk of 64 tokens, k^ = rk k,
// q^ = rq q (norms as row factors, so that fp16 inputs stay as they are) and S the state at its start:
//   A_ij = beta_i e^(G_i - G_j) k^_i.k^_j  (i > j),     T = (I + A)^-1
//   d = T diag(beta) (V - diag(e^G) K^ S),              o = scale (diag(e^G) Q^ S + tril(e^(G_i - G_j) q^_i.k^_j) d)
//   S <- e^(G_64) S + sum_j e^(G_64 - G_j) k^_j d_j
// T, the masked score matrix P and the row factors do not depend on S: gdn_chunk_prep_kernel makes them for
// all chunks of a segment at once. gdn_chunk_scan_kernel then walks the chunks; its products with S, d and T
// run on the tensor cores (mma m16n8k16).
//
// Precision. The state has to stay an fp32 state, and fp16 products of a rounded S would leave 2^-12 in it. So every
// fp32 operand enters as two fp16 parts, x 2^-e = hi + 2^-11 lo (lo stored 2^11 times as large, so it is not cut
// off), and a product takes hi*hi, hi*lo and, where both operands are split, lo*hi: 22 bits. k and q of fp16
// calls are one part and exact. The exponents e are per value column (columns never mix), P and T have one each.
// Running sums never live in a tensor-core accumulator for longer than a chunk (its sums are cut off towards
// zero): S is updated in fp32 registers.
//
// Infinities and NaN. A masked product is 0 times a later token's value, which is no 0 where that is infinite or NaN,
// and one such value would set the exponent of its whole column. So they are taken out: an infinite or NaN k, g
// (not -inf) or beta ends the chunk's matrices before its token, an infinite or NaN element of X (from a v, or from a
// state that is so already) is replaced by 0, and what follows from them (all later outputs and the state, of the head or
// of the column) is set to NaN. A q reaches its own row only.
// ----------------------------------------------------------------------------------------------------
constexpr int kGdnChunk = 64;
constexpr float kGdnLo = 2048.f;
constexpr float kGdnFinite = 3.402823466e38f;  // the largest finite number: neither an infinity nor a NaN is <= it

// A (chunk, value head)'s part of the workspace. Matrices as mma A fragments, 16 bytes per lane: fragment
// (m-tile i, k-step j <= i) at index i * (i + 1) / 2 + j, 512 bytes each.
struct GdnChunkData {
    uint4 t_hi[10][32], t_lo[10][32];
    uint4 p[20][32];  // hi parts, then lo parts
    float a[64], b[64], c[64];      // row factors of K S, Q S and d
    float decay, t_up, p_up, pad;   // e^(G_64), 2^e of T and of P
};

__device__ __forceinline__ void mma_f16(float (&d)[4], const uint4& a, uint32_t b0, uint32_t b1) {
    const uint32_t x[4] = {a.x, a.y, a.z, a.w};
    mma_f16(d, x, b0, b1);
}
__device__ __forceinline__ void gdn_split(float x, float y, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn((x - f.x) * kGdnLo, (y - f.y) * kGdnLo);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
}
// e with |x| < 2^e for a finite x, within [-100, 120]
__device__ __forceinline__ int gdn_exp(float x) {
    const int e = (int)((__float_as_uint(x) >> 23) & 0xFF) - 126;
    return e < -100 ? -100 : (e > 120 ? 120 : e);
}
__device__ __forceinline__ float gdn_exp2i(int e) { return __int_as_float((e + 127) << 23); }

// A (chunk, k head)'s K and Q as the scan's shared memory holds them (rows padded by 16 bytes, missing tokens zero), so
// that one bulk copy fetches them: 64 rows by cp.async took the scan's load/store unit 450 cycles per chunk, and
// a bulk copy per row far longer. fp32 inputs as two fp16 parts each.
template <bool kSplit, int HD>
struct GdnKq {
    static constexpr int kLd = HD + 8;
    __half k[kSplit ? 2 : 1][64 * kLd], q[kSplit ? 2 : 1][64 * kLd];
};

struct GdnPrepArgs {
    GdnDeltaArgs x;
    int64_t t0;     // first token of the segment
    uint8_t* data;  // [chunks, v_heads] GdnChunkData
    uint8_t* kq;    // [chunks, k_heads] GdnKq
};

template <typename T, int HD>
struct GdnPrepSmem {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kLd = HD + 8;
    GdnKq<kSplit, HD> kq;
    float A[64][68];
    float tm[64][68];
    float rk[64], rq[64], beta[64], ghi[64], glo[64];
    unsigned int amax[2];
    unsigned int k_bad[2];  // bit per token: k is infinite or NaN
    int first_bad;          // of the value head: the first token from which everything is NaN, 64 for none
};

// The rows of k that hold an infinity or a NaN become 0 in the chunk's images; k_bad names them.
template <typename T, int HD>
__device__ __noinline__ void gdn_zero_bad_k(const GdnPrepArgs& p, GdnPrepSmem<T, HD>& sm, GdnKq<sizeof(T) == 4, HD>& image, int64_t tok0, int hk,
                                            int n) {
    constexpr int kParts = sizeof(T) == 4 ? 2 : 1;
    bool bad = false;
    const int r = threadIdx.x;
    if (r < n) {
        const T* const k = static_cast<const T*>(p.x.k) + (tok0 + r) * p.x.k_row + hk * HD;
        for (int i = 0; i < HD; ++i) bad = bad || !(fabsf((float)k[i]) <= kGdnFinite);
        for (int part = 0; bad && part < kParts; ++part)
            for (int i = 0; i < HD; ++i) sm.kq.k[part][r * (HD + 8) + i] = image.k[part][r * (HD + 8) + i] = __float2half_rn(0.f);
        if (bad) sm.rk[r] = 0.f;
    }
    const unsigned int bits = __ballot_sync(0xffffffffu, bad);
    __syncthreads();
    if (r < 64 && r % 32 == 0) sm.k_bad[r / 32] = bits;
    __syncthreads();
}

// One CTA of 4 warps per (chunk, k head), over the value heads that share it. Warp w owns rows 16w .. 16w+15.
// T by blocks of 16: a diagonal block's inverse by forward substitution (a lane per column), then the column
// block j below it by warp j: T_ij = -T_ii sum_k A_ik T_kj, fp32 FMA. Bound by the latency of those short dependent
// sums at 3 CTAs per SM (168 registers): 64 chunks of 16/32 heads of 128, fp16, 73 us, 30 % of the call's time.
// Halving (the 64 rows as 32 + 32, those as 16 + 16) has longer sums and shorter chains, but needs 209 registers: 2 CTAs
// per SM, 6 % slower.
// The least CTAs per SM that the registers have to leave room for (0: the compiler's choice, which is 168 registers too):
// shared memory holds two of fp32 with head_dim 128. us at 8192 tokens of 16/32 (fp32: 16/48) heads: fp32, 128: 1148 with
// two, 1193 with the compiler's choice; fp16, 128: 490 with its choice, 496 with three (more spills), 506 with one; fp16,
// 64: 391 with three, 414 with its choice (172 registers); fp32, 64: 536 and 580.
template <typename T, int HD>
constexpr int gdn_prep_ctas() {
    return HD == 64 ? 3 : (sizeof(T) == 4 ? 2 : 0);
}
template <typename T, int HD>
__global__ void __launch_bounds__(128, gdn_prep_ctas<T, HD>()) gdn_chunk_prep_kernel(const GdnPrepArgs p) {
    pdl_begin();
    using S = GdnPrepSmem<T, HD>;
    constexpr bool kSplit = S::kSplit;
    constexpr int kLd = S::kLd;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    S& sm = *reinterpret_cast<S*>(smem_raw);
    const GdnDeltaArgs& a = p.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t4 = lane & 3;
    const int chunk = blockIdx.x / a.k_heads, hk = blockIdx.x % a.k_heads;
    const int64_t tok0 = p.t0 + (int64_t)chunk * kGdnChunk;
    const int n = (int)(a.T - tok0 < kGdnChunk ? a.T - tok0 : kGdnChunk);
    constexpr int kL = HD / 8;  // lanes per row
    GdnKq<kSplit, HD>& image = reinterpret_cast<GdnKq<kSplit, HD>*>(p.kq)[(int64_t)chunk * a.k_heads + hk];

    if (tid < 2) sm.k_bad[tid] = 0u;
    __syncthreads();
    for (int r0 = 0; r0 < 64; r0 += 128 / kL) {
        const int r = r0 + tid / kL, col = (tid % kL) * 8;
        float x[2][8];
        float f[2];
#pragma unroll
        for (int m = 0; m < 2; ++m) {
            const T* src = static_cast<const T*>(m ? a.q : a.k) + (tok0 + r) * (m ? a.q_row : a.k_row) + hk * HD + col;
            if (r < n) {
                Vec8<T>::load_ro(src, x[m]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[m][i] = 0.f;
            }
            float ss = 0.f, am = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                ss = fmaf(x[m][i], x[m][i], ss);
                am = fmaxf(am, fabsf(x[m][i]));
            }
            ss = group_sum<kL>(ss);
            if (m == 0 && col == 0 && !(ss <= kGdnFinite)) sm.k_bad[r >> 5] = 1u;  // infinite or NaN, or too large to be squared
            f[m] = r < n ? (a.l2norm ? rsqrtf(ss + a.l2_eps) : 1.f) : 0.f;
            __half* const hi = (m ? sm.kq.q[0] : sm.kq.k[0]) + r * kLd + col;
            if constexpr (kSplit) {
#pragma unroll
                for (int o = kL / 2; o > 0; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
                const int e = am == 0.f ? 0 : gdn_exp(am);
                const float down = gdn_exp2i(-e);
                f[m] *= gdn_exp2i(e);
                uint32_t h[4], l[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) gdn_split(x[m][2 * i] * down, x[m][2 * i + 1] * down, h[i], l[i]);
                const uint4 vh = make_uint4(h[0], h[1], h[2], h[3]), vl = make_uint4(l[0], l[1], l[2], l[3]);
                *reinterpret_cast<uint4*>(hi) = vh;
                *reinterpret_cast<uint4*>((m ? sm.kq.q[kSplit] : sm.kq.k[kSplit]) + r * kLd + col) = vl;
                *reinterpret_cast<uint4*>((m ? image.q[0] : image.k[0]) + r * kLd + col) = vh;
                *reinterpret_cast<uint4*>((m ? image.q[kSplit] : image.k[kSplit]) + r * kLd + col) = vl;
            } else {
                const uint4 v = Vec8<__half>::from_f32(x[m]);
                *reinterpret_cast<uint4*>(hi) = v;
                *reinterpret_cast<uint4*>((m ? image.q[0] : image.k[0]) + r * kLd + col) = v;
            }
        }
        if (col == 0) {
            sm.rk[r] = f[0];
            sm.rq[r] = f[1] * a.scale;
        }
    }
    __syncthreads();
    if ((sm.k_bad[0] | sm.k_bad[1]) != 0u) gdn_zero_bad_k<T, HD>(p, sm, image, tok0, hk, n);

    // raw k.k and q.k of this warp's rows, columns up to the diagonal block
    float kk[8][4], qk[8][4];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        float (&acc)[8][4] = m ? qk : kk;
        const __half* const xh = m ? sm.kq.q[0] : sm.kq.k[0];
        const __half* const xl = m ? sm.kq.q[kSplit] : sm.kq.k[kSplit];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) acc[i][c] = 0.f;
        const int arow = warp * 16 + (lane & 15), acol = (lane >> 4) * 8;
        const int brow = (lane & 7) + ((lane >> 4) << 3), bcol = ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int part = kSplit ? 1 : 0; part >= 0; --part) {
#pragma unroll
            for (int ks = 0; ks < HD / 16; ++ks) {
                uint32_t fa[4], fl[4];
                ldmatrix_x4(fa, xh + arow * kLd + ks * 16 + acol);
                if (part == 1) ldmatrix_x4(fl, xl + arow * kLd + ks * 16 + acol);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (i > warp) break;  // warp-uniform
                    uint32_t fb[4];
                    if (part == 1) {
                        ldmatrix_x4(fb, sm.kq.k[kSplit] + (i * 16 + brow) * kLd + ks * 16 + bcol);
                        mma_f16(acc[2 * i], fa, fb[0], fb[1]);
                        mma_f16(acc[2 * i + 1], fa, fb[2], fb[3]);
                    }
                    ldmatrix_x4(fb, sm.kq.k[0] + (i * 16 + brow) * kLd + ks * 16 + bcol);
                    if (part == 1) {
                        mma_f16(acc[2 * i], fl, fb[0], fb[1]);
                        mma_f16(acc[2 * i + 1], fl, fb[2], fb[3]);
                    } else {
                        mma_f16(acc[2 * i], fa, fb[0], fb[1]);
                        mma_f16(acc[2 * i + 1], fa, fb[2], fb[3]);
                    }
                }
            }
            if (part == 1) {
#pragma unroll
                for (int i = 0; i < 8; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) acc[i][c] *= 1.f / kGdnLo;
            }
        }
    }

    const int per = a.v_heads / a.k_heads;
    float gx[2] = {0.f, 0.f}, bx[2] = {0.f, 0.f};  // warp 0: g and beta of tokens 2 * lane, + 1, a head ahead
    auto load_gb = [&](int h) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            if (2 * lane + i < n) {
                gx[i] = __ldg(a.g + (tok0 + 2 * lane + i) * a.v_heads + h);
                bx[i] = __ldg(a.beta + (tok0 + 2 * lane + i) * a.v_heads + h);
            }
    };
    if (warp == 0) load_gb(hk * per);
    for (int hv = 0; hv < per; ++hv) {
        const int h = hk * per + hv;
        GdnChunkData& out = reinterpret_cast<GdnChunkData*>(p.data)[(int64_t)chunk * a.v_heads + h];
        if (warp == 0) {
            // running sums in fp64, held as two fp32 parts in log2 units: differences of close tokens keep their
            // precision after strong decays. A decay below e^-120 is 0 in fp32 either way (so -inf is as well).
            double s0 = 0., s1 = 0.;
            bool bad[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                bad[i] = !(gx[i] <= kGdnFinite) || !(fabsf(bx[i]) <= kGdnFinite) || (sm.k_bad[lane >> 4] >> ((2 * lane + i) & 31) & 1u);
            int first = 64;
            if (__any_sync(0xffffffffu, bad[0] || bad[1])) {
                first = __reduce_min_sync(0xffffffffu, bad[0] ? 2 * lane : (bad[1] ? 2 * lane + 1 : 64));
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (2 * lane + i >= first) gx[i] = bx[i] = 0.f;
            }
            if (lane == 0) sm.first_bad = first;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                sm.beta[2 * lane + i] = bx[i];
                (i ? s1 : s0) = (double)(gx[i] < -120.f ? -120.f : gx[i]) * 1.4426950408889634;
            }
            if (hv + 1 < per) load_gb(h + 1);
            s1 += s0;
            double run = s1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += y;
            }
            s0 += run - s1;
            s1 = run;
            sm.ghi[2 * lane] = (float)s0;
            sm.glo[2 * lane] = (float)(s0 - (float)s0);
            sm.ghi[2 * lane + 1] = (float)s1;
            sm.glo[2 * lane + 1] = (float)(s1 - (float)s1);
            if (lane < 2) sm.amax[lane] = 0u;
        }
        __syncthreads();
        float pv[8][4];
        float p_max = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i > 2 * warp + 1) break;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = warp * 16 + g + (c >> 1) * 8, col = i * 8 + 2 * t4 + (c & 1);
                const float d = ex2_approx((sm.ghi[r] - sm.ghi[col]) + (sm.glo[r] - sm.glo[col]));
                sm.A[r][col] = r > col ? sm.beta[r] * (kk[i][c] * (sm.rk[r] * sm.rk[col]) * d) : 0.f;
                pv[i][c] = r >= col ? qk[i][c] * (sm.rq[r] * sm.rk[col]) * d : 0.f;
                p_max = fmaxf(p_max, fabsf(pv[i][c]));
            }
        }
        if (tid < 64) {
            const float e = ex2_approx(sm.ghi[tid] + sm.glo[tid]);
            out.a[tid] = sm.rk[tid] * e;
            out.b[tid] = tid < sm.first_bad ? sm.rq[tid] * e : __int_as_float(0x7FC00000);
            out.c[tid] = sm.rk[tid] * ex2_approx((sm.ghi[63] - sm.ghi[tid]) + (sm.glo[63] - sm.glo[tid]));
        }
        __syncwarp();
        {  // inverse of the diagonal block: lane = column (the upper 16 lanes repeat the lower)
            const int b0 = warp * 16, j = lane & 15;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float s = 0.f;
#pragma unroll
                for (int k = 0; k < 16; ++k)
                    if (k < i) s = fmaf(sm.A[b0 + i][b0 + k], x[k], s);
                x[i] = (i == j ? 1.f : 0.f) - s;
            }
            if (lane < 16) {
#pragma unroll
                for (int i = 0; i < 16; ++i) sm.tm[b0 + i][b0 + j] = x[i];
            }
        }
        __syncthreads();
        {  // the blocks below it: lane = 2 rows x 4 columns
            const int rr = (lane >> 2) * 2, cc = warp * 16 + (lane & 3) * 4;
            for (int i = warp + 1; i < 4; ++i) {
                float y[2][4] = {};
                for (int k = warp; k < i; ++k) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float4 b = *reinterpret_cast<const float4*>(&sm.tm[k * 16 + e][cc]);
#pragma unroll
                        for (int r = 0; r < 2; ++r) {
                            const float x = sm.A[i * 16 + rr + r][k * 16 + e];
                            y[r][0] = fmaf(x, b.x, y[r][0]);
                            y[r][1] = fmaf(x, b.y, y[r][1]);
                            y[r][2] = fmaf(x, b.z, y[r][2]);
                            y[r][3] = fmaf(x, b.w, y[r][3]);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    *reinterpret_cast<float4*>(&sm.tm[i * 16 + rr + r][cc]) = make_float4(y[r][0], y[r][1], y[r][2], y[r][3]);
                __syncwarp();
                float z[2][4] = {};
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const float4 b = *reinterpret_cast<const float4*>(&sm.tm[i * 16 + e][cc]);
#pragma unroll
                    for (int r = 0; r < 2; ++r) {
                        const float x = sm.tm[i * 16 + rr + r][i * 16 + e];
                        z[r][0] = fmaf(x, b.x, z[r][0]);
                        z[r][1] = fmaf(x, b.y, z[r][1]);
                        z[r][2] = fmaf(x, b.z, z[r][2]);
                        z[r][3] = fmaf(x, b.w, z[r][3]);
                    }
                }
                __syncwarp();
#pragma unroll
                for (int r = 0; r < 2; ++r)
                    *reinterpret_cast<float4*>(&sm.tm[i * 16 + rr + r][cc]) = make_float4(-z[r][0], -z[r][1], -z[r][2], -z[r][3]);
                __syncwarp();
            }
        }
        __syncthreads();
        // T diag(beta) and P as fragments, their largest element scaled to [2^13, 2^14): the bits that fp16 parts hold do
        // not depend on the sizes of beta, of the caller's scale or of an unnormed q
        float tv[8][4];
        float t_max = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (i > 2 * warp + 1) break;
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int r = warp * 16 + g + (c >> 1) * 8, col = i * 8 + 2 * t4 + (c & 1);
                tv[i][c] = sm.tm[r][col] * sm.beta[col];
                t_max = fmaxf(t_max, fabsf(tv[i][c]));
            }
        }
        if (p_max > kGdnFinite) {  // an infinite q: its rows are alone with it
            p_max = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (i > 2 * warp + 1) break;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (fabsf(pv[i][c]) <= kGdnFinite) p_max = fmaxf(p_max, fabsf(pv[i][c]));
            }
        }
        const unsigned int tb = __reduce_max_sync(0xffffffffu, __float_as_uint(t_max));
        const unsigned int pb = __reduce_max_sync(0xffffffffu, __float_as_uint(p_max));
        if (lane == 0) {
            atomicMax(&sm.amax[0], tb);
            atomicMax(&sm.amax[1], pb);
        }
        __syncthreads();
        const int et = gdn_exp(__uint_as_float(sm.amax[0])) - 14, ep = gdn_exp(__uint_as_float(sm.amax[1])) - 14;
        const float td = gdn_exp2i(-et), pd = gdn_exp2i(-ep);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (j > warp) break;
            const int at = warp * (warp + 1) / 2 + j;
            uint32_t h[4], l[4];
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                gdn_split(tv[2 * j + b][0] * td, tv[2 * j + b][1] * td, h[2 * b], l[2 * b]);
                gdn_split(tv[2 * j + b][2] * td, tv[2 * j + b][3] * td, h[2 * b + 1], l[2 * b + 1]);
            }
            out.t_hi[at][lane] = make_uint4(h[0], h[1], h[2], h[3]);
            out.t_lo[at][lane] = make_uint4(l[0], l[1], l[2], l[3]);
#pragma unroll
            for (int b = 0; b < 2; ++b) {
                gdn_split(pv[2 * j + b][0] * pd, pv[2 * j + b][1] * pd, h[2 * b], l[2 * b]);
                gdn_split(pv[2 * j + b][2] * pd, pv[2 * j + b][3] * pd, h[2 * b + 1], l[2 * b + 1]);
            }
            out.p[at][lane] = make_uint4(h[0], h[1], h[2], h[3]);
            out.p[10 + at][lane] = make_uint4(l[0], l[1], l[2], l[3]);
        }
        if (tid == 0) {
            out.decay = sm.first_bad < 64 ? __int_as_float(0x7FC00000) : ex2_approx(sm.ghi[63] + sm.glo[63]);
            out.t_up = gdn_exp2i(et);
            out.p_up = gdn_exp2i(ep);
            out.pad = 0.f;
        }
        __syncthreads();
    }
}

struct GdnScanArgs {
    GdnDeltaArgs x;
    int64_t t0, t1;  // the segment's tokens
    const float* state_in;
    const uint8_t* data;
    const uint8_t* kq;
};

template <typename T, int HD>
struct GdnScanStage {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kLd = HD + 8, kVLd = 32 + 16 / sizeof(T);
    GdnKq<kSplit, HD> kq;
    GdnChunkData d;
    T v[64 * kVLd];
};

// Two column exponents per lane (columns 2*t4, 2*t4 + 1 of its warp), alike over the lanes of a column: values
// scaled by 2^-e stay below 2^14. `force` sets them anew (every 16 chunks, so they follow a shrinking state
// down too); otherwise they move only when a value would pass 2^14. `m`: the lane's largest magnitudes.
__device__ __forceinline__ bool gdn_exp_moves(const float (&m)[2], const int (&e)[2], bool force) {
    const bool over = !(m[0] * gdn_exp2i(-e[0]) <= 16384.f) || !(m[1] * gdn_exp2i(-e[1]) <= 16384.f);
    return __any_sync(0xffffffffu, over) || force;
}
__device__ __forceinline__ void gdn_move_exp(float (&m)[2], int (&e)[2], bool force) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) m[i] = fmaxf(m[i], __shfl_xor_sync(0xffffffffu, m[i], o));
        if (force || m[i] * gdn_exp2i(-e[i]) > 16384.f) {
            const int n = gdn_exp(m[i]) - 8;
            e[i] = n < -100 ? -100 : n;
        }
    }
}
template <int N>
__device__ __forceinline__ void gdn_col_exp(const float (&x)[N][4], int (&e)[2], bool force) {
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) m[c & 1] = fmaxf(m[c & 1], fabsf(x[i][c]));
    if (gdn_exp_moves(m, e, force)) gdn_move_exp(m, e, force);
}
// The largest magnitude of three, NaN where one is.
__device__ __forceinline__ float max3_abs_nan(float a, float x, float y) {
    float z;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(z) : "f"(a), "f"(x), "f"(y));
    return z;
}
// For X: also the first infinite or NaN row of each of the two columns (unchanged where there is none, which is to say
// always); such elements become 0.
__device__ __forceinline__ void gdn_clean_exp(float (&x)[4][4], int (&e)[2], bool force, int (&first)[2], int g) {
    float m[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int c = 0; c < 2; ++c) m[c] = max3_abs_nan(m[c], x[i][c], x[i][c + 2]);
    if (!gdn_exp_moves(m, e, force)) return;
    if (__any_sync(0xffffffffu, !(m[0] <= kGdnFinite) || !(m[1] <= kGdnFinite))) {
        m[0] = m[1] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                if (!(fabsf(x[i][c]) <= kGdnFinite)) {
                    first[c & 1] = min(first[c & 1], 16 * i + g + (c >> 1) * 8);
                    x[i][c] = 0.f;
                }
                m[c & 1] = fmaxf(m[c & 1], fabsf(x[i][c]));
            }
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
            for (int o = 4; o < 32; o <<= 1) first[c] = min(first[c], __shfl_xor_sync(0xffffffffu, first[c], o));
    }
    gdn_move_exp(m, e, force);
}

// Accumulator layout (rows g, g + 8 of each 16-row tile; columns 2*t4, 2*t4 + 1) to the second operand's (16 rows
// per step, columns g): packed fp16 pairs through 8x8 register transposes.
template <int N>
__device__ __forceinline__ void gdn_operand(const float (&x)[N][4], const int (&e)[2], uint32_t (&hi)[N][2],
                                            uint32_t (&lo)[N][2]) {
    const float d0 = gdn_exp2i(-e[0]), d1 = gdn_exp2i(-e[1]);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            uint32_t h, l;
            gdn_split(x[i][2 * b] * d0, x[i][2 * b + 1] * d1, h, l);
            hi[i][b] = transpose8(h);
            lo[i][b] = transpose8(l);
        }
}

// What a state warp hands to its output warp: S at the chunk's start as a second operand (per step of 16: hi, hi,
// lo, lo) with the scales of a lane's two columns, and d as fp32 accumulator tiles (the output warp has the time to
// make an operand of it, the state warp's chain has not).
template <int HD>
struct GdnHandOver {
    uint4 s[HD / 16][32];
    float4 d[4][32];
    float2 s_up[32];
    int2 first_bad[32];  // the first rows of a lane's two columns from which o is NaN, 64 for none
};
// All of a scan CTA's shared memory; the launch asks for its size, so no part of it can lie outside.
template <typename T, int HD>
struct GdnScanSmem {
    GdnScanStage<T, HD> st[2];
    GdnHandOver<HD> hand[4];  // one per pair of warps
    uint64_t full[2];         // a chunk's copies have landed
};
static_assert(sizeof(GdnScanSmem<float, 128>) <= 227 * 1024, "the largest instance fits one CTA per SM");
template <int N>
__device__ __forceinline__ void gdn_hand(uint4 (&to)[N][32], const uint32_t (&hi)[N][2], const uint32_t (&lo)[N][2], int lane) {
#pragma unroll
    for (int i = 0; i < N; ++i) to[i][lane] = make_uint4(hi[i][0], hi[i][1], lo[i][0], lo[i][1]);
}
__device__ __forceinline__ void named_bar_arrive(int id, int nthreads) {
    asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(nthreads) : "memory");
}

// 8 value columns of a head belong to two warps from the first chunk to the last. The state warp keeps its part of S
// in its registers as fp32 accumulator tiles; S, X = V - e^G K S and d = T X pass from product to product inside it
// (columns never mix), so its chain, which is what the chunks wait for, needs no barrier but the one per chunk. The
// output warp takes S and d from it when T X is done and makes o = e^G Q S + P d beside the rest of the chunk and the
// start of the next one (one warp for both took 1.5 times as long). The CTA's four pairs share the chunk's K, Q, T and
// P in shared memory; a ninth warp fetches the next chunk's meanwhile.
// Bound: the state warp's chain per chunk of 64 tokens, about 5000 cycles (fp16) or 6500 (fp32), the tensor pipe of an SM
// that has a CTA busy 49 % of it. 16/32 heads of 128, fp16: 32,768 tokens with the prep 1900 us. One CTA per SM: 128 CTAs hold 32
// heads; 48 heads are two waves.
template <typename T, int HD>
__global__ void __launch_bounds__(288, 1) gdn_chunk_scan_kernel(const GdnScanArgs p) {
    pdl_begin();
    using Stage = GdnScanStage<T, HD>;
    constexpr bool kSplit = Stage::kSplit;
    constexpr int kLd = Stage::kLd, kVLd = Stage::kVLd, kM = HD / 16;
    extern __shared__ __align__(16) uint8_t smem_raw[];
    GdnScanSmem<T, HD>& sm = *reinterpret_cast<GdnScanSmem<T, HD>*>(smem_raw);
    Stage* const st = sm.st;
    const GdnDeltaArgs& a = p.x;
    const int tid = threadIdx.x, lane = tid & 31, pair = (tid >> 5) & 3, g = lane >> 2, t4 = lane & 3;
    const int role = tid >> 7;  // 0 state, 1 output, 2 fetch
    GdnHandOver<HD>& hand = sm.hand[pair];
    const int h = blockIdx.x / (HD / 32), c0 = (blockIdx.x % (HD / 32)) * 32;
    const int hk = h / (a.v_heads / a.k_heads);
    const int chunks = (int)((p.t1 - p.t0 + kGdnChunk - 1) / kGdnChunk);

    uint64_t* const full = sm.full;
    if (tid == 0) {
        mbar_init(&full[0], 1);
        mbar_init(&full[1], 1);
        fence_mbar_init();
    }
    __syncthreads();

    // named barriers: chunk ready (fetch, state), buffers free (fetch, output), handed over and taken (each pair)
    constexpr int kBarReady = 1, kBarFree = 2, kBarHand = 3, kBarTaken = 7;
    if (role == 2) {
        const uint64_t policy = policy_evict_normal();
        int lost = -1;  // the chunk whose wait gave up: no wait and no copy follows, the results are void (and reported)
        for (int ch = 0; ch <= chunks; ++ch) {  // chunk ch is fetched while ch - 1 is worked through
            if (ch > 0) {
                cp_async_wait<0>();
                if (lost < 0 && !mbar_wait(&full[(ch - 1) & 1], ((ch - 1) >> 1) & 1)) lost = ch - 1;
                named_bar_sync(kBarReady, 160);  // chunk ch - 1 is there for the state warps
                // the output warps have begun chunk ch - 1, so nobody reads chunk ch - 2's buffers any more; the state
                // warps are past the products that the copies would slow down
                named_bar_sync(kBarFree, 160);
            }
            if (ch == chunks) break;
            Stage& s = st[ch & 1];
            if (lane == 0 && lost < 0) {
                constexpr int kKq = sizeof(GdnKq<kSplit, HD>), kData = sizeof(GdnChunkData);
                mbar_arrive_expect_tx(&full[ch & 1], kKq + kData);
                bulk_load(&s.kq, p.kq + ((int64_t)ch * a.k_heads + hk) * kKq, kKq, &full[ch & 1], policy);
                bulk_load(&s.d, p.data + ((int64_t)ch * a.v_heads + h) * kData, kData, &full[ch & 1], policy);
            }
            const int64_t tok0 = p.t0 + (int64_t)ch * kGdnChunk;
            const int n = (int)(p.t1 - tok0 < kGdnChunk ? p.t1 - tok0 : kGdnChunk);
            constexpr int kVC = 32 * sizeof(T) / 16, kVE = 16 / sizeof(T);
#pragma unroll 4
            for (int i = lane; i < 64 * kVC; i += 32) {
                const int r = i / kVC, cv = (i % kVC) * kVE;
                T* const dst = s.v + r * kVLd + cv;
                if (r < n)
                    cp_async16(dst, static_cast<const T*>(a.v) + (tok0 + r) * a.v_row + h * HD + c0 + cv);
                else
                    *reinterpret_cast<uint4*>(dst) = make_uint4(0, 0, 0, 0);
            }
            cp_async_commit();
        }
        // that chunk's copies are the only ones that can still be in flight
        if (lost >= 0) mbar_wait_until(&full[lost & 1], (lost >> 1) & 1, globaltimer_ns() + kWaitLimitNs);
        return;
    }
    const int col = c0 + pair * 8 + 2 * t4;  // this lane's columns col, col + 1
    const int arow = lane & 15, acol = (lane >> 4) * 8;
    if (role == 1) {
        int ed[2] = {0, 0};
        for (int ch = 0; ch < chunks; ++ch) {
            const Stage& z = st[ch & 1];
            named_bar_sync(kBarHand + pair, 64);  // S and d (and, through the state warp, the chunk's data)
            named_bar_arrive(kBarFree, 160);
            uint4 so[kM];
            float d[4][4];
#pragma unroll
            for (int i = 0; i < kM; ++i) so[i] = hand.s[i][lane];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 y = hand.d[i][lane];
                d[i][0] = y.x;
                d[i][1] = y.y;
                d[i][2] = y.z;
                d[i][3] = y.w;
            }
            const float2 su = hand.s_up[lane];
            const int2 first_bad = hand.first_bad[lane];
            named_bar_arrive(kBarTaken + pair, 64);
            float o[4][4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float qh[4] = {}, ql[4] = {};
#pragma unroll
                for (int ks = 0; ks < kM; ++ks) {
                    uint32_t fq[4];
                    ldmatrix_x4(fq, z.kq.q[0] + (i * 16 + arow) * kLd + ks * 16 + acol);
                    mma_f16(qh, fq, so[ks].x, so[ks].y);
                    mma_f16(ql, fq, so[ks].z, so[ks].w);
                    if constexpr (kSplit) {
                        ldmatrix_x4(fq, z.kq.q[kSplit] + (i * 16 + arow) * kLd + ks * 16 + acol);
                        mma_f16(ql, fq, so[ks].x, so[ks].y);
                    }
                }
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    o[i][c] = z.d.b[16 * i + g + (c >> 1) * 8] * (c & 1 ? su.y : su.x) * fmaf(ql[c], 1.f / kGdnLo, qh[c]);
            }
            uint32_t dh[4][2], dl[4][2];
            gdn_col_exp(d, ed, (ch & 15) == 0);
            gdn_operand(d, ed, dh, dl);
            const float2 up = make_float2(gdn_exp2i(ed[0]) * z.d.p_up, gdn_exp2i(ed[1]) * z.d.p_up);
            const int64_t tok0 = p.t0 + (int64_t)ch * kGdnChunk;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float oh[4] = {}, ol[4] = {};
#pragma unroll
                for (int j = 0; j <= i; ++j) {
                    const uint4 ph = z.d.p[i * (i + 1) / 2 + j][lane];
                    mma_f16(oh, ph, dh[j][0], dh[j][1]);
                    mma_f16(ol, ph, dl[j][0], dl[j][1]);
                    mma_f16(ol, z.d.p[10 + i * (i + 1) / 2 + j][lane], dh[j][0], dh[j][1]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) o[i][c] = fmaf(c & 1 ? up.y : up.x, fmaf(ol[c], 1.f / kGdnLo, oh[c]), o[i][c]);
#pragma unroll
                for (int b = 0; b < 2; ++b) {
                    const int64_t t = tok0 + 16 * i + g + 8 * b;
                    if (t < p.t1) {
                        T* const dst = static_cast<T*>(a.o) + t * a.o_row + h * HD + col;
                        if constexpr (kSplit)
                            *reinterpret_cast<float2*>(dst) = make_float2(o[i][2 * b], o[i][2 * b + 1]);
                        else
                            *reinterpret_cast<__half2*>(dst) = __floats2half2_rn(o[i][2 * b], o[i][2 * b + 1]);
                    }
                }
            }
            if (min(first_bad.x, first_bad.y) < 64) {  // over what was stored
#pragma unroll 1
                for (int r = g; r < 64 && tok0 + r < p.t1; r += 8) {
                    T* const dst = static_cast<T*>(a.o) + (tok0 + r) * a.o_row + h * HD + col;
                    if (r >= first_bad.x) dst[0] = (T)__int_as_float(0x7FC00000);
                    if (r >= first_bad.y) dst[1] = (T)__int_as_float(0x7FC00000);
                }
            }
        }
        return;
    }

    float s[kM][4];  // S: rows k = 16*i + g, + 8
    const float* const sin = p.state_in + ((int64_t)h * HD + col) * HD;
#pragma unroll
    for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c)
            s[i][c] = p.state_in != nullptr ? sin[(c & 1) * HD + 16 * i + g + (c >> 1) * 8] : 0.f;
    int es[2] = {0, 0}, ex[2] = {0, 0}, ec[2] = {0, 0};
    bool was_bad = false;
    hand.first_bad[lane] = make_int2(64, 64);
    for (int ch = 0; ch < chunks; ++ch) {
        named_bar_sync(kBarReady, 160);
        const Stage& z = st[ch & 1];
        const bool force = (ch & 15) == 0;

        uint32_t sh[kM][2], sl[kM][2];
        gdn_col_exp(s, es, force);
        gdn_operand(s, es, sh, sl);
        const float su[2] = {gdn_exp2i(es[0]), gdn_exp2i(es[1])};
        if (ch > 0) named_bar_sync(kBarTaken + pair, 64);
        gdn_hand(hand.s, sh, sl, lane);
        hand.s_up[lane] = make_float2(su[0], su[1]);
        float x[4][4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {  // two row tiles at a time: four independent chains of products
            float kh[2][4] = {}, kl[2][4] = {};
#pragma unroll
            for (int ks = 0; ks < kM; ++ks)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t fk[4];
                    ldmatrix_x4(fk, z.kq.k[0] + ((i + j) * 16 + arow) * kLd + ks * 16 + acol);
                    mma_f16(kh[j], fk, sh[ks][0], sh[ks][1]);
                    mma_f16(kl[j], fk, sl[ks][0], sl[ks][1]);
                    if constexpr (kSplit) {
                        ldmatrix_x4(fk, z.kq.k[kSplit] + ((i + j) * 16 + arow) * kLd + ks * 16 + acol);
                        mma_f16(kl[j], fk, sh[ks][0], sh[ks][1]);
                    }
                }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int r = 16 * (i + j) + g + (c >> 1) * 8;
                    const float v = (float)z.v[r * kVLd + pair * 8 + 2 * t4 + (c & 1)];
                    x[i + j][c] = v - z.d.a[r] * su[c & 1] * fmaf(kl[j][c], 1.f / kGdnLo, kh[j][c]);
                }
        }
        // d = T X
        uint32_t xh[4][2], xl[4][2];
        int first_bad[2] = {64, 64};
        gdn_clean_exp(x, ex, force, first_bad, g);
        gdn_operand(x, ex, xh, xl);
        const float xu[2] = {gdn_exp2i(ex[0]) * z.d.t_up, gdn_exp2i(ex[1]) * z.d.t_up};
        float d[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float dh[4] = {}, dl[4] = {}, dm[4] = {};
#pragma unroll
            for (int j = 0; j <= i; ++j) {
                const uint4 th = z.d.t_hi[i * (i + 1) / 2 + j][lane], tl = z.d.t_lo[i * (i + 1) / 2 + j][lane];
                mma_f16(dh, th, xh[j][0], xh[j][1]);
                mma_f16(dl, th, xl[j][0], xl[j][1]);
                mma_f16(dm, tl, xh[j][0], xh[j][1]);
            }
#pragma unroll
            for (int c = 0; c < 4; ++c) d[i][c] = xu[c & 1] * fmaf(dl[c] + dm[c], 1.f / kGdnLo, dh[c]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) hand.d[i][lane] = make_float4(d[i][0], d[i][1], d[i][2], d[i][3]);
        const bool bad = min(first_bad[0], first_bad[1]) < 64;
        if (bad || was_bad) hand.first_bad[lane] = make_int2(first_bad[0], first_bad[1]);
        was_bad = bad;
        named_bar_arrive(kBarHand + pair, 64);
        // S <- e^G S + K^T (c d)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int c = 0; c < 4; ++c) d[i][c] *= z.d.c[16 * i + g + (c >> 1) * 8];
        uint32_t dh[4][2], dl[4][2];
        gdn_col_exp(d, ec, force);
        gdn_operand(d, ec, dh, dl);
        const float cu[2] = {gdn_exp2i(ec[0]), gdn_exp2i(ec[1])};
        float decay[2] = {z.d.decay, z.d.decay};
        if (bad) {
            if (first_bad[0] < 64) decay[0] = __int_as_float(0x7FC00000);
            if (first_bad[1] < 64) decay[1] = __int_as_float(0x7FC00000);
        }
        const int krow = (lane & 7) + ((lane >> 4) << 3), kcol = ((lane >> 3) & 1) * 8;
#pragma unroll
        for (int i = 0; i < kM; i += 2) {
            float nh[2][4] = {}, nl[2][4] = {};
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    uint32_t fk[4];
                    ldmatrix_x4_t(fk, z.kq.k[0] + (j * 16 + krow) * kLd + (i + e) * 16 + kcol);
                    mma_f16(nh[e], fk, dh[j][0], dh[j][1]);
                    mma_f16(nl[e], fk, dl[j][0], dl[j][1]);
                    if constexpr (kSplit) {
                        ldmatrix_x4_t(fk, z.kq.k[kSplit] + (j * 16 + krow) * kLd + (i + e) * 16 + kcol);
                        mma_f16(nl[e], fk, dh[j][0], dh[j][1]);
                    }
                }
#pragma unroll
            for (int e = 0; e < 2; ++e)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    s[i + e][c] = fmaf(decay[c & 1], s[i + e][c], cu[c & 1] * fmaf(nl[e][c], 1.f / kGdnLo, nh[e][c]));
        }
    }
    float* const sout = a.state_out + ((int64_t)h * HD + col) * HD;
#pragma unroll
    for (int i = 0; i < kM; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) sout[(c & 1) * HD + 16 * i + g + (c >> 1) * 8] = s[i][c];
}

// Tokens per segment: what the prep kernel writes for a segment is still in L2 when the scan reads it.
constexpr int64_t kGdnSegBytes = int64_t(96) << 20;
static int64_t gdn_chunk_bytes(bool f32, int k_heads, int v_heads, int head_dim) {
    const int64_t row = 2 * 64 * (head_dim + 8) * (int64_t)sizeof(__half);  // of a GdnKq, K and Q
    return v_heads * (int64_t)sizeof(GdnChunkData) + k_heads * (f32 ? 2 * row : row);
}
static int64_t gdn_most_chunks(bool f32, int64_t T, int k_heads, int v_heads, int head_dim) {
    const int64_t n = kGdnSegBytes / gdn_chunk_bytes(f32, k_heads, v_heads, head_dim), all = (T + kGdnChunk - 1) / kGdnChunk;
    return n < 1 ? 1 : (all < n ? all : n);
}
// Chunks per segment, at most that many: segments of one size, as a short last one costs as much as a long one's start.
static int64_t gdn_seg_chunks(bool f32, int64_t T, int k_heads, int v_heads, int head_dim) {
    const int64_t most = gdn_most_chunks(f32, T, k_heads, v_heads, head_dim), all = (T + kGdnChunk - 1) / kGdnChunk;
    const int64_t segs = (all + most - 1) / most;
    return (all + segs - 1) / segs;
}
// Calls of at least this many tokens take the chunked form. Chunked / token by token, us per call: fp16 16/32 heads of
// 128, 64 tokens 22 / 21, 96 26 / 30, 256 34 / 78; fp32 16/48 heads 64 tokens 38 / 32, 96 45 / 47; fp32 2/6 heads of
// 64, 96 tokens 28 / 23, 128 28 / 31 (one rule for all: the smallest models lose up to 5 us there).
constexpr int64_t kGdnChunkedFrom = 96;

template <typename T, int HD>
static int launch_gdn_chunked(const GdnDeltaArgs& a, uint8_t* ws, cudaStream_t stream) {
    constexpr bool kSplit = sizeof(T) == 4;
    const int64_t seg = gdn_seg_chunks(kSplit, a.T, a.k_heads, a.v_heads, HD);
    const auto prep = gdn_chunk_prep_kernel<T, HD>;
    const auto scan = gdn_chunk_scan_kernel<T, HD>;
    const int prep_smem = (int)sizeof(GdnPrepSmem<T, HD>), scan_smem = (int)sizeof(GdnScanSmem<T, HD>);
    int rc = ensure_smem((const void*)prep, prep_smem);
    if (rc == WZYB_OK) rc = ensure_smem((const void*)scan, scan_smem);
    if (rc != WZYB_OK) return rc;
    GdnPrepArgs pa;
    GdnScanArgs sa;
    pa.x = sa.x = a;
    pa.data = ws;
    pa.kq = ws + seg * a.v_heads * (int64_t)sizeof(GdnChunkData);
    sa.data = pa.data;
    sa.kq = pa.kq;
    sa.state_in = a.state_in;
    for (int64_t t0 = 0; t0 < a.T; t0 += seg * kGdnChunk) {
        const int64_t t1 = t0 + seg * kGdnChunk < a.T ? t0 + seg * kGdnChunk : a.T;
        pa.t0 = sa.t0 = t0;
        sa.t1 = t1;
        const int64_t chunks = (t1 - t0 + kGdnChunk - 1) / kGdnChunk;
        launch_k(prep, (unsigned)(chunks * a.k_heads), 128, prep_smem, stream, pa);
        launch_k(scan, a.v_heads * (HD / 32), 288, scan_smem, stream, sa);
        sa.state_in = a.state_out;
    }
    return launch_status();
}

template <typename T>
static int gdn_delta_entry(const wzyb_gdn_delta_args* p, int64_t T_, cudaStream_t stream) {
    if (p == nullptr) return WZYB_ERR_NULL;
    const wzyb_gdn_delta_args& x = *p;
    if (!x.state_out || (T_ != 0 && (!x.q || !x.k || !x.v || !x.g || !x.beta || !x.o))) return WZYB_ERR_NULL;
    if (T_ < 0 || T_ > (int64_t(1) << 31) || (x.head_dim != 64 && x.head_dim != 128) || x.k_heads < 1 ||
        x.v_heads < 1 || x.v_heads > 1024 || x.v_heads % x.k_heads != 0)
        return WZYB_ERR_SHAPE;
    const int64_t kw = (int64_t)x.k_heads * x.head_dim, vw = (int64_t)x.v_heads * x.head_dim;
    if (T_ > 1 && (x.q_row_stride < kw || x.k_row_stride < kw || x.v_row_stride < vw || x.o_row_stride < vw))
        return WZYB_ERR_SHAPE;
    constexpr int64_t kB = sizeof(T);
    if (!aligned16(x.q) || !aligned16(x.k) || !aligned16(x.v) || !aligned16(x.o) || !aligned16(x.state_in) ||
        !aligned16(x.state_out) || !aligned16(x.state_snaps) ||
        (T_ > 1 && ((x.q_row_stride | x.k_row_stride | x.v_row_stride | x.o_row_stride) * kB) % 16 != 0))
        return WZYB_ERR_ALIGN;
    if ((((uintptr_t)x.g | (uintptr_t)x.beta) & 3) != 0) return WZYB_ERR_ALIGN;
    if (T_ == 0 && x.state_in == x.state_out) return WZYB_OK;
    DeviceInfo di;
    const int rc = device_info(&di);
    if (rc != WZYB_OK) return rc;
    GdnDeltaArgs a;
    a.q = x.q;
    a.k = x.k;
    a.v = x.v;
    a.q_row = x.q_row_stride;
    a.k_row = x.k_row_stride;
    a.v_row = x.v_row_stride;
    a.o_row = x.o_row_stride;
    a.g = x.g;
    a.beta = x.beta;
    a.state_in = x.state_in;
    a.state_out = x.state_out;
    a.snaps = x.state_snaps;
    a.o = x.o;
    a.T = T_;
    a.k_heads = x.k_heads;
    a.v_heads = x.v_heads;
    a.scale = x.scale;
    a.l2norm = x.qk_l2norm;
    a.l2_eps = x.l2_eps;
    if (T_ >= kGdnChunkedFrom && x.state_snaps == nullptr) {
        if (!x.workspace) return WZYB_ERR_NULL;
        if (!aligned16(x.workspace)) return WZYB_ERR_ALIGN;
        if (x.workspace_bytes < wzyb_gdn_delta_rule_workspace(T_, x.k_heads, x.v_heads, x.head_dim)) return WZYB_ERR_SHAPE;
        uint8_t* const ws = static_cast<uint8_t*>(x.workspace);
        return x.head_dim == 64 ? launch_gdn_chunked<T, 64>(a, ws, stream) : launch_gdn_chunked<T, 128>(a, ws, stream);
    }
    const int grid = x.v_heads * (x.head_dim / 32);
    if (x.head_dim == 64)
        launch_k(gdn_recurrent_kernel<T, 64>, grid, 256, 0, stream, a);
    else
        launch_k(gdn_recurrent_kernel<T, 128>, grid, 256, 0, stream, a);
    return launch_status();
}

}  // namespace wzyb

extern "C" {

int64_t wzyb_gdn_delta_rule_workspace(int64_t T, int k_heads, int v_heads, int head_dim) {
    if (T < wzyb::kGdnChunkedFrom || k_heads < 1 || v_heads < 1 || head_dim < 1) return 0;
    int64_t most = 0;
    for (int f32 = 0; f32 < 2; ++f32) {
        const int64_t bytes = wzyb::gdn_most_chunks(f32 != 0, T, k_heads, v_heads, head_dim) *
                              wzyb::gdn_chunk_bytes(f32 != 0, k_heads, v_heads, head_dim);
        most = bytes > most ? bytes : most;
    }
    return most;
}
int wzyb_gdn_delta_rule_f16(const wzyb_gdn_delta_args* a, int64_t T, wzyb_stream_t stream) {
    return wzyb::gdn_delta_entry<__half>(a, T, (cudaStream_t)stream);
}
int wzyb_gdn_delta_rule_f32(const wzyb_gdn_delta_args* a, int64_t T, wzyb_stream_t stream) {
    return wzyb::gdn_delta_entry<float>(a, T, (cudaStream_t)stream);
}

}  // extern "C"
