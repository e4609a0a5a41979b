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
    (void)T, (void)k_heads, (void)v_heads, (void)head_dim;
    return 0;
}
int wzyb_gdn_delta_rule_f16(const wzyb_gdn_delta_args* a, int64_t T, wzyb_stream_t stream) {
    return wzyb::gdn_delta_entry<__half>(a, T, (cudaStream_t)stream);
}
int wzyb_gdn_delta_rule_f32(const wzyb_gdn_delta_args* a, int64_t T, wzyb_stream_t stream) {
    return wzyb::gdn_delta_entry<float>(a, T, (cudaStream_t)stream);
}

}  // extern "C"
