// Gated linear recurrence along tokens, forward and backward (include/mv2.h mv2_gateloop_forward / mv2_gateloop_backward):
//     h_t = g_t h_{t-1} + kv_t,   g_t = sigmoid(a_t) (0 where a document starts),   y_t = q_t h_t
// and, with D_t the gradient that arrives at h_t,
//     D_t = q_t dy_t + g_{t+1} D_{t+1} (+ dh_last at the last token),  dq = h dy,  dkv = D,  da = D h_{t-1} g (1 - g),  dh0 = g_0 D_0.
// Everything between the loads and the stores is fp32; only y, dq, dkv, da are rounded to the storage type.
#include <algorithm>
#include <initializer_list>
#include "rowvec.h"

// sigmoid(a) and its slope g (1 - g) = e / (1 + e)^2 with e = exp(-|a|): no cancellation for either sign, no overflow, NaN stays NaN.
// bf16 storage: hardware exp / rcp (1 ulp each, far below the stores' 2^-9); fp32: the library's exp and an exact division.
template <typename E> struct Gate;
template <> struct Gate<BF16> {
    static __device__ __forceinline__ float recip(float v) { return __builtin_amdgcn_rcpf(v); }
    static __device__ __forceinline__ float ex(float v) { return __expf(v); }
};
template <> struct Gate<F32> {
    static __device__ __forceinline__ float recip(float v) { return 1.f / v; }
    static __device__ __forceinline__ float ex(float v) { return expf(v); }
};
template <typename E> __device__ __forceinline__ float sigm(float a) { return Gate<E>::recip(1.f + Gate<E>::ex(-a)); }
template <typename E> __device__ __forceinline__ void sigm_slope(float a, float& g, float& slope) {
    const float e = Gate<E>::ex(-fabsf(a)), r = Gate<E>::recip(1.f + e), er = e * r;
    g = a < 0.f ? er : r;
    slope = er * r;
}

struct LoopArgs {
    int B, T, P, C;
    int64_t sb, st, sp;            // q, kv, a
    int64_t gb, gt, gp;            // dq, dkv, da
    const int32_t* lengths;
    const unsigned char* resets;
    int nstate;                    // kept states per sequence (mv2_gateloop_states)
};

#define LOOP_STEPS 8               // tokens between two kept states of the walking kernels

__device__ __forceinline__ int live_tokens(const LoopArgs& A, int b) {
    if (!A.lengths) return A.T;
    const int n = A.lengths[b];
    return n < 0 ? 0 : (n > A.T ? A.T : n);
}

// --------------------------------------------------------------------------- one thread per chunk of channels walks its tokens
template <typename E, int V>
__global__ __launch_bounds__(256) void loop_walk_fwd_kernel(LoopArgs A, const void* __restrict__ q, const void* __restrict__ kv, const void* __restrict__ a,
                                                            const float* h0, void* __restrict__ y, float* hlast, float* __restrict__ states) {
    const int cpr = A.C / V;
    const int64_t total = (int64_t)A.B * A.P * cpr;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t seq = i / cpr;
    const int c = (int)(i - seq * cpr) * V;
    const int b = (int)(seq / A.P), p = (int)(seq - (int64_t)b * A.P);
    const int n = live_tokens(A, b);
    const int64_t in0 = b * A.sb + p * A.sp + c;
    const int64_t yt = (int64_t)A.P * A.C, y0 = (int64_t)b * A.T * yt + (int64_t)p * A.C + c;
    const unsigned char* rs = A.resets ? A.resets + (int64_t)b * A.T : nullptr;
    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = h0 ? h0[seq * A.C + c + k] : 0.f;
    int t = 0;
    for (; t + LOOP_STEPS <= n; t += LOOP_STEPS) {
        RowVec<E, V> vq[LOOP_STEPS], vk[LOOP_STEPS], va[LOOP_STEPS];
#pragma unroll
        for (int s = 0; s < LOOP_STEPS; ++s) {
            const int64_t at = in0 + (t + s) * A.st;
            vk[s].load(kv, at); va[s].load(a, at); vq[s].load(q, at);
        }
        if (states && t > 0) {
            float* o = states + (((int64_t)b * A.nstate + t / LOOP_STEPS - 1) * A.P + p) * A.C + c;
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = h[k];
        }
#pragma unroll
        for (int s = 0; s < LOOP_STEPS; ++s) {
            float fq[V], fk[V], fa[V];
            vq[s].get(fq); vk[s].get(fk); va[s].get(fa);
            const bool cut = rs && rs[t + s];
#pragma unroll
            for (int k = 0; k < V; ++k) {
                h[k] = cut ? fk[k] : fmaf(sigm<E>(fa[k]), h[k], fk[k]);
                fq[k] *= h[k];
            }
            RowVec<E, V>::store(y, y0 + (t + s) * yt, fq);
        }
    }
    if (states && t > 0 && t < n) {
        float* o = states + (((int64_t)b * A.nstate + t / LOOP_STEPS - 1) * A.P + p) * A.C + c;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = h[k];
    }
    for (; t < n; ++t) {
        RowVec<E, V> vq, vk, va;
        const int64_t at = in0 + t * A.st;
        vk.load(kv, at); va.load(a, at); vq.load(q, at);
        float fq[V], fk[V], fa[V];
        vq.get(fq); vk.get(fk); va.get(fa);
        const bool cut = rs && rs[t];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            h[k] = cut ? fk[k] : fmaf(sigm<E>(fa[k]), h[k], fk[k]);
            fq[k] *= h[k];
        }
        RowVec<E, V>::store(y, y0 + t * yt, fq);
    }
    float zero[V];
#pragma unroll
    for (int k = 0; k < V; ++k) zero[k] = 0.f;
    for (; t < A.T; ++t) RowVec<E, V>::store(y, y0 + t * yt, zero);
    if (hlast) {
#pragma unroll
        for (int k = 0; k < V; ++k) hlast[seq * A.C + c + k] = h[k];
    }
}

template <typename E, int V>
__global__ __launch_bounds__(256) void loop_walk_bwd_kernel(LoopArgs A, const void* __restrict__ q, const void* __restrict__ kv, const void* __restrict__ a,
                                                            const float* __restrict__ h0, const float* __restrict__ states, const void* __restrict__ dy,
                                                            const float* __restrict__ dhlast, void* __restrict__ dq, void* __restrict__ dkv,
                                                            void* __restrict__ da, float* __restrict__ dh0) {
    const int cpr = A.C / V;
    const int64_t total = (int64_t)A.B * A.P * cpr;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int64_t seq = i / cpr;
    const int c = (int)(i - seq * cpr) * V;
    const int b = (int)(seq / A.P), p = (int)(seq - (int64_t)b * A.P);
    const int n = live_tokens(A, b);
    const int64_t in0 = b * A.sb + p * A.sp + c, g0 = b * A.gb + p * A.gp + c;
    const int64_t yt = (int64_t)A.P * A.C, y0 = (int64_t)b * A.T * yt + (int64_t)p * A.C + c;
    const unsigned char* rs = A.resets ? A.resets + (int64_t)b * A.T : nullptr;
    float back[V], zero[V];                         // what h_{t+1} passes back to h_t
#pragma unroll
    for (int k = 0; k < V; ++k) { back[k] = dhlast ? dhlast[seq * A.C + c + k] : 0.f; zero[k] = 0.f; }
    for (int t = n; t < A.T; ++t) {
        const int64_t at = g0 + t * A.gt;
        RowVec<E, V>::store(dq, at, zero); RowVec<E, V>::store(dkv, at, zero); RowVec<E, V>::store(da, at, zero);
    }
    for (int blk = (n + LOOP_STEPS - 1) / LOOP_STEPS - 1; blk >= 0; --blk) {
        const int t0 = blk * LOOP_STEPS;
        RowVec<E, V> vq[LOOP_STEPS], vk[LOOP_STEPS], va[LOOP_STEPS], vy[LOOP_STEPS];
#pragma unroll
        for (int s = 0; s < LOOP_STEPS; ++s)
            if (t0 + s < n) {
                const int64_t at = in0 + (t0 + s) * A.st;
                vk[s].load(kv, at); va[s].load(a, at); vq[s].load(q, at); vy[s].load(dy, y0 + (t0 + s) * yt);
            }
        float h[LOOP_STEPS + 1][V];                 // h[s] = state before token t0 + s
        const float* hin = blk > 0 ? states + (((int64_t)b * A.nstate + blk - 1) * A.P + p) * A.C + c : (h0 ? h0 + seq * A.C + c : nullptr);
#pragma unroll
        for (int k = 0; k < V; ++k) h[0][k] = hin ? hin[k] : 0.f;
#pragma unroll
        for (int s = 0; s < LOOP_STEPS; ++s)
            if (t0 + s < n) {
                float fk[V], fa[V];
                vk[s].get(fk); va[s].get(fa);
                const bool cut = rs && rs[t0 + s];
#pragma unroll
                for (int k = 0; k < V; ++k) h[s + 1][k] = cut ? fk[k] : fmaf(sigm<E>(fa[k]), h[s][k], fk[k]);
            }
#pragma unroll
        for (int s = LOOP_STEPS - 1; s >= 0; --s)
            if (t0 + s < n) {
                float fq[V], fa[V], fy[V], oq[V], oa[V], ok[V];
                vq[s].get(fq); va[s].get(fa); vy[s].get(fy);
                const bool cut = rs && rs[t0 + s];
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    float g, slope;
                    sigm_slope<E>(fa[k], g, slope);
                    const float d = fmaf(fq[k], fy[k], back[k]);
                    oq[k] = h[s + 1][k] * fy[k];
                    ok[k] = d;
                    oa[k] = cut ? 0.f : d * h[s][k] * slope;
                    back[k] = cut ? 0.f : g * d;
                }
                const int64_t at = g0 + (t0 + s) * A.gt;
                RowVec<E, V>::store(dq, at, oq); RowVec<E, V>::store(dkv, at, ok); RowVec<E, V>::store(da, at, oa);
            }
    }
    if (dh0) {
#pragma unroll
        for (int k = 0; k < V; ++k) dh0[seq * A.C + c + k] = back[k];
    }
}

// --------------------------------------------------------------------------- host side
// refuses what a launch could not address: sizes, strides that run backwards, products that leave 63 bits
static int loop_check(const mv2_gateloop_desc* d) {
    if (!d) return MV2_EINVAL;
    if (d->dtype != MV2_BF16 && d->dtype != MV2_F32) return MV2_EINVAL;
    if (d->B <= 0 || d->T < 0 || d->P <= 0 || d->C <= 0) return MV2_EINVAL;
    const int64_t lim = (int64_t)1 << 30;
    if (d->T > lim || d->P > lim || d->C > (1 << 24) || d->B > lim) return MV2_ETOOLARGE;
    const int64_t s[6] = {d->in_b, d->in_t, d->in_p, d->grad_b, d->grad_t, d->grad_p};
    for (int i = 0; i < 6; ++i) if (s[i] < 0) return MV2_EINVAL;
    const double far = (double)((int64_t)1 << 60);
    if ((double)d->B * d->T * d->P * d->C > far) return MV2_ETOOLARGE;
    if ((double)d->B * d->in_b + (double)d->T * d->in_t + (double)d->P * d->in_p > far) return MV2_ETOOLARGE;
    if ((double)d->B * d->grad_b + (double)d->T * d->grad_t + (double)d->P * d->grad_p > far) return MV2_ETOOLARGE;
    if (((double)d->B * d->P * d->C + 255) / 256 > 2147483647.0) return MV2_ETOOLARGE;
    return MV2_OK;
}

extern "C" int64_t mv2_gateloop_states(const mv2_gateloop_desc* d) {
    if (loop_check(d) != MV2_OK) return MV2_EINVAL;
    return d->T > 0 ? (d->T - 1) / LOOP_STEPS : 0;
}

extern "C" size_t mv2_gateloop_workspace_bytes(const mv2_gateloop_desc* d, int backward) {
    (void)d; (void)backward;
    return 0;
}

static LoopArgs loop_args(const mv2_gateloop_desc* d, const int32_t* lengths, const unsigned char* resets) {
    LoopArgs A;
    A.B = d->B; A.T = d->T; A.P = d->P; A.C = d->C;
    A.sb = d->in_b; A.st = d->in_t; A.sp = d->in_p; A.gb = d->grad_b; A.gt = d->grad_t; A.gp = d->grad_p;
    A.lengths = lengths; A.resets = resets;
    A.nstate = (int)mv2_gateloop_states(d);
    return A;
}

extern "C" int mv2_gateloop_forward(const mv2_gateloop_desc* d, const void* q, const void* kv, const void* a, const float* h0, const int32_t* lengths,
                                    const unsigned char* resets, void* y, float* h_last, float* states, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = loop_check(d);
    if (rc != MV2_OK) return rc;
    if (d->T > 0 && (!q || !kv || !a || !y)) return MV2_EINVAL;
    if (workspace_bytes < mv2_gateloop_workspace_bytes(d, 0)) return MV2_EWORKSPACE;
    const LoopArgs A = loop_args(d, lengths, resets);
    const int kvec = d->dtype == MV2_BF16 ? 8 : 4;
    const bool wide = d->C % kvec == 0 && d->in_b % kvec == 0 && d->in_t % kvec == 0 && d->in_p % kvec == 0 && rows_aligned16({q, kv, a, y});
    const int64_t n = (int64_t)d->B * d->P * (d->C / (wide ? kvec : 1));
    const dim3 grid((unsigned)((n + 255) / 256));
    hipStream_t st = (hipStream_t)stream;
#define GO(E, V) hipLaunchKernelGGL((loop_walk_fwd_kernel<E, V>), grid, dim3(256), 0, st, A, q, kv, a, h0, y, h_last, states)
    if (d->dtype == MV2_BF16) { if (wide) GO(BF16, 8); else GO(BF16, 1); }
    else { if (wide) GO(F32, 4); else GO(F32, 1); }
#undef GO
    MV2_LAUNCH_CHECK();
    return MV2_OK;
}

extern "C" int mv2_gateloop_backward(const mv2_gateloop_desc* d, const void* q, const void* kv, const void* a, const float* h0, const int32_t* lengths,
                                     const unsigned char* resets, const float* states, const void* dy, const float* dh_last, void* dq, void* dkv, void* da,
                                     float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = loop_check(d);
    if (rc != MV2_OK) return rc;
    if (d->T > 0 && (!q || !kv || !a || !dy || !dq || !dkv || !da)) return MV2_EINVAL;
    if (workspace_bytes < mv2_gateloop_workspace_bytes(d, 1)) return MV2_EWORKSPACE;
    const LoopArgs A = loop_args(d, lengths, resets);
    if (A.nstate > 0 && !states) return MV2_EINVAL;
    const int kvec = d->dtype == MV2_BF16 ? 8 : 4;
    const bool wide = d->C % kvec == 0 && d->in_b % kvec == 0 && d->in_t % kvec == 0 && d->in_p % kvec == 0 && d->grad_b % kvec == 0 &&
                      d->grad_t % kvec == 0 && d->grad_p % kvec == 0 && rows_aligned16({q, kv, a, dy, dq, dkv, da});
    const int64_t n = (int64_t)d->B * d->P * (d->C / (wide ? kvec : 1));
    const dim3 grid((unsigned)((n + 255) / 256));
    hipStream_t st = (hipStream_t)stream;
#define GO(E, V) hipLaunchKernelGGL((loop_walk_bwd_kernel<E, V>), grid, dim3(256), 0, st, A, q, kv, a, h0, states, dy, dh_last, dq, dkv, da, dh0)
    if (d->dtype == MV2_BF16) { if (wide) GO(BF16, 8); else GO(BF16, 1); }
    else { if (wide) GO(F32, 4); else GO(F32, 1); }
#undef GO
    MV2_LAUNCH_CHECK();
    return MV2_OK;
}
