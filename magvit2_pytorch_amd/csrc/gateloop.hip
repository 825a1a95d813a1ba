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
#define SPAN_KEEP 128              // and of the spans

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

// --------------------------------------------------------------------------- spans of tokens joined along the sequence
// The walking kernels above leave the chip empty where there are few channels and many tokens.  Here a workgroup of WAVES waves owns
// WAVES * 32 tokens of CL * V channels of one sequence (a "block"): a lane holds L consecutive tokens of V channels in registers (every
// element is read once), CL lanes side by side read whole 128-byte pieces of rows, and the 64 / CL lane rows of a wave, the waves, and the
// blocks of a sequence are joined through the pair (A, H) of a span: it takes the state h in front of it to A h + H, and spans join as
// (A1, H1) (A2, H2) -> (A1 A2, A2 H1 + H2).
// Between workgroups: a block publishes its pair and reads the pairs of the blocks before it in its group of LOOP_GROUP blocks, and the
// state that the last block of the group before published: always the same pairs in the same order, so results do not depend on timing.
// Every wait ends: a block's place in the order is the ticket it draws when it starts, blocks wait for lower tickets only - for workgroups
// that are running - and a pair is published before its block waits for anything.
#define LOOP_GROUP 32
#define LOOP_CUT 2.f               // A of a span in which a document starts (products of decays are <= 1 or NaN): nothing passes through it
typedef unsigned long long u64;

// a pair in one 8-byte word, written and read whole; the sign of A is the mark that it is there (the words are zero before the launch)
__device__ __forceinline__ u64 pair_word(float A, float H) { return ((u64)(__float_as_uint(A) | 0x80000000u) << 32) | __float_as_uint(H); }
__device__ __forceinline__ bool pair_there(u64 w) { return (w >> 63) != 0; }
__device__ __forceinline__ float pair_A(u64 w) { return __uint_as_float((unsigned)(w >> 32) & 0x7fffffffu); }
__device__ __forceinline__ float pair_H(u64 w) { return __uint_as_float((unsigned)w); }
__device__ __forceinline__ void publish(u64* p, float A, float H) { __hip_atomic_store(p, pair_word(A, H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// (A, H) := (A, H) then (A2, H2)
__device__ __forceinline__ void join(float& A, float& H, float A2, float H2) {
    const bool cut2 = A2 == LOOP_CUT;
    H = cut2 ? H2 : fmaf(A2, H, H2);
    A = (cut2 || A == LOOP_CUT) ? LOOP_CUT : A * A2;
}

struct SpanWork {
    unsigned* ticket;
    u64* pairs;                    // [block][tile][channel of the tile]
    u64* states;                   // [group][tile][channel of the tile]: the state behind a whole group
    int nblk, ntile, ctiles;
};

// What a workgroup's channels receive from the blocks before this one (in the direction of the recurrence): block `kb` counts in that
// direction, `first` is what block 0 starts from.  Entered by all threads with (A, H) of the whole block in totA / totH (LDS, published here);
// on return carry[ch] holds the state in front of the block.
template <int NCH, int THREADS>
__device__ __forceinline__ void span_carry(const SpanWork& W, int kb, int tile, bool ok, float first, const float* totA, const float* totH, float* carry,
                                           float (*partA)[NCH], float (*partH)[NCH]) {
    constexpr int SLOTS = THREADS / NCH, M = LOOP_GROUP / SLOTS;
    static_assert(SLOTS * M == LOOP_GROUP, "slots share a group evenly");
    const int tid = threadIdx.x, ch = tid % NCH, slot = tid / NCH;
    if (W.nblk == 1) {
        if (tid < NCH) carry[ch] = first;
        __syncthreads();
        return;
    }
    u64* mine = W.pairs + ((int64_t)kb * W.ntile + tile) * NCH;
    if (tid < NCH && ok) {
        // block 0 publishes a state rather than a pair: whoever depends on it does not read `first` again, which may be overwritten by then
        if (kb == 0) publish(mine + ch, LOOP_CUT, totA[ch] == LOOP_CUT ? totH[ch] : fmaf(totA[ch], first, totH[ch]));
        else publish(mine + ch, totA[ch], totH[ch]);
    }
    const int grp = kb / LOOP_GROUP, in = kb % LOOP_GROUP;
    const int lead = grp > 0 ? 1 : 0, count = lead + in;      // the group before, then the blocks of this group
    float A = 1.f, H = 0.f;
    if (ok && kb > 0) {
        u64 w[M];
#pragma unroll
        for (int j = 0; j < M; ++j) w[j] = 0;
        bool all;
        do {
            all = true;
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const int e = slot * M + j;
                if (e < count && !pair_there(w[j])) {
                    const u64* p = e < lead ? W.states + ((int64_t)(grp - 1) * W.ntile + tile) * NCH
                                            : W.pairs + ((int64_t)(grp * LOOP_GROUP + e - lead) * W.ntile + tile) * NCH;
                    w[j] = __hip_atomic_load(p + ch, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    all = all && pair_there(w[j]);
                }
            }
            if (!all) __builtin_amdgcn_s_sleep(1);
        } while (!all);
#pragma unroll
        for (int j = 0; j < M; ++j)
            if (slot * M + j < count) join(A, H, pair_A(w[j]), pair_H(w[j]));
    }
    partA[slot][ch] = A; partH[slot][ch] = H;
    __syncthreads();
    if (tid < NCH) {
        float h = first;
        if (kb > 0) {
            A = 1.f; H = 0.f;
#pragma unroll
            for (int s = 0; s < SLOTS; ++s) join(A, H, partA[s][ch], partH[s][ch]);
            h = H;                                            // the first entry is a state: nothing in front of it counts
        }
        carry[ch] = h;
        if (ok && in == LOOP_GROUP - 1 && kb + 1 < W.nblk)
            publish(W.states + ((int64_t)grp * W.ntile + tile) * NCH + ch, LOOP_CUT, totA[ch] == LOOP_CUT ? totH[ch] : fmaf(totA[ch], h, totH[ch]));
    }
    __syncthreads();
}

// pairs of the waves -> what is in front of each wave; totals of the block.  In the direction of the recurrence (REV: last wave first).
template <int NCH, int WAVES, bool REV>
__device__ __forceinline__ void wave_prefix(float (*sA)[NCH], float (*sH)[NCH], float* totA, float* totH) {
    const int ch = threadIdx.x;
    if (ch < NCH) {
        float A = 1.f, H = 0.f;
#pragma unroll
        for (int i = 0; i < WAVES; ++i) {
            const int w = REV ? WAVES - 1 - i : i;
            const float a2 = sA[w][ch], h2 = sH[w][ch];
            sA[w][ch] = A; sH[w][ch] = H;
            join(A, H, a2, h2);
        }
        totA[ch] = A; totH[ch] = H;
    }
}

// joins the lane rows of a wave: on entry a lane's own pair, on return the pair in front of the lane; the wave's whole pair goes to LDS
template <int V, int CL, bool REV>
__device__ __forceinline__ void lane_prefix(float* A, float* H, float* waveA, float* waveH) {
    constexpr int TL = 64 / CL;
    const int lane = threadIdx.x & 63, r = REV ? TL - 1 - lane / CL : lane / CL, cl = lane % CL;
#pragma unroll
    for (int d = 1; d < TL; d *= 2) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float a0 = REV ? __shfl_down(A[k], d * CL, 64) : __shfl_up(A[k], d * CL, 64);
            float h0 = REV ? __shfl_down(H[k], d * CL, 64) : __shfl_up(H[k], d * CL, 64);
            if (r >= d) { join(a0, h0, A[k], H[k]); A[k] = a0; H[k] = h0; }
        }
    }
    if (r == TL - 1)
#pragma unroll
        for (int k = 0; k < V; ++k) { waveA[cl * V + k] = A[k]; waveH[cl * V + k] = H[k]; }
    if (TL > 1) {
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float a0 = REV ? __shfl_down(A[k], CL, 64) : __shfl_up(A[k], CL, 64);
            const float h0 = REV ? __shfl_down(H[k], CL, 64) : __shfl_up(H[k], CL, 64);
            A[k] = r == 0 ? 1.f : a0; H[k] = r == 0 ? 0.f : h0;
        }
    } else {
#pragma unroll
        for (int k = 0; k < V; ++k) { A[k] = 1.f; H[k] = 0.f; }
    }
}

// (block in the direction of the recurrence, tile) of this workgroup
__device__ __forceinline__ void span_place(const SpanWork& W, int& kb, int& tile) {
    __shared__ unsigned drawn;
    if (W.nblk == 1) { kb = 0; tile = blockIdx.x; return; }
    if (threadIdx.x == 0) drawn = __hip_atomic_fetch_add(W.ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    kb = (int)(drawn / (unsigned)W.ntile); tile = (int)(drawn % (unsigned)W.ntile);
}

__global__ __launch_bounds__(256) void span_clear_kernel(u64* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

template <typename E, int V, int CL, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void loop_span_fwd_kernel(LoopArgs A, SpanWork W, const void* __restrict__ q, const void* __restrict__ kv,
                                                                   const void* __restrict__ a, const float* h0, void* __restrict__ y, float* hlast,
                                                                   float* __restrict__ states) {
    constexpr int TL = 64 / CL, L = 32 / TL, NCH = CL * V, SPAN = WAVES * 32;
    __shared__ float sA[WAVES][NCH], sH[WAVES][NCH], totA[NCH], totH[NCH], carry[NCH], partA[WAVES * 64 / NCH][NCH], partH[WAVES * 64 / NCH][NCH];
    int kb, tile;
    span_place(W, kb, tile);
    const int ct = tile % W.ctiles, seq = tile / W.ctiles, b = seq / A.P, p = seq % A.P;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, cl = lane % CL;
    const int n = live_tokens(A, b), t0 = kb * SPAN + wave * 32 + (lane / CL) * L;
    const int c = ct * NCH + cl * V;
    const bool cok = c < A.C;
    const int cc = cok ? c : 0;
    const unsigned char* rs = A.resets ? A.resets + (int64_t)b * A.T : nullptr;

    RowVec<E, V> vq[L], vk[L];
    float g[L][V];
    unsigned cuts = 0;
    {
        RowVec<E, V> va[L];
        const int64_t in0 = (int64_t)b * A.sb + (int64_t)p * A.sp + cc;
        if (kb * SPAN < n) {
#pragma unroll
            for (int i = 0; i < L; ++i) {                     // rows behind the last token are not read: the last one stands in for them
                const int64_t at = in0 + (int64_t)min(t0 + i, n - 1) * A.st;
                va[i].load(a, at); vk[i].load(kv, at); vq[i].load(q, at);
            }
            if (rs)
#pragma unroll
                for (int i = 0; i < L; ++i) cuts |= (t0 + i < n && rs[min(t0 + i, n - 1)]) ? 1u << i : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i) { va[i].clear(); vk[i].clear(); vq[i].clear(); }
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            float fa[V];
            va[i].get(fa);
#pragma unroll
            for (int k = 0; k < V; ++k) g[i][k] = t0 + i < n ? sigm<E>(fa[k]) : 1.f;
        }
    }
    float pa[V], ph[V];
#pragma unroll
    for (int k = 0; k < V; ++k) { pa[k] = 1.f; ph[k] = 0.f; }
#pragma unroll
    for (int i = 0; i < L; ++i) {
        float fk[V];
        vk[i].get(fk);
        const bool cut = cuts >> i & 1, on = t0 + i < n;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float x = on ? fk[k] : 0.f;
            ph[k] = cut ? x : fmaf(g[i][k], ph[k], x);
            pa[k] *= g[i][k];
        }
    }
    if (cuts)
#pragma unroll
        for (int k = 0; k < V; ++k) pa[k] = LOOP_CUT;
    lane_prefix<V, CL, false>(pa, ph, sA[wave], sH[wave]);
    __syncthreads();
    wave_prefix<NCH, WAVES, false>(sA, sH, totA, totH);
    __syncthreads();
    const int chn = threadIdx.x % NCH;
    const bool chok = ct * NCH + chn < A.C;
    float first = 0.f;
    if (kb == 0 && h0 && chok && threadIdx.x < NCH) first = h0[(int64_t)seq * A.C + ct * NCH + chn];
    span_carry<NCH, WAVES * 64>(W, kb, tile, chok, first, totA, totH, carry, partA, partH);

    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int ch = cl * V + k;
        float wa = sA[wave][ch], wh = sH[wave][ch];
        join(wa, wh, pa[k], ph[k]);
        h[k] = wa == LOOP_CUT ? wh : fmaf(wa, carry[ch], wh);
    }
    if (states && cok && t0 > 0 && t0 < n && t0 % SPAN_KEEP == 0) {
        float* o = states + (((int64_t)b * A.nstate + t0 / SPAN_KEEP - 1) * A.P + p) * A.C + c;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = h[k];
    }
    const int64_t yt = (int64_t)A.P * A.C, y0 = ((int64_t)b * A.T * A.P + p) * A.C + c;
#pragma unroll
    for (int i = 0; i < L; ++i) {
        float fk[V], fq[V];
        vk[i].get(fk); vq[i].get(fq);
        const bool cut = cuts >> i & 1, on = t0 + i < n;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float x = on ? fk[k] : 0.f;
            h[k] = cut ? x : fmaf(g[i][k], h[k], x);
            fq[k] = on ? fq[k] * h[k] : 0.f;
        }
        if (cok && t0 + i < A.T) RowVec<E, V>::store(y, y0 + (t0 + i) * yt, fq);
    }
    if (hlast && cok && kb == W.nblk - 1 && wave == WAVES - 1 && lane / CL == TL - 1) {
#pragma unroll
        for (int k = 0; k < V; ++k) hlast[(int64_t)seq * A.C + c + k] = h[k];
    }
}

// The same from the last token to the first for D; the states in front of a block's tokens are formed again from the kept state
template <typename E, int V, int CL, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void loop_span_bwd_kernel(LoopArgs A, SpanWork W, const void* __restrict__ q, const void* __restrict__ kv,
                                                                   const void* __restrict__ a, const float* __restrict__ h0, const float* __restrict__ states,
                                                                   const void* __restrict__ dy, const float* __restrict__ dhlast, void* __restrict__ dq,
                                                                   void* __restrict__ dkv, void* __restrict__ da, float* __restrict__ dh0) {
    constexpr int TL = 64 / CL, L = 32 / TL, NCH = CL * V, SPAN = WAVES * 32;
    static_assert(SPAN == SPAN_KEEP, "a block begins at a kept state");
    __shared__ float sA[WAVES][NCH], sH[WAVES][NCH], bA[WAVES][NCH], bH[WAVES][NCH], totA[NCH], totH[NCH], carry[NCH];
    __shared__ float partA[WAVES * 64 / NCH][NCH], partH[WAVES * 64 / NCH][NCH];
    int back_kb, tile;
    span_place(W, back_kb, tile);
    const int kb = W.nblk - 1 - back_kb;
    const int ct = tile % W.ctiles, seq = tile / W.ctiles, b = seq / A.P, p = seq % A.P;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, cl = lane % CL;
    const int n = live_tokens(A, b), t0 = kb * SPAN + wave * 32 + (lane / CL) * L;
    const int c = ct * NCH + cl * V;
    const bool cok = c < A.C;
    const int cc = cok ? c : 0;
    const unsigned char* rs = A.resets ? A.resets + (int64_t)b * A.T : nullptr;
    const int64_t yt = (int64_t)A.P * A.C, y0 = ((int64_t)b * A.T * A.P + p) * A.C + cc;

    RowVec<E, V> vq[L], vk[L], va[L], vy[L];
    float hin[V];                                             // the block's kept state
    unsigned cuts = 0;
#pragma unroll
    for (int k = 0; k < V; ++k) hin[k] = 0.f;
    if (kb * SPAN < n) {
        const int64_t in0 = (int64_t)b * A.sb + (int64_t)p * A.sp + cc;
#pragma unroll
        for (int i = 0; i < L; ++i) {
            const int t = min(t0 + i, n - 1);
            const int64_t at = in0 + (int64_t)t * A.st;
            va[i].load(a, at); vk[i].load(kv, at); vq[i].load(q, at); vy[i].load(dy, y0 + t * yt);
        }
        if (rs)
#pragma unroll
            for (int i = 0; i < L; ++i) cuts |= (t0 + i < n && rs[min(t0 + i, n - 1)]) ? 1u << i : 0u;
        const float* hp = kb > 0 ? states + (((int64_t)b * A.nstate + kb - 1) * A.P + p) * A.C + cc : (h0 ? h0 + (int64_t)seq * A.C + cc : nullptr);
        if (hp)
#pragma unroll
            for (int k = 0; k < V; ++k) hin[k] = hp[k];
    } else {
#pragma unroll
        for (int i = 0; i < L; ++i) { va[i].clear(); vk[i].clear(); vq[i].clear(); vy[i].clear(); }
    }
    float g[L][V];
#pragma unroll
    for (int i = 0; i < L; ++i) {
        float fa[V];
        va[i].get(fa);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float slope;
            sigm_slope<E>(fa[k], g[i][k], slope);
            if (t0 + i >= n) g[i][k] = 1.f;
        }
    }
    float pa[V], ph[V], ba[V], bh[V];
#pragma unroll
    for (int k = 0; k < V; ++k) { pa[k] = ba[k] = 1.f; ph[k] = bh[k] = 0.f; }
#pragma unroll
    for (int i = 0; i < L; ++i) {
        float fk[V];
        vk[i].get(fk);
        const bool cut = cuts >> i & 1, on = t0 + i < n;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float x = on ? fk[k] : 0.f;
            ph[k] = cut ? x : fmaf(g[i][k], ph[k], x);
            pa[k] *= g[i][k];
        }
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
        float fq[V], fy[V];
        vq[i].get(fq); vy[i].get(fy);
        const bool cut = cuts >> i & 1, on = t0 + i < n;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float d = on ? fmaf(fq[k], fy[k], bh[k]) : bh[k];
            bh[k] = cut ? 0.f : g[i][k] * d;
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) { if (cuts) pa[k] = LOOP_CUT; ba[k] = pa[k]; }
    lane_prefix<V, CL, false>(pa, ph, sA[wave], sH[wave]);
    lane_prefix<V, CL, true>(ba, bh, bA[wave], bH[wave]);
    __syncthreads();
    wave_prefix<NCH, WAVES, false>(sA, sH, totA, totH);       // the forward totals are not needed
    wave_prefix<NCH, WAVES, true>(bA, bH, totA, totH);
    __syncthreads();
    const int chn = threadIdx.x % NCH;
    const bool chok = ct * NCH + chn < A.C;
    float first = 0.f;
    if (back_kb == 0 && dhlast && chok && threadIdx.x < NCH) first = dhlast[(int64_t)seq * A.C + ct * NCH + chn];
    span_carry<NCH, WAVES * 64>(W, back_kb, tile, chok, first, totA, totH, carry, partA, partH);

    float h[L + 1][V], back[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        const int ch = cl * V + k;
        float wa = sA[wave][ch], wh = sH[wave][ch];
        join(wa, wh, pa[k], ph[k]);
        h[0][k] = wa == LOOP_CUT ? wh : fmaf(wa, hin[k], wh);
        wa = bA[wave][ch], wh = bH[wave][ch];
        join(wa, wh, ba[k], bh[k]);
        back[k] = wa == LOOP_CUT ? wh : fmaf(wa, carry[ch], wh);
    }
#pragma unroll
    for (int i = 0; i < L; ++i) {
        float fk[V];
        vk[i].get(fk);
        const bool cut = cuts >> i & 1, on = t0 + i < n;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float x = on ? fk[k] : 0.f;
            h[i + 1][k] = cut ? x : fmaf(g[i][k], h[i][k], x);
        }
    }
    const int64_t g0 = (int64_t)b * A.gb + (int64_t)p * A.gp + c;
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
        float fq[V], fy[V], fa[V], ok[V], oa[V];
        vq[i].get(fq); vy[i].get(fy); va[i].get(fa);
        const bool cut = cuts >> i & 1, on = t0 + i < n;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float gg, slope;
            sigm_slope<E>(fa[k], gg, slope);
            const float d = fmaf(fq[k], fy[k], back[k]);
            fq[k] = on ? h[i + 1][k] * fy[k] : 0.f;
            ok[k] = on ? d : 0.f;
            oa[k] = on && !cut ? d * h[i][k] * slope : 0.f;
            back[k] = on ? (cut ? 0.f : g[i][k] * d) : back[k];
        }
        if (cok && t0 + i < A.T) {
            const int64_t at = g0 + (t0 + i) * A.gt;
            RowVec<E, V>::store(dq, at, fq); RowVec<E, V>::store(dkv, at, ok); RowVec<E, V>::store(da, at, oa);
        }
    }
    if (dh0 && cok && kb == 0 && wave == 0 && lane / CL == 0) {
#pragma unroll
        for (int k = 0; k < V; ++k) dh0[(int64_t)seq * A.C + c + k] = back[k];
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

// Which form runs: one thread per chunk where the tokens are few or the channels many, spans otherwise.  A function of the sizes alone (the
// backward pass finds the states that the forward pass kept).
static bool loop_walks(const mv2_gateloop_desc* d) {
    const int kvec = d->dtype == MV2_BF16 ? 8 : 4;
    const double chunks = (double)d->B * d->P * ((d->C + kvec - 1) / kvec);
    return d->T <= 16 || chunks >= 131072;
}

extern "C" int64_t mv2_gateloop_states(const mv2_gateloop_desc* d) {
    const int rc = loop_check(d);
    if (rc != MV2_OK) return rc;
    return d->T > 0 ? (d->T - 1) / (loop_walks(d) ? LOOP_STEPS : SPAN_KEEP) : 0;
}

struct SpanShape { int64_t nblk, ctiles, ntile, words; };
static SpanShape span_shape(const mv2_gateloop_desc* d, int nch, int span) {
    SpanShape s;
    s.nblk = (d->T + span - 1) / span;
    s.ctiles = (d->C + nch - 1) / nch;
    s.ntile = s.ctiles * d->B * d->P;
    s.words = s.nblk > 1 ? 2 + (s.nblk + (s.nblk + LOOP_GROUP - 1) / LOOP_GROUP) * s.ntile * nch : 0;
    return s;
}
#define SPAN_FWD_WAVES 8
#define SPAN_BWD_WAVES 4
// channels of a workgroup: 128-byte pieces of rows (64 bf16 or 32 fp32), 64 single elements where rows are not whole 16-byte chunks
static int span_channels(const mv2_gateloop_desc* d, bool wide) { return wide && d->dtype == MV2_F32 ? 32 : 64; }

extern "C" size_t mv2_gateloop_workspace_bytes(const mv2_gateloop_desc* d, int backward) {
    if (loop_check(d) != MV2_OK || loop_walks(d)) return 0;
    const int span = 32 * (backward ? SPAN_BWD_WAVES : SPAN_FWD_WAVES);
    int64_t words = 0;
    for (int wide = 0; wide < 2; ++wide) words = std::max(words, span_shape(d, span_channels(d, wide), span).words);      // whichever the addresses allow
    return (size_t)words * sizeof(u64);
}

static LoopArgs loop_args(const mv2_gateloop_desc* d, const int32_t* lengths, const unsigned char* resets) {
    LoopArgs A;
    A.B = d->B; A.T = d->T; A.P = d->P; A.C = d->C;
    A.sb = d->in_b; A.st = d->in_t; A.sp = d->in_p; A.gb = d->grad_b; A.gt = d->grad_t; A.gp = d->grad_p;
    A.lengths = lengths; A.resets = resets;
    A.nstate = (int)mv2_gateloop_states(d);
    return A;
}

// the pairs' words, cleared by a kernel (a captured memset would not do: the launch may be recorded into a graph)
static int span_work(const mv2_gateloop_desc* d, bool wide, int waves, void* workspace, size_t workspace_bytes, hipStream_t st, SpanWork& W, unsigned& grid) {
    const int nch = span_channels(d, wide);
    const SpanShape s = span_shape(d, nch, waves * 32);
    if ((double)s.nblk * s.ntile > 2147483647.0) return MV2_ETOOLARGE;
    W.nblk = (int)s.nblk; W.ntile = (int)s.ntile; W.ctiles = (int)s.ctiles;
    grid = (unsigned)(s.nblk * s.ntile);
    W.ticket = nullptr; W.pairs = W.states = nullptr;
    if (s.words == 0) return MV2_OK;
    if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < s.words * sizeof(u64)) return MV2_EWORKSPACE;
    W.ticket = (unsigned*)workspace;
    W.pairs = (u64*)workspace + 2;
    W.states = W.pairs + s.nblk * s.ntile * nch;
    hipLaunchKernelGGL(span_clear_kernel, dim3((unsigned)std::min<int64_t>((s.words + 255) / 256, 2048)), dim3(256), 0, st, (u64*)workspace, s.words);
    MV2_LAUNCH_CHECK();
    return MV2_OK;
}

extern "C" int mv2_gateloop_forward(const mv2_gateloop_desc* d, const void* q, const void* kv, const void* a, const float* h0, const int32_t* lengths,
                                    const unsigned char* resets, void* y, float* h_last, float* states, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = loop_check(d);
    if (rc != MV2_OK) return rc;
    if (d->T > 0 && (!q || !kv || !a || !y)) return MV2_EINVAL;
    const LoopArgs A = loop_args(d, lengths, resets);
    const int kvec = d->dtype == MV2_BF16 ? 8 : 4;
    const bool wide = d->C % kvec == 0 && d->in_b % kvec == 0 && d->in_t % kvec == 0 && d->in_p % kvec == 0 && rows_aligned16({q, kv, a, y});
    hipStream_t st = (hipStream_t)stream;
    if (loop_walks(d)) {
        const int64_t n = (int64_t)d->B * d->P * (d->C / (wide ? kvec : 1));
        const dim3 grid((unsigned)((n + 255) / 256));
#define GO(E, V) hipLaunchKernelGGL((loop_walk_fwd_kernel<E, V>), grid, dim3(256), 0, st, A, q, kv, a, h0, y, h_last, states)
        if (d->dtype == MV2_BF16) { if (wide) GO(BF16, 8); else GO(BF16, 1); }
        else { if (wide) GO(F32, 4); else GO(F32, 1); }
#undef GO
    } else {
        SpanWork W;
        unsigned grid;
        rc = span_work(d, wide, SPAN_FWD_WAVES, workspace, workspace_bytes, st, W, grid);
        if (rc != MV2_OK) return rc;
#define GO(E, V, CL) hipLaunchKernelGGL((loop_span_fwd_kernel<E, V, CL, SPAN_FWD_WAVES>), dim3(grid), dim3(64 * SPAN_FWD_WAVES), 0, st, A, W, q, kv, a, h0, y, h_last, states)
        if (d->dtype == MV2_BF16) { if (wide) GO(BF16, 8, 8); else GO(BF16, 1, 64); }
        else { if (wide) GO(F32, 4, 8); else GO(F32, 1, 64); }
#undef GO
    }
    MV2_LAUNCH_CHECK();
    return MV2_OK;
}

extern "C" int mv2_gateloop_backward(const mv2_gateloop_desc* d, const void* q, const void* kv, const void* a, const float* h0, const int32_t* lengths,
                                     const unsigned char* resets, const float* states, const void* dy, const float* dh_last, void* dq, void* dkv, void* da,
                                     float* dh0, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = loop_check(d);
    if (rc != MV2_OK) return rc;
    if (d->T > 0 && (!q || !kv || !a || !dy || !dq || !dkv || !da)) return MV2_EINVAL;
    const LoopArgs A = loop_args(d, lengths, resets);
    if (A.nstate > 0 && !states) return MV2_EINVAL;
    const int kvec = d->dtype == MV2_BF16 ? 8 : 4;
    const bool wide = d->C % kvec == 0 && d->in_b % kvec == 0 && d->in_t % kvec == 0 && d->in_p % kvec == 0 && d->grad_b % kvec == 0 &&
                      d->grad_t % kvec == 0 && d->grad_p % kvec == 0 && rows_aligned16({q, kv, a, dy, dq, dkv, da});
    hipStream_t st = (hipStream_t)stream;
    if (loop_walks(d)) {
        const int64_t n = (int64_t)d->B * d->P * (d->C / (wide ? kvec : 1));
        const dim3 grid((unsigned)((n + 255) / 256));
#define GO(E, V) hipLaunchKernelGGL((loop_walk_bwd_kernel<E, V>), grid, dim3(256), 0, st, A, q, kv, a, h0, states, dy, dh_last, dq, dkv, da, dh0)
        if (d->dtype == MV2_BF16) { if (wide) GO(BF16, 8); else GO(BF16, 1); }
        else { if (wide) GO(F32, 4); else GO(F32, 1); }
#undef GO
    } else {
        SpanWork W;
        unsigned grid;
        rc = span_work(d, wide, SPAN_BWD_WAVES, workspace, workspace_bytes, st, W, grid);
        if (rc != MV2_OK) return rc;
#define GO(E, V, CL)                                                                                                                                    \
    hipLaunchKernelGGL((loop_span_bwd_kernel<E, V, CL, SPAN_BWD_WAVES>), dim3(grid), dim3(64 * SPAN_BWD_WAVES), 0, st, A, W, q, kv, a, h0, states, dy, dh_last, dq, dkv, da, dh0)
        if (d->dtype == MV2_BF16) { if (wide) GO(BF16, 8, 8); else GO(BF16, 1, 64); }
        else { if (wide) GO(F32, 4, 8); else GO(F32, 1, 64); }
#undef GO
    }
    MV2_LAUNCH_CHECK();
    return MV2_OK;
}
