// The norms before and after a residual block with its gate and scale, forward and backward (include/mv2.h mv2_block_norm_*):
//     out = x + s act(gate) N(branch; w1),   n = N(out; w2),   N(v; w) = v r sqrt(C) w,  r = 1 / max(|v|, 1e-12)
// Backward, with dn' = sqrt(C) w2 dn, o = out r2:   D = dout + r2 (dn' - o (o . dn'))         (gradient that arrives at out; the second term
//     dx = D,   dgate = D s act'(gate) u,   ds = sum_rows D act(gate) u                        without its projection where |out| < 1e-12)
//     dbranch = r1 (d' - b (b . d')),  d' = sqrt(C) w1 D s act(gate),  b = branch r1          (likewise),
//     dw1 = sqrt(C) sum_rows D s act(gate) b,   dw2 = sqrt(C) sum_rows dn o.
// A group of G threads (a power of two) owns a row and keeps it in registers: every tensor is read once and written once.  out is not saved:
// the backward pass forms it again from x, branch and gate, unrounded, as the forward pass had it.  Memory-bound: a workgroup walks many
// rows with the parameters in registers, R rows at a time so that their loads and their sums' latencies overlap.
// Measured on one MI355X, us and TB/s of the rows read and written, kernels alone (a copy in 16-byte accesses: 5.9 TB/s):
//     16384 x 2048 bf16, all parts   forward 63 (5.3), backward 116 (4.6) + 4 for the column sums' second kernel
//     69632 x 256 bf16, add and norm forward 25 (5.7, part of it from the last-level cache), backward 40 (4.4)
//     65536 x 512 bf16               forward 62 (5.4), backward 109 (4.9)        8192 x 2048 fp32  forward 60 (5.6), backward 100 (5.4)
//     16384 x 1001 bf16, ragged      forward 41 (4.0), backward 79 (3.3)         4097 x 501 fp32   forward 14, backward 23
//     6250 x 5120 bf16               forward 67 (4.8), backward 177 (2.9)        6251 x 5119 bf16, ragged  90 (3.6), 225 (2.3)
//     2000 x 16384 bf16              forward 73 (4.5), backward 265 (2.0)
// Forward it is the memory; backward also the 160 to 200 registers, which leave two or three waves on a SIMD, and beyond 8192 wide, where 1024 threads
// have 128 registers each, the spills (bf16 157, ragged 212; fp32 185, ragged 306, and 189 in its ragged forward kernel; tools/check_spills.sh).  32 rows take 5 us: latency.
#include <algorithm>
#include <initializer_list>
#include "rowvec.h"

struct NormArgs {
    int64_t rows;
    int C, act;
    int64_t xs, bs, gs;
    float root;                    // sqrt(C)
};

// Sums over the G threads of a row's group of N values at a time, in every thread.  Groups of more than a wave meet in LDS: `red` has two buffers
// that calls use in turn, so one barrier a call is enough (a buffer is written again behind the barrier of the call in between).
template <int BLOCK, int N> struct GroupSum {
    float (*red)[N][BLOCK / 64];
    int turn;
    __device__ __forceinline__ void operator()(float (&v)[N], int G) {
        lanes_sum(v, G);
        if (G <= 64) return;
        const int wave = threadIdx.x >> 6, nw = G / 64, first = wave / nw * nw;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[turn][i][wave] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float s = 0.f;
            for (int j = 0; j < nw; ++j) s += red[turn][i][first + j];
            v[i] = s;
        }
        turn ^= 1;
    }
};

// the gate's activation and its derivative
template <typename E> __device__ __forceinline__ float gate_act(int act, float g) {
    if (act == MV2_ACT_NONE) return g;
    const float s = sigm<E>(g);
    return act == MV2_ACT_SILU ? g * s : s;
}
// exp(-|g|) down to the smallest numbers: the hardware's exp2 flushes results below 2^-126, but silu's slope multiplies them by |g|
template <typename E> __device__ __forceinline__ float exp_tail(float g);
template <> __device__ __forceinline__ float exp_tail<BF16>(float g) {
    const float t = -fabsf(g) * 1.44269504088896340736f;
    const bool small = t < -126.f;
    return ldexpf(__builtin_amdgcn_exp2f(small ? t + 64.f : t), small ? -64 : 0);
}
template <> __device__ __forceinline__ float exp_tail<F32>(float g) { return expf(-fabsf(g)); }
template <typename E> __device__ __forceinline__ void gate_act_slope(int act, float g, float& v, float& d) {
    if (act == MV2_ACT_NONE) { v = g; d = 1.f; return; }
    const float e = exp_tail<E>(g), r = Gate<E>::recip(1.f + e), er = e * r;
    const float s = g < 0.f ? er : r, ds = er * r;
    if (act == MV2_ACT_SIGMOID) { v = s; d = ds; }
    else { v = g * s; d = fmaf(g, ds, s); }
}
// 1 / max(|v|, 1e-12) from the sum of squares; NaN stays NaN (fmaxf would drop it, and the row's other elements would come out finite)
__device__ __forceinline__ float inv_norm(float ss) {
    const float n = sqrtf(ss);
    return 1.f / (n < 1e-12f ? 1e-12f : n);
}

// a thread's parameters, f times w, or ones where there are none: in registers for all the rows (7000 x 4096 bf16, 16 a thread: 60 us forward;
// read again with every row 136)
template <int NC, int V> struct Params {
    float r[NC][V];
    __device__ __forceinline__ Params(const float* w, float f, int l, int G, int C) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int c = (l + j * G) * V;
#pragma unroll
            for (int k = 0; k < V; ++k) r[j][k] = 1.f;
            if (w && c + V <= C) {
#pragma unroll
                for (int k = 0; k < V; ++k) r[j][k] = f * w[c + k];
            } else if (w) {
#pragma unroll
                for (int k = 0; k < V; ++k) if (c + k < C) r[j][k] = f * w[c + k];
            }
        }
    }
};

// (four waves on a SIMD: up to 128 registers; without the bound the compiler takes at most one more in any shape)
template <typename E, int V, bool RAG, int NC, int R, int BLOCK, bool S>
__global__ __launch_bounds__(BLOCK, 4) void block_norm_fwd_kernel(NormArgs A, int G, const void* x, const void* __restrict__ branch, const void* __restrict__ gate,
                                                               const float* __restrict__ w1, const float* __restrict__ sc, const float* __restrict__ w2,
                                                               void* out, void* __restrict__ normed, float* __restrict__ rstd) {
    __shared__ float red[2][R][BLOCK / 64];
    GroupSum<BLOCK, R> sum{red, 0};
    // rows of more than one chunk a thread have a workgroup of their own, of G threads (whole waves), others a power of two of threads
    const int l = NC > 1 ? threadIdx.x : threadIdx.x & (G - 1), per = NC > 1 ? 1 : BLOCK / G, mine = NC > 1 ? 0 : threadIdx.x / G;
    const int nch = (A.C + V - 1) / V;
    const Params<NC, V> p1(w1, A.root, l, G, A.C), ps(sc, 1.f, l, G, A.C), p2(w2, A.root, l, G, A.C);
    const int64_t step = (int64_t)per * R;
    for (int64_t base = blockIdx.x * step; base < A.rows; base += gridDim.x * step) {
        int64_t row[R];
        bool on[R];
        RowVec<E, V, RAG> vx[R][NC], vb[R][NC], vg[R][NC];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            row[i] = base + i * per + mine;
            on[i] = row[i] < A.rows;
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int ch = l + j * G;
                if (on[i] && ch < nch) {
                    vx[i][j].template load<S>(x, row[i] * A.xs + ch * V, min(V, A.C - ch * V));
                    if (branch) vb[i][j].template load<S>(branch, row[i] * A.bs + ch * V, min(V, A.C - ch * V));
                    if (gate) vg[i][j].template load<S>(gate, row[i] * A.gs + ch * V, min(V, A.C - ch * V));
                } else { vx[i][j].clear(); vb[i][j].clear(); vg[i][j].clear(); }
            }
        }
        if (RAG)
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int ch = l + j * G, nv = ch < nch ? min(V, A.C - ch * V) : V;
#pragma unroll
                for (int i = 0; i < R; ++i) { vx[i][j].settle(nv); vb[i][j].settle(nv); vg[i][j].settle(nv); }
            }
        float r1[R], r2[R];
        if (w1) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                r1[i] = 0.f;
#pragma unroll
                for (int j = 0; j < NC; ++j) {
                    float f[V]; vb[i][j].get(f);
#pragma unroll
                    for (int k = 0; k < V; ++k) r1[i] = fmaf(f[k], f[k], r1[i]);
                }
            }
            sum(r1, G);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                r1[i] = inv_norm(r1[i]);
                if (rstd && on[i] && l == 0) rstd[row[i]] = r1[i];
            }
        }
        float o[R][NC][V];
#pragma unroll
        for (int i = 0; i < R; ++i) r2[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const float (&f1)[V] = p1.r[j], (&fs)[V] = ps.r[j];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int ch = l + j * G;
                vx[i][j].get(o[i][j]);
                if (branch) {
                    float fb[V], fg[V];
                    vb[i][j].get(fb); vg[i][j].get(fg);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        float u = fb[k];
                        if (w1) u *= r1[i] * f1[k];
                        if (gate) u *= gate_act<E>(A.act, fg[k]);
                        o[i][j][k] = fmaf(fs[k], u, o[i][j][k]);
                    }
                    if (on[i] && ch < nch) RowVec<E, V, RAG>::template store<S>(out, row[i] * A.C + ch * V, o[i][j], min(V, A.C - ch * V));
                }
                if (on[i] && ch < nch)
#pragma unroll
                    for (int k = 0; k < V; ++k) r2[i] = fmaf(o[i][j][k], o[i][j][k], r2[i]);
            }
        }
        if (!w2) continue;
        sum(r2, G);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            r2[i] = inv_norm(r2[i]);
            if (rstd && on[i] && l == 0) rstd[A.rows + row[i]] = r2[i];
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const float (&f2)[V] = p2.r[j];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int ch = l + j * G;
#pragma unroll
                for (int k = 0; k < V; ++k) o[i][j][k] *= r2[i] * f2[k];
                if (on[i] && ch < nch) RowVec<E, V, RAG>::template store<S>(normed, row[i] * A.C + ch * V, o[i][j], min(V, A.C - ch * V));
            }
        }
    }
}

// parts: [gridDim.x][3][C] column sums of a workgroup's rows (dw1, ds, dw2), summed in workgroup order by block_norm_cols_kernel
template <typename E, int V, bool RAG, int NC, int R, int BLOCK, bool S>
__global__ __launch_bounds__(BLOCK, NC == 1 ? 3 : 1) void block_norm_bwd_kernel(NormArgs A, int G, const void* __restrict__ x, const void* __restrict__ branch,
                                                               const void* __restrict__ gate, const float* __restrict__ w1, const float* __restrict__ sc,
                                                               const float* __restrict__ w2, const float* __restrict__ rstd, const void* __restrict__ dout,
                                                               const void* __restrict__ dn, void* __restrict__ dx, void* __restrict__ dbranch,
                                                               void* __restrict__ dgate, float* __restrict__ parts) {
    __shared__ float red[2][R][BLOCK / 64];
    GroupSum<BLOCK, R> sum{red, 0};
    // rows of more than one chunk a thread have a workgroup of their own, of G threads (whole waves), others a power of two of threads
    const int l = NC > 1 ? threadIdx.x : threadIdx.x & (G - 1), per = NC > 1 ? 1 : BLOCK / G, mine = NC > 1 ? 0 : threadIdx.x / G;
    const int nch = (A.C + V - 1) / V;
    const Params<NC, V> p1(w1, A.root, l, G, A.C), ps(sc, 1.f, l, G, A.C), p2(w2, A.root, l, G, A.C);
    const int64_t step = (int64_t)per * R;
    float s1[NC][V], s2[NC][V], s3[NC][V];
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) s1[j][k] = s2[j][k] = s3[j][k] = 0.f;
    for (int64_t base = blockIdx.x * step; base < A.rows; base += gridDim.x * step) {
        int64_t row[R];
        bool on[R];
        RowVec<E, V, RAG> vx[R][NC], vb[R][NC], vg[R][NC], vo[R][NC], vn[R][NC];
        float r1[R], r2[R];
#pragma unroll
        for (int i = 0; i < R; ++i) {
            row[i] = base + i * per + mine;
            on[i] = row[i] < A.rows;
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int ch = l + j * G;
                vx[i][j].clear(); vb[i][j].clear(); vg[i][j].clear(); vo[i][j].clear(); vn[i][j].clear();
                if (on[i] && ch < nch) {
                    if (w2 && dn) { vx[i][j].template load<S>(x, row[i] * A.xs + ch * V, min(V, A.C - ch * V)); vn[i][j].template load<S>(dn, row[i] * A.C + ch * V, min(V, A.C - ch * V)); }
                    if (branch) vb[i][j].template load<S>(branch, row[i] * A.bs + ch * V, min(V, A.C - ch * V));
                    if (gate) vg[i][j].template load<S>(gate, row[i] * A.gs + ch * V, min(V, A.C - ch * V));
                    if (dout) vo[i][j].template load<S>(dout, row[i] * A.C + ch * V, min(V, A.C - ch * V));
                }
            }
            r1[i] = on[i] && branch && w1 ? rstd[row[i]] : 0.f;
            r2[i] = on[i] && w2 ? rstd[A.rows + row[i]] : 0.f;
        }
        if (RAG)
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int ch = l + j * G, nv = ch < nch ? min(V, A.C - ch * V) : V;
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    vx[i][j].settle(nv); vb[i][j].settle(nv); vg[i][j].settle(nv); vo[i][j].settle(nv); vn[i][j].settle(nv);
                }
            }
        float D[R][NC][V];                             // gradient that arrives at out
        float dot[R];
#pragma unroll
        for (int i = 0; i < R; ++i) dot[i] = 0.f;
        if (w2 && dn) {
            float o[R][NC][V];                         // out r2
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const float (&f1)[V] = p1.r[j], (&fs)[V] = ps.r[j], (&f2)[V] = p2.r[j];
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    float fb[V], fg[V], fn[V];
                    vx[i][j].get(o[i][j]); vn[i][j].get(fn); vb[i][j].get(fb); vg[i][j].get(fg);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        if (branch) {
                            float u = fb[k];
                            if (w1) u *= r1[i] * f1[k];
                            if (gate) u *= gate_act<E>(A.act, fg[k]);
                            o[i][j][k] = fmaf(fs[k], u, o[i][j][k]);
                        }
                        o[i][j][k] *= r2[i];
                        s3[j][k] = fmaf(fn[k], o[i][j][k], s3[j][k]);
                        D[i][j][k] = fn[k] * f2[k];
                        dot[i] = fmaf(o[i][j][k], D[i][j][k], dot[i]);
                    }
                }
            }
            sum(dot, G);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                if (r2[i] >= 1e12f) dot[i] = 0.f;      // |out| below the floor: N is linear there
#pragma unroll
                for (int j = 0; j < NC; ++j)
#pragma unroll
                    for (int k = 0; k < V; ++k) D[i][j][k] = r2[i] * (D[i][j][k] - o[i][j][k] * dot[i]);
            }
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int j = 0; j < NC; ++j)
#pragma unroll
                    for (int k = 0; k < V; ++k) D[i][j][k] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) dot[i] = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const float (&f1)[V] = p1.r[j], (&fs)[V] = ps.r[j];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int ch = l + j * G;
                const bool in = on[i] && ch < nch;
                float fo[V];
                vo[i][j].get(fo);
#pragma unroll
                for (int k = 0; k < V; ++k) D[i][j][k] += fo[k];
                if (dx && in) RowVec<E, V, RAG>::template store<S>(dx, row[i] * A.C + ch * V, D[i][j], min(V, A.C - ch * V));
                if (branch) {
                    float fb[V], fg[V], og[V];
                    vb[i][j].get(fb); vg[i][j].get(fg);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const float b = w1 ? fb[k] * r1[i] : fb[k];
                        const float u = b * f1[k], d = D[i][j][k];
                        float act = 1.f, slope = 0.f;
                        if (gate) gate_act_slope<E>(A.act, fg[k], act, slope);
                        og[k] = d * fs[k] * u * slope;
                        s2[j][k] = fmaf(d * act, u, s2[j][k]);
                        const float db = d * fs[k] * act;
                        s1[j][k] = fmaf(db, b, s1[j][k]);
                        D[i][j][k] = db * f1[k];
                        dot[i] = fmaf(D[i][j][k], b, dot[i]);
                    }
                    if (dgate && in) RowVec<E, V, RAG>::template store<S>(dgate, row[i] * A.C + ch * V, og, min(V, A.C - ch * V));
                }
            }
        }
        if (!branch || !dbranch) continue;
        if (w1) sum(dot, G);
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (r1[i] >= 1e12f) dot[i] = 0.f;
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int ch = l + j * G;
                if (w1) {
                    float fb[V]; vb[i][j].get(fb);
#pragma unroll
                    for (int k = 0; k < V; ++k) D[i][j][k] = r1[i] * (D[i][j][k] - fb[k] * r1[i] * dot[i]);
                }
                if (on[i] && ch < nch) RowVec<E, V, RAG>::template store<S>(dbranch, row[i] * A.C + ch * V, D[i][j], min(V, A.C - ch * V));
            }
        }
    }
    if (!parts) return;
    float* o = parts + (int64_t)blockIdx.x * 3 * A.C;
    if (per == 1) {
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int ch = l + j * G;
            if (ch < nch)
#pragma unroll
                for (int k = 0; k < V; ++k)
                    if (!RAG || ch * V + k < A.C) {
                        o[ch * V + k] = s1[j][k] * A.root; o[A.C + ch * V + k] = s2[j][k]; o[2 * A.C + ch * V + k] = s3[j][k] * A.root;
                    }
        }
    } else if (NC == 1) {                              // several groups per workgroup (then NC is 1): their sums meet in LDS, group after group
        __shared__ float meet[NC == 1 ? 3 * V : 1][NC == 1 ? BLOCK : 1];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            meet[k][threadIdx.x] = s1[0][k] * A.root; meet[V + k][threadIdx.x] = s2[0][k]; meet[2 * V + k][threadIdx.x] = s3[0][k] * A.root;
        }
        __syncthreads();
        for (int e = threadIdx.x; e < 3 * V * G; e += BLOCK) {
            const int w = e / (V * G), c = e % (V * G), kk = w * V + c % V, ll = c / V;      // column c = ll * V + k of sum w
            float s = 0.f;
            for (int g = 0; g < per; ++g) s += meet[kk][g * G + ll];
            if (c < A.C) o[w * A.C + c] = s;
        }
    }
}

// column sums of `n` parts: 32 columns per workgroup, 16 interleaved shares of the parts, eight loads in flight a thread
__global__ __launch_bounds__(512) void block_norm_cols_kernel(const float* __restrict__ parts, int n, int C, float* __restrict__ dw1, float* __restrict__ ds,
                                                              float* __restrict__ dw2) {
    __shared__ float red[16][33];
    const int cl = threadIdx.x & 31, share = threadIdx.x >> 5, c = blockIdx.x * 32 + cl, which = blockIdx.y;
    float* out = which == 0 ? dw1 : which == 1 ? ds : dw2;
    if (!out) return;
    float s = 0.f;
    if (c < C) {
        const float* p = parts + (int64_t)which * C + c;
        const int64_t pitch = (int64_t)3 * C;
        int i = share;
        for (; i + 7 * 16 < n; i += 8 * 16) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = p[(i + 16 * k) * pitch];
#pragma unroll
            for (int k = 0; k < 8; ++k) s += v[k];
        }
        for (; i < n; i += 16) s += p[i * pitch];
    }
    red[share][cl] = s;
    __syncthreads();
    if (share == 0 && c < C) {
        s = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) s += red[i][cl];
        out[c] = s;
    }
}

// --------------------------------------------------------------------------- host side
#define NORM_R 2                   // rows at a time, one chunk per thread: 16384 x 2048 bf16 65 us forward and 118 backward, one row 69 and 118, four 119 and 245;
                                   // 65536 x 512 62 and 109, one row 68 and 112
#define NORM_GROUPS 1024           // workgroups from which on rows are taken NORM_R at a time
#define NORM_BWD_MOST 768          // workgroups of a backward pass at most
static int norm_check(const mv2_block_norm_desc* d) {
    if (!d || d->reserved != 0) return MV2_EINVAL;
    if (d->dtype != MV2_BF16 && d->dtype != MV2_F32) return MV2_EINVAL;
    if (d->gate_act != MV2_ACT_NONE && d->gate_act != MV2_ACT_SILU && d->gate_act != MV2_ACT_SIGMOID) return MV2_EINVAL;
    if (d->rows < 0 || d->C <= 0 || d->x_stride < 0 || d->branch_stride < 0 || d->gate_stride < 0) return MV2_EINVAL;
    if (d->C > 16384 || d->rows > ((int64_t)1 << 40)) return MV2_ETOOLARGE;
    const int64_t lim = (int64_t)1 << 20;
    if (d->x_stride > lim || d->branch_stride > lim || d->gate_stride > lim) return MV2_ETOOLARGE;
    return MV2_OK;
}

// threads per row G, chunks per thread NC, rows at a time R: the row's chunks spread over up to 256 threads first, then over two registers, then over
// up to 1024 threads (and four registers); R > 1 once every workgroup of a full chip has that many rows.  Rows of more than 256 chunks take as many
// whole waves as they fill (6250 x 5120 bf16 67 us forward, 70 with a power of two; ragged 6251 x 5119 90 and 96), but a power of two backward, where the
// registers leave one workgroup on a CU either way (177 us, whole waves 180; ragged 225 and 239)
struct NormShape { int access, NC, R, block, G; bool stream; };
static NormShape norm_shape(const mv2_block_norm_desc* d, int access, int tensors, bool backward) {
    const int es = d->dtype == MV2_BF16 ? 2 : 4, V = access ? 16 / es : 1, nch = (d->C + V - 1) / V;
    NormShape s{access, 1, 1, 256, 1, access == 2 && calls_stream((double)d->rows * d->C * tensors * es)};
    while (s.G < nch && s.G < 256) s.G *= 2;
    if (nch > 256) {
        s.NC = nch <= 2048 ? 2 : 4;
        s.G = ((nch + s.NC - 1) / s.NC + 63) / 64 * 64;
        while (backward && (s.G < 256 || (s.G & (s.G - 1)))) s.G += 64;
        s.block = s.G;
    }
    if (s.NC == 1 && d->rows / (s.block / s.G) >= (int64_t)NORM_R * NORM_GROUPS) s.R = NORM_R;
    return s;
}

static int norm_access(const mv2_block_norm_desc* d, const void* branch, const void* gate, std::initializer_list<const void*> ps) {
    const int es = d->dtype == MV2_BF16 ? 2 : 4;
    return rows_access(d->dtype, d->C, ps, {d->x_stride * es, branch ? d->branch_stride * es : 0, gate ? d->gate_stride * es : 0});
}

static unsigned norm_grid(const mv2_block_norm_desc* d, const NormShape& s, int64_t most) {
    const int64_t per = (int64_t)s.block / s.G * s.R, groups = (d->rows + per - 1) / per;
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(groups, most));
}

// Workgroups of the backward pass: each leaves 3 C partial column sums, so two turns of the loop at least (1000 x 2048 bf16 25 us, one turn 28;
// 4097 x 501 fp32 26 us, three turns 32, one 25), and no more than the chip holds at once by the registers of the shapes (up to 168 with two rows of
// one 16-byte chunk, 200 with one row of two; 16384 x 2048 bf16 118 us with 768, 126 with 512, 132 with 1280; 8000 x 2048 70, 72, 78).
static int64_t norm_bwd_grid(const mv2_block_norm_desc* d, const NormShape& s) {
    const int64_t most = s.block > 256 ? 256 : s.NC == 1 ? NORM_BWD_MOST : 512;
    return std::min(most, std::max<int64_t>(256, d->rows / ((int64_t)s.block / s.G * s.R) / 2));
}

extern "C" size_t mv2_block_norm_workspace_bytes(const mv2_block_norm_desc* d) {
    if (norm_check(d) != MV2_OK) return 0;
    return (size_t)NORM_BWD_MOST * 3 * d->C * sizeof(float);
}

static NormArgs norm_args(const mv2_block_norm_desc* d) {
    NormArgs A;
    A.rows = d->rows; A.C = d->C; A.act = d->gate_act; A.xs = d->x_stride; A.bs = d->branch_stride; A.gs = d->gate_stride;
    A.root = sqrtf((float)d->C);
    return A;
}

// one launch of KERNEL<E, V, RAGGED, NC, R, BLOCK, S> for the shape; S, past the caches: where the call is large, and always at widths beyond 512 chunks
// (a row of a thousand and more threads: 2000 x 16384 73 us forward, 78 through the caches)
#define NORM_CASES(KERNEL, ...)                                                                                   \
    do {                                                                                                          \
        if (d->dtype == MV2_BF16) { NORM_ACCESS(KERNEL, BF16, 8, __VA_ARGS__) }                                   \
        else { NORM_ACCESS(KERNEL, F32, 4, __VA_ARGS__) }                                                         \
    } while (0)
#define NORM_ACCESS(KERNEL, E, V, ...)                                                                            \
        if (s.access == 2 && s.stream && s.NC == 1 && s.R > 1) NORM_GO(KERNEL, E, V, false, 1, NORM_R, 256, true, __VA_ARGS__);         \
        else if (s.access == 2 && s.stream && s.NC == 2 && s.block <= 256) NORM_GO(KERNEL, E, V, false, 2, 1, 256, true, __VA_ARGS__);  \
        else if (s.access == 2) { NORM_SHAPES(KERNEL, E, V, false, true, __VA_ARGS__) }                           \
        else if (s.access == 1) { NORM_SHAPES(KERNEL, E, V, true, false, __VA_ARGS__) }                           \
        else if (s.R == 1) NORM_GO(KERNEL, E, 1, false, 1, 1, 256, false, __VA_ARGS__);                           \
        else NORM_GO(KERNEL, E, 1, false, 1, NORM_R, 256, false, __VA_ARGS__);
#define NORM_SHAPES(KERNEL, E, V, RAG, S, ...)                                                                    \
        if (s.NC == 1 && s.R == 1) NORM_GO(KERNEL, E, V, RAG, 1, 1, 256, false, __VA_ARGS__);                     \
        else if (s.NC == 1) NORM_GO(KERNEL, E, V, RAG, 1, NORM_R, 256, false, __VA_ARGS__);                       \
        else if (s.block <= 256) NORM_GO(KERNEL, E, V, RAG, 2, 1, 256, false, __VA_ARGS__);                       \
        else if (s.block <= 512) NORM_GO(KERNEL, E, V, RAG, 2, 1, 512, S, __VA_ARGS__);                           \
        else if (s.NC == 2) NORM_GO(KERNEL, E, V, RAG, 2, 1, 1024, S, __VA_ARGS__);                               \
        else NORM_GO(KERNEL, E, V, RAG, V == 4 ? 4 : 2, 1, 1024, S, __VA_ARGS__);
#define NORM_GO(KERNEL, E, V, RAG, NC, R, BLOCK, S, ...) hipLaunchKernelGGL((KERNEL<E, V, RAG, NC, R, BLOCK, S>), dim3(grid), dim3((NC) > 1 ? s.block : BLOCK), 0, st, A, s.G, __VA_ARGS__)

extern "C" int mv2_block_norm_forward(const mv2_block_norm_desc* d, const void* x, const void* branch, const void* gate, const float* post_gamma,
                                      const float* scale, const float* pre_gamma, void* out, void* normed, float* rstd, void* stream) {
    const int rc = norm_check(d);
    if (rc != MV2_OK) return rc;
    if (!branch && (gate || post_gamma || scale || !pre_gamma)) return MV2_EINVAL;
    if (d->rows == 0) return MV2_OK;
    if (!x || (branch && !out) || (pre_gamma && !normed)) return MV2_EINVAL;
    const int access = norm_access(d, branch, gate, {x, branch, gate, out, normed});
    const NormShape s = norm_shape(d, access, 1 + !!branch * 2 + !!gate + !!pre_gamma, false);
    const NormArgs A = norm_args(d);
    // as many workgroups as the chip holds at once: 4 waves on a SIMD by the registers of the shapes, 6 of those of aligned fp32 chunks (6250 x 5120
    // bf16 67 us with 512 workgroups of 5 waves, 84 with 768; 16384 x 2048 65, and 65 with twice as many)
    const int held = s.NC > 1 && d->dtype == MV2_F32 && access == 2 ? 6 : 4;
    const unsigned grid = norm_grid(d, s, 256 * std::max(1, held / ((s.block + 255) / 256)));
    hipStream_t st = (hipStream_t)stream;
    NORM_CASES(block_norm_fwd_kernel, x, branch, gate, post_gamma, scale, pre_gamma, out, normed, rstd);
    MV2_LAUNCH_CHECK();
    return MV2_OK;
}

extern "C" int mv2_block_norm_backward(const mv2_block_norm_desc* d, const void* x, const void* branch, const void* gate, const float* post_gamma,
                                       const float* scale, const float* pre_gamma, const float* rstd, const void* dout, const void* dn, void* dx,
                                       void* dbranch, void* dgate, float* dpost, float* dscale, float* dpre, void* workspace, size_t workspace_bytes,
                                       void* stream) {
    const int rc = norm_check(d);
    if (rc != MV2_OK) return rc;
    if (!branch && (gate || post_gamma || scale || !pre_gamma || dbranch || dgate || dpost || dscale)) return MV2_EINVAL;
    if ((dgate && !gate) || (dpost && !post_gamma) || (dscale && !scale) || (dpre && !pre_gamma) || (dn && !pre_gamma)) return MV2_EINVAL;
    if (d->rows > 0 && (!x || ((pre_gamma || post_gamma) && !rstd))) return MV2_EINVAL;
    const bool cols = dpost || dscale || dpre;
    if (cols && (!workspace || ((uintptr_t)workspace & 3) || workspace_bytes < mv2_block_norm_workspace_bytes(d))) return MV2_EWORKSPACE;
    const int access = norm_access(d, branch, gate, {x, branch, gate, dout, dn, dx, dbranch, dgate});
    const NormShape s = norm_shape(d, access, !!dout + !!dn * 2 + !!branch + !!gate + !!dx + !!dbranch + !!dgate, true);
    const NormArgs A = norm_args(d);
    const unsigned grid = norm_grid(d, s, norm_bwd_grid(d, s));
    float* parts = cols ? (float*)workspace : nullptr;
    hipStream_t st = (hipStream_t)stream;
    NORM_CASES(block_norm_bwd_kernel, x, branch, gate, post_gamma, scale, pre_gamma, rstd, dout, dn, dx, dbranch, dgate, parts);
    MV2_LAUNCH_CHECK();
    if (cols) {
        hipLaunchKernelGGL(block_norm_cols_kernel, dim3((unsigned)((d->C + 31) / 32), 3), dim3(512), 0, st, (const float*)parts, (int)grid, (int)d->C, dpost,
                           dscale, dpre);
        MV2_LAUNCH_CHECK();
    }
    return MV2_OK;
}
