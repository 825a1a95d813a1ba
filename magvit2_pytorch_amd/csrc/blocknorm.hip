// The norms before and after a residual block with its gate and scale, forward and backward (include/mv2.h mv2_block_norm_*):
//     out = x + s act(gate) N(branch; w1),   n = N(out; w2),   N(v; w) = v r sqrt(C) w,  r = 1 / max(|v|, 1e-12)
// Backward, with dn' = sqrt(C) w2 dn, o = out r2:   D = dout + r2 (dn' - o (o . dn'))         (gradient that arrives at out; the second term
//     dx = D,   dgate = D s act'(gate) u,   ds = sum_rows D act(gate) u                        without its projection where |out| < 1e-12)
//     dbranch = r1 (d' - b (b . d')),  d' = sqrt(C) w1 D s act(gate),  b = branch r1          (likewise),
//     dw1 = sqrt(C) sum_rows D s act(gate) b,   dw2 = sqrt(C) sum_rows dn o.
// A group of G threads (a power of two) owns a row and keeps it in registers: every tensor is read once and written once.  out is not saved:
// the backward pass forms it again from x, branch and gate, unrounded, as the forward pass had it.
#include <algorithm>
#include <initializer_list>
#include "rowvec.h"

struct NormArgs {
    int64_t rows;
    int C, act;
    int64_t xs, bs, gs;
    float root;                    // sqrt(C)
};

// sum over the G threads of a row's group; every thread of the workgroup takes part (groups of more than a wave meet in LDS)
template <int BLOCK> __device__ __forceinline__ float group_sum(float v, int G, float* red) {
    const int w = G < 64 ? G : 64;
    for (int o = w >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    if (G <= 64) return v;
    __syncthreads();                                   // the previous sum has been read
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    const int nw = G / 64, first = (threadIdx.x >> 6) / nw * nw;
    float s = 0.f;
    for (int i = 0; i < nw; ++i) s += red[first + i];
    return s;
}

__device__ __forceinline__ float sigmoid_f(float g) { return 1.f / (1.f + expf(-g)); }
__device__ __forceinline__ float gate_act(int act, float g) {
    if (act == MV2_ACT_NONE) return g;
    const float s = sigmoid_f(g);
    return act == MV2_ACT_SILU ? g * s : s;
}
// act and its derivative; s (1 - s) as e / (1 + e)^2 with e = exp(-|g|): no cancellation
__device__ __forceinline__ void gate_act_slope(int act, float g, float& v, float& d) {
    if (act == MV2_ACT_NONE) { v = g; d = 1.f; return; }
    const float e = expf(-fabsf(g)), r = 1.f / (1.f + e), er = e * r;
    const float s = g < 0.f ? er : r, ds = er * r;
    if (act == MV2_ACT_SIGMOID) { v = s; d = ds; }
    else { v = g * s; d = fmaf(g, ds, s); }
}

template <typename E, int V, int NC, int BLOCK>
__global__ __launch_bounds__(BLOCK) void block_norm_fwd_kernel(NormArgs A, int G, const void* x, const void* __restrict__ branch, const void* __restrict__ gate,
                                                               const float* __restrict__ w1, const float* __restrict__ sc, const float* __restrict__ w2,
                                                               void* out, void* __restrict__ normed, float* __restrict__ rstd) {
    __shared__ float red[BLOCK / 64];
    const int l = threadIdx.x & (G - 1), per = BLOCK / G;
    const int nch = A.C / V;
    const int64_t groups = (A.rows + per - 1) / per;
    for (int64_t blk = blockIdx.x; blk < groups; blk += gridDim.x) {
        const int64_t row = blk * per + threadIdx.x / G;
        const bool on = row < A.rows;
        RowVec<E, V> vx[NC], vb[NC], vg[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int ch = l + j * G;
            if (on && ch < nch) {
                vx[j].load(x, row * A.xs + (int64_t)ch * V);
                if (branch) vb[j].load(branch, row * A.bs + (int64_t)ch * V);
                if (gate) vg[j].load(gate, row * A.gs + (int64_t)ch * V);
            }
        }
        float r1 = 1.f;
        if (branch && (w1 || rstd)) {
            float ss = 0.f;
#pragma unroll
            for (int j = 0; j < NC; ++j)
                if (on && l + j * G < nch) {
                    float f[V]; vb[j].get(f);
#pragma unroll
                    for (int k = 0; k < V; ++k) ss = fmaf(f[k], f[k], ss);
                }
            r1 = 1.f / fmaxf(sqrtf(group_sum<BLOCK>(ss, G, red)), 1e-12f);
            if (rstd && on && l == 0) rstd[row] = r1;
        }
        float o[NC][V], ss = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int ch = l + j * G;
            if (on && ch < nch) {
                vx[j].get(o[j]);
                if (branch) {
                    float fb[V], fg[V];
                    vb[j].get(fb);
                    if (gate) vg[j].get(fg);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const int c = ch * V + k;
                        float u = fb[k];
                        if (w1) u *= r1 * (A.root * w1[c]);
                        if (gate) u *= gate_act(A.act, fg[k]);
                        o[j][k] = sc ? fmaf(sc[c], u, o[j][k]) : o[j][k] + u;
                    }
                    RowVec<E, V>::store(out, row * A.C + (int64_t)ch * V, o[j]);
                }
#pragma unroll
                for (int k = 0; k < V; ++k) ss = fmaf(o[j][k], o[j][k], ss);
            }
        }
        if (!w2) continue;
        const float r2 = 1.f / fmaxf(sqrtf(group_sum<BLOCK>(ss, G, red)), 1e-12f);
        if (rstd && on && l == 0) rstd[A.rows + row] = r2;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int ch = l + j * G;
            if (on && ch < nch) {
#pragma unroll
                for (int k = 0; k < V; ++k) o[j][k] *= r2 * (A.root * w2[ch * V + k]);
                RowVec<E, V>::store(normed, row * A.C + (int64_t)ch * V, o[j]);
            }
        }
    }
}

// parts: [gridDim.x][3][C] column sums of a workgroup's rows (dw1, ds, dw2), summed in workgroup order by block_norm_cols_kernel
template <typename E, int V, int NC, int BLOCK>
__global__ __launch_bounds__(BLOCK) void block_norm_bwd_kernel(NormArgs A, int G, const void* __restrict__ x, const void* __restrict__ branch,
                                                               const void* __restrict__ gate, const float* __restrict__ w1, const float* __restrict__ sc,
                                                               const float* __restrict__ w2, const float* __restrict__ rstd, const void* __restrict__ dout,
                                                               const void* __restrict__ dn, void* __restrict__ dx, void* __restrict__ dbranch,
                                                               void* __restrict__ dgate, float* __restrict__ parts) {
    __shared__ float red[BLOCK / 64];
    const int l = threadIdx.x & (G - 1), per = BLOCK / G;
    const int nch = A.C / V;
    const int64_t groups = (A.rows + per - 1) / per;
    float s1[NC][V], s2[NC][V], s3[NC][V];
#pragma unroll
    for (int j = 0; j < NC; ++j)
#pragma unroll
        for (int k = 0; k < V; ++k) s1[j][k] = s2[j][k] = s3[j][k] = 0.f;
    for (int64_t blk = blockIdx.x; blk < groups; blk += gridDim.x) {
        const int64_t row = blk * per + threadIdx.x / G;
        const bool on = row < A.rows;
        RowVec<E, V> vx[NC], vb[NC], vg[NC], vo[NC], vn[NC];
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int ch = l + j * G;
            if (on && ch < nch) {
                if (w2) vx[j].load(x, row * A.xs + (int64_t)ch * V);
                if (branch) vb[j].load(branch, row * A.bs + (int64_t)ch * V);
                if (gate) vg[j].load(gate, row * A.gs + (int64_t)ch * V);
                if (dout) vo[j].load(dout, row * A.C + (int64_t)ch * V);
                if (w2 && dn) vn[j].load(dn, row * A.C + (int64_t)ch * V);
            }
        }
        const float r1 = (on && branch && w1) ? rstd[row] : 0.f, r2 = (on && w2) ? rstd[A.rows + row] : 0.f;
        float D[NC][V];                                // gradient that arrives at out
        float dot = 0.f;
        float o[NC][V];                                // out r2
        if (w2 && dn) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int ch = l + j * G;
                if (on && ch < nch) {
                    float fb[V], fg[V], fn[V];
                    vx[j].get(o[j]); vn[j].get(fn);
                    if (branch) { vb[j].get(fb); if (gate) vg[j].get(fg); }
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const int c = ch * V + k;
                        if (branch) {
                            float u = fb[k];
                            if (w1) u *= r1 * (A.root * w1[c]);
                            if (gate) u *= gate_act(A.act, fg[k]);
                            o[j][k] = sc ? fmaf(sc[c], u, o[j][k]) : o[j][k] + u;
                        }
                        o[j][k] *= r2;
                        s3[j][k] = fmaf(fn[k], o[j][k], s3[j][k]);
                        D[j][k] = fn[k] * (A.root * w2[c]);
                        dot = fmaf(o[j][k], D[j][k], dot);
                    }
                }
            }
            dot = group_sum<BLOCK>(dot, G, red);
            if (r2 >= 1e12f) dot = 0.f;                // |out| below the floor: N is linear there
#pragma unroll
            for (int j = 0; j < NC; ++j)
                if (on && l + j * G < nch)
#pragma unroll
                    for (int k = 0; k < V; ++k) D[j][k] = r2 * (D[j][k] - o[j][k] * dot);
        } else {
#pragma unroll
            for (int j = 0; j < NC; ++j)
#pragma unroll
                for (int k = 0; k < V; ++k) D[j][k] = 0.f;
        }
        float dot1 = 0.f;
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int ch = l + j * G;
            if (on && ch < nch) {
                if (dout) {
                    float fo[V]; vo[j].get(fo);
#pragma unroll
                    for (int k = 0; k < V; ++k) D[j][k] += fo[k];
                }
                if (dx) RowVec<E, V>::store(dx, row * A.C + (int64_t)ch * V, D[j]);
                if (branch) {
                    float fb[V], fg[V], og[V];
                    vb[j].get(fb);
                    if (gate) vg[j].get(fg);
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const int c = ch * V + k;
                        const float b = w1 ? fb[k] * r1 : fb[k];
                        const float rw = w1 ? A.root * w1[c] : 1.f;
                        const float u = b * rw, s = sc ? sc[c] : 1.f;
                        float act = 1.f, slope = 0.f;
                        if (gate) gate_act_slope(A.act, fg[k], act, slope);
                        const float d = D[j][k];
                        og[k] = d * s * u * slope;
                        s2[j][k] = fmaf(d * act, u, s2[j][k]);
                        const float db = d * s * act;
                        s1[j][k] = fmaf(db, b, s1[j][k]);
                        D[j][k] = db * rw;
                        dot1 = fmaf(D[j][k], b, dot1);
                    }
                    if (dgate) RowVec<E, V>::store(dgate, row * A.C + (int64_t)ch * V, og);
                }
            }
        }
        if (!branch || !dbranch) continue;
        if (w1) {
            dot1 = group_sum<BLOCK>(dot1, G, red);
            if (r1 >= 1e12f) dot1 = 0.f;
        }
#pragma unroll
        for (int j = 0; j < NC; ++j) {
            const int ch = l + j * G;
            if (on && ch < nch) {
                if (w1) {
                    float fb[V]; vb[j].get(fb);
#pragma unroll
                    for (int k = 0; k < V; ++k) D[j][k] = r1 * (D[j][k] - fb[k] * r1 * dot1);
                }
                RowVec<E, V>::store(dbranch, row * A.C + (int64_t)ch * V, D[j]);
            }
        }
    }
    if (!parts) return;
    // one group of the workgroup after the other adds its rows' sums
    float* o = parts + (int64_t)blockIdx.x * 3 * A.C;
    for (int g = 0; g < per; ++g) {
        if ((int)threadIdx.x / G == g) {
#pragma unroll
            for (int j = 0; j < NC; ++j) {
                const int ch = l + j * G;
                if (ch < nch)
#pragma unroll
                    for (int k = 0; k < V; ++k) {
                        const int c = ch * V + k;
                        const float a = s1[j][k] * A.root, b = s2[j][k], e = s3[j][k] * A.root;
                        o[c] = g ? o[c] + a : a;
                        o[A.C + c] = g ? o[A.C + c] + b : b;
                        o[2 * A.C + c] = g ? o[2 * A.C + c] + e : e;
                    }
            }
        }
        __syncthreads();
    }
}

// column sums of `n` parts, 64 columns x 4 interleaved quarters per workgroup
__global__ __launch_bounds__(256) void block_norm_cols_kernel(const float* __restrict__ parts, int n, int C, float* __restrict__ dw1, float* __restrict__ ds,
                                                              float* __restrict__ dw2) {
    __shared__ float red[4][64];
    const int c = blockIdx.x * 64 + (threadIdx.x & 63), quarter = threadIdx.x >> 6, which = blockIdx.y;
    float* out = which == 0 ? dw1 : which == 1 ? ds : dw2;
    float s = 0.f;
    if (out && c < C)
        for (int i = quarter; i < n; i += 4) s += parts[((int64_t)i * 3 + which) * C + c];
    red[quarter][threadIdx.x & 63] = s;
    __syncthreads();
    if (quarter == 0 && out && c < C) out[c] = (red[0][threadIdx.x] + red[1][threadIdx.x]) + (red[2][threadIdx.x] + red[3][threadIdx.x]);
}

// --------------------------------------------------------------------------- host side
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

// threads per row G and chunks per thread NC: the row's chunks spread over up to 256 threads first, then over registers
struct NormShape { int V, NC, block, G; };
static NormShape norm_shape(int C, int V) {
    const int nch = C / V;
    NormShape s{V, 1, 256, 1};
    while (s.G < nch && s.G < 256) s.G *= 2;
    if (nch > 256) {
        if (V > 1) s.NC = nch <= 512 ? 2 : 4;
        else s.NC = nch <= 1024 ? 4 : 16;
        if (nch > 256 * s.NC) s.block = s.G = 1024;
    }
    return s;
}

static unsigned norm_grid(const mv2_block_norm_desc* d, const NormShape& s, int64_t most) {
    const int64_t per = s.block / s.G, groups = (d->rows + per - 1) / per;
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>(groups, most));
}
#define NORM_BWD_GRID 512          // workgroups of the backward pass at most: each leaves 3 C partial column sums

extern "C" size_t mv2_block_norm_workspace_bytes(const mv2_block_norm_desc* d) {
    if (norm_check(d) != MV2_OK) return 0;
    return (size_t)NORM_BWD_GRID * 3 * d->C * sizeof(float);
}

static NormArgs norm_args(const mv2_block_norm_desc* d) {
    NormArgs A;
    A.rows = d->rows; A.C = d->C; A.act = d->gate_act; A.xs = d->x_stride; A.bs = d->branch_stride; A.gs = d->gate_stride;
    A.root = sqrtf((float)d->C);
    return A;
}

// one launch of KERNEL<E, V, NC, BLOCK> for the shape
#define NORM_CASES(KERNEL, ...)                                                                                   \
    do {                                                                                                          \
        if (d->dtype == MV2_BF16) {                                                                               \
            if (s.V == 8) {                                                                                       \
                if (s.block == 1024) NORM_GO(KERNEL, BF16, 8, 4, 1024, __VA_ARGS__);                              \
                else if (s.NC == 1) NORM_GO(KERNEL, BF16, 8, 1, 256, __VA_ARGS__);                                \
                else if (s.NC == 2) NORM_GO(KERNEL, BF16, 8, 2, 256, __VA_ARGS__);                                \
                else NORM_GO(KERNEL, BF16, 8, 4, 256, __VA_ARGS__);                                               \
            } else {                                                                                              \
                if (s.block == 1024) NORM_GO(KERNEL, BF16, 1, 16, 1024, __VA_ARGS__);                             \
                else if (s.NC == 1) NORM_GO(KERNEL, BF16, 1, 1, 256, __VA_ARGS__);                                \
                else if (s.NC == 4) NORM_GO(KERNEL, BF16, 1, 4, 256, __VA_ARGS__);                                \
                else NORM_GO(KERNEL, BF16, 1, 16, 256, __VA_ARGS__);                                              \
            }                                                                                                     \
        } else {                                                                                                  \
            if (s.V == 4) {                                                                                       \
                if (s.block == 1024) NORM_GO(KERNEL, F32, 4, 4, 1024, __VA_ARGS__);                               \
                else if (s.NC == 1) NORM_GO(KERNEL, F32, 4, 1, 256, __VA_ARGS__);                                 \
                else if (s.NC == 2) NORM_GO(KERNEL, F32, 4, 2, 256, __VA_ARGS__);                                 \
                else NORM_GO(KERNEL, F32, 4, 4, 256, __VA_ARGS__);                                                \
            } else {                                                                                              \
                if (s.block == 1024) NORM_GO(KERNEL, F32, 1, 16, 1024, __VA_ARGS__);                              \
                else if (s.NC == 1) NORM_GO(KERNEL, F32, 1, 1, 256, __VA_ARGS__);                                 \
                else if (s.NC == 4) NORM_GO(KERNEL, F32, 1, 4, 256, __VA_ARGS__);                                 \
                else NORM_GO(KERNEL, F32, 1, 16, 256, __VA_ARGS__);                                               \
            }                                                                                                     \
        }                                                                                                         \
    } while (0)
#define NORM_GO(KERNEL, E, V, NC, BLOCK, ...) hipLaunchKernelGGL((KERNEL<E, V, NC, BLOCK>), dim3(grid), dim3(BLOCK), 0, st, A, s.G, __VA_ARGS__)

extern "C" int mv2_block_norm_forward(const mv2_block_norm_desc* d, const void* x, const void* branch, const void* gate, const float* post_gamma,
                                      const float* scale, const float* pre_gamma, void* out, void* normed, float* rstd, void* stream) {
    const int rc = norm_check(d);
    if (rc != MV2_OK) return rc;
    if (!branch && (gate || post_gamma || scale || !pre_gamma)) return MV2_EINVAL;
    if (d->rows == 0) return MV2_OK;
    if (!x || (branch && !out) || (pre_gamma && !normed)) return MV2_EINVAL;
    const int kvec = d->dtype == MV2_BF16 ? 8 : 4;
    const bool wide = d->C % kvec == 0 && d->x_stride % kvec == 0 && (!branch || d->branch_stride % kvec == 0) && (!gate || d->gate_stride % kvec == 0) &&
                      rows_aligned16({x, branch, gate, out, normed});
    const NormShape s = norm_shape(d->C, wide ? kvec : 1);
    const NormArgs A = norm_args(d);
    const unsigned grid = norm_grid(d, s, 8192);
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
    const int kvec = d->dtype == MV2_BF16 ? 8 : 4;
    const bool wide = d->C % kvec == 0 && d->x_stride % kvec == 0 && (!branch || d->branch_stride % kvec == 0) && (!gate || d->gate_stride % kvec == 0) &&
                      rows_aligned16({x, branch, gate, dout, dn, dx, dbranch, dgate});
    const NormShape s = norm_shape(d->C, wide ? kvec : 1);
    const NormArgs A = norm_args(d);
    const unsigned grid = norm_grid(d, s, NORM_BWD_GRID);
    float* parts = cols ? (float*)workspace : nullptr;
    hipStream_t st = (hipStream_t)stream;
    NORM_CASES(block_norm_bwd_kernel, x, branch, gate, post_gamma, scale, pre_gamma, rstd, dout, dn, dx, dbranch, dgate, parts);
    MV2_LAUNCH_CHECK();
    if (cols) {
        hipLaunchKernelGGL(block_norm_cols_kernel, dim3((unsigned)((d->C + 63) / 64), 3), dim3(256), 0, st, (const float*)parts, (int)grid, (int)d->C, dpost,
                           dscale, dpre);
        MV2_LAUNCH_CHECK();
    }
    return MV2_OK;
}
