// Gated linear recurrence along tokens, forward and backward (include/mv2.h mv2_gateloop_forward / mv2_gateloop_backward):
//     h_t = g_t h_{t-1} + kv_t,   g_t = sigmoid(a_t) (0 where a document starts),   y_t = q_t h_t
// and, with D_t the gradient that arrives at h_t,
//     D_t = q_t dy_t + g_{t+1} D_{t+1} (+ dh_last at the last token),  dq = h dy,  dkv = D,  da = D h_{t-1} g (1 - g),  dh0 = g_0 D_0.
// Everything between the loads and the stores is fp32; only y, dq, dkv, da are rounded to the storage type (on their stores, once).
// One or two flops a byte: the work is to read every element once (4 tensors forward, 7 backward) and to keep the chip's memory busy.  A copy of
// 256 MB in 16-byte accesses runs at 5.9 TB/s.  Measured on one MI355X, us and TB/s of those tensors, kernels alone:
//     walks   4 x 17 tokens x 1024 x 256 bf16       forward 25 (5.7; part of it from the last-level cache), backward 52 (4.8)
//     spans   8 x 2048 x 2048 bf16                  forward 55 (4.9), backward 96 (4.9); with document starts 54 and 105
//             1 x 131072 x 512 bf16                 forward 106 (5.1), backward 193 (4.9); 1 x 100000 x 64 23 and 36
//             6 x 4095 x 1000 bf16, rows off lines  forward 53 (3.7), backward 92 (3.7)
//             16 x 60000 x 16 bf16                  forward 70 (1.8), backward 137 (1.6): two lanes of a row's eight hold data
//             3 x 1023 x 777 fp32                   forward 14, backward 18 (9.5 MB a tensor: as much latency as bandwidth)
// and 2.6 us for a single token of 512 channels, 4.4 us for one of 192 x 2048, where launch and load latency are all there is.
#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include "rowvec.h"

struct LoopArgs {
    int B, T, P, C;
    int64_t sb, st, sp;            // q, kv, a
    int64_t gb, gt, gp;            // dq, dkv, da
    const int32_t* lengths;
    const unsigned char* resets;
    int nstate, keep;              // kept states per sequence (mv2_gateloop_states), tokens between them
};

#define LOOP_STEPS 8               // tokens between two kept states of the walking kernels

__device__ __forceinline__ int live_tokens(const LoopArgs& A, int b) {
    if (!A.lengths) return A.T;
    const int n = A.lengths[b];
    return n < 0 ? 0 : (n > A.T ? A.T : n);
}

// --------------------------------------------------------------------------- one thread per chunk of channels walks its tokens
// chunk i -> sequence, chunk of its row, sample, pixel (divisions in 32 bits where they do: a quarter of a single token's kernel otherwise)
__device__ __forceinline__ void walk_place(const LoopArgs& A, int64_t i, int64_t total, int cpr, int64_t& seq, int& chunk, int& b, int& p) {
    if (total <= 0x7fffffff) {
        const unsigned s = (unsigned)i / (unsigned)cpr;
        chunk = (int)((unsigned)i - s * (unsigned)cpr);
        b = (int)(s / (unsigned)A.P); p = (int)(s - (unsigned)b * (unsigned)A.P);
        seq = s;
    } else {
        seq = i / cpr;
        chunk = (int)(i - seq * cpr);
        b = (int)(seq / A.P); p = (int)(seq - (int64_t)b * A.P);
    }
}

// the marks of 8 tokens from t on, a byte each (0 behind token T - 1).  Asked for before the tokens' rows, which may then still be on their way when
// the marks are needed (4 x 33 x 512 x 256 bf16 28 us, read behind the rows 34)
typedef unsigned long long Marks __attribute__((aligned(1)));
__device__ __forceinline__ unsigned long long eight_marks(const unsigned char* rs, int t, int T) {
    if (t + LOOP_STEPS <= T) return *(const Marks*)(rs + t);
    unsigned long long w = 0;
#pragma unroll
    for (int s = 0; s < LOOP_STEPS; ++s)
        if (t + s < T) w |= (unsigned long long)rs[t + s] << 8 * s;
    return w;
}
__device__ __forceinline__ bool mark(unsigned long long w, int s) { return (unsigned)(w >> 8 * s) & 0xff; }

template <typename E, int V, bool S>
__global__ __launch_bounds__(256) void loop_walk_fwd_kernel(LoopArgs A, const void* __restrict__ q, const void* __restrict__ kv, const void* __restrict__ a,
                                                            const float* h0, void* __restrict__ y, float* hlast, float* __restrict__ states) {
    const int cpr = A.C / V;
    const int64_t total = (int64_t)A.B * A.P * cpr;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    int64_t seq;
    int c, b, p;
    walk_place(A, i, total, cpr, seq, c, b, p);
    c *= V;
    const int n = live_tokens(A, b);
    const int64_t in0 = b * A.sb + p * A.sp + c;
    const int64_t yt = (int64_t)A.P * A.C, y0 = (int64_t)b * A.T * yt + (int64_t)p * A.C + c;
    const unsigned char* rs = A.resets ? A.resets + (int64_t)b * A.T : nullptr;
    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = h0 ? h0[seq * A.C + c + k] : 0.f;
    int t = 0;
    // `most` tokens at a time, all loaded before the first is worked on; up to `most` of them exist if GUARD
    auto batch = [&](auto most, auto guard) {
        constexpr int M = decltype(most)::value;
        constexpr bool GUARD = decltype(guard)::value;
        RowVec<E, V> vq[M], vk[M], va[M];
        const unsigned long long cuts = rs ? eight_marks(rs, t, A.T) : 0;
#pragma unroll
        for (int s = 0; s < M; ++s)
            if (!GUARD || t + s < n) {
                const int64_t at = in0 + (t + s) * A.st;
                vk[s].template load<S>(kv, at); va[s].template load<S>(a, at); vq[s].template load<S>(q, at);
            }
        if (states && t > 0) {
            float* o = states + (((int64_t)b * A.nstate + t / LOOP_STEPS - 1) * A.P + p) * A.C + c;
#pragma unroll
            for (int k = 0; k < V; ++k) o[k] = h[k];
        }
#pragma unroll
        for (int s = 0; s < M; ++s)
            if (!GUARD || t + s < n) {
                float fq[V], fk[V], fa[V];
                vq[s].get(fq); vk[s].get(fk); va[s].get(fa);
#pragma unroll
                for (int k = 0; k < V; ++k) {
                    h[k] = mark(cuts, s) ? fk[k] : fmaf(sigm<E>(fa[k]), h[k], fk[k]);
                    fq[k] *= h[k];
                }
                RowVec<E, V>::template store<S>(y, y0 + (t + s) * yt, fq);
            }
        t = min(t + M, n);
    };
    while (t + LOOP_STEPS <= n) batch(std::integral_constant<int, LOOP_STEPS>(), std::false_type());
    if (n - t > 1) batch(std::integral_constant<int, LOOP_STEPS - 1>(), std::true_type());      // (12 tokens of 8192 chunks: 6.6 us, one by one 8.5; 15 of 131072, where the memory bounds it, 23.2 and 21.7)
    else if (n - t == 1) batch(std::integral_constant<int, 1>(), std::false_type());
    float zero[V];
#pragma unroll
    for (int k = 0; k < V; ++k) zero[k] = 0.f;
    for (; t < A.T; ++t) RowVec<E, V>::template store<S>(y, y0 + t * yt, zero);
    if (hlast) {
#pragma unroll
        for (int k = 0; k < V; ++k) hlast[seq * A.C + c + k] = h[k];
    }
}

template <typename E, int V, bool RAG>
__global__ __launch_bounds__(256) void loop_walk_bwd_kernel(LoopArgs A, const void* __restrict__ q, const void* __restrict__ kv, const void* __restrict__ a,
                                                            const float* __restrict__ h0, const float* __restrict__ states, const void* __restrict__ dy,
                                                            const float* __restrict__ dhlast, void* __restrict__ dq, void* __restrict__ dkv,
                                                            void* __restrict__ da, float* __restrict__ dh0) {
    const int cpr = (A.C + V - 1) / V;
    const int64_t total = (int64_t)A.B * A.P * cpr;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    int64_t seq;
    int c, b, p;
    walk_place(A, i, total, cpr, seq, c, b, p);
    c *= V;
    const int nv = RAG ? min(V, A.C - c) : V;       // elements of the chunk
    const int n = live_tokens(A, b);
    const int64_t in0 = b * A.sb + p * A.sp + c, g0 = b * A.gb + p * A.gp + c;
    const int64_t yt = (int64_t)A.P * A.C, y0 = (int64_t)b * A.T * yt + (int64_t)p * A.C + c;
    const unsigned char* rs = A.resets ? A.resets + (int64_t)b * A.T : nullptr;
    float back[V], zero[V];                         // what h_{t+1} passes back to h_t
#pragma unroll
    for (int k = 0; k < V; ++k) { back[k] = dhlast && k < nv ? dhlast[seq * A.C + c + k] : 0.f; zero[k] = 0.f; }
    for (int t = n; t < A.T; ++t) {
        const int64_t at = g0 + t * A.gt;
        RowVec<E, V, RAG>::store(dq, at, zero, nv); RowVec<E, V, RAG>::store(dkv, at, zero, nv); RowVec<E, V, RAG>::store(da, at, zero, nv);
    }
    for (int blk = (n + LOOP_STEPS - 1) / LOOP_STEPS - 1; blk >= 0; --blk) {
        const int t0 = blk * LOOP_STEPS;
        RowVec<E, V, RAG> vq[LOOP_STEPS], vk[LOOP_STEPS], va[LOOP_STEPS], vy[LOOP_STEPS];
        const unsigned long long cuts = rs ? eight_marks(rs, t0, A.T) : 0;
#pragma unroll
        for (int s = 0; s < LOOP_STEPS; ++s)
            if (t0 + s < n) {
                const int64_t at = in0 + (t0 + s) * A.st;
                vk[s].load(kv, at, nv); va[s].load(a, at, nv); vq[s].load(q, at, nv); vy[s].load(dy, y0 + (t0 + s) * yt, nv);
            } else { vk[s].clear(); va[s].clear(); vq[s].clear(); vy[s].clear(); }
#pragma unroll
        for (int s = 0; s < LOOP_STEPS; ++s) { vk[s].settle(nv); va[s].settle(nv); vq[s].settle(nv); vy[s].settle(nv); }
        float h[LOOP_STEPS + 1][V];                 // h[s] = state before token t0 + s
        const float* hin = blk > 0 ? states + (((int64_t)b * A.nstate + blk - 1) * A.P + p) * A.C + c : (h0 ? h0 + seq * A.C + c : nullptr);
#pragma unroll
        for (int k = 0; k < V; ++k) h[0][k] = hin && k < nv ? hin[k] : 0.f;
#pragma unroll
        for (int s = 0; s < LOOP_STEPS; ++s)
            if (t0 + s < n) {
                float fk[V], fa[V];
                vk[s].get(fk); va[s].get(fa);
                const bool cut = mark(cuts, s);
#pragma unroll
                for (int k = 0; k < V; ++k) h[s + 1][k] = cut ? fk[k] : fmaf(sigm<E>(fa[k]), h[s][k], fk[k]);
            }
#pragma unroll
        for (int s = LOOP_STEPS - 1; s >= 0; --s)
            if (t0 + s < n) {
                float fq[V], fa[V], fy[V], oq[V], oa[V], ok[V];
                vq[s].get(fq); va[s].get(fa); vy[s].get(fy);
                const bool cut = mark(cuts, s);
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
                RowVec<E, V, RAG>::store(dq, at, oq, nv); RowVec<E, V, RAG>::store(dkv, at, ok, nv); RowVec<E, V, RAG>::store(da, at, oa, nv);
            }
    }
    if (dh0) {
#pragma unroll
        for (int k = 0; k < V; ++k) if (k < nv) dh0[seq * A.C + c + k] = back[k];
    }
}

// --------------------------------------------------------------------------- spans of tokens joined along the sequence
// (What bounds them: a workgroup lives through load, join, wait and store one after the other, and two of them share a CU; the rest of the
// distance to the copy is those phases where both wait.)
// The walking kernels above leave the chip empty where there are few channels and many tokens.  Here a workgroup owns WAVES * TW tokens of
// CL * V channels of one sequence (a "block"): a lane holds L consecutive tokens of V channels in registers (every element is read once),
// CL lanes side by side read whole 128-byte pieces of rows.  Lane rows and blocks are joined through the pair (A, H) of a span: it takes the
// state h in front of it to A h + H, and spans join as (A1, H1) (A2, H2) -> (A1 A2, A2 H1 + H2).  Within the workgroup the pairs meet in LDS,
// where thread (channel, segment) takes a run of lane rows, and come back as the state in front of each lane row.
// Between workgroups: a block publishes its pair and reads the pairs of the blocks before it in its group; the last block of a group publishes
// the group's pair, and groups are joined likewise in sets, whose last block publishes the state behind the set.  A block reads at most 7 pairs,
// 7 groups' pairs and one state, always the same in the same order, so results do not depend on timing, and states are handed on once every 64
// blocks.  bf16, us forward / backward, measured in turn: 1 x 100000 x 64 23 / 35, states handed on from group to group of 16 blocks 36 / 58 (1 x 131072 x 512 108 / 193
// and 107 / 188); groups and sets of 16 21 / 34, but every block reads twice as much: 16 x 60000 x 16 68 / 140 against 65 / 136.
// Every wait ends: a block's place in the order is the ticket it draws when it starts, blocks wait for lower tickets only - for workgroups
// that are running; a block's pair is published before it waits for anything, a group's before its block waits for other groups.
#define LOOP_GROUP 8                // blocks
#define LOOP_SET 8                  // groups
#define LOOP_CUT 2.f               // A of a span in which a document starts (products of decays are <= 1 or NaN): nothing passes through it
typedef unsigned long long u64;

// a pair in one 8-byte word, written and read whole; the sign of A is the mark that it is there (the words are zero before the launch)
__device__ __forceinline__ u64 pair_word(float A, float H) { return ((u64)(__float_as_uint(A) | 0x80000000u) << 32) | __float_as_uint(H); }
__device__ __forceinline__ bool pair_there(u64 w) { return (w >> 63) != 0; }
__device__ __forceinline__ float pair_A(u64 w) { return __uint_as_float((unsigned)(w >> 32) & 0x7fffffffu); }
__device__ __forceinline__ float pair_H(u64 w) { return __uint_as_float((unsigned)w); }
__device__ __forceinline__ void publish(u64* p, float A, float H) { __hip_atomic_store(p, pair_word(A, H), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// A of joined spans stays above 0 where all of theirs are (low: the least of them, as bits): a product below the smallest number, 1.4e-45, becomes that
// number (no further off than the rounding of any product down there), so that an infinite state stays infinite as it does token by token; a decay of
// exactly 0 makes it NaN in either form.  The bits of numbers that are not negative are ordered as the numbers are, NaN highest: it stays.
__device__ __forceinline__ float above_zero(float A, unsigned low) { return __uint_as_float(max(__float_as_uint(A), min(low, 1u))); }
// the same for the product of a lane's L decays, g(i, k) of channel k: looked at again only where one came out as 0
template <int L, int V, typename G> __device__ __forceinline__ void lane_decay(float (&pa)[V], G g) {
    unsigned least = __float_as_uint(pa[0]);
#pragma unroll
    for (int k = 1; k < V; ++k) least = min(least, __float_as_uint(pa[k]));
    if (least == 0)
#pragma unroll
        for (int k = 0; k < V; ++k) {
            unsigned low = 1;
#pragma unroll
            for (int i = 0; i < L; ++i) low = min(low, __float_as_uint(g(i, k)));
            pa[k] = above_zero(pa[k], low);
        }
}

// state behind a span, from the state in front of it; CUTS: may documents start in it?
template <bool CUTS> __device__ __forceinline__ float pass(float A, float H, float h) {
    const float r = fmaf(A, h, H);
    return CUTS && A == LOOP_CUT ? H : r;
}
// (A, H) := (A, H) then (A2, H2).  A run of spans keeps the least A on the way and looks at the product at its end (above_zero): one step of a chain less.
template <bool CUTS> __device__ __forceinline__ void join(float& A, float& H, float A2, float H2, unsigned& low) {
    H = pass<CUTS>(A2, H2, H);
    low = min(low, __float_as_uint(A2));
    const float r = A * A2;
    A = CUTS && (A == LOOP_CUT || A2 == LOOP_CUT) ? LOOP_CUT : r;
}
template <bool CUTS> __device__ __forceinline__ void join(float& A, float& H, float A2, float H2) {
    unsigned low = __float_as_uint(A);
    join<CUTS>(A, H, A2, H2, low);
    A = above_zero(A, low);
}

// Tiles are dealt to `nq` queues of neighbours, workgroup i draws from queue i % nq: with 8 queues neighbouring tiles, which share cache lines
// where rows are not whole lines, stay on one XCD (workgroups go to the XCDs in turn; nothing but speed depends on it).
struct SpanWork {
    unsigned* ticket;              // one per queue, 64 bytes apart
    u64* pairs;                    // [block][tile][channel of the tile]
    u64* groups;                   // [1 + group][tile][channel of the tile]: the pair of the group, or behind the last group of a set the state
    int nblk, ntile, ctiles, nq;
};

// (block in the direction of the recurrence, tile) of this workgroup; false: its queue is empty, the workgroup ends
__device__ __forceinline__ bool span_place(const SpanWork& W, int& kb, int& tile) {
    __shared__ unsigned drawn;
    if (W.nblk == 1) { kb = 0; tile = blockIdx.x; return true; }
    const unsigned x = blockIdx.x % (unsigned)W.nq;
    if (threadIdx.x == 0) drawn = __hip_atomic_fetch_add(W.ticket + 16 * x, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    const unsigned each = (unsigned)W.ntile / (unsigned)W.nq, more = (unsigned)W.ntile % (unsigned)W.nq;      // the first `more` queues hold one tile more
    const unsigned cnt = each + (x < more), lo = each * x + min(x, more);
    kb = (int)(drawn / cnt); tile = (int)(lo + drawn % cnt);
    return kb < W.nblk;
}

// State of the recurrence in front of this workgroup's block for channel ch (thread = (ch, seg), SEGS threads per channel).  kb counts blocks in
// the direction of the recurrence, (A, H) is the whole block's pair (known to the threads of the last segment, which publish it), `first` what
// block 0 starts from (the same threads).  nearA, nearH: scratch.  All threads enter; everyone gets the state.
template <int NCH, int SEGS, bool CUTS>
__device__ __forceinline__ float span_carry(const SpanWork& W, int kb, int tile, int ch, int seg, bool ok, float first, float A, float H,
                                            float (*nearA)[NCH], float (*nearH)[NCH]) {
    __shared__ float farA[SEGS][NCH], farH[SEGS][NCH];
    const bool tail = seg == SEGS - 1;
    const unsigned pitch = (unsigned)W.ntile * NCH, mine = (unsigned)tile * NCH + ch;      // words: 32 bits by the launch's limit on workgroups
    if (kb == 0) {
        if (tail) {
            nearH[0][ch] = first;
            // block 0 publishes a state rather than a pair: whoever depends on it does not read `first` again, which may be overwritten by then
            if (ok && W.nblk > 1) publish(W.pairs + mine, LOOP_CUT, pass<CUTS>(A, H, first));
        }
        __syncthreads();
        return nearH[0][ch];
    }
    const int grp = kb / LOOP_GROUP, in = kb % LOOP_GROUP, set = grp / LOOP_SET, gin = grp % LOOP_SET;
    const bool last = in == LOOP_GROUP - 1;
    if (ok && tail && !last) publish(W.pairs + ((unsigned)kb * pitch + mine), A, H);
    // waits for the entries from .. to - 1 of those at `row` of `words`, this thread's share of them, and leaves their join in (a, h)
    float a, h;
    auto gather = [&](auto most, const u64* words, int row, int from, int to) {
        constexpr int M = (decltype(most)::value + SEGS - 1) / SEGS;
        a = 1.f; h = 0.f;
        if (!ok) return;
        u64 w[M];
#pragma unroll
        for (int j = 0; j < M; ++j) w[j] = 0;
        bool all;
        do {
            all = true;
#pragma unroll
            for (int j = 0; j < M; ++j) {
                const int e = seg * M + j;
                if (e >= from && e < to && !pair_there(w[j])) {
                    w[j] = __hip_atomic_load(words + ((unsigned)(row + e) * pitch + mine), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    all = all && pair_there(w[j]);
                }
            }
            if (!all) __builtin_amdgcn_s_sleep(1);
        } while (!all);
#pragma unroll
        for (int j = 0; j < M; ++j)
            if (pair_there(w[j])) join<true>(a, h, pair_A(w[j]), pair_H(w[j]));
    };
    const bool behind = last && kb + 1 < W.nblk && ok && tail;      // publishes what lies behind the group
    gather(std::integral_constant<int, LOOP_GROUP>(), W.pairs, grp * LOOP_GROUP, 0, in);
    nearA[seg][ch] = a; nearH[seg][ch] = h;
    if (last) {
        __syncthreads();
        if (behind && gin < LOOP_SET - 1) {
            a = 1.f; h = 0.f;
            for (int s = 0; s < SEGS; ++s) join<true>(a, h, nearA[s][ch], nearH[s][ch]);
            join<true>(a, h, A, H);
            publish(W.groups + ((unsigned)(grp + 1) * pitch + mine), a, h);
        }
    }
    if (grp > 0) {
        gather(std::integral_constant<int, LOOP_SET>(), W.groups, set * LOOP_SET, set > 0 ? 0 : 1, gin + 1);
        farA[seg][ch] = a; farH[seg][ch] = h;
    }
    __syncthreads();
    h = 0.f;                                                  // the first entry of all is a state: nothing in front of it counts
    if (grp > 0)
#pragma unroll
        for (int s = 0; s < SEGS; ++s) h = pass<true>(farA[s][ch], farH[s][ch], h);
#pragma unroll
    for (int s = 0; s < SEGS; ++s) h = pass<true>(nearA[s][ch], nearH[s][ch], h);
    if (behind && gin == LOOP_SET - 1) publish(W.groups + ((unsigned)(grp + 1) * pitch + mine), LOOP_CUT, pass<CUTS>(A, H, h));
    return h;
}

// Lane rows of a workgroup, ROWS of them, in LDS: row r's pair at rowA[r], rowH[r].  Replaces rowH[r] by the state in front of row r (REV: the
// recurrence runs from the last row to the first).  partA / partH: SEGS rows of scratch each.  All threads enter, after a barrier; leaves behind one.
template <int NCH, int SEGS, int ROWS, bool REV, bool CUTS>
__device__ __forceinline__ void span_join(const SpanWork& W, int kb, int tile, bool ok, float first, const float (*rowA)[NCH], float (*rowH)[NCH],
                                          float (*partA)[NCH], float (*partH)[NCH], float (*prevA)[NCH], float (*prevH)[NCH]) {
    constexpr int RPS = ROWS / SEGS;
    const int ch = threadIdx.x % NCH, seg = threadIdx.x / NCH;
    float A = 1.f, H = 0.f;
    unsigned low = 1;
#pragma unroll
    for (int j = 0; j < RPS; ++j) {
        const int r = REV ? ROWS - 1 - (seg * RPS + j) : seg * RPS + j;
        join<CUTS>(A, H, rowA[r][ch], rowH[r][ch], low);
    }
    A = above_zero(A, low);
    partA[seg][ch] = A; partH[seg][ch] = H;
    __syncthreads();
    float fa = 1.f, fh = 0.f;                                 // everything in front of this segment
    for (int s = 0; s < seg; ++s) join<CUTS>(fa, fh, partA[s][ch], partH[s][ch]);
    join<CUTS>(A = fa, H = fh, partA[seg][ch], partH[seg][ch]);
    const float h0 = span_carry<NCH, SEGS, CUTS>(W, kb, tile, ch, seg, ok, first, A, H, prevA, prevH);
    float h = pass<CUTS>(fa, fh, h0);
#pragma unroll
    for (int j = 0; j < RPS; ++j) {
        const int r = REV ? ROWS - 1 - (seg * RPS + j) : seg * RPS + j;
        const float pA = rowA[r][ch], pH = rowH[r][ch];       // read again: held over the wait they would be 16 registers
        rowH[r][ch] = h;
        h = pass<CUTS>(pA, pH, h);
    }
    __syncthreads();
}

__global__ __launch_bounds__(256) void span_clear_kernel(u64* p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

template <typename E, int V, bool RAG, int CL, int WAVES, int TW, bool CUTS, bool S>
__global__ __launch_bounds__(WAVES * 64) void loop_span_fwd_kernel(LoopArgs A, SpanWork W, const void* __restrict__ q, const void* __restrict__ kv,
                                                                   const void* __restrict__ a, const float* h0, void* __restrict__ y, float* hlast,
                                                                   float* __restrict__ states) {
    constexpr int TL = 64 / CL, L = TW / TL, NCH = CL * V, SPAN = WAVES * TW, ROWS = WAVES * TL, SEGS = WAVES * 64 / NCH;
    __shared__ __attribute__((aligned(16))) float rowA[ROWS][NCH], rowH[ROWS][NCH];
    __shared__ float partA[SEGS][NCH], partH[SEGS][NCH], prevA[SEGS][NCH], prevH[SEGS][NCH];
    int kb, tile;
    if (!span_place(W, kb, tile)) return;
    const int ct = tile % W.ctiles, seq = tile / W.ctiles, b = seq / A.P, p = seq % A.P;
    const int row = threadIdx.x / CL, cl = threadIdx.x % CL;
    const int n = live_tokens(A, b), b0 = kb * SPAN, t0 = b0 + row * L;
    const int c = ct * NCH + cl * V;
    const bool cok = c < A.C, whole = b0 + SPAN <= n;         // whole: every token of the block exists
    const int cc = cok ? c : 0, nv = RAG ? min(V, A.C - cc) : V;      // elements of the chunk

    RowVec<E, V, RAG> vq[L], vk[L], va[L];
    unsigned cuts = 0;
    if (b0 < n) {
        const int64_t in0 = (int64_t)b * A.sb + (int64_t)p * A.sp + cc;
        unsigned char start[L];                               // read first: rows may still be on their way when these are needed (read behind them 60 us, 55)
        if (CUTS)
#pragma unroll
            for (int i = 0; i < L; ++i) start[i] = A.resets[(int64_t)b * A.T + min(t0 + i, n - 1)];
#pragma unroll
        for (int i = 0; i < L; ++i) {                         // rows behind the last token are not read: the last one stands in for them
            const int64_t at = in0 + (int64_t)min(t0 + i, n - 1) * A.st;
            va[i].template load<S>(a, at, nv); vk[i].template load<S>(kv, at, nv); vq[i].template load<S>(q, at, nv);
        }
#pragma unroll
        for (int i = 0; i < L; ++i) { va[i].settle(nv); vk[i].settle(nv); vq[i].settle(nv); }
        if (CUTS)
#pragma unroll
            for (int i = 0; i < L; ++i) cuts |= (t0 + i < n && start[i]) ? 1u << i : 0u;
    } else {
#pragma unroll
        for (int i = 0; i < L; ++i) { va[i].clear(); vk[i].clear(); vq[i].clear(); }
    }
    if (!whole) {                                             // a token that does not exist lets the state pass: decay 1, nothing added
#pragma unroll
        for (int i = 0; i < L; ++i)
            if (t0 + i >= n) { va[i].infinite(); vk[i].clear(); }
    }
    float g[L][V];
    {
        float pa[V], ph[V];
#pragma unroll
        for (int k = 0; k < V; ++k) { pa[k] = 1.f; ph[k] = 0.f; }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            float fk[V], fa[V];
            vk[i].get(fk); va[i].get(fa);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                g[i][k] = sigm<E>(fa[k]);
                pa[k] *= g[i][k];
            }
#pragma unroll
            for (int k = 0; k < V; ++k) ph[k] = fmaf(g[i][k], ph[k], fk[k]);
            if (CUTS)
#pragma unroll
                for (int k = 0; k < V; ++k) ph[k] = cuts >> i & 1 ? fk[k] : ph[k];
        }
        lane_decay<L, V>(pa, [&](int i, int k) { return g[i][k]; });
#pragma unroll
        for (int k = 0; k < V; ++k) { rowA[row][cl * V + k] = CUTS && cuts ? LOOP_CUT : pa[k]; rowH[row][cl * V + k] = ph[k]; }
    }
    __syncthreads();
    const int chn = threadIdx.x % NCH, chc = ct * NCH + chn;
    const bool chok = chc < A.C;
    const float first = kb == 0 && h0 && chok && threadIdx.x >= (SEGS - 1) * NCH ? h0[(int64_t)seq * A.C + chc] : 0.f;
    span_join<NCH, SEGS, ROWS, false, CUTS>(W, kb, tile, chok, first, rowA, rowH, partA, partH, prevA, prevH);

    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = rowH[row][cl * V + k];
    if (states && cok && t0 > 0 && t0 < n && (t0 & (A.keep - 1)) == 0) {      // a block of the backward pass begins here
        float* o = states + (((int64_t)b * A.nstate + t0 / A.keep - 1) * A.P + p) * A.C + c;
#pragma unroll
        for (int k = 0; k < V; ++k) if (k < nv) o[k] = h[k];
    }
    const int64_t yt = (int64_t)A.P * A.C, y0 = ((int64_t)b * A.T * A.P + p) * A.C + c;
#pragma unroll
    for (int i = 0; i < L; ++i) {
        float fk[V], fq[V];
        vk[i].get(fk); vq[i].get(fq);
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = fmaf(g[i][k], h[k], fk[k]);
        if (CUTS)
#pragma unroll
            for (int k = 0; k < V; ++k) h[k] = cuts >> i & 1 ? fk[k] : h[k];
#pragma unroll
        for (int k = 0; k < V; ++k) fq[k] *= h[k];
        if (!whole && t0 + i >= n)
#pragma unroll
            for (int k = 0; k < V; ++k) fq[k] = 0.f;
        if (cok && t0 + i < A.T) RowVec<E, V, RAG>::template store<S>(y, y0 + (t0 + i) * yt, fq, nv);
    }
    if (hlast && cok && kb == W.nblk - 1 && row == ROWS - 1) {
#pragma unroll
        for (int k = 0; k < V; ++k) if (k < nv) hlast[(int64_t)seq * A.C + c + k] = h[k];
    }
}

// The same from the last token to the first for D.  The states in front of a block's tokens are formed again from the kept state.  Held per
// element: m = min(g, 1 - g) with the sign of a, from which g and g (1 - g) follow without a cancellation and without another exponential.
template <typename E, int V, bool RAG, int CL, int WAVES, int TW, bool CUTS, bool S>
__global__ __launch_bounds__(WAVES * 64, 4) void loop_span_bwd_kernel(LoopArgs A, SpanWork W, const void* __restrict__ q, const void* __restrict__ kv,
                                                                   const void* __restrict__ a, const float* __restrict__ h0, const float* __restrict__ states,
                                                                   const void* __restrict__ dy, const float* __restrict__ dhlast, void* __restrict__ dq,
                                                                   void* __restrict__ dkv, void* __restrict__ da, float* __restrict__ dh0) {
    constexpr int TL = 64 / CL, L = TW / TL, NCH = CL * V, SPAN = WAVES * TW, ROWS = WAVES * TL, SEGS = WAVES * 64 / NCH, RPS = ROWS / SEGS;
    __shared__ __attribute__((aligned(16))) float rowA[ROWS][NCH], rowH[ROWS][NCH], rowU[ROWS][NCH];
    __shared__ float partA[SEGS][NCH], partH[SEGS][NCH], prevA[SEGS][NCH], prevH[SEGS][NCH];
    int back_kb, tile;
    if (!span_place(W, back_kb, tile)) return;
    const int kb = W.nblk - 1 - back_kb;
    const int ct = tile % W.ctiles, seq = tile / W.ctiles, b = seq / A.P, p = seq % A.P;
    const int row = threadIdx.x / CL, cl = threadIdx.x % CL;
    const int n = live_tokens(A, b), b0 = kb * SPAN, t0 = b0 + row * L;
    const int c = ct * NCH + cl * V;
    const bool cok = c < A.C, whole = b0 + SPAN <= n;
    const int cc = cok ? c : 0, nv = RAG ? min(V, A.C - cc) : V;      // elements of the chunk
    const int chn = threadIdx.x % NCH, seg = threadIdx.x / NCH, chc = ct * NCH + chn;
    const bool chok = chc < A.C;
    const int64_t yt = (int64_t)A.P * A.C, y0 = ((int64_t)b * A.T * A.P + p) * A.C + cc;

    RowVec<E, V, RAG> vq[L], vk[L], vy[L];
    float m[L][V];
    unsigned cuts = 0;
    float hin = 0.f;                                          // kept state in front of the block, channel chn
    {
        RowVec<E, V, RAG> va[L];
        if (b0 < n) {
            const int64_t in0 = (int64_t)b * A.sb + (int64_t)p * A.sp + cc;
            unsigned char start[L];
            if (CUTS)
#pragma unroll
                for (int i = 0; i < L; ++i) start[i] = A.resets[(int64_t)b * A.T + min(t0 + i, n - 1)];
#pragma unroll
            for (int i = 0; i < L; ++i) {
                const int t = min(t0 + i, n - 1);
                const int64_t at = in0 + (int64_t)t * A.st;
                va[i].template load<S>(a, at, nv); vk[i].template load<S>(kv, at, nv); vq[i].template load<S>(q, at, nv); vy[i].template load<S>(dy, y0 + t * yt, nv);
            }
#pragma unroll
            for (int i = 0; i < L; ++i) { va[i].settle(nv); vk[i].settle(nv); vq[i].settle(nv); vy[i].settle(nv); }
            if (CUTS)
#pragma unroll
                for (int i = 0; i < L; ++i) cuts |= (t0 + i < n && start[i]) ? 1u << i : 0u;
            if (chok) {
                if (kb > 0) hin = states[(((int64_t)b * A.nstate + kb - 1) * A.P + p) * A.C + chc];
                else if (h0) hin = h0[(int64_t)seq * A.C + chc];
            }
        } else {
#pragma unroll
            for (int i = 0; i < L; ++i) { va[i].clear(); vk[i].clear(); vq[i].clear(); vy[i].clear(); }
        }
        if (!whole) {                                         // a token that does not exist: decay 1, nothing added in either direction
#pragma unroll
            for (int i = 0; i < L; ++i)
                if (t0 + i >= n) { va[i].infinite(); vk[i].clear(); vq[i].clear(); vy[i].clear(); }
        }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            float fa[V];
            va[i].get(fa);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float e = Gate<E>::ex(-fabsf(fa[k]));
                m[i][k] = copysignf(e * Gate<E>::recip(1.f + e), fa[k]);
            }
        }
    }
    auto decay = [&](int i, int k) { const float v = m[i][k]; return signbit(v) ? -v : 1.f - v; };
    {
        float pa[V], ph[V], pu[V];
#pragma unroll
        for (int k = 0; k < V; ++k) { pa[k] = 1.f; ph[k] = pu[k] = 0.f; }
#pragma unroll
        for (int i = 0; i < L; ++i) {
            float fk[V];
            vk[i].get(fk);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const float g = decay(i, k);
                ph[k] = fmaf(g, ph[k], fk[k]);
                pa[k] *= g;
            }
            if (CUTS)
#pragma unroll
                for (int k = 0; k < V; ++k) ph[k] = cuts >> i & 1 ? fk[k] : ph[k];
        }
#pragma unroll
        for (int i = L - 1; i >= 0; --i) {
            float fq[V], fy[V];
            vq[i].get(fq); vy[i].get(fy);
#pragma unroll
            for (int k = 0; k < V; ++k) pu[k] = decay(i, k) * fmaf(fq[k], fy[k], pu[k]);
            if (CUTS)
#pragma unroll
                for (int k = 0; k < V; ++k) pu[k] = cuts >> i & 1 ? 0.f : pu[k];
        }
        lane_decay<L, V>(pa, decay);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            rowA[row][cl * V + k] = CUTS && cuts ? LOOP_CUT : pa[k];
            rowH[row][cl * V + k] = ph[k]; rowU[row][cl * V + k] = pu[k];
        }
    }
    __syncthreads();
    {   // states in front of the lane rows: from the kept state
        float ra[RPS], rh[RPS], pA = 1.f, pH = 0.f;
        unsigned low = 1;
#pragma unroll
        for (int j = 0; j < RPS; ++j) {
            ra[j] = rowA[seg * RPS + j][chn]; rh[j] = rowH[seg * RPS + j][chn];
            join<CUTS>(pA, pH, ra[j], rh[j], low);
        }
        prevA[seg][chn] = above_zero(pA, low); prevH[seg][chn] = pH;
        __syncthreads();
        float h = hin;
        for (int s = 0; s < seg; ++s) h = pass<CUTS>(prevA[s][chn], prevH[s][chn], h);
#pragma unroll
        for (int j = 0; j < RPS; ++j) {
            rowH[seg * RPS + j][chn] = h;
            h = pass<CUTS>(ra[j], rh[j], h);
        }
    }
    const float first = back_kb == 0 && dhlast && chok && seg == SEGS - 1 ? dhlast[(int64_t)seq * A.C + chc] : 0.f;
    // (the barrier inside, between its use of partA and of prevA, keeps prevA apart from its use above)
    span_join<NCH, SEGS, ROWS, true, CUTS>(W, back_kb, tile, chok, first, rowA, rowU, partA, partH, prevA, prevH);

    float h[L + 1][V], back[V];
#pragma unroll
    for (int k = 0; k < V; ++k) { h[0][k] = rowH[row][cl * V + k]; back[k] = rowU[row][cl * V + k]; }
    const int64_t g0 = (int64_t)b * A.gb + (int64_t)p * A.gp + c;
#pragma unroll
    for (int i = 0; i < L; ++i) {
        float fk[V], fy[V];
        vk[i].get(fk); vy[i].get(fy);
#pragma unroll
        for (int k = 0; k < V; ++k) h[i + 1][k] = fmaf(decay(i, k), h[i][k], fk[k]);
        if (CUTS)
#pragma unroll
            for (int k = 0; k < V; ++k) h[i + 1][k] = cuts >> i & 1 ? fk[k] : h[i + 1][k];
#pragma unroll
        for (int k = 0; k < V; ++k) fy[k] *= h[i + 1][k];
        if (!whole && t0 + i >= n)
#pragma unroll
            for (int k = 0; k < V; ++k) fy[k] = 0.f;
        if (cok && t0 + i < A.T) RowVec<E, V, RAG>::template store<S>(dq, g0 + (t0 + i) * A.gt, fy, nv);
    }
#pragma unroll
    for (int i = L - 1; i >= 0; --i) {
        float fq[V], fy[V], oa[V];
        vq[i].get(fq); vy[i].get(fy);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            const float s = fabsf(m[i][k]);
            fq[k] = fmaf(fq[k], fy[k], back[k]);
            oa[k] = fq[k] * h[i][k] * (s * (1.f - s));
            back[k] = decay(i, k) * fq[k];
        }
        if (CUTS)
#pragma unroll
            for (int k = 0; k < V; ++k) {
                oa[k] = cuts >> i & 1 ? 0.f : oa[k];
                back[k] = cuts >> i & 1 ? 0.f : back[k];
            }
        if (!whole && t0 + i >= n)
#pragma unroll
            for (int k = 0; k < V; ++k) { back[k] = fq[k]; fq[k] = 0.f; oa[k] = 0.f; }
        if (cok && t0 + i < A.T) {
            const int64_t at = g0 + (t0 + i) * A.gt;
            RowVec<E, V, RAG>::template store<S>(dkv, at, fq, nv); RowVec<E, V, RAG>::template store<S>(da, at, oa, nv);
        }
    }
    if (dh0 && cok && kb == 0 && row == 0) {
#pragma unroll
        for (int k = 0; k < V; ++k) if (k < nv) dh0[(int64_t)seq * A.C + c + k] = back[k];
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
    if ((double)d->B * d->P * d->C > 4294967040.0) return MV2_ETOOLARGE;      // threads of a launch: 32 bits
    return MV2_OK;
}

// Which form runs: one thread per chunk where the tokens are few for that many channels, spans otherwise.  A function of the sizes alone (the
// backward pass finds the states that the forward pass kept), counted in the spans' tiles of 8 chunks, which rows shorter than a tile leave partly
// empty.  A walk takes 0.35 us a token (backward 0.65) until the memory is busy, a span of up to 256 tokens some 5 us and as much again for every 512
// (256) tiles.  Above 8192 tiles walks are near the memory's rate at any length.  Measured, bf16, us forward / backward, walk : span:
//     64 tiles, 8 tokens 4.8 / 6.1 : 5.2 / 5.9        16 tokens 7.0 / 10 : 5.2 / 5.8
//   2048 tiles, 40 tokens 16 / 27 : 22 / 27           48 tokens 18 / 34 : 22 / 28
//   6144 tiles, 96 tokens 63 / 124 : 71 / 111         200 tokens 124 / 249 : 128 / 224
//   8192 tiles, 192 tokens 159 / 303 : 165 / 281      1024 tokens 809 / 1570 : 721 / 1271
//   4096 rows of 8 channels, 40 tokens 15 / 24 : 38 / 46, 200 tokens 58 / 121 : 50 / 132
//  16384 rows of 5 channels, 200 tokens 60 / 175 : 505 / 619, 1000 tokens 285 / 871 : 2097 / 2602
// The last bound is for the narrow rows; whole tiles of so many channels over hundreds of tokens are some 15 % slower than spans for it.
static bool loop_walks(const mv2_gateloop_desc* d) {
    const int nch = d->dtype == MV2_BF16 ? 64 : 32;
    const int64_t tiles = (int64_t)d->B * d->P * ((d->C + nch - 1) / nch);
    return tiles >= 8192 || d->T <= 8 + tiles / 64;
}

// Spans are of SPAN_WAVES waves of 32 tokens forward, and backward of 16 tokens where that lets two workgroups live on a CU by their registers
// (128 against 216 in bf16: 8 x 2048 x 2048 97 us, 106 with 32 tokens, 1 x 131072 x 512 196 and 207; fp32 fits with 32: 8 x 2048 x 1024 94 us, 96
// with 16, 1 x 131072 x 256 169 and 177, but 3 x 1023 x 776 19.4 and 18.4) and for rows shorter than a chunk.
#define SPAN_WAVES 8
static int span_tokens(const mv2_gateloop_desc* d, bool backward) {
    return SPAN_WAVES * (!backward || (d->dtype == MV2_F32 && d->C >= 4) ? 32 : 16);
}
static int loop_keep(const mv2_gateloop_desc* d) { return loop_walks(d) ? LOOP_STEPS : span_tokens(d, true); }

extern "C" int64_t mv2_gateloop_states(const mv2_gateloop_desc* d) {
    const int rc = loop_check(d);
    if (rc != MV2_OK) return rc;
    return d->T > 0 ? (d->T - 1) / loop_keep(d) : 0;
}

struct SpanShape { int64_t nblk, ctiles, ntile, nq, words; };
static SpanShape span_shape(const mv2_gateloop_desc* d, int nch, bool backward) {
    SpanShape s;
    const int span = span_tokens(d, backward);
    s.nblk = (d->T + span - 1) / span;
    s.ctiles = (d->C + nch - 1) / nch;
    s.ntile = s.ctiles * d->B * d->P;
    // queues per XCD, forward: 4 x 8192 x 768 bf16 48 us against 50 from one queue, rows that are not whole lines 6 x 4095 x 1000 53 against 61;
    // backward for those (92 us against 108); whole lines are drawn from one there, 1 to 4 % behind eight (8 x 2048 x 2048 97 us and 95, 4 x 8192 x
    // 768 79 and 76).  Few tiles would leave XCDs idle.
    const int64_t es = d->dtype == MV2_BF16 ? 2 : 4;
    s.nq = s.ntile >= 32 && (!backward || d->in_t * es % 128 != 0) ? 8 : 1;
    s.words = s.nblk > 1 ? 64 + (s.nblk + s.nblk / LOOP_GROUP + 1) * s.ntile * nch : 0;
    return s;
}
// channels of a workgroup: 128-byte pieces of rows (64 bf16 or, in chunks of four, 32 fp32), 64 single elements of rows that are not whole chunks
static int span_channels(bool fours) { return fours ? 32 : 64; }

extern "C" size_t mv2_gateloop_workspace_bytes(const mv2_gateloop_desc* d, int backward) {
    if (loop_check(d) != MV2_OK || loop_walks(d)) return 0;
    int64_t words = 0;
    for (int fours = 0; fours < 2; ++fours) words = std::max(words, span_shape(d, span_channels(fours), backward != 0).words);      // whichever the addresses allow
    return (size_t)words * sizeof(u64);
}

static int loop_access(const mv2_gateloop_desc* d, bool backward, std::initializer_list<const void*> ps) {
    const int64_t es = d->dtype == MV2_BF16 ? 2 : 4, g = backward ? es : 0;
    return rows_access(d->dtype, d->C, ps, {d->in_b * es, d->in_t * es, d->in_p * es, d->grad_b * g, d->grad_t * g, d->grad_p * g});
}

// past the caches: large calls whose rows are whole lines (where lines are shared by tiles, the caches bring the second half: 6 x 4095 x 1000 bf16
// 52 us forward through them, 65 past)
static bool loop_streams(const mv2_gateloop_desc* d, int tensors) {
    const int64_t es = d->dtype == MV2_BF16 ? 2 : 4;
    return d->C * es % 128 == 0 && d->in_t * es % 128 == 0 && calls_stream((double)d->B * d->T * d->P * d->C * es * tensors);
}

static LoopArgs loop_args(const mv2_gateloop_desc* d, const int32_t* lengths, const unsigned char* resets) {
    LoopArgs A;
    A.B = d->B; A.T = d->T; A.P = d->P; A.C = d->C;
    A.sb = d->in_b; A.st = d->in_t; A.sp = d->in_p; A.gb = d->grad_b; A.gt = d->grad_t; A.gp = d->grad_p;
    A.lengths = lengths; A.resets = resets;
    A.nstate = (int)mv2_gateloop_states(d); A.keep = loop_keep(d);
    return A;
}

// threads of a launch, and with them the words' indexes: 32 bits
static bool span_fits(const SpanShape& s) { return (double)s.nblk * (s.ntile + 8) * 64 * SPAN_WAVES <= 4294967040.0; }

// the pairs' words, cleared by a kernel (a captured memset would not do: the launch may be recorded into a graph)
static int span_work(const mv2_gateloop_desc* d, bool fours, bool backward, void* workspace, size_t workspace_bytes, hipStream_t st, SpanWork& W, unsigned& grid) {
    const int nch = span_channels(fours);
    const SpanShape s = span_shape(d, nch, backward);
    if (!span_fits(s)) return MV2_ETOOLARGE;
    W.nblk = (int)s.nblk; W.ntile = (int)s.ntile; W.ctiles = (int)s.ctiles;
    W.nq = (int)s.nq;
    grid = (unsigned)(s.nblk > 1 ? s.nblk * s.nq * ((s.ntile + s.nq - 1) / s.nq) : s.ntile);
    W.ticket = nullptr; W.pairs = W.groups = nullptr;
    if (s.words == 0) return MV2_OK;
    if (!workspace || ((uintptr_t)workspace & 7) || workspace_bytes < s.words * sizeof(u64)) return MV2_EWORKSPACE;
    W.ticket = (unsigned*)workspace;
    W.pairs = (u64*)workspace + 64;
    W.groups = W.pairs + s.nblk * s.ntile * nch;
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
    const int access = loop_access(d, false, {q, kv, a, y});
    const bool stream_past = loop_streams(d, 4);
    hipStream_t st = (hipStream_t)stream;
    if (loop_walks(d)) {
        const int V = access == 2 ? (d->dtype == MV2_BF16 ? 8 : 4) : 1;      // (ragged chunks: 4 x 17 x 1024 x 251 bf16 41 us, single elements 31)
        const int64_t n = (int64_t)d->B * d->P * (d->C / V);
        const dim3 grid((unsigned)((n + 255) / 256));
#define GO(E, V, S) hipLaunchKernelGGL((loop_walk_fwd_kernel<E, V, S>), grid, dim3(256), 0, st, A, q, kv, a, h0, y, h_last, states)
        if (d->dtype == MV2_BF16) { if (access == 2 && stream_past) GO(BF16, 8, true); else if (access == 2) GO(BF16, 8, false); else GO(BF16, 1, false); }
        else { if (access == 2 && stream_past) GO(F32, 4, true); else if (access == 2) GO(F32, 4, false); else GO(F32, 1, false); }
#undef GO
    } else {
        SpanWork W;
        unsigned grid;
        // states are kept for a backward pass, whose blocks are shorter: it is refused here rather than after the forward pass
        if (states && !span_fits(span_shape(d, span_channels(d->dtype == MV2_F32 && (int64_t)d->C * 4 >= 16), true))) return MV2_ETOOLARGE;
        rc = span_work(d, d->dtype == MV2_F32 && access, false, workspace, workspace_bytes, st, W, grid);
        if (rc != MV2_OK) return rc;
#define GO(E, V, RAG, CL, CUTS, S) hipLaunchKernelGGL((loop_span_fwd_kernel<E, V, RAG, CL, SPAN_WAVES, 32, CUTS, S>), dim3(grid), dim3(64 * SPAN_WAVES), 0, st, A, W, q, kv, a, h0, y, h_last, states)
#define GO2(E, V, RAG, CL, S) do { if (resets) GO(E, V, RAG, CL, true, S); else GO(E, V, RAG, CL, false, S); } while (0)
        if (d->dtype == MV2_BF16) { if (access == 2 && stream_past) GO2(BF16, 8, false, 8, true); else if (access == 2) GO2(BF16, 8, false, 8, false); else if (access) GO2(BF16, 8, true, 8, false); else GO2(BF16, 1, false, 64, false); }
        else { if (access == 2 && stream_past) GO2(F32, 4, false, 8, true); else if (access == 2) GO2(F32, 4, false, 8, false); else if (access) GO2(F32, 4, true, 8, false); else GO2(F32, 1, false, 64, false); }
#undef GO2
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
    const int access = loop_access(d, true, {q, kv, a, dy, dq, dkv, da});
    const bool stream_past = loop_streams(d, 7);
    hipStream_t st = (hipStream_t)stream;
    if (loop_walks(d)) {
        const int V = access ? (d->dtype == MV2_BF16 ? 4 : 2) : 1;
        const int64_t n = (int64_t)d->B * d->P * ((d->C + V - 1) / V);
        const dim3 grid((unsigned)((n + 255) / 256));
#define GO(E, V, RAG) hipLaunchKernelGGL((loop_walk_bwd_kernel<E, V, RAG>), grid, dim3(256), 0, st, A, q, kv, a, h0, states, dy, dh_last, dq, dkv, da, dh0)
        if (d->dtype == MV2_BF16) { if (access == 2) GO(BF16, 4, false); else if (access) GO(BF16, 4, true); else GO(BF16, 1, false); }
        else { if (access == 2) GO(F32, 2, false); else if (access) GO(F32, 2, true); else GO(F32, 1, false); }
#undef GO
    } else {
        SpanWork W;
        unsigned grid;
        rc = span_work(d, d->dtype == MV2_F32 && access, true, workspace, workspace_bytes, st, W, grid);
        if (rc != MV2_OK) return rc;
#define GO(E, V, RAG, CL, TW, CUTS, S)                                                                                                                                 \
    hipLaunchKernelGGL((loop_span_bwd_kernel<E, V, RAG, CL, SPAN_WAVES, TW, CUTS, S>), dim3(grid), dim3(64 * SPAN_WAVES), 0, st, A, W, q, kv, a, h0, states, dy, dh_last, dq, dkv, da, dh0)
#define GO2(E, V, RAG, CL, TW, S) do { if (resets) GO(E, V, RAG, CL, TW, true, S); else GO(E, V, RAG, CL, TW, false, S); } while (0)
        if (d->dtype == MV2_BF16) { if (access == 2 && stream_past) GO2(BF16, 8, false, 8, 16, true); else if (access == 2) GO2(BF16, 8, false, 8, 16, false); else if (access) GO2(BF16, 8, true, 8, 16, false); else GO2(BF16, 1, false, 64, 16, false); }
        else { if (access == 2 && stream_past) GO2(F32, 4, false, 8, 32, true); else if (access == 2) GO2(F32, 4, false, 8, 32, false); else if (access) GO2(F32, 4, true, 8, 32, false); else GO2(F32, 1, false, 64, 16, false); }
#undef GO2
#undef GO
    }
    MV2_LAUNCH_CHECK();
    return MV2_OK;
}
