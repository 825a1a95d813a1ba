// Row access of the kernels that serve any width and any strides: V elements of storage type E as one access.
//   RowVec<E, kVec>        16-byte chunks of rows, strides and addresses that are whole such chunks
//   RowVec<E, kVec, true>  ragged: 16-byte accesses at any element (the memory pipe takes them at the same rate: a copy of 256 MB runs at
//                          5.7 - 6.0 TB/s whatever the offsets); a row's last chunk holds nv < V elements and is read as the row's last V
//                          elements, moved down, with zeros behind them, and written in pieces of 8, 4 and 2 bytes.  Rows of V elements at least.
//   V = kVec / 2           half of either, for kernels that hold many rows in registers
//   V = 1                  single elements: rows shorter than a chunk, and kernels whose every wave would hold a row's end
// STREAM: past the caches, for calls that move more than the last-level cache holds (calls_stream).
#pragma once
#include "common.h"

template <int BYTES> struct RowBits;
template <> struct RowBits<16> { typedef i32x4 T; typedef i32x4 __attribute__((aligned(2))) Any; };
template <> struct RowBits<8> { typedef i32x2 T; typedef i32x2 __attribute__((aligned(2))) Any; };

typedef int __attribute__((aligned(2))) RowWord;

// N words moved down by `bytes` (of 4 N; whole words, or half words too if HALVES), zeros behind them.  By selects: written as one wide shift this
// becomes 64-bit shifts by a variable amount, and with the amount in a wave's last register those have given wrong results here (tools/check_spills.sh
// counts them: no kernel of the library holds one with its amount in a vector register).
template <int N, bool HALVES, typename W> __device__ __forceinline__ W moved_down(W v, int bytes) {
#pragma unroll
    for (int d = 1; d < N; d *= 2) {
        const bool by = bytes & 4 * d;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = by ? (i + d < N ? v[i + d < N ? i + d : i] : 0) : v[i];
    }
    if (HALVES) {
        const bool by = bytes & 2;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = by ? (int)__builtin_amdgcn_alignbit(i + 1 < N ? v[i + 1 < N ? i + 1 : i] : 0, v[i], 16) : v[i];
    }
    return v;
}

template <typename E, int V, bool RAGGED = false> struct RowVec {
    static constexpr int kBytes = V * E::kBytes;
    typedef RowBits<kBytes> B;
    typename B::T v;
    __device__ __forceinline__ void clear() { v = 0; }
    __device__ __forceinline__ void infinite() { v = E::kBytes == 2 ? 0x7f807f80 : 0x7f800000; }
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, int64_t i, int nv = V) {
        if (!RAGGED) {
            const typename B::T* q = (const typename B::T*)((const typename E::T*)p + i);
            v = STREAM ? __builtin_nontemporal_load(q) : *q;
        } else {
            v = *(const typename B::Any*)((const typename E::T*)p + i - (V - nv));
        }
    }
    // after the loads that belong together have been asked for, before any get()
    __device__ __forceinline__ void settle(int nv) {
        if (RAGGED && __any(nv < V)) v = moved_down<kBytes / 4, E::kBytes == 2>(v, E::kBytes * (V - nv));
    }
    __device__ __forceinline__ void get(float* f) const {
        if constexpr (kBytes == 16) Chunk<E>::unpack(v, f);
        else if constexpr (E::kBytes == 2) ld4<BF16>(&v, 0, f);
        else { f[0] = __int_as_float(v[0]); f[1] = __int_as_float(v[1]); }
    }
    static __device__ __forceinline__ typename B::T pack(const float* f) {
        if constexpr (kBytes == 16) return Chunk<E>::pack(f);
        else if constexpr (E::kBytes == 2) { typename B::T w; st4<BF16>(&w, 0, f); return w; }
        else return typename B::T{__float_as_int(f[0]), __float_as_int(f[1])};
    }
    template <bool STREAM = false> static __device__ __forceinline__ void store(void* p, int64_t i, const float* f, int nv = V) {
        if (!RAGGED) {
            typename B::T* q = (typename B::T*)((typename E::T*)p + i);
            if (STREAM) __builtin_nontemporal_store(pack(f), q);
            else *q = pack(f);
        } else if (nv == V) {
            *(typename B::Any*)((typename E::T*)p + i) = pack(f);
        } else {                                       // 8, 4 and 2 bytes of what there is
            typename B::T w = pack(f);
            char* q = (char*)((typename E::T*)p + i);
            const int bytes = nv * E::kBytes;
            if (kBytes == 16 && (bytes & 8)) {
                *(typename RowBits<8>::Any*)q = i32x2{w[0], w[1]};
                w = moved_down<kBytes / 4, false>(w, 8);
                q += 8;
            }
            if (bytes & 4) {
                *(RowWord*)q = w[0];
                w = moved_down<kBytes / 4, false>(w, 4);
                q += 4;
            }
            if (E::kBytes == 2 && (bytes & 2)) *(unsigned short*)q = (unsigned short)w[0];
        }
    }
};
template <typename E> struct RowVec<E, 1, false> {
    typename E::T v;
    __device__ __forceinline__ void clear() { v = 0; }
    __device__ __forceinline__ void infinite() { st_elem<E>(&v, 0, __uint_as_float(0x7f800000u)); }
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, int64_t i, int = 1) { v = ((const typename E::T*)p)[i]; }
    __device__ __forceinline__ void settle(int) {}
    __device__ __forceinline__ void get(float* f) const { f[0] = ld_elem<E>(&v, 0); }
    template <bool STREAM = false> static __device__ __forceinline__ void store(void* p, int64_t i, const float* f, int = 1) { st_elem<E>(p, i, f[0]); }
};

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

// Does a call that moves this many bytes go past the caches (16-byte accesses only)?  From what the 256 MB last-level cache holds on: what a
// smaller call reads may still be there, and what it writes is read there next.  Measured, whole lines: block norm of 16384 x 2048 bf16 71 us
// forward and 123 backward through the caches, 65 and 118 past them; gate loop of 8 x 2048 x 2048 59 and 101, 55 and 97.
static inline bool calls_stream(double bytes) { return bytes >= 256.0 * 1024 * 1024; }

// how rows of C elements are accessed: whole 16-byte chunks (2), 16 bytes at any element (1), single elements (0).  `bytes`: everything that has to
// be whole chunks for the first.
static inline int rows_access(int dtype, int C, std::initializer_list<const void*> ps, std::initializer_list<int64_t> bytes) {
    const int es = dtype == MV2_BF16 ? 2 : 4;
    uintptr_t any = (uintptr_t)C * es;
    for (const void* p : ps) any |= (uintptr_t)p;
    for (int64_t b : bytes) any |= (uintptr_t)b;
    return !(any & 15) ? 2 : C * es >= 16 ? 1 : 0;
}

// Sum over a group of G neighbouring lanes (a power of two up to 64), in every lane, without LDS: pairs, quads, eights and rows of 16 by DPP,
// 16 and 32 apart by the row swaps of gfx950 (a register swapped with itself holds the value and its partner's).
__device__ __forceinline__ float dpp_add(float v, const int ctrl) {
    switch (ctrl) {
        case 0: return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0xB1, 0xf, 0xf, true));      // quad_perm 1 0 3 2
        case 1: return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x4E, 0xf, 0xf, true));      // quad_perm 2 3 0 1
        case 2: return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x141, 0xf, 0xf, true));     // row_half_mirror
        default: return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x140, 0xf, 0xf, true));    // row_mirror
    }
}
template <int N> __device__ __forceinline__ void lanes_sum(float (&v)[N], int G) {
#pragma unroll
    for (int step = 0; step < 4; ++step)
        if (G >> (step + 1))
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = dpp_add(v[i], step);
    if (G >= 32)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
            v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
    if (G >= 64)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[i]), __float_as_uint(v[i]), false, false);
            v[i] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
        }
}
