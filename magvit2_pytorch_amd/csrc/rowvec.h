// Row access of the kernels that serve any width and any strides: V elements of storage type E as one access - 16 bytes where the
// rows, strides and addresses are whole 16-byte chunks (V = E::kVec; V = E::kVec / 2: 8 bytes, half a chunk, for kernels that hold many rows
// in registers), pairs of 16-bit elements where only 4 bytes are whole (V = 2), one element otherwise (V = 1).
#pragma once
#include "common.h"

template <typename E, int V> struct RowVec {
    static_assert(V == E::kVec, "a 16-byte chunk or one element");
    i32x4 v;
    __device__ __forceinline__ void clear() { v = i32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void infinite() { const int w = E::kBytes == 2 ? 0x7f807f80 : 0x7f800000; v = i32x4{w, w, w, w}; }
    // STREAM: past the caches, for calls that move more than the last-level cache holds (calls_stream)
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, int64_t i) {
        const i32x4* q = (const i32x4*)((const typename E::T*)p + i);
        v = STREAM ? __builtin_nontemporal_load(q) : *q;
    }
    __device__ __forceinline__ void get(float* f) const { Chunk<E>::unpack(v, f); }
    template <bool STREAM = false> static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) {
        i32x4* q = (i32x4*)((typename E::T*)p + i);
        if (STREAM) __builtin_nontemporal_store(Chunk<E>::pack(f), q);
        else *q = Chunk<E>::pack(f);
    }
};
struct RowHalf {
    i32x2 v;
    __device__ __forceinline__ void clear() { v = i32x2{0, 0}; }
    template <typename T> __device__ __forceinline__ void load_at(const void* p, int64_t i) { v = *(const i32x2*)((const T*)p + i); }
};
template <> struct RowVec<BF16, 4> : RowHalf {
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, int64_t i) { load_at<unsigned short>(p, i); }
    __device__ __forceinline__ void get(float* f) const { ld4<BF16>(&v, 0, f); }
    template <bool STREAM = false> static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { st4<BF16>(p, i, f); }
};
template <> struct RowVec<F32, 2> : RowHalf {
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, int64_t i) { load_at<float>(p, i); }
    __device__ __forceinline__ void get(float* f) const { f[0] = __int_as_float(v[0]); f[1] = __int_as_float(v[1]); }
    template <bool STREAM = false> static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) {
        *(i32x2*)((float*)p + i) = i32x2{__float_as_int(f[0]), __float_as_int(f[1])};
    }
};
template <> struct RowVec<BF16, 2> {
    unsigned v;
    __device__ __forceinline__ void clear() { v = 0; }
    __device__ __forceinline__ void infinite() { v = 0x7f807f80u; }
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, int64_t i) { v = *(const unsigned*)((const unsigned short*)p + i); }
    __device__ __forceinline__ void get(float* f) const { f[0] = __uint_as_float(v << 16); f[1] = __uint_as_float(v & 0xffff0000u); }
    template <bool STREAM = false> static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) {
        *(unsigned*)((unsigned short*)p + i) = (unsigned)f2bf(f[0]) | ((unsigned)f2bf(f[1]) << 16);
    }
};
template <typename E> struct RowVec<E, 1> {
    typename E::T v;
    __device__ __forceinline__ void clear() { v = 0; }
    __device__ __forceinline__ void infinite() { st_elem<E>(&v, 0, __uint_as_float(0x7f800000u)); }
    template <bool STREAM = false> __device__ __forceinline__ void load(const void* p, int64_t i) { v = ((const typename E::T*)p)[i]; }
    __device__ __forceinline__ void get(float* f) const { f[0] = ld_elem<E>(&v, 0); }
    template <bool STREAM = false> static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { st_elem<E>(p, i, f[0]); }
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
// smaller call reads may still be there, and what it writes is read there next.  Measured, whole lines: block norm of 16384 x 2048 bf16 73 us
// forward and 128 backward through the caches, 65 and 118 past them; gate loop of 8 x 2048 x 2048 59 and 114, 55 and 108.
static inline bool calls_stream(double bytes) { return bytes >= 256.0 * 1024 * 1024; }

// the widest access (16, 4 or 1 bytes) that all the addresses and all the lengths in bytes are multiples of; null pointers are
static inline int rows_access(std::initializer_list<const void*> ps, std::initializer_list<int64_t> bytes) {
    uintptr_t any = 0;
    for (const void* p : ps) any |= (uintptr_t)p;
    for (int64_t b : bytes) any |= (uintptr_t)b;
    return any & 3 ? 1 : any & 15 ? 4 : 16;
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
