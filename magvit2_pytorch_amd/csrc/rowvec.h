// Row access of the kernels that serve any width and any strides: V elements of storage type E as one access - 16 bytes where the
// rows, strides and addresses are whole 16-byte chunks (V = E::kVec; V = E::kVec / 2: 8 bytes, half a chunk, for kernels that hold many rows
// in registers), one element otherwise (V = 1).
#pragma once
#include "common.h"

template <typename E, int V> struct RowVec {
    static_assert(V == E::kVec, "a 16-byte chunk or one element");
    i32x4 v;
    __device__ __forceinline__ void clear() { v = i32x4{0, 0, 0, 0}; }
    __device__ __forceinline__ void infinite() { const int w = E::kBytes == 2 ? 0x7f807f80 : 0x7f800000; v = i32x4{w, w, w, w}; }
    __device__ __forceinline__ void load(const void* p, int64_t i) { v = *(const i32x4*)((const typename E::T*)p + i); }
    __device__ __forceinline__ void get(float* f) const { Chunk<E>::unpack(v, f); }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { *(i32x4*)((typename E::T*)p + i) = Chunk<E>::pack(f); }
};
struct RowHalf {
    i32x2 v;
    __device__ __forceinline__ void clear() { v = i32x2{0, 0}; }
    template <typename T> __device__ __forceinline__ void load_at(const void* p, int64_t i) { v = *(const i32x2*)((const T*)p + i); }
};
template <> struct RowVec<BF16, 4> : RowHalf {
    __device__ __forceinline__ void load(const void* p, int64_t i) { load_at<unsigned short>(p, i); }
    __device__ __forceinline__ void get(float* f) const { ld4<BF16>(&v, 0, f); }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { st4<BF16>(p, i, f); }
};
template <> struct RowVec<F32, 2> : RowHalf {
    __device__ __forceinline__ void load(const void* p, int64_t i) { load_at<float>(p, i); }
    __device__ __forceinline__ void get(float* f) const { f[0] = __int_as_float(v[0]); f[1] = __int_as_float(v[1]); }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) {
        *(i32x2*)((float*)p + i) = i32x2{__float_as_int(f[0]), __float_as_int(f[1])};
    }
};
template <typename E> struct RowVec<E, 1> {
    typename E::T v;
    __device__ __forceinline__ void clear() { v = 0; }
    __device__ __forceinline__ void infinite() { st_elem<E>(&v, 0, __uint_as_float(0x7f800000u)); }
    __device__ __forceinline__ void load(const void* p, int64_t i) { v = ((const typename E::T*)p)[i]; }
    __device__ __forceinline__ void get(float* f) const { f[0] = ld_elem<E>(&v, 0); }
    static __device__ __forceinline__ void store(void* p, int64_t i, const float* f) { st_elem<E>(p, i, f[0]); }
};

static inline bool rows_aligned16(std::initializer_list<const void*> ps) {
    for (const void* p : ps) if ((uintptr_t)p & 15) return false;
    return true;
}
