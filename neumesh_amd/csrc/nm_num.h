// nm_num.h -- device: element types and conversions of the free-standing operators (nm_dense.hip, nm_scan.hip).
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/neumesh_hip.h"

typedef __bf16 nm_v8b __attribute__((ext_vector_type(8)));
typedef _Float16 nm_v8h __attribute__((ext_vector_type(8)));
typedef float nm_v4f __attribute__((ext_vector_type(4)));
typedef float nm_v16f __attribute__((ext_vector_type(16)));

template <int DT> struct NmType;
template <> struct NmType<NM_F32> { typedef float elem; };
template <> struct NmType<NM_F16> { typedef _Float16 elem; };
template <> struct NmType<NM_BF16> { typedef __bf16 elem; };

template <int DT>
__device__ __forceinline__ float nm_to_float(typename NmType<DT>::elem e) { return (float)e; }
template <int DT>
__device__ __forceinline__ typename NmType<DT>::elem nm_from_float(float f) { return (typename NmType<DT>::elem)f; }

static inline bool nm_dtype_ok(int dt) { return dt == NM_F32 || dt == NM_F16 || dt == NM_BF16; }
static inline int nm_dtype_size(int dt) { return dt == NM_F32 ? 4 : 2; }

// Eight consecutive elements, at any element-aligned address (one or two 16-byte accesses: global memory takes them unaligned).
template <int DT> struct NmOct { uint4 v[DT == NM_F32 ? 2 : 1]; };

template <int DT>
__device__ __forceinline__ NmOct<DT> nm_oct_load(const typename NmType<DT>::elem* p) {
    NmOct<DT> o;
    __builtin_memcpy(&o, p, sizeof(o));
    return o;
}
template <int DT>
__device__ __forceinline__ NmOct<DT> nm_oct_zero() {
    NmOct<DT> o;
    o.v[0] = make_uint4(0, 0, 0, 0);
    if constexpr (DT == NM_F32) o.v[1] = make_uint4(0, 0, 0, 0);
    return o;
}
// n < 8 elements, the rest zero, one after the other (rows shorter than eight)
template <int DT>
__device__ __forceinline__ NmOct<DT> nm_oct_load_short(const typename NmType<DT>::elem* p, long long n) {
    constexpr int W = DT == NM_F32 ? 8 : 4;                  // dwords
    unsigned w[W];
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0u;
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        if constexpr (DT == NM_F32) {
            unsigned e;
            __builtin_memcpy(&e, p + i, 4);
#pragma unroll
            for (int k = 0; k < W; ++k) w[k] = k == i ? e : w[k];
        } else {
            unsigned short e;
            __builtin_memcpy(&e, p + i, 2);
#pragma unroll
            for (int k = 0; k < W; ++k) w[k] |= k == (i >> 1) ? (unsigned)e << (16 * (i & 1)) : 0u;
        }
    }
    NmOct<DT> o;
    __builtin_memcpy(&o, w, sizeof(o));
    return o;
}
// an oct with its first `sh` elements cleared (sh >= 8: all of them)
template <int DT>
__device__ __forceinline__ NmOct<DT> nm_oct_clear_first(NmOct<DT> o, int sh) {
    constexpr int W = DT == NM_F32 ? 8 : 4;
    unsigned w[W];
    __builtin_memcpy(w, &o, sizeof(o));
#pragma unroll
    for (int i = 0; i < W; ++i) {
        if constexpr (DT == NM_F32) w[i] = i >= sh ? w[i] : 0u;
        else w[i] &= (2 * i >= sh ? 0xffffu : 0u) | (2 * i + 1 >= sh ? 0xffff0000u : 0u);
    }
    __builtin_memcpy(&o, w, sizeof(o));
    return o;
}
// elements q .. q + 7 of a row of Q, zero from Q on.  The last piece of a row is the row's last eight elements shifted down, so that nothing beyond
// the row is touched; rows shorter than eight go element by element.  (Both forms are a few instructions: this sits in unrolled loops.)
template <int DT>
__device__ __forceinline__ NmOct<DT> nm_oct_load_row(const typename NmType<DT>::elem* row, long long q, long long Q) {
    if (q + 8 <= Q) return nm_oct_load<DT>(row + q);
    NmOct<DT> o = nm_oct_zero<DT>();
    if (q >= Q) return o;
    constexpr int W = DT == NM_F32 ? 8 : 4;                  // dwords
    unsigned w[W];
    if (Q >= 8) {
        o = nm_oct_load<DT>(row + Q - 8);
        __builtin_memcpy(w, &o, sizeof(o));
        const int sh = (int)(q + 8 - Q);                     // 1 .. 7 elements
        if constexpr (DT == NM_F32) {
#pragma unroll
            for (int b = 4; b > 0; b >>= 1)
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = (sh & b) ? (i + b < 8 ? w[i + b] : 0u) : w[i];
        } else {
#pragma unroll
            for (int b = 2; b > 0; b >>= 1)
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = (sh & (2 * b)) ? (i + b < 4 ? w[i + b] : 0u) : w[i];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = (sh & 1) ? (w[i] >> 16) | (i < 3 ? w[i + 1] << 16 : 0u) : w[i];
        }
        __builtin_memcpy(&o, w, sizeof(o));
        return o;
    }
    return nm_oct_load_short<DT>(row + q, Q - q);
}
template <int DT>
__device__ __forceinline__ void nm_oct_to_float(const NmOct<DT>& o, float (&f)[8]) {
    typename NmType<DT>::elem e[8];
    __builtin_memcpy(e, &o, sizeof(o));
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = nm_to_float<DT>(e[i]);
}
// the first `n` of eight values, rounded once to the element type
template <int DT>
__device__ __forceinline__ void nm_oct_store_n(typename NmType<DT>::elem* p, const float (&f)[8], long long n) {
    typename NmType<DT>::elem e[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = nm_from_float<DT>(f[i]);
    if (n >= 8) {
        __builtin_memcpy(p, e, sizeof(e));
        return;
    }
    constexpr int W = DT == NM_F32 ? 8 : 4;
    unsigned w[W];
    __builtin_memcpy(w, e, sizeof(e));
#pragma unroll 1
    for (int i = 0; i < n; ++i) {
        if constexpr (DT == NM_F32) {
            __builtin_memcpy(p + i, &w[0], 4);
#pragma unroll
            for (int k = 0; k < 7; ++k) w[k] = w[k + 1];
        } else {
            const unsigned short lo = (unsigned short)w[0];
            __builtin_memcpy(p + i, &lo, 2);
#pragma unroll
            for (int k = 0; k < 4; ++k) w[k] = (w[k] >> 16) | (k < 3 ? w[k + 1] << 16 : 0u);
        }
    }
}
