// Element types of the token-head operators (linear.hip, normgate.hip, gradclip.hip): loads to f32, stores with one
// rounding, and vectors whose address is aligned to one element only (the hardware takes such 16-byte accesses
// anywhere in global memory, so odd row lengths and views into larger buffers need no path of their own).
#pragma once
#include "pclip_common.h"

template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) PclipPack { T v[V]; };

// elements of one 16-byte access
template <typename T> struct PclipVec { static constexpr int N = 16 / (int)sizeof(T); };

// `valid` (any value) elements from p, the rest of out zero; nothing past p[valid - 1] is read
template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* __restrict__ p, int valid, float (&out)[V]) {
    if (valid >= V) {
        const PclipPack<T, V> a = *(const PclipPack<T, V>*)p;
#pragma unroll
        for (int i = 0; i < V; i++) out[i] = (float)a.v[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; i++) out[i] = i < valid ? (float)p[i] : 0.f;
    }
}
template <typename T, int V>
__device__ __forceinline__ void store_f32(T* p, int valid, const float (&v)[V]) {
    if (valid >= V) {
        PclipPack<T, V> a;
#pragma unroll
        for (int i = 0; i < V; i++) a.v[i] = (T)v[i];
        *(PclipPack<T, V>*)p = a;
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < valid) p[i] = (T)v[i];
    }
}
// 8, 16 or 32 bytes past the L2 (results that nobody reads back soon: they would push out what the kernel still reads)
template <typename P>
__device__ __forceinline__ void store_past_l2(void* p, const P& a) {
    static_assert(sizeof(P) == 32 || sizeof(P) == 16 || sizeof(P) == 8, "one access or two");
    typedef unsigned __attribute__((ext_vector_type(sizeof(P) == 8 ? 2 : 4), aligned(1))) Any;
    struct Parts { Any part[sizeof(P) / sizeof(Any)]; };
    const Parts all = __builtin_bit_cast(Parts, a);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(P) / sizeof(Any)); i++) __builtin_nontemporal_store(all.part[i], (Any*)p + i);
}
template <typename T, int V>
__device__ __forceinline__ void stream_f32(T* p, int valid, const float (&v)[V]) {
    if (valid >= V) {
        PclipPack<T, V> a;
#pragma unroll
        for (int i = 0; i < V; i++) a.v[i] = (T)v[i];
        store_past_l2(p, a);
    } else {
#pragma unroll
        for (int i = 0; i < V; i++)
            if (i < valid) p[i] = (T)v[i];
    }
}

inline int pclip_dtype_size(int dtype) { return dtype == PCLIP_DT_F32 ? 4 : 2; }
inline bool pclip_dtype_ok(int dtype) { return dtype == PCLIP_DT_F32 || dtype == PCLIP_DT_BF16 || dtype == PCLIP_DT_F16; }
