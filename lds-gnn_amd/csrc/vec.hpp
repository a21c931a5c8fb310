// Element types, vector loads / stores and the keyed dropout mask of the block
// operators (dropout, group norm, 8-bit product).
//
// A tensor element is fp32, bf16 or fp16 (include/ldsgnn.h LDS_F32 / LDS_BF16 /
// LDS_F16); all arithmetic is fp32 and a result is rounded once, to nearest
// even, when it is stored.
#pragma once

#include "common.hpp"
#include "../../include/ldsgnn.h"

namespace lds {

using bf16_t = __bf16;
using f16_t = _Float16;

// V consecutive elements as one load or store.  Rows of an odd length start at
// any multiple of the element size: the type carries the element's alignment,
// and gfx950's global memory takes a 16-byte access at any address.
template <typename T, int V>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
template <typename T>
struct VecOf<T, 1> {
    typedef T type;
};

template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&f)[V]) {
    if constexpr (V == 1) {
        f[0] = (float)p[0];
    } else {
        const auto v = *reinterpret_cast<const typename VecOf<T, V>::type*>(p);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (float)v[e];
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&f)[V]) {
    if constexpr (V == 1) {
        p[0] = (T)f[0];
    } else {
        typename VecOf<T, V>::type v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)f[e];
        *reinterpret_cast<typename VecOf<T, V>::type*>(p) = v;
    }
}

// A vector whose first w <= V elements exist (a row's last, partial one).
template <typename T, int V>
__device__ __forceinline__ void load_part(const T* __restrict__ p, int w, float (&f)[V]) {
    if (w >= V) {
        load_vec<T, V>(p, f);
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = e < w ? (float)p[e] : 0.f;
}
template <typename T, int V>
__device__ __forceinline__ void store_part(T* __restrict__ p, int w, const float (&f)[V]) {
    if (w >= V) {
        store_vec<T, V>(p, f);
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e)
        if (e < w) p[e] = (T)f[e];
}

// One element of a parameter vector stored as `code` (LDS_F32 / BF16 / F16).
__device__ __forceinline__ float load_param(const void* p, int code, int64_t i) {
    if (code == LDS_F32) return reinterpret_cast<const float*>(p)[i];
    if (code == LDS_BF16) return (float)reinterpret_cast<const bf16_t*>(p)[i];
    return (float)reinterpret_cast<const f16_t*>(p)[i];
}

// The mask of the RNG contract (include/ldsgnn.h) at V neighbouring columns
// and the four rows of a row quad: bit (4 e + r) of the result is set where
// u(4 rq + r, col + e) < keep.  u < keep is a comparison of whole numbers:
// u = (w >> 8) 2^-24 < keep  <=>  w < ceil(keep 2^24) 256 = `thr` (keep < 1).
struct DropKey {
    uint32_t k0, k1, tag, counter, thr;
    float scale;
};

template <int V>
__device__ __forceinline__ uint32_t keep_bits(const DropKey& k, uint32_t col, uint32_t rq) {
    uint32_t bits = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const U32x4 o = philox4x32_10(U32x4{col + e, rq, k.tag, k.counter}, k.k0, k.k1);
        bits |= (o.x < k.thr ? 1u : 0u) << (4 * e);
        bits |= (o.y < k.thr ? 2u : 0u) << (4 * e);
        bits |= (o.z < k.thr ? 4u : 0u) << (4 * e);
        bits |= (o.w < k.thr ? 8u : 0u) << (4 * e);
    }
    return bits;
}

// keep in [0, 1] -> the threshold; false when every element is kept.
inline bool drop_key(float keep, float scale, uint64_t seed, uint32_t tag, uint32_t counter, DropKey* k) {
    const double t = ceil((double)keep * 16777216.0);
    k->k0 = (uint32_t)seed;
    k->k1 = (uint32_t)(seed >> 32);
    k->tag = tag;
    k->counter = counter;
    k->scale = scale;
    k->thr = t >= 16777216.0 ? 0u : (uint32_t)t * 256u;
    return t < 16777216.0;
}

// A compile-time int as a value.
template <int N>
struct IntC {
    static constexpr int value = N;
};

// Calls f with a value of the element type.
template <typename F>
inline int with_type(int code, F&& f) {
    if (code == LDS_F32) return f(float{});
    if (code == LDS_BF16) return f(bf16_t{});
    if (code == LDS_F16) return f(f16_t{});
    return (int)hipErrorInvalidValue;
}

}  // namespace lds
