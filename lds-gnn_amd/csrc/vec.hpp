// Element types, vector loads / stores and the keyed dropout mask of the block
// operators (dropout, group norm, 8-bit product).
//
// A tensor element is fp32, bf16 or fp16 (include/ldsgnn.h LDS_F32 / LDS_BF16 /
// LDS_F16); all arithmetic is fp32 and a result is rounded once, to nearest
// even, when it is stored.
#pragma once

#include <type_traits>

#include "common.hpp"
#include "../../include/ldsgnn.h"

namespace lds {

using bf16_t = __bf16;
using f16_t = _Float16;

// The cache between the memory and the chip's L2s.
constexpr int64_t kMemorySideCache = (int64_t)256 << 20;

// The bytes from a block's first element to its last.
struct ByteSpan {
    uintptr_t lo, hi;
    ByteSpan(const void* p, int64_t elements, size_t size)
        : lo((uintptr_t)p), hi(lo + (uintptr_t)elements * size) {}
    bool meets(const ByteSpan& o) const { return lo < o.hi && o.lo < hi; }
};

// The helpers' pointers are not __restrict__: a caller may write its result over an
// input (include/ldsgnn.h says which).
//
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
__device__ __forceinline__ void load_vec(const T* p, float (&f)[V]) {
    if constexpr (V == 1) {
        f[0] = (float)p[0];
    } else {
        const auto v = *reinterpret_cast<const typename VecOf<T, V>::type*>(p);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (float)v[e];
    }
}

// PAST: a store that leaves the caches to others.
template <typename T, int V, bool PAST = false>
__device__ __forceinline__ void store_vec(T* p, const float (&f)[V]) {
    if constexpr (V == 1) {
        p[0] = (T)f[0];
    } else {
        typename VecOf<T, V>::type v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)f[e];
        if constexpr (PAST)
            __builtin_nontemporal_store(v, reinterpret_cast<typename VecOf<T, V>::type*>(p));
        else
            *reinterpret_cast<typename VecOf<T, V>::type*>(p) = v;
    }
}

// A vector whose first w <= V elements exist (a row's last, partial one).
template <typename T, int V>
__device__ __forceinline__ void load_part(const T* p, int w, float (&f)[V]) {
    if (w >= V) {
        load_vec<T, V>(p, f);
        return;
    }
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = e < w ? (float)p[e] : 0.f;
}
template <typename T, int V>
__device__ __forceinline__ void store_part(T* p, int w, const float (&f)[V]) {
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

// V consecutive elements as they lie in memory, and as fp32.
template <typename T, int V>
using Raw = typename VecOf<T, V>::type;
// PAST: a last read, which leaves the caches to others.
template <typename T, int V, bool PAST = false>
__device__ __forceinline__ Raw<T, V> load_raw(const T* p) {
    if constexpr (PAST)
        return __builtin_nontemporal_load(reinterpret_cast<const Raw<T, V>*>(p));
    else
        return *reinterpret_cast<const Raw<T, V>*>(p);
}
template <typename T, int V>
__device__ __forceinline__ float elem(const Raw<T, V>& v, int e) {
    if constexpr (V == 1)
        return (float)v;
    else
        return (float)v[e];
}

// The mask of the RNG contract (include/ldsgnn.h): u(row, col) < keep, with
// u = (w >> 8) 2^-24, as a comparison of whole numbers,
// w < ceil(keep 2^24) 256 = `thr` (keep < 1).
struct DropKey {
    uint32_t k0, k1, tag, counter, thr;
    float scale;
};

constexpr uint32_t kPhiloxM0 = 0xD2511F53u, kPhiloxM1 = 0xCD9E8D57u, kPhiloxW0 = 0x9E3779B9u,
                   kPhiloxW1 = 0xBB67AE85u;

__device__ __forceinline__ void mul_wide(uint32_t m, uint32_t x, uint32_t& hi, uint32_t& lo) {
    uint64_t p, cc;  // one v_mad_u64_u32 (common.hpp philox4x32_10)
    asm("v_mad_u64_u32 %0, %1, %2, %3, 0" : "=v"(p), "=s"(cc) : "s"(m), "v"(x));
    (void)cc;
    hi = (uint32_t)(p >> 32);
    lo = (uint32_t)p;
}

// Philox4x32-10 at V neighbouring columns and any row quads.  Of the counter
// (column, row quad, tag, draw) only the row quad changes along a thread's
// rows, so the products of the first three rounds that do not see it are
// taken once: 15.1 wide products a quad and column are left of 20.
//   round 1:  a = (M1·tag hi ^ rq ^ k0,  M1·tag lo,  M0·col hi ^ draw ^ k1,  M0·col lo)
//   round 2:  q0 = M0·a0 (row quad only),  q1 = M1·a2 (column only)
//   round 3:  r0 = M0·(q1 hi ^ a1 ^ k0) (column only),  r1 = M1·(q0 hi ^ a3 ^ k1)
template <int V>
struct ColumnKeep {
    uint32_t a3[V], b1[V], r0h[V], r0l[V];
    uint32_t u0;

    __device__ __forceinline__ void init(const DropKey& k, uint32_t col) {
        uint32_t th, tl;
        mul_wide(kPhiloxM1, k.tag, th, tl);
        u0 = th ^ k.k0;
        const uint32_t k0b = k.k0 + kPhiloxW0, k1b = k.k1 + kPhiloxW1;
        const uint32_t k0c = k0b + kPhiloxW0, k1c = k1b + kPhiloxW1;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            uint32_t hi, lo, qh, ql, rh, rl;
            mul_wide(kPhiloxM0, col + e, hi, lo);
            a3[e] = lo ^ k1b;
            mul_wide(kPhiloxM1, hi ^ k.counter ^ k.k1, qh, ql);
            b1[e] = ql ^ k0c;
            mul_wide(kPhiloxM0, qh ^ tl ^ k0b, rh, rl);
            r0h[e] = rh ^ k1c;
            r0l[e] = rl;
        }
    }

    // kept[r][e]: the element of row 4 rq + r at column col + e is kept
    __device__ __forceinline__ void quad(const DropKey& k, uint32_t rq, bool (&kept)[4][V]) const {
        uint32_t qh, ql;
        mul_wide(kPhiloxM0, u0 ^ rq, qh, ql);
        uint32_t c0[V], c1[V], c2[V], c3[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            uint32_t hi;
            mul_wide(kPhiloxM1, qh ^ a3[e], hi, c1[e]);
            c0[e] = hi ^ b1[e];
            c2[e] = r0h[e] ^ ql;
            c3[e] = r0l[e];
        }
        uint32_t k0 = k.k0 + 3 * kPhiloxW0, k1 = k.k1 + 3 * kPhiloxW1;
#pragma unroll
        for (int r = 3; r < 10; ++r) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                uint32_t h0, l0, h1, l1;
                mul_wide(kPhiloxM0, c0[e], h0, l0);
                mul_wide(kPhiloxM1, c2[e], h1, l1);
                asm("v_bitop3_b32 %0, %1, %2, %3 bitop3:0x96" : "=v"(c0[e]) : "v"(h1), "v"(c1[e]), "s"(k0));
                asm("v_bitop3_b32 %0, %1, %2, %3 bitop3:0x96" : "=v"(c2[e]) : "v"(h0), "v"(c3[e]), "s"(k1));
                c1[e] = l1;
                c3[e] = l0;
            }
            k0 += kPhiloxW0;
            k1 += kPhiloxW1;
        }
#pragma unroll
        for (int e = 0; e < V; ++e) {
            kept[0][e] = c0[e] < k.thr;
            kept[1][e] = c1[e] < k.thr;
            kept[2][e] = c2[e] < k.thr;
            kept[3][e] = c3[e] < k.thr;
        }
    }
};

// A quad's mask as a word, and back.
template <int V>
__device__ __forceinline__ uint32_t pack_kept(const bool (&kept)[4][V]) {
    uint32_t bits = 0;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) bits |= kept[r][e] ? 1u << (r * V + e) : 0u;
    return bits;
}
template <int V>
__device__ __forceinline__ void unpack_kept(uint32_t bits, bool (&kept)[4][V]) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) kept[r][e] = (bits >> (r * V + e)) & 1u;
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

// A launch counts its threads along x in 32 bits, and one with more runs in part,
// with no error: no launch has more.
inline bool grid_fits(int64_t blocks, int threads) { return blocks <= 0xffffffffll / threads; }
// f(first block, blocks) for the launches that `blocks` of them take: whole
// rounds of the eight XCDs each.
template <typename F>
inline void in_launches(int64_t blocks, int threads, F&& f) {
    const int64_t most = 0xffffffffll / threads / 8 * 8;
    for (int64_t first = 0; first < blocks; first += most)
        f(first, (unsigned)(blocks - first < most ? blocks - first : most));
}

// A pointer that no other argument's memory overlaps (RESTRICT), or that one may.
template <typename T, bool RESTRICT>
using Pointer = std::conditional_t<RESTRICT, T* __restrict__, T*>;

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
