// Group norm with an activation, channels last: the pieces that the forward
// (norm_fwd.hip) and the backward (norm_bwd.hip) share.
//
// A thread owns V neighbouring channels of one group (V divides the channels
// per group) and walks row quads: four rows whose flat indices s·n + i differ in
// their two low bits, the unit in which the keyed dropout mask is drawn.
#pragma once

#include "vec.hpp"

namespace lds {

constexpr int kNormThreads = 256;

// How the channels of a row are cut: a block takes `lanes` vectors of V
// channels and `ty` rows at a time; `chunks` blocks cover a row.  A chunk
// holds whole groups, or (a group wider than 256 vectors) one of the `sub`
// parts of a group.
struct NormCut {
    int v, lanes, ty, chunks, lpg, sub;
};

inline NormCut norm_cut(int c, int groups, int v) {
    NormCut k;
    const int cg = c / groups;
    k.v = v;
    const int lpg = cg / v;  // vectors per group
    if (lpg <= kNormThreads) {
        int per = kNormThreads / lpg;
        if (per > groups) per = groups;
        k.chunks = (groups + per - 1) / per;
        per = (groups + k.chunks - 1) / k.chunks;  // even chunks
        k.chunks = (groups + per - 1) / per;
        k.lanes = per * lpg;
        k.lpg = lpg;
        k.sub = 1;
    } else {
        k.sub = (lpg + kNormThreads - 1) / kNormThreads;
        k.lanes = (lpg + k.sub - 1) / k.sub;
        k.lpg = k.lanes;
        k.chunks = groups * k.sub;
    }
    k.ty = kNormThreads / k.lanes;
    return k;
}

// The widest vector (<= 16 bytes) that lies in one group: 1, 2, 4 or 8 channels.
inline int norm_vec(int c, int groups, int elem_bytes) {
    const int cg = c / groups;
    for (int v = 16 / elem_bytes; v > 1; v /= 2)
        if (cg % v == 0) return v;
    return 1;
}

struct NormArgs {
    int64_t samples, n, sx, ldx;
    int c, groups, cg;
    int lanes, ty, chunks, lpg, sub;
    int parts;        // row parts per sample
    int64_t part_q;   // row quads per part
    const void* weight;
    const void* bias;
    int ptype;
    DropKey key;
};

// What a thread of a block works on.
struct NormPlace {
    int64_t s;            // sample
    int part, chunk;
    int tx, row0, stride;  // vector in the chunk, first quad of the thread, quads per step
    int group, c0;         // the thread's group and its first channel
    bool live;
    int64_t q0, q1;        // the part's row quads (flat index / 4)
    int64_t f0, f1;        // the sample's flat rows
};

__device__ __forceinline__ NormPlace norm_place(const NormArgs& a, int v) {
    NormPlace p;
    int64_t b = blockIdx.x;
    p.chunk = (int)(b % a.chunks);
    b /= a.chunks;
    p.part = (int)(b % a.parts);
    p.s = b / a.parts;
    const int t = threadIdx.x;
    p.row0 = t / a.lanes;
    p.tx = t - p.row0 * a.lanes;
    p.stride = a.ty;
    if (a.sub == 1) {
        const int per = a.lanes / a.lpg;
        const int gi = p.tx / a.lpg;
        p.group = p.chunk * per + gi;
        p.c0 = p.group * a.cg + (p.tx - gi * a.lpg) * v;
        p.live = p.row0 < a.ty && p.group < a.groups;
    } else {
        p.group = p.chunk / a.sub;
        const int at = ((p.chunk - p.group * a.sub) * a.lanes + p.tx) * v;
        p.c0 = p.group * a.cg + at;
        p.live = p.row0 < a.ty && at < a.cg;
    }
    p.f0 = p.s * a.n;
    p.f1 = p.f0 + a.n;
    p.q0 = (p.f0 >> 2) + (int64_t)p.part * a.part_q;
    const int64_t qe = ((p.f1 - 1) >> 2) + 1;
    p.q1 = p.q0 + a.part_q < qe ? p.q0 + a.part_q : qe;
    return p;
}

// Merges the values of a row quad (rows with in[r]) into running moments.
template <int V>
__device__ __forceinline__ void quad_moments(const float (&v)[4][V], const bool (&in)[4], double& mean, float& m2,
                                             float& cnt) {
    float k = 0.f, m = 0.f;
#pragma unroll
    for (int r = 3; r >= 0; --r) {
        k = in[r] ? v[r][0] : k;
        m += in[r] ? (float)V : 0.f;
    }
    if (m == 0.f) return;
    float d[4][V], s1 = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            d[r][e] = in[r] ? v[r][e] - k : 0.f;
            s1 += d[r][e];
        }
    const float mq = s1 * __builtin_amdgcn_rcpf(m);
    float s2 = 0.f;
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float t = in[r] ? d[r][e] - mq : 0.f;
            s2 = __builtin_fmaf(t, t, s2);
        }
    const double delta = ((double)k + (double)mq) - mean;
    const float part = m * __builtin_amdgcn_rcpf(cnt + m);
    mean += delta * (double)part;
    m2 += __builtin_fmaf((float)delta * (float)delta, cnt * part, s2);
    cnt += m;
}

// silu'(z) and friends.  v_exp_f32 and v_rcp_f32 are good to about one unit in
// the last place of fp32, below the rounding of z itself.
__device__ __forceinline__ float sigmoid_f(float z) { return __builtin_amdgcn_rcpf(1.f + __expf(-z)); }

template <int ACT>
__device__ __forceinline__ float act_f(float z) {
    if constexpr (ACT == LDS_ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
    if constexpr (ACT == LDS_ACT_SILU) return z * sigmoid_f(z);
    return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
    if constexpr (ACT == LDS_ACT_RELU) return z <= 0.f ? 0.f : 1.f;
    if constexpr (ACT == LDS_ACT_SILU) {
        const float s = sigmoid_f(z);
        return s * (1.f + z * (1.f - s));
    }
    return 1.f;
}

// Calls f with an integral constant for the activation.
template <typename F>
inline int with_act(int act, F&& f) {
    if (act == LDS_ACT_NONE) return f(IntC<LDS_ACT_NONE>{});
    if (act == LDS_ACT_RELU) return f(IntC<LDS_ACT_RELU>{});
    if (act == LDS_ACT_SILU) return f(IntC<LDS_ACT_SILU>{});
    return (int)hipErrorInvalidValue;
}
template <int MAXV, typename F>
inline int with_vec(int v, F&& f) {
    if constexpr (MAXV >= 8)
        if (v == 8) return f(IntC<8>{});
    if (v == 4) return f(IntC<4>{});
    if (v == 2) return f(IntC<2>{});
    return f(IntC<1>{});
}

// The sizes that both directions accept; false: hipErrorInvalidValue.
inline bool norm_sizes_ok(int64_t samples, int64_t n, int c, int groups) {
    if (samples < 0 || n < 0 || c < 0 || groups < 1 || c % groups) return false;
    if (samples > 0x7fffffff || n > 0x7fffffff) return false;
    return samples * n <= (int64_t)0x7fffffff;
}

constexpr int kNormBlocks = 2048;  // blocks of a pass: eight per CU

// Row parts per sample: about `want` blocks in all, and not less than eight
// quads to a thread where there are that many.
inline void norm_parts(int64_t samples, int64_t n, const NormCut& k, int want, int* parts, int64_t* part_q) {
    const int64_t quads = n / 4 + 2;  // a sample's quads, its partial first and last one among them
    int64_t p = want / (samples * k.chunks > 0 ? samples * k.chunks : 1);
    const int64_t most = (quads + 8 * k.ty - 1) / (8 * k.ty);
    if (p > most) p = most;
    if (p < 1) p = 1;
    *part_q = (quads + p - 1) / p;
    *parts = (int)((quads + *part_q - 1) / *part_q);
}

inline void norm_fill(NormArgs* a, const NormCut& k, int64_t samples, int64_t n, int c, int groups, int64_t sx,
                      int64_t ldx, const void* weight, const void* bias, int ptype) {
    a->samples = samples;
    a->n = n;
    a->sx = sx;
    a->ldx = ldx;
    a->c = c;
    a->groups = groups;
    a->cg = c / groups;
    a->lanes = k.lanes;
    a->ty = k.ty;
    a->chunks = k.chunks;
    a->lpg = k.lpg;
    a->sub = k.sub;
    norm_parts(samples, n, k, kNormBlocks, &a->parts, &a->part_q);
    a->weight = weight;
    a->bias = bias;
    a->ptype = ptype;
}

}  // namespace lds
