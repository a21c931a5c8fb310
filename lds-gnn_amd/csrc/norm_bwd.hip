// Group norm + activation + keyed dropout, channels last, backward
// (include/ldsgnn.h lds_group_norm_backward).
//
//   h = dy · mask · act'(z),  dβ_c = Σ h,  dγ_c = Σ h x̂,
//   dx = r (γ h - mean_g(γ h) - x̂ mean_g(γ h x̂))
// Three launches: the per-channel sums of every row part; the group means and
// dγ / dβ from them; the elementwise pass.  z, x̂ and the mask are recomputed.
#include "norm.hpp"

namespace lds {

template <typename T, int V, int ACT, bool DROP>
struct NormBack {
    float mu, rs;
    float w[V], b[V];

    __device__ __forceinline__ void load(const NormArgs& a, const NormPlace& p, const float* mean,
                                         const float* rstd) {
        mu = mean[p.s * a.groups + p.group];
        rs = rstd[p.s * a.groups + p.group];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            w[e] = a.weight ? load_param(a.weight, a.ptype, p.c0 + e) : 1.f;
            b[e] = a.bias ? load_param(a.bias, a.ptype, p.c0 + e) : 0.f;
        }
    }
    // x -> x̂, g -> h
    __device__ __forceinline__ void eval(float& x, float& g, int e, bool kept, float scale) const {
        x = (x - mu) * rs;
        if constexpr (DROP) g = kept ? g * scale : 0.f;
        if constexpr (ACT == LDS_ACT_RELU) {
            g = __builtin_fmaf(x, w[e], b[e]) <= 0.f ? 0.f : g;
        } else if constexpr (ACT != LDS_ACT_NONE) {
            g *= act_grad<ACT>(__builtin_fmaf(x, w[e], b[e]));
        }
    }
};

template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_sums_kernel(const T* __restrict__ dy, int64_t sdy,
                                                                   int64_t lddy, const T* __restrict__ x, NormArgs a,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd,
                                                                   float2* __restrict__ out) {
    __shared__ float2 red[V][kNormThreads];
    const NormPlace p = norm_place(a, V);
    float sh[V] = {}, sx[V] = {};
    if (p.live) {
        NormBack<T, V, ACT, DROP> k;
        k.load(a, p, mean, rstd);
        const T* xs = x + p.s * a.sx + p.c0;
        const T* gs = dy + p.s * sdy + p.c0;
        for (int64_t q = p.q0 + p.row0; q < p.q1; q += p.stride) {
            float v[4][V], g[4][V];
            bool in[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t f = 4 * q + r;
                in[r] = f >= p.f0 && f < p.f1;
                if (in[r]) {
                    load_vec<T, V>(xs + (f - p.f0) * a.ldx, v[r]);
                    load_vec<T, V>(gs + (f - p.f0) * lddy, g[r]);
                }
            }
            const uint32_t keep = DROP ? keep_bits<V>(a.key, (uint32_t)p.c0, (uint32_t)q) : 0u;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (!in[r]) continue;
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    k.eval(v[r][e], g[r][e], e, (keep >> (4 * e + r)) & 1u, a.key.scale);
                    sh[e] += g[r][e];
                    sx[e] = __builtin_fmaf(g[r][e], v[r][e], sx[e]);
                }
            }
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) red[e][threadIdx.x] = make_float2(sh[e], sx[e]);
    __syncthreads();
    // the ty rows of every channel of the chunk, a thread per channel
    const int first = a.sub == 1 ? p.chunk * a.lanes * V
                                 : (p.chunk / a.sub) * a.cg + (p.chunk % a.sub) * a.lanes * V;
    const int last = a.sub == 1 ? a.c : (p.chunk / a.sub + 1) * a.cg;
    for (int i = threadIdx.x; i < a.lanes * V; i += kNormThreads) {
        if (first + i >= last) break;
        float h = 0.f, hx = 0.f;
        for (int r = 0; r < a.ty; ++r) {
            const float2 t = red[i % V][r * a.lanes + i / V];
            h += t.x;
            hx += t.y;
        }
        out[(p.s * a.parts + p.part) * a.c + first + i] = make_float2(h, hx);
    }
}

// Blocks [0, pairs): a (sample, group)'s two means.  The blocks after them:
// 16 channels each, summed over every sample and part.
__global__ __launch_bounds__(kNormThreads) void gn_bwd_combine_kernel(const float2* __restrict__ sums, NormArgs a,
                                                                      int64_t pairs, float2* __restrict__ means,
                                                                      float* __restrict__ dweight,
                                                                      float* __restrict__ dbias) {
    __shared__ double red[2][kNormThreads];
    const int t = threadIdx.x;
    double h = 0.0, hx = 0.0;
    if ((int64_t)blockIdx.x < pairs) {
        const int64_t s = blockIdx.x / a.groups;
        const int g = (int)(blockIdx.x - s * a.groups);
        const int64_t items = (int64_t)a.parts * a.cg;
        for (int64_t i = t; i < items; i += kNormThreads) {
            const int64_t part = i / a.cg;
            const int c = g * a.cg + (int)(i - part * a.cg);
            const float2 v = sums[(s * a.parts + part) * a.c + c];
            const float w = a.weight ? load_param(a.weight, a.ptype, c) : 1.f;
            h += (double)(w * v.x);
            hx += (double)(w * v.y);
        }
        h = wave_sum(h);
        hx = wave_sum(hx);
        if (wave_lane() == 0) {
            red[0][wave_id()] = h;
            red[1][wave_id()] = hx;
        }
        __syncthreads();
        if (t == 0) {
            const double m = (double)a.n * (double)a.cg;
            means[blockIdx.x] = make_float2((float)((red[0][0] + red[0][1] + red[0][2] + red[0][3]) / m),
                                            (float)((red[1][0] + red[1][1] + red[1][2] + red[1][3]) / m));
        }
        return;
    }
    const int c = (int)(blockIdx.x - pairs) * 16 + (t & 15);
    const int64_t rows = a.samples * a.parts;
    if (c < a.c)
        for (int64_t i = t >> 4; i < rows; i += kNormThreads / 16) {
            const float2 v = sums[i * a.c + c];
            h += (double)v.x;
            hx += (double)v.y;
        }
    red[0][t] = h;
    red[1][t] = hx;
    __syncthreads();
    if (t < 16 && c < a.c) {
        for (int i = t + 16; i < kNormThreads; i += 16) {
            h += red[0][i];
            hx += red[1][i];
        }
        if (dbias) dbias[c] = (float)h;
        if (dweight) dweight[c] = (float)hx;
    }
}

template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_dx_kernel(const T* __restrict__ dy, int64_t sdy, int64_t lddy,
                                                                 const T* __restrict__ x, NormArgs a,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd,
                                                                 const float2* __restrict__ means,
                                                                 T* __restrict__ dx) {
    const NormPlace p = norm_place(a, V);
    if (!p.live) return;
    NormBack<T, V, ACT, DROP> k;
    k.load(a, p, mean, rstd);
    const float2 m = means[p.s * a.groups + p.group];
    const T* xs = x + p.s * a.sx + p.c0;
    const T* gs = dy + p.s * sdy + p.c0;
    T* ds = dx + p.f0 * a.c + p.c0;
    for (int64_t q = p.q0 + p.row0; q < p.q1; q += p.stride) {
        float v[4][V], g[4][V];
        bool in[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t f = 4 * q + r;
            in[r] = f >= p.f0 && f < p.f1;
            if (in[r]) {
                load_vec<T, V>(xs + (f - p.f0) * a.ldx, v[r]);
                load_vec<T, V>(gs + (f - p.f0) * lddy, g[r]);
            }
        }
        const uint32_t keep = DROP ? keep_bits<V>(a.key, (uint32_t)p.c0, (uint32_t)q) : 0u;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (!in[r]) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                k.eval(v[r][e], g[r][e], e, (keep >> (4 * e + r)) & 1u, a.key.scale);
                v[r][e] = k.rs * (__builtin_fmaf(k.w[e], g[r][e], -m.x) - v[r][e] * m.y);
            }
            store_vec<T, V>(ds + (4 * q + r - p.f0) * a.c, v[r]);
        }
    }
}

}  // namespace lds

using namespace lds;

extern "C" int lds_group_norm_backward(const void* dy, int64_t sdy, int64_t lddy, const void* x, int64_t sx,
                                       int64_t ldx, int64_t samples, int64_t n, int c, int groups, int dtype,
                                       const void* weight, const void* bias, int ptype, int act, float keep_prob,
                                       float scale, uint64_t seed, uint32_t tag, uint32_t counter, const float* mean,
                                       const float* rstd, void* dx, float* dweight, float* dbias, void* ws,
                                       void* stream) {
    LDS_CHECK_ARG(norm_sizes_ok(samples, n, c, groups));
    LDS_CHECK_ARG(keep_prob >= 0.f && ptype >= LDS_F32 && ptype <= LDS_F16);
    LDS_CHECK_ARG(act >= LDS_ACT_NONE && act <= LDS_ACT_SILU && dtype >= LDS_F32 && dtype <= LDS_F16);
    // with no rows the sums are the caller's zeros to write
    if (samples == 0 || n == 0 || c == 0) return 0;
    LDS_CHECK_ARG(dy && x && mean && rstd && ws && ldx >= c && lddy >= c);
    LDS_CHECK_ARG(samples == 1 || (sx >= 0 && sdy >= 0));
    hipStream_t st = (hipStream_t)stream;
    NormArgs a{};
    const bool drop = keep_prob < 1.f && drop_key(keep_prob, scale, seed, tag, counter, &a.key);
    const int v = norm_vec(c, groups, dtype == LDS_F32 ? 4 : 2);
    const NormCut k = norm_cut(c, groups, v);
    norm_fill(&a, k, samples, n, c, groups, sx, ldx, weight, bias, ptype);
    const int64_t blocks = samples * a.parts * a.chunks;
    const int64_t pairs = dx ? samples * groups : 0;
    const int64_t cblocks = pairs + ((dweight || dbias) ? (c + 15) / 16 : 0);
    LDS_CHECK_ARG(blocks < (int64_t)1 << 31 && cblocks < (int64_t)1 << 31);
    if (cblocks == 0) return 0;
    float2* sums = (float2*)ws;
    float2* means = sums + samples * a.parts * (int64_t)c;
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        return with_vec<16 / (int)sizeof(T)>(v, [&](auto vc) -> int {
            constexpr int V = decltype(vc)::value;
            return with_act(act, [&](auto ac) -> int {
                constexpr int ACT = decltype(ac)::value;
                auto go = [&](auto dr) {
                    constexpr bool DROP = decltype(dr)::value;
                    hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, ACT, DROP>), dim3((unsigned)blocks),
                                       dim3(kNormThreads), 0, st, (const T*)dy, sdy, lddy, (const T*)x, a, mean,
                                       rstd, sums);
                    hipLaunchKernelGGL(gn_bwd_combine_kernel, dim3((unsigned)cblocks), dim3(kNormThreads), 0, st,
                                       sums, a, pairs, means, dweight, dbias);
                    if (dx)
                        hipLaunchKernelGGL((gn_bwd_dx_kernel<T, V, ACT, DROP>), dim3((unsigned)blocks),
                                           dim3(kNormThreads), 0, st, (const T*)dy, sdy, lddy, (const T*)x, a, mean,
                                           rstd, means, (T*)dx);
                };
                drop ? go(BoolC<true>{}) : go(BoolC<false>{});
                LDS_RETURN_LAST_ERROR();
            });
        });
    });
}
