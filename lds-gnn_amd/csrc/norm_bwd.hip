// Group norm + activation + keyed dropout, channels last, backward
// (include/ldsgnn.h lds_group_norm_backward).
//
//   h = dy · mask · act'(z),  dβ_c = Σ h,  dγ_c = Σ h x̂,
//   dx = r (γ h - mean_g(γ h) - x̂ mean_g(γ h x̂))
// z, x̂ and the mask are recomputed from x, the statistics and the key.
#include "norm.hpp"

namespace lds {

// x - mean and h / scale of a quad.
template <typename T, int V, int ACT, bool DROP, bool SPAN>
struct BackQuad {
    float d[4][V], h[4][V];

    __device__ __forceinline__ void eval(const Quad<T, V>& x, const Quad<T, V>& g, const NormParams<V>& par,
                                         const GroupValue<V, SPAN>& mu, const bool (&kept)[4][V]) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                d[r][e] = elem<T, V>(x.row[r], e) - mu[e];
                float t = elem<T, V>(g.row[r], e);
                if constexpr (DROP) t = kept[r][e] ? t : 0.f;
                if constexpr (ACT == LDS_ACT_RELU) {
                    t = __builtin_fmaf(d[r][e], par.rw[e], par.b[e]) <= 0.f ? 0.f : t;
                } else if constexpr (ACT != LDS_ACT_NONE) {
                    t *= act_grad<ACT>(__builtin_fmaf(d[r][e], par.rw[e], par.b[e]));
                }
                h[r][e] = t;
            }
    }
    // Σ h and Σ h (x - mean), both over scale
    __device__ __forceinline__ void sums(const QuadRows& in, float (&sh)[V], float (&sx)[V]) const {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r < in.lo || r >= in.hi) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                sh[e] += h[r][e];
                sx[e] = __builtin_fmaf(h[r][e], d[r][e], sx[e]);
            }
        }
    }
    // dx = (γ rstd scale) h + (-(rstd² m2) (x - mean) - rstd m1)
    template <bool PAST>
    __device__ __forceinline__ void store(const QuadRows& in, const float (&rws)[V], const GroupValue<V, SPAN>& k0,
                                          const GroupValue<V, SPAN>& k1, T* at, int64_t ld,
                                          int skip) const {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (r < in.lo || r >= in.hi) continue;
            float o[V];
#pragma unroll
            for (int e = 0; e < V; ++e) o[e] = __builtin_fmaf(rws[e], h[r][e], __builtin_fmaf(k1[e], d[r][e], k0[e]));
            store_own<T, V, SPAN, PAST>(at + r * ld, skip, o);
        }
    }
};

template <typename T, int V>
struct QuadPair {
    Quad<T, V> x, g;
};

// A thread's channel sums from those of BackQuad::sums.
template <int V, bool SPAN>
__device__ __forceinline__ void finish_sums(float (&sh)[V], float (&sx)[V], float scale,
                                            const GroupValue<V, SPAN>& rs) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        sh[e] *= scale;
        sx[e] *= scale * rs[e];
    }
}

// The two sums of every channel of a block's chunk over its ty rows: value
// i of a thread at red[i][thread], V values at a time.  Channel i of the chunk
// is summed by a team of lanes in a fixed order; f(i, h, hx).
template <int V, int NT, typename F>
__device__ __forceinline__ void channel_sums(const float (&sh)[V], const float (&sx)[V], const NormArgs& a,
                                             float2 (*red)[NT], int threads, F&& f) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < V; ++e) red[e][threadIdx.x] = make_float2(sh[e], sx[e]);
    __syncthreads();
    const int channels = a.lanes * V;
    int team = 16;
    while (team > 1 && (team / 2 >= a.ty || channels * team > 2 * threads)) team /= 2;
    const int lane = threadIdx.x & (team - 1);
    for (int i = threadIdx.x / team; i < channels; i += threads / team) {
        float h = 0.f, hx = 0.f;
        for (int r = lane; r < a.ty; r += team) {
            const float2 t = red[i % V][r * a.lanes + i / V];
            h += t.x;
            hx += t.y;
        }
        for (int o = team / 2; o > 0; o >>= 1) {
            h += __shfl_xor(h, o);
            hx += __shfl_xor(hx, o);
        }
        if (lane == 0) f(i, h, hx);
    }
}

// The chunk's first channel and the end of those it may write.
__device__ __forceinline__ int chunk_first(const NormArgs& a, int chunk, int v) {
    return a.sub == 1 ? chunk * a.lanes * v : (chunk / a.sub) * a.cg + (chunk % a.sub) * a.lanes * v;
}
__device__ __forceinline__ int chunk_last(const NormArgs& a, int chunk) {
    return a.sub == 1 ? a.c : (chunk / a.sub + 1) * a.cg;
}

// ---------------------------------------------------------------------------
// slab: x and dy in registers, Q quads a thread
// ---------------------------------------------------------------------------

template <typename T, int V, int ACT, bool DROP, int Q>
__global__ __launch_bounds__(kBackwardSlabThreads) void gn_bwd_slab_kernel(
    const T* dy, int64_t sdy, int64_t lddy, const T* x, NormArgs a, const float* __restrict__ mean,
    const float* __restrict__ rstd, float2* __restrict__ sums, float* __restrict__ dweight, float* __restrict__ dbias,
    T* dx) {
    constexpr int NT = kBackwardSlabThreads;
    __shared__ float2 chan[V][NT];
    __shared__ float2 red[2 * NT];
    int64_t s;
    int chunk;
    if (!slab_place(a, s, chunk)) return;
    const NormPlace p = norm_place(a, V, s, 0, chunk);
    const T* xs = x + s * a.sx + p.c0;
    const T* gs = dy + s * sdy + p.c0;
    uint32_t masks[Q];
    if constexpr (DROP) slab_masks<V, Q>(a, p, masks);
    Quad<T, V> v[Q], g[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int64_t q = p.q0 + p.ty + k * a.ty;
        if (p.live && q < p.q1) {
            const QuadRows in = quad_rows(p, q);
            v[k].load(xs, a.ldx, p, q, in);
            g[k].load(gs, lddy, p, q, in);
        }
    }
    GroupValue<V, false> mu{}, rs{};
    NormParams<V> par{};
    const float scale = DROP ? a.key.scale : 1.f;
    float sh[V] = {}, sx[V] = {};
    if (p.live) {
        mu.f[0] = mean[s * a.groups + p.group];
        rs.f[0] = rstd[s * a.groups + p.group];
        par.load(a, p.c0);
        par.times(rs);
    }
    BackQuad<T, V, ACT, DROP, false> b;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int64_t q = p.q0 + p.ty + k * a.ty;
        if (!p.live || q >= p.q1) continue;
        bool kept[4][V];
        if constexpr (DROP) unpack_kept<V>(masks[k], kept);
        b.eval(v[k], g[k], par, mu, kept);
        b.sums(quad_rows(p, q), sh, sx);
    }
    finish_sums<V>(sh, sx, scale, rs);
    if (sums || dweight || dbias) {
        const int c0 = chunk_first(a, chunk, V), c1 = chunk_last(a, chunk);
        channel_sums<V, NT>(sh, sx, a, chan, blockDim.x, [&](int i, float h, float hx) {
            if (c0 + i >= c1) return;
            if (sums) {
                sums[s * a.c + c0 + i] = make_float2(h, hx);
            } else {  // one sample: the sums are the gradients
                if (dbias) dbias[c0 + i] = h;
                if (dweight) dweight[c0 + i] = hx;
            }
        });
    }
    if (!dx) return;
    float2 m = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < V; ++e) {
        m.x = __builtin_fmaf(par.rw[e], sh[e], m.x);
        m.y = __builtin_fmaf(par.rw[e], sx[e], m.y);
    }
    m = group_sum<float2, NT>(m, a, p, red, blockDim.x);
    const float inv = 1.f / ((float)a.n * (float)a.cg);
    if (!p.live) return;
    // of γ rstd: one rstd is in the sums
    const GroupValue<V, false> k0{{-m.x * inv}}, k1{{-rs[0] * (m.y * inv)}};
#pragma unroll
    for (int e = 0; e < V; ++e) par.rw[e] *= Q > 1 ? 1.f : scale;
    T* ds = dx + p.c0;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int64_t q = p.q0 + p.ty + k * a.ty;
        if (q >= p.q1) continue;
        if constexpr (Q > 1) {
            bool kept[4][V];
            if constexpr (DROP) unpack_kept<V>(masks[k], kept);
            b.eval(v[k], g[k], par, mu, kept);
        }
        float rws[V];
#pragma unroll
        for (int e = 0; e < V; ++e) rws[e] = Q > 1 ? par.rw[e] * scale : par.rw[e];
        b.template store<false>(quad_rows(p, q), rws, k0, k1, ds + 4 * q * a.c, a.c, 0);
    }
}

// ---------------------------------------------------------------------------
// parts.  8 x 20000 x 256 bf16, silu and dropout: sums 37 us for 164 MB (26 vector
// operations a value, two waves a SIMD), result 44 us for 246 MB (5.6 TB/s).
// ---------------------------------------------------------------------------

template <typename T, int V, int ACT, bool DROP, bool SPAN>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_sums_kernel(const T* __restrict__ dy, int64_t sdy,
                                                                   int64_t lddy, const T* __restrict__ x, NormArgs a,
                                                                   const float* __restrict__ mean,
                                                                   const float* __restrict__ rstd,
                                                                   float2* __restrict__ out) {
    __shared__ float2 red[V][kNormThreads];
    const NormPlace p = norm_part_place(a, V);
    float sh[V] = {}, sx[V] = {};
    if (p.live) {
        GroupValue<V, SPAN> mu, rs;
        mu.fill(a, p, [&](int g) { return mean[p.s * a.groups + g]; });
        rs.fill(a, p, [&](int g) { return rstd[p.s * a.groups + g]; });
        NormParams<V> par;
        par.load(a, p.c0);
        ColumnKeep<V> columns;
        if constexpr (DROP) columns.init(a.key, (uint32_t)p.c0);
        const T* xs = x + p.s * a.sx + p.c0;
        const T* gs = dy + p.s * sdy + p.c0;
        par.times(rs);
        each_quad_ahead<QuadPair<T, V>>(
            a, p,
            [&](QuadPair<T, V>& d, int64_t q, const QuadRows in) {
                d.x.load(xs, a.ldx, p, q, in);
                d.g.load(gs, lddy, p, q, in);
            },
            [&](const QuadPair<T, V>& d, int64_t q, const QuadRows in) {
            bool kept[4][V];
            if constexpr (DROP) columns.quad(a.key, (uint32_t)q, kept);
            BackQuad<T, V, ACT, DROP, SPAN> b;
            b.eval(d.x, d.g, par, mu, kept);
            b.sums(in, sh, sx);
        });
        finish_sums<V>(sh, sx, DROP ? a.key.scale : 1.f, rs);
    }
    float2* sums = out + (p.s * a.parts + p.part) * a.c;
    if constexpr (SPAN) {
        channel_sums<V, kNormThreads>(sh, sx, a, red, kNormThreads, [&](int i, float h, float hx) {
            const int at = i - i % V, first = at < a.c - V ? at : a.c - V, c = first + i % V;
            if (c >= at) sums[c] = make_float2(h, hx);  // a channel's owner
        });
    } else {
        const int c0 = chunk_first(a, p.chunk, V), c1 = chunk_last(a, p.chunk);
        channel_sums<V, kNormThreads>(sh, sx, a, red, kNormThreads, [&](int i, float h, float hx) {
            if (c0 + i < c1) sums[c0 + i] = make_float2(h, hx);
        });
    }
}

// Blocks [0, pairs): a (sample, group)'s two means.  The blocks after them: four
// channels each, summed over every sample and part.
__global__ __launch_bounds__(kNormThreads) void gn_bwd_combine_kernel(const float2* __restrict__ sums, NormArgs a,
                                                                      int64_t pairs, float2* __restrict__ means,
                                                                      float* __restrict__ dweight,
                                                                      float* __restrict__ dbias) {
    __shared__ double red[2][kNormThreads];
    const int t = threadIdx.x;
    const unsigned b = blockIdx.x + a.first;
    double h = 0.0, hx = 0.0;
    if ((int64_t)b < pairs) {
        const int64_t s = b / (unsigned)a.groups;
        const int g = (int)(b - s * a.groups);
        const int64_t items = (int64_t)a.parts * a.cg;
#pragma unroll 4
        for (int64_t i = t; i < items; i += kNormThreads) {
            const int64_t part = items <= 0xffffffffll ? (uint32_t)i / (uint32_t)a.cg : i / a.cg;
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
            means[b] = make_float2((float)((red[0][0] + red[0][1] + red[0][2] + red[0][3]) / m),
                                            (float)((red[1][0] + red[1][1] + red[1][2] + red[1][3]) / m));
        }
        return;
    }
    const int c = (int)(b - pairs) * 4 + (t & 3);
    const int64_t rows = a.samples * a.parts;
    if (c < a.c) {
#pragma unroll 4
        for (int64_t i = t >> 2; i < rows; i += kNormThreads / 4) {
            const float2 v = sums[i * a.c + c];
            h += (double)v.x;
            hx += (double)v.y;
        }
    }
    for (int o = 4; o < kWave; o <<= 1) {  // the wave's 16 rows
        h += __shfl_xor(h, o);
        hx += __shfl_xor(hx, o);
    }
    if (wave_lane() < 4) {
        red[0][wave_id() * 4 + (t & 3)] = h;
        red[1][wave_id() * 4 + (t & 3)] = hx;
    }
    __syncthreads();
    if (t < 4 && c < a.c) {
        if (dbias) dbias[c] = (float)(red[0][t] + red[0][4 + t] + red[0][8 + t] + red[0][12 + t]);
        if (dweight) dweight[c] = (float)(red[1][t] + red[1][4 + t] + red[1][8 + t] + red[1][12 + t]);
    }
}

// PAST: x and dy are read past the caches (1), dx is stored past them too (2).
template <typename T, int V, int ACT, bool DROP, bool SPAN, int PAST>
__global__ __launch_bounds__(kNormThreads) void gn_bwd_dx_kernel(const T* dy, int64_t sdy, int64_t lddy, const T* x,
                                                                 NormArgs a,
                                                                 const float* __restrict__ mean,
                                                                 const float* __restrict__ rstd,
                                                                 const float2* __restrict__ means, T* dx) {
    const NormPlace p = norm_part_place(a, V);
    if (!p.live) return;
    GroupValue<V, SPAN> mu, rs, k0, k1;
    mu.fill(a, p, [&](int g) { return mean[p.s * a.groups + g]; });
    rs.fill(a, p, [&](int g) { return rstd[p.s * a.groups + g]; });
    NormParams<V> par;
    par.load(a, p.c0);
    ColumnKeep<V> columns;
    if constexpr (DROP) columns.init(a.key, (uint32_t)p.c0);
    const T* xs = x + p.s * a.sx + p.c0;
    const T* gs = dy + p.s * sdy + p.c0;
    T* ds = dx + p.c0;
    par.times(rs);
    float rws[V];
#pragma unroll
    for (int e = 0; e < V; ++e) rws[e] = DROP ? par.rw[e] * a.key.scale : par.rw[e];
    k0.fill(a, p, [&](int g) { return -rstd[p.s * a.groups + g] * means[p.s * a.groups + g].x; });
    k1.fill(a, p, [&](int g) {
        const float r = rstd[p.s * a.groups + g];
        return -r * r * means[p.s * a.groups + g].y;
    });
    each_quad_ahead<QuadPair<T, V>>(
        a, p,
        [&](QuadPair<T, V>& d, int64_t q, const QuadRows in) {
            d.x.template load<(PAST > 0)>(xs, a.ldx, p, q, in);
            d.g.template load<(PAST > 0)>(gs, lddy, p, q, in);
        },
        [&](const QuadPair<T, V>& d, int64_t q, const QuadRows in) {
        bool kept[4][V];
        if constexpr (DROP) columns.quad(a.key, (uint32_t)q, kept);
        BackQuad<T, V, ACT, DROP, SPAN> b;
        b.eval(d.x, d.g, par, mu, kept);
        b.template store<(PAST > 1)>(in, rws, k0, k1, ds + 4 * q * a.c, a.c, p.skip);
    });
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
    LDS_CHECK_ARG(dy && x && mean && rstd && ldx >= c && lddy >= c);
    LDS_CHECK_ARG(samples == 1 || (sx >= 0 && sdy >= 0));
    if (!dx && !dweight && !dbias) return 0;
    hipStream_t st = (hipStream_t)stream;
    NormPlan k = norm_plan(samples, n, c, groups, dtype, kBackwardSlabThreads);
    NormArgs& a = k.a;
    LDS_CHECK_ARG(ws || backward_ws(a, k.slab) == 0);
    const bool drop = keep_prob < 1.f && drop_key(keep_prob, scale, seed, tag, counter, &a.key);
    a.sx = sx;
    a.ldx = ldx;
    a.weight = weight;
    a.bias = bias;
    a.ptype = ptype;
    const int size = norm_elem(dtype);
    a.whole = dx && whole_store(dx, samples, n, c, size, x, sx, ldx) &&
              whole_store(dx, samples, n, c, size, dy, sdy, lddy);
    const int64_t blocks = k.slab ? slab_blocks(a) : samples * a.parts * a.chunks;
    const int64_t pairs = dx && !k.slab ? samples * groups : 0;
    const bool params = dweight || dbias;
    const int64_t cblocks = pairs + (params && !(k.slab && samples == 1) ? (c + 3) / 4 : 0);
    LDS_CHECK_ARG(blocks < (int64_t)1 << 31 && cblocks < (int64_t)1 << 31);
    float2* sums = (float2*)ws;
    float2* means = k.slab ? nullptr : sums + samples * a.parts * (int64_t)c;
    const bool lines = whole_lines(x, samples, sx, ldx, c, size) && whole_lines(dy, samples, sdy, lddy, c, size) &&
                       whole_lines(dx, 1, 0, c, c, size);
    const int past = !lines ? 0 : past_caches(samples * n * c * size) ? 2 : 1;
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        return with_vec<16 / (int)sizeof(T)>(k.v, a.span, [&](auto vc, auto sc) -> int {
            constexpr int V = decltype(vc)::value;
            constexpr bool SPAN = decltype(sc)::value, WIDE = !SPAN && V * sizeof(T) == 16;
            return with_act(act, [&](auto ac) -> int {
                constexpr int ACT = decltype(ac)::value;
                auto go = [&](auto dr) {
                    constexpr bool DROP = decltype(dr)::value;
                    auto slab = [&](auto qc) {
                        const bool direct = samples == 1;
                        norm_launches(a, blocks, k.threads, [&](const NormArgs& l, unsigned count) {
                            hipLaunchKernelGGL((gn_bwd_slab_kernel<T, V, ACT, DROP, decltype(qc)::value>), dim3(count),
                                               dim3(k.threads), 0, st, (const T*)dy, sdy, lddy, (const T*)x, l, mean,
                                               rstd, params && !direct ? sums : nullptr, direct ? dweight : nullptr,
                                               direct ? dbias : nullptr, (T*)dx);
                        });
                    };
                    if (!k.slab)
                        norm_launches(a, blocks, kNormThreads, [&](const NormArgs& l, unsigned count) {
                            hipLaunchKernelGGL((gn_bwd_sums_kernel<T, V, ACT, DROP, SPAN>), dim3(count),
                                               dim3(kNormThreads), 0, st, (const T*)dy, sdy, lddy, (const T*)x, l, mean,
                                               rstd, sums);
                        });
                    else if constexpr (!SPAN)
                        with_quads<V>(k.quads, slab);
                    norm_launches(a, cblocks, kNormThreads, [&](const NormArgs& l, unsigned count) {
                        hipLaunchKernelGGL(gn_bwd_combine_kernel, dim3(count), dim3(kNormThreads), 0, st,
                                           (const float2*)sums, l, pairs, means, dweight, dbias);
                    });
                    auto second = [&](auto ps) {
                        norm_launches(a, blocks, kNormThreads, [&](const NormArgs& l, unsigned count) {
                            hipLaunchKernelGGL(
                                (gn_bwd_dx_kernel<T, V, ACT, DROP, SPAN, WIDE ? decltype(ps)::value : 0>),
                                dim3(count), dim3(kNormThreads), 0, st, (const T*)dy, sdy, lddy, (const T*)x, l, mean,
                                rstd, (const float2*)means, (T*)dx);
                        });
                    };
                    if (!k.slab && dx) past == 2 ? second(IntC<2>{}) : past ? second(IntC<1>{}) : second(IntC<0>{});
                };
                drop ? go(BoolC<true>{}) : go(BoolC<false>{});
                LDS_RETURN_LAST_ERROR();
            });
        });
    });
}
