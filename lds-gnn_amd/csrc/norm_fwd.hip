// Group norm + activation + keyed dropout, channels last, forward
// (include/ldsgnn.h lds_group_norm_forward).
#include "norm.hpp"

namespace lds {

struct Moments {
    double mean;  // to more than fp32's last bit: parts of data far from 0 are compared
    float count, m2;
};

// y of a quad from x.
template <typename T, int V, int ACT, bool DROP, bool SPAN, bool PAST = false>
__device__ __forceinline__ void apply_quad(const Quad<T, V>& x, const QuadRows& in, const NormParams<V>& par,
                                           const GroupValue<V, SPAN>& mu, const bool (&kept)[4][V], float scale,
                                           T* at, int64_t ld, int skip) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (r < in.lo || r >= in.hi) continue;
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float z = __builtin_fmaf(elem<T, V>(x.row[r], e) - mu[e], par.rw[e], par.b[e]);
            o[e] = act_f<ACT>(z);
            if constexpr (DROP) o[e] = kept[r][e] ? o[e] * scale : 0.f;
        }
        store_own<T, V, SPAN, PAST>(at + r * ld, skip, o);
    }
}

// ---------------------------------------------------------------------------
// slab: one block, a sample's rows of a few groups, Q quads a thread.  Bound by
// its chain of latencies (one load, two block sums, one store): one node of 32
// groups of 8, bf16, 4.6 us; 2708 x 4 groups of 4, fp32 with dropout, 8.7.
// ---------------------------------------------------------------------------

template <typename T, int V, int ACT, bool DROP, int Q>
__global__ __launch_bounds__(1024) void gn_slab_kernel(const T* x, NormArgs a, float eps, T* y,
                                                       float* __restrict__ mean, float* __restrict__ rstd) {
    __shared__ float2 red[2][2 * 1024];
    int64_t s;
    int chunk;
    if (!slab_place(a, s, chunk)) return;
    const NormPlace p = norm_place(a, V, s, 0, chunk);
    const T* xs = x + s * a.sx + p.c0;
    uint32_t masks[Q];
    if constexpr (DROP) slab_masks<V, Q>(a, p, masks);
    Quad<T, V> v[Q];
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int64_t q = p.q0 + p.ty + k * a.ty;
        if (p.live && q < p.q1) v[k].load(xs, a.ldx, p, q, quad_rows(p, q));
    }
    // The mean of the values about the group's first one, so that an offset of
    // the data costs no digits; then, about that mean, the squares and what
    // the mean is still off by (the first value may be an outlier).
    const float first = p.live ? (float)x[s * a.sx + (int64_t)p.group * a.cg] : 0.f;
    NormParams<V> par;
    if (p.live) par.load(a, p.c0);
    const float inv = 1.f / ((float)a.n * (float)a.cg);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int64_t q = p.q0 + p.ty + k * a.ty;
        if (!p.live || q >= p.q1) continue;
        const QuadRows in = quad_rows(p, q);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r >= in.lo && r < in.hi) {
#pragma unroll
                for (int e = 0; e < V; ++e) sum += elem<T, V>(v[k].row[r], e) - first;
            }
    }
    const float m0 = first + group_sum<float, 1024>(sum, a, p, (float*)red[0], blockDim.x) * inv;
    float2 d2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int64_t q = p.q0 + p.ty + k * a.ty;
        if (!p.live || q >= p.q1) continue;
        const QuadRows in = quad_rows(p, q);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (r >= in.lo && r < in.hi) {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float d = elem<T, V>(v[k].row[r], e) - m0;
                    d2.x += d;
                    d2.y = __builtin_fmaf(d, d, d2.y);
                }
            }
    }
    d2 = group_sum<float2, 1024>(d2, a, p, red[1], blockDim.x);
    const float off = d2.x * inv, mu = m0 + off;
    const float rs = 1.f / sqrtf(fmaxf(__builtin_fmaf(-off, off, d2.y * inv), 0.f) + eps);
    if (!p.live) return;
    GroupValue<V, false> gmu{{mu}};
    par.times(GroupValue<V, false>{{rs}});
    if (p.ty == 0 && p.c0 == p.group * a.cg) {
        mean[s * a.groups + p.group] = mu;
        rstd[s * a.groups + p.group] = rs;
    }
    T* ys = y + p.c0;
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        const int64_t q = p.q0 + p.ty + k * a.ty;
        if (q >= p.q1) continue;
        bool kept[4][V];
        if constexpr (DROP) unpack_kept<V>(masks[k], kept);
        apply_quad<T, V, ACT, DROP, false>(v[k], quad_rows(p, q), par, gmu, kept, a.key.scale, ys + 4 * q * a.c, a.c,
                                           0);
    }
}

// ---------------------------------------------------------------------------
// parts.  Bound by memory: 8 x 20000 x 256 bf16 (82 MB) statistics 17.3 us, result
// 27.0 (x comes from the memory-side cache the second time); with dropout 34,
// bound by the vector units (24 operations a value, half of them the mask).
// ---------------------------------------------------------------------------

// Statistics of one part.  A thread takes the 4 V values of a row quad at a
// time: their mean, about the first of them, then the squares about that mean,
// then one merge into the thread's running moments,
//   mean' = mean + δ m/(n+m),  m2' = m2 + m2_quad + δ² n m/(n+m).
// No difference of large sums is taken, so neither an offset of the data nor an
// outlier costs digits; means are carried in fp64.
template <typename T, int V>
__device__ __forceinline__ void quad_moments(const Quad<T, V>& v, const QuadRows& in, double& mean, float& m2,
                                             float& cnt) {
    float f[4][V], s1 = 0.f, s2 = 0.f;
    // rows outside the sample repeat its nearest row: out of the sums by a factor
    const float k = elem<T, V>(v.row[0], 0);
    const float m = (float)((in.hi - in.lo) * V);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float use = r >= in.lo && r < in.hi ? 1.f : 0.f;
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            f[r][e] = elem<T, V>(v.row[r], e) - k;
            t += f[r][e];
        }
        s1 = __builtin_fmaf(t, use, s1);
    }
    const float mq = s1 * __builtin_amdgcn_rcpf(m);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const float use = r >= in.lo && r < in.hi ? 1.f : 0.f;
        float t = 0.f;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const float d = f[r][e] - mq;
            t = __builtin_fmaf(d, d, t);
        }
        s2 = __builtin_fmaf(t, use, s2);
    }
    const double delta = ((double)k + (double)mq) - mean;
    const float part = m * __builtin_amdgcn_rcpf(cnt + m);
    mean += delta * (double)part;
    m2 += __builtin_fmaf((float)delta * (float)delta, cnt * part, s2);
    cnt += m;
}

template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void gn_stats_kernel(const T* __restrict__ x, NormArgs a,
                                                                Moments* __restrict__ out) {
    __shared__ double red[3][2 * kNormThreads];
    const NormPlace p = norm_part_place(a, V);
    double mean = 0.0;
    float m2 = 0.f, cnt = 0.f;
    if (p.live) {
        const T* xs = x + p.s * a.sx + p.c0;
        each_quad(a, p, [&](int64_t q, const QuadRows in) {
            Quad<T, V> v;
            v.load(xs, a.ldx, p, q, in);
            quad_moments<T, V>(v, in, mean, m2, cnt);
        });
    }
    const double c = group_sum<double, kNormThreads>((double)cnt, a, p, red[0], kNormThreads);
    const double gm =
        group_sum<double, kNormThreads>((double)cnt * mean, a, p, red[1], kNormThreads) / (c > 0.0 ? c : 1.0);
    const float d = (float)(mean - gm);
    const double g2 = group_sum<double, kNormThreads>(cnt > 0.f ? (double)(m2 + cnt * d * d) : 0.0, a, p, red[2],
                                                      kNormThreads);
    const int at = a.sub == 1 ? 0 : p.chunk - p.group * a.sub;
    if (p.live && p.ty == 0 && (a.sub == 1 ? p.tx % a.lpg == 0 : p.tx == 0))
        out[(p.s * a.groups + p.group) * ((int64_t)a.parts * a.sub) + p.part * a.sub + at] =
            Moments{gm, (float)c, (float)g2};
}

// The same where vectors lie across groups: running moments per channel, about
// the channel's first value, put together per group at the end.
template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void gn_stats_span_kernel(const T* __restrict__ x, NormArgs a,
                                                                     Moments* __restrict__ out) {
    __shared__ double s_mean[V][kNormThreads];
    __shared__ float s_m2[V][kNormThreads], s_cnt[kNormThreads];
    const NormPlace p = norm_part_place(a, V);
    float k[V], mean[V] = {}, m2[V] = {}, cnt = 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) k[e] = 0.f;
    if (p.live) {
        const T* xs = x + p.s * a.sx + p.c0;
        each_quad(a, p, [&](int64_t q, const QuadRows in) {
            Quad<T, V> v;
            v.load(xs, a.ldx, p, q, in);
            if (cnt == 0.f) {
#pragma unroll
                for (int e = 0; e < V; ++e) k[e] = elem<T, V>(v.row[0], e);
            }
            const float m = (float)(in.hi - in.lo), over = __builtin_amdgcn_rcpf(m);
            const float part = m * __builtin_amdgcn_rcpf(cnt + m), both = cnt * part;
            float use[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) use[r] = r >= in.lo && r < in.hi ? 1.f : 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                float d[4], s1 = 0.f, s2 = 0.f;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    d[r] = elem<T, V>(v.row[r], e) - k[e];
                    s1 = __builtin_fmaf(use[r], d[r], s1);
                }
                const float mq = s1 * over;
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float t = use[r] * (d[r] - mq);
                    s2 = __builtin_fmaf(t, t, s2);
                }
                const float delta = mq - mean[e];
                mean[e] = __builtin_fmaf(delta, part, mean[e]);
                m2[e] += __builtin_fmaf(delta * delta, both, s2);
            }
            cnt += m;
        });
    }
    s_cnt[threadIdx.x] = cnt;
#pragma unroll
    for (int e = 0; e < V; ++e) {
        s_mean[e][threadIdx.x] = (double)k[e] + (double)mean[e];
        s_m2[e][threadIdx.x] = m2[e];
    }
    __syncthreads();
    // a team of lanes per group over its channels in the ty rows of threads
    const int members = a.ty * a.cg;
    int team = kWave;
    while (team > 1 && (team / 2 >= members || a.groups * team > 2 * kNormThreads)) team /= 2;
    const int lane = threadIdx.x & (team - 1);
    const int end = (a.lanes - 1) * V;  // the last vector ends with the row
    for (int g = threadIdx.x / team; g < a.groups; g += kNormThreads / team) {
        const auto each = [&](auto&& f) {
            for (int i = lane; i < members; i += team) {
                const int r = (int)((unsigned)i / (unsigned)a.cg), c = g * a.cg + (i - r * a.cg);
                const int vec = c < end ? c / V : a.lanes - 1, e = c < end ? c % V : c - (a.c - V);
                const int t = r * a.lanes + vec;
                if (s_cnt[t] > 0.f) f(s_cnt[t], s_mean[e][t], s_m2[e][t]);
            }
        };
        double n = 0.0, mu = 0.0, v = 0.0;
        each([&](float c, double m, float) {
            n += (double)c;
            mu += (double)c * m;
        });
        for (int o = team / 2; o > 0; o >>= 1) {
            n += __shfl_xor(n, o);
            mu += __shfl_xor(mu, o);
        }
        mu /= n > 0.0 ? n : 1.0;
        each([&](float c, double m, float q) {
            const double d = m - mu;
            v += (double)q + (double)c * d * d;
        });
        for (int o = team / 2; o > 0; o >>= 1) v += __shfl_xor(v, o);
        if (lane == 0) out[(p.s * a.groups + g) * (int64_t)a.parts + p.part] = Moments{mu, (float)n, (float)v};
    }
}

// One wave per (sample, group): its parts combined in fp64.
__global__ __launch_bounds__(kNormThreads) void gn_combine_kernel(const Moments* __restrict__ in, int64_t total,
                                                                  int parts, float eps, float* __restrict__ mean,
                                                                  float* __restrict__ rstd) {
    const int64_t i = (int64_t)blockIdx.x * (kNormThreads / kWave) + wave_id();
    if (i >= total) return;
    const Moments* m = in + i * parts;
    double c = 0.0, s = 0.0;
#pragma unroll 4
    for (int j = wave_lane(); j < parts; j += kWave) {
        c += (double)m[j].count;
        s += (double)m[j].count * m[j].mean;
    }
    c = wave_sum(c);
    s = wave_sum(s);
    const double mu = s / c;
    double v = 0.0;
#pragma unroll 4
    for (int j = wave_lane(); j < parts; j += kWave) {
        const double d = m[j].mean - mu;
        v += m[j].count > 0.f ? (double)m[j].m2 + (double)m[j].count * d * d : 0.0;
    }
    v = wave_sum(v);
    if (wave_lane() == 0) {
        mean[i] = (float)mu;
        rstd[i] = (float)(1.0 / sqrt(v / c + (double)eps));
    }
}

// PAST: x is read and y stored past the caches, and they do not overlap (16 x 20000 x
// 256 fp32 with dropout 109 us; 122 where the compiler cannot know it).
template <typename T, int V, int ACT, bool DROP, bool SPAN, bool PAST>
__global__ __launch_bounds__(kNormThreads) void gn_apply_kernel(Pointer<const T, PAST> x, NormArgs a,
                                                                const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, Pointer<T, PAST> y) {
    const NormPlace p = norm_part_place(a, V);
    if (!p.live) return;
    GroupValue<V, SPAN> mu, rs;
    mu.fill(a, p, [&](int g) { return mean[p.s * a.groups + g]; });
    rs.fill(a, p, [&](int g) { return rstd[p.s * a.groups + g]; });
    NormParams<V> par;
    par.load(a, p.c0);
    ColumnKeep<V> columns;
    if constexpr (DROP) columns.init(a.key, (uint32_t)p.c0);
    const T* xs = x + p.s * a.sx + p.c0;
    T* ys = y + p.c0;
    par.times(rs);
    each_quad(a, p, [&](int64_t q, const QuadRows in) {
        Quad<T, V> v;
        v.template load<PAST>(xs, a.ldx, p, q, in);
        bool kept[4][V];
        if constexpr (DROP) columns.quad(a.key, (uint32_t)q, kept);
        apply_quad<T, V, ACT, DROP, SPAN, PAST>(v, in, par, mu, kept, a.key.scale, ys + 4 * q * a.c, a.c, p.skip);
    });
}

}  // namespace lds

using namespace lds;

extern "C" int64_t lds_group_norm_ws_bytes(int64_t samples, int64_t n, int c, int groups, int dtype, int backward) {
    if (!norm_sizes_ok(samples, n, c, groups) || dtype < LDS_F32 || dtype > LDS_F16) return -1;
    if (samples == 0 || n == 0 || c == 0) return 0;
    const NormPlan k = norm_plan(samples, n, c, groups, dtype, backward ? kBackwardSlabThreads : kForwardSlabThreads);
    if (backward) return backward_ws(k.a, k.slab);
    return k.slab ? 0 : samples * groups * k.a.parts * k.a.sub * (int64_t)sizeof(Moments);
}

extern "C" int lds_group_norm_forward(const void* x, int64_t sx, int64_t ldx, int64_t samples, int64_t n, int c,
                                      int groups, int dtype, const void* weight, const void* bias, int ptype,
                                      float eps, int act, float keep_prob, float scale, uint64_t seed, uint32_t tag,
                                      uint32_t counter, void* y, float* mean, float* rstd, void* ws, void* stream) {
    LDS_CHECK_ARG(norm_sizes_ok(samples, n, c, groups) && eps >= 0.f);
    LDS_CHECK_ARG(keep_prob >= 0.f && ptype >= LDS_F32 && ptype <= LDS_F16);
    LDS_CHECK_ARG(act >= LDS_ACT_NONE && act <= LDS_ACT_SILU && dtype >= LDS_F32 && dtype <= LDS_F16);
    if (samples == 0 || n == 0 || c == 0) return 0;
    LDS_CHECK_ARG(x && y && mean && rstd && ldx >= c && (samples == 1 || sx >= 0));
    hipStream_t st = (hipStream_t)stream;
    NormPlan k = norm_plan(samples, n, c, groups, dtype, kForwardSlabThreads);
    NormArgs& a = k.a;
    LDS_CHECK_ARG(k.slab || ws);
    const bool drop = keep_prob < 1.f && drop_key(keep_prob, scale, seed, tag, counter, &a.key);
    a.sx = sx;
    a.ldx = ldx;
    a.weight = weight;
    a.bias = bias;
    a.ptype = ptype;
    const int size = norm_elem(dtype);
    a.whole = whole_store(y, samples, n, c, size, x, sx, ldx);
    NormArgs b = a;  // the second pass of the parts form
    if (!k.slab) {
        const NormArgs cut = norm_plan(samples, n, c, groups, dtype, kForwardSlabThreads, kApplyBlocks).a;
        b.parts = cut.parts;
        b.part_q = cut.part_q;
    }
    const int64_t blocks = k.slab ? slab_blocks(a) : samples * a.parts * a.chunks;
    const int64_t pairs = samples * groups;
    LDS_CHECK_ARG(blocks < (int64_t)1 << 31 && samples * b.parts * b.chunks < (int64_t)1 << 31);
    LDS_CHECK_ARG(pairs < (int64_t)1 << 32);
    const bool past = a.whole && past_caches(samples * n * c * size) && whole_lines(x, samples, sx, ldx, c, size) &&
                      whole_lines(y, 1, 0, c, c, size);
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        return with_vec<16 / (int)sizeof(T)>(k.v, a.span, [&](auto vc, auto sc) -> int {
            constexpr int V = decltype(vc)::value;
            constexpr bool SPAN = decltype(sc)::value, WIDE = !SPAN && V * sizeof(T) == 16;
            if (!k.slab) {
                norm_launches(a, blocks, kNormThreads, [&](const NormArgs& l, unsigned count) {
                    if constexpr (SPAN)
                        hipLaunchKernelGGL((gn_stats_span_kernel<T, V>), dim3(count), dim3(kNormThreads), 0, st,
                                           (const T*)x, l, (Moments*)ws);
                    else
                        hipLaunchKernelGGL((gn_stats_kernel<T, V>), dim3(count), dim3(kNormThreads), 0, st,
                                           (const T*)x, l, (Moments*)ws);
                });
                in_launches((pairs + 3) / 4, kNormThreads, [&](int64_t first, unsigned count) {
                    const int64_t i = first * 4, each = (int64_t)a.parts * a.sub;
                    hipLaunchKernelGGL(gn_combine_kernel, dim3(count), dim3(kNormThreads), 0, st,
                                       (const Moments*)ws + i * each, pairs - i, (int)each, eps, mean + i, rstd + i);
                });
            }
            return with_act(act, [&](auto ac) -> int {
                constexpr int ACT = decltype(ac)::value;
                auto go = [&](auto dr) {
                    constexpr bool DROP = decltype(dr)::value;
                    auto slab = [&](auto qc) {
                        norm_launches(a, blocks, k.threads, [&](const NormArgs& l, unsigned count) {
                            hipLaunchKernelGGL((gn_slab_kernel<T, V, ACT, DROP, decltype(qc)::value>), dim3(count),
                                               dim3(k.threads), 0, st, (const T*)x, l, eps, (T*)y, mean, rstd);
                        });
                    };
                    auto apply = [&](auto ps) {
                        norm_launches(b, samples * b.parts * b.chunks, kNormThreads,
                                      [&](const NormArgs& l, unsigned count) {
                            hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, DROP, SPAN, WIDE && decltype(ps)::value>),
                                               dim3(count), dim3(kNormThreads), 0, st, (const T*)x, l, mean, rstd,
                                               (T*)y);
                        });
                    };
                    if (!k.slab)
                        past ? apply(BoolC<true>{}) : apply(BoolC<false>{});
                    else if constexpr (!SPAN)
                        with_quads<V>(k.quads, slab);
                };
                drop ? go(BoolC<true>{}) : go(BoolC<false>{});
                LDS_RETURN_LAST_ERROR();
            });
        });
    });
}
