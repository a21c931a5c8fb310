// Group norm + activation + keyed dropout, channels last, forward
// (include/ldsgnn.h lds_group_norm_forward).
//
// Three launches: (count, mean, centred squares) of every row part and group;
// their combination per (sample, group); the elementwise pass.
#include "norm.hpp"

namespace lds {

struct Moments {
    double mean;  // to more than fp32's last bit: parts of data far from 0 are compared
    float count, m2;
};

// Statistics of one part.  A thread takes the 4 V values of a row quad at a
// time: their mean, about the first of them, then the squares about that mean,
// then one merge into the thread's running moments,
//   mean' = mean + δ m/(n+m),  m2' = m2 + m2_quad + δ² n m/(n+m).
// No difference of large sums is taken, so neither an offset of the data nor an
// outlier costs digits; means are carried in fp64.
template <typename T, int V>
__global__ __launch_bounds__(kNormThreads) void gn_stats_kernel(const T* __restrict__ x, NormArgs a,
                                                                Moments* __restrict__ out) {
    __shared__ double s_mean[kNormThreads];
    __shared__ float s_cnt[kNormThreads], s_m2[kNormThreads];
    const NormPlace p = norm_place(a, V);
    double mean = 0.0;
    float m2 = 0.f, cnt = 0.f;
    if (p.live) {
        const T* xs = x + p.s * a.sx + p.c0;
        for (int64_t q = p.q0 + p.row0; q < p.q1; q += p.stride) {
            float v[4][V];
            bool in[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int64_t f = 4 * q + r;
                in[r] = f >= p.f0 && f < p.f1;
                if (in[r]) load_vec<T, V>(xs + (f - p.f0) * a.ldx, v[r]);
            }
            quad_moments<V>(v, in, mean, m2, cnt);
        }
    }
    s_cnt[threadIdx.x] = cnt;
    s_mean[threadIdx.x] = mean;
    s_m2[threadIdx.x] = m2;
    __syncthreads();
    // one wave per group of the chunk over its ty x lpg threads
    const int per = a.sub == 1 ? a.lanes / a.lpg : 1;
    const int members = a.ty * a.lpg;
    for (int gi = wave_id(); gi < per; gi += kNormThreads / kWave) {
        const int g = a.sub == 1 ? p.chunk * per + gi : p.chunk / a.sub;
        if (g >= a.groups) break;
        float c = 0.f, g2 = 0.f;
        double m = 0.0;
        for (int i = wave_lane(); i < members; i += kWave) {
            const int t = (i / a.lpg) * a.lanes + gi * a.lpg + i % a.lpg;
            c += s_cnt[t];
            m += (double)s_cnt[t] * s_mean[t];
        }
        c = wave_sum(c);
        m = wave_sum(m);
        const double gm = c > 0.f ? m / (double)c : 0.0;
        for (int i = wave_lane(); i < members; i += kWave) {
            const int t = (i / a.lpg) * a.lanes + gi * a.lpg + i % a.lpg;
            const float d = (float)(s_mean[t] - gm);
            g2 += s_cnt[t] > 0.f ? s_m2[t] + s_cnt[t] * d * d : 0.f;
        }
        g2 = wave_sum(g2);
        if (wave_lane() == 0) {
            const int j = p.part * a.sub + (a.sub == 1 ? 0 : p.chunk - g * a.sub);
            out[(p.s * a.groups + g) * ((int64_t)a.parts * a.sub) + j] = Moments{gm, c, g2};
        }
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
    for (int j = wave_lane(); j < parts; j += kWave) {
        c += (double)m[j].count;
        s += (double)m[j].count * m[j].mean;
    }
    c = wave_sum(c);
    s = wave_sum(s);
    const double mu = s / c;
    double v = 0.0;
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

template <typename T, int V, int ACT, bool DROP>
__global__ __launch_bounds__(kNormThreads) void gn_apply_kernel(const T* __restrict__ x, NormArgs a,
                                                                const float* __restrict__ mean,
                                                                const float* __restrict__ rstd, T* __restrict__ y) {
    const NormPlace p = norm_place(a, V);
    if (!p.live) return;
    const float mu = mean[p.s * a.groups + p.group];
    const float rs = rstd[p.s * a.groups + p.group];
    float w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        w[e] = a.weight ? load_param(a.weight, a.ptype, p.c0 + e) : 1.f;
        b[e] = a.bias ? load_param(a.bias, a.ptype, p.c0 + e) : 0.f;
    }
    const T* xs = x + p.s * a.sx + p.c0;
    T* ys = y + p.f0 * a.c + p.c0;
    for (int64_t q = p.q0 + p.row0; q < p.q1; q += p.stride) {
        float v[4][V];
        bool in[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int64_t f = 4 * q + r;
            in[r] = f >= p.f0 && f < p.f1;
            if (in[r]) load_vec<T, V>(xs + (f - p.f0) * a.ldx, v[r]);
        }
        const uint32_t keep = DROP ? keep_bits<V>(a.key, (uint32_t)p.c0, (uint32_t)q) : 0u;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (!in[r]) continue;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float z = __builtin_fmaf((v[r][e] - mu) * rs, w[e], b[e]);
                float o = act_f<ACT>(z);
                if constexpr (DROP) o = (keep >> (4 * e + r)) & 1u ? o * a.key.scale : 0.f;
                v[r][e] = o;
            }
            store_vec<T, V>(ys + (4 * q + r - p.f0) * a.c, v[r]);
        }
    }
}

}  // namespace lds

using namespace lds;

namespace {

int elem_bytes(int dtype) { return dtype == LDS_F32 ? 4 : 2; }

}  // namespace

extern "C" int64_t lds_group_norm_ws_bytes(int64_t samples, int64_t n, int c, int groups, int dtype, int backward) {
    if (!norm_sizes_ok(samples, n, c, groups) || dtype < LDS_F32 || dtype > LDS_F16) return -1;
    if (samples == 0 || n == 0 || c == 0) return 0;
    const NormCut k = norm_cut(c, groups, norm_vec(c, groups, elem_bytes(dtype)));
    int parts;
    int64_t part_q;
    norm_parts(samples, n, k, kNormBlocks, &parts, &part_q);
    if (!backward) return samples * groups * parts * k.sub * (int64_t)sizeof(Moments);
    // per channel sums of the parts, then the two group means
    return samples * parts * (int64_t)c * 8 + samples * groups * 8;
}

extern "C" int lds_group_norm_forward(const void* x, int64_t sx, int64_t ldx, int64_t samples, int64_t n, int c,
                                      int groups, int dtype, const void* weight, const void* bias, int ptype,
                                      float eps, int act, float keep_prob, float scale, uint64_t seed, uint32_t tag,
                                      uint32_t counter, void* y, float* mean, float* rstd, void* ws, void* stream) {
    LDS_CHECK_ARG(norm_sizes_ok(samples, n, c, groups) && eps >= 0.f);
    LDS_CHECK_ARG(keep_prob >= 0.f && ptype >= LDS_F32 && ptype <= LDS_F16);
    LDS_CHECK_ARG(act >= LDS_ACT_NONE && act <= LDS_ACT_SILU && dtype >= LDS_F32 && dtype <= LDS_F16);
    if (samples == 0 || n == 0 || c == 0) return 0;
    LDS_CHECK_ARG(x && y && mean && rstd && ws && ldx >= c && (samples == 1 || sx >= 0));
    hipStream_t st = (hipStream_t)stream;
    NormArgs a{};
    const bool drop = keep_prob < 1.f && drop_key(keep_prob, scale, seed, tag, counter, &a.key);
    const int v = norm_vec(c, groups, elem_bytes(dtype));
    const NormCut k = norm_cut(c, groups, v);
    norm_fill(&a, k, samples, n, c, groups, sx, ldx, weight, bias, ptype);
    const int64_t blocks = samples * a.parts * a.chunks;
    const int64_t pairs = samples * groups;
    LDS_CHECK_ARG(blocks < (int64_t)1 << 31 && pairs < (int64_t)1 << 32);
    Moments* mom = (Moments*)ws;
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        return with_vec<16 / (int)sizeof(T)>(v, [&](auto vc) -> int {
            constexpr int V = decltype(vc)::value;
            hipLaunchKernelGGL((gn_stats_kernel<T, V>), dim3((unsigned)blocks), dim3(kNormThreads), 0, st,
                               (const T*)x, a, mom);
            hipLaunchKernelGGL(gn_combine_kernel, dim3((unsigned)((pairs + 3) / 4)), dim3(kNormThreads), 0, st, mom,
                               pairs, a.parts * a.sub, eps, mean, rstd);
            return with_act(act, [&](auto ac) -> int {
                constexpr int ACT = decltype(ac)::value;
                if (drop)
                    hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, true>), dim3((unsigned)blocks),
                                       dim3(kNormThreads), 0, st, (const T*)x, a, mean, rstd, (T*)y);
                else
                    hipLaunchKernelGGL((gn_apply_kernel<T, V, ACT, false>), dim3((unsigned)blocks),
                                       dim3(kNormThreads), 0, st, (const T*)x, a, mean, rstd, (T*)y);
                LDS_RETURN_LAST_ERROR();
            });
        });
    });
}
