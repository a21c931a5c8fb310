// 8-bit integer product with row and channel scales, and the row quantiser
// (include/ldsgnn.h lds_quantize_rows, lds_int8_matmul).
//
//   y_ij = (Σ_k xq_ik wq_jk) xs_i ws_j + bias_j
// The sum runs on the int8 matrix cores (16 x 16 x 64 a wave instruction), exact in
// int32.  Lane l of an operand holds row l % 16 and the 16 bytes of k that start at
// 16 (l / 16); of a result, column l % 16 and rows 4 (l / 16) .. + 3.
#include "vec.hpp"

namespace lds {

typedef int v4i __attribute__((ext_vector_type(4)));

// q = x / s to the nearest integer, ties to even, of the exact quotient: the
// sign of x - (q ± ½) s, one fused operation, decides next to a half.
__device__ __forceinline__ int quant_exact(float x, float s, float inv) {
    const float t = x * inv;
    float q = rintf(t);
    const float d = t - q;
    if (fabsf(d) > 0.4999f) {
        const float h = q + (d < 0.f ? -0.5f : 0.5f);
        const float r = __builtin_fmaf(-h, s, x);
        q = r > 0.f ? h + 0.5f : r < 0.f ? h - 0.5f : rintf(h);
    }
    return (int)fminf(fmaxf(q, -127.f), 127.f);
}

// A row's scale from the bits of its largest |x|, and what quantises its values.
struct RowScale {
    float s, su, inv, up;
    bool zero;  // every q is 0

    __device__ __forceinline__ explicit RowScale(uint32_t top) {
        const bool finite = top < 0x7f800000u;
        s = finite ? __uint_as_float(top) / 127.f : __uint_as_float(0x7fc00000u);
        zero = !finite || s == 0.f;
        // the quotient is unchanged when both sides grow by 2^64: 1/s stays finite
        // for the smallest scales
        up = s < 1e-30f ? 18446744073709551616.f : 1.f;
        su = s * up;
        inv = zero ? 0.f : 1.f / su;
    }
    // V values as bytes.  Adding 1.5 2^23 rounds x (1/s) to an integer (ties to
    // even) that then stands in the low bits.  x (1/s) is within 127 2^-22 of the
    // quotient, so only a vector with a value that close to a half (one in a
    // few thousand), or of a row with a tiny scale, is done again exactly.
    // |q| <= 127 needs no clamp: the largest quotient is 127 to within 2^-16.
    template <int V>
    __device__ __forceinline__ void put(signed char* __restrict__ q, const float (&f)[V]) const {
        constexpr float kRound = 12582912.f;
        static_assert(V % 4 == 0, "whole words");
        uint32_t o[V / 4];
        float off = up != 1.f ? 1.f : 0.f;
#pragma unroll
        for (int w = 0; w < V / 4; ++w) {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float r = __builtin_fmaf(f[4 * w + e], inv, kRound);
                off = fmaxf(off, fabsf(__builtin_fmaf(f[4 * w + e], inv, -(r - kRound))));
                y[e] = __float_as_uint(r);
            }
            const uint32_t lo = __builtin_amdgcn_perm(y[1], y[0], 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(y[3], y[2], 0x04000c0cu);
            o[w] = lo | hi;
        }
        if (off > 0.4999f) {
#pragma unroll
            for (int w = 0; w < V / 4; ++w) {
                o[w] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    o[w] |= ((uint32_t)quant_exact(f[4 * w + e] * up, su, inv) & 0xffu) << (8 * e);
            }
        }
        typedef uint32_t words __attribute__((ext_vector_type(V / 4)));
        words v;
#pragma unroll
        for (int w = 0; w < V / 4; ++w) v[w] = zero ? 0u : o[w];
        *reinterpret_cast<words*>(q) = v;
    }
};
template <int V>
__device__ __forceinline__ uint32_t top_bits(uint32_t top, const float (&f)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) {
        const uint32_t b = __float_as_uint(f[e]) & 0x7fffffffu;
        top = b > top ? b : top;
    }
    return top;
}

__device__ __forceinline__ uint32_t umax(uint32_t a, uint32_t b) { return a > b ? a : b; }
// The largest of G neighbouring lanes (16, 32 or 64), in each of them: within
// rows of 16 lanes by DPP, across them by the lane swaps; no LDS round trips.
template <int G>
__device__ __forceinline__ uint32_t lanes_max(uint32_t v) {
    v = umax(v, (uint32_t)dpp_int<0x128>((int)v));  // row_ror:8, 4, 2, 1
    v = umax(v, (uint32_t)dpp_int<0x124>((int)v));
    v = umax(v, (uint32_t)dpp_int<0x122>((int)v));
    v = umax(v, (uint32_t)dpp_int<0x121>((int)v));
    if constexpr (G >= 32) {
        const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
        v = umax(r[0], r[1]);
    }
    if constexpr (G >= 64) {
        const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
        v = umax(r[0], r[1]);
    }
    return v;
}

// The V values of a row from j < cols on, zeros behind its end: one whole load that
// ends with the row at most, moved down by what lies before j.  cols >= V.  (Element
// by element, 20000 rows of 4095 bf16 took 71 us to quantise, so 44; of 4096 alike.)
template <typename T, int V>
__device__ __forceinline__ void load_to_end(const T* __restrict__ row, int j, int cols, float (&f)[V]) {
    static_assert(V * sizeof(T) == 16, "two 64-bit halves");
    union {
        Raw<T, V> raw;
        uint64_t half[2];
    } u;
    const int at = min(j, cols - V);
    u.raw = load_raw<T, V>(row + at);
    if (const int bits = (j - at) * 8 * (int)sizeof(T)) {  // j - at < V: fewer than 128
        if (bits < 64) {
            u.half[0] = u.half[0] >> bits | u.half[1] << (64 - bits);
            u.half[1] >>= bits;
        } else {
            u.half[0] = u.half[1] >> (bits - 64);
            u.half[1] = 0;
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = elem<T, V>(u.raw, e);
}

// Bound by memory where rows are long (20000 x 4096 bf16: 43 to 50 us by the clock,
// 5.7 to 4.9 TB/s), by the waves' latency where they are short (20000 x 128: 4.6 us).
// G lanes per row (a power of two up to the block), R vectors of V values a lane
// held in registers between the two uses of a row; a row longer than G R V is
// read again.  The largest |x| is found on the bits, so that an infinity or a
// NaN is the largest.
template <typename T, int V, int G, int R>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int64_t rows,
                                                            int cols, signed char* __restrict__ q, int64_t ldq,
                                                            float* __restrict__ scale) {
    __shared__ uint32_t red[4];
    const int64_t row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
    const bool live = row < rows;
    const int t = threadIdx.x % G;
    const T* xr = x + (live ? row : 0) * ldx;
    uint32_t top = 0;
    float v[R][V];
    if (cols >= V) {
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int j = (t + i * G) * V;
            if (j < cols) {
                load_to_end<T, V>(xr, j, cols, v[i]);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) v[i][e] = 0.f;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < R; ++i) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int j = (t + i * G) * V + e;
                v[i][e] = j < cols ? (float)xr[j] : 0.f;
            }
        }
    }
#pragma unroll
    for (int i = 0; i < R; ++i) top = top_bits<V>(top, v[i]);
    for (int64_t j = (int64_t)(t + R * G) * V; j < cols; j += G * V) {
        float f[V];
        load_to_end<T, V>(xr, (int)j, cols, f);
        top = top_bits<V>(top, f);
    }
    top = lanes_max<(G < 64 ? G : 64)>(top);
    if constexpr (G > 64) {
        if (wave_lane() == 0) red[wave_id()] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) top = umax(top, red[i]);
    }
    if (!live) return;
    const RowScale k(top);
    if (t == 0) scale[row] = k.s;
    signed char* qr = q + row * ldq;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int j = (t + i * G) * V;
        if (j < ldq) k.put<V>(qr + j, v[i]);  // ldq is a multiple of 16, V divides it
    }
    for (int64_t j = (int64_t)(t + R * G) * V; j < ldq; j += G * V) {
        float f[V];
        if (j < cols) {
            load_to_end<T, V>(xr, (int)j, cols, f);
        } else {  // padding: the row may be shorter than a vector, or empty
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = 0.f;
        }
        k.put<V>(qr + j, f);
    }
}

// The 16 bytes of a row from k on; nothing of what lies at or past kend.
__device__ __forceinline__ v4i load_k(const signed char* __restrict__ row, int k, int kend) {
    v4i v = {0, 0, 0, 0};
    if (k < kend) v = *reinterpret_cast<const v4i*>(row + k);
    return v;
}
__device__ __forceinline__ v4i mask_k(v4i v, int k, int kend) {
    const int left = kend - k;  // bytes that count
    if (left >= 16) return v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = left - 4 * i;
        v[i] &= b >= 4 ? -1 : b <= 0 ? 0 : (int)((1u << (8 * b)) - 1u);
    }
    return v;
}

struct Int8Args {
    const signed char* xq;
    const signed char* wq;
    const float* xs;
    const float* ws;
    const void* bias;
    int64_t ldx, ldw, ldy, m;
    int n, k, ptype;
};

template <typename T>
__device__ __forceinline__ void put_y(const Int8Args& a, T* __restrict__ y, int64_t i, int j, int acc) {
    const float b = a.bias ? load_param(a.bias, a.ptype, j) : 0.f;
    y[i * a.ldy + j] = (T)((float)acc * a.xs[i] * a.ws[j] + b);
}

// A 16 MF x 16 NF tile of y per block; its W waves take W slices of k, four steps of
// 64 bytes in flight, and meet in LDS.  For few rows, where the weights' bytes
// are the bound: 1 x 4096 x 4096 4.5 us (3.7 TB/s), 64 rows 8.4 us.
template <typename T, int MF, int NF, int W>
__global__ __launch_bounds__(64 * W) void int8_split_kernel(Int8Args a, T* __restrict__ y) {
    constexpr int kAhead = 4;
    __shared__ int red[W][MF * NF * 256];
    const int nt = (a.n + 16 * NF - 1) / (16 * NF);
    const int64_t bm = blockIdx.x / nt;
    const int bn = (int)(blockIdx.x - bm * nt);
    const int lane = wave_lane(), w = wave_id();
    const int r = lane & 15, kc = (lane >> 4) * 16;
    const signed char* xr[MF];
    const signed char* wr[NF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
        const int64_t row = bm * (16 * MF) + 16 * i + r;
        xr[i] = a.xq + (row < a.m ? row : a.m - 1) * a.ldx + kc;
    }
#pragma unroll
    for (int j = 0; j < NF; ++j) {
        const int row = bn * (16 * NF) + 16 * j + r;
        wr[j] = a.wq + (int64_t)(row < a.n ? row : a.n - 1) * a.ldw + kc;
    }
    v4i acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    auto mul = [&](const v4i (&xf)[MF], const v4i (&wf)[NF]) {
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[i], wf[j], acc[i][j], 0, 0, 0);
    };
    const int steps = (a.k + 63) / 64, per = (steps + W - 1) / W;
    const int last = (w + 1) * per < steps ? (w + 1) * per : steps;
    const int full = a.k / 64 < last ? a.k / 64 : last;  // steps before this hold 64 bytes of k
    int t = w * per;
    for (; t + kAhead <= full; t += kAhead) {
        v4i xf[kAhead][MF], wf[kAhead][NF];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
#pragma unroll
            for (int j = 0; j < NF; ++j) wf[u][j] = *reinterpret_cast<const v4i*>(wr[j] + (t + u) * 64);
#pragma unroll
            for (int i = 0; i < MF; ++i) xf[u][i] = *reinterpret_cast<const v4i*>(xr[i] + (t + u) * 64);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) mul(xf[u], wf[u]);
    }
    if (t < last) {
        v4i xf[kAhead][MF], wf[kAhead][NF];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k0 = (t + u) * 64, end = t + u < last ? a.k - kc : 0;
#pragma unroll
            for (int j = 0; j < NF; ++j) wf[u][j] = load_k(wr[j], k0, end);
#pragma unroll
            for (int i = 0; i < MF; ++i) xf[u][i] = mask_k(load_k(xr[i], k0, end), k0, end);
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) mul(xf[u], wf[u]);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
            *reinterpret_cast<v4i*>(&red[w][((i * NF + j) * 64 + lane) * 4]) = acc[i][j];
    __syncthreads();
    for (int e = threadIdx.x; e < MF * NF * 256; e += 64 * W) {
        int sum = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) sum += red[i][e];
        const int f = e >> 8, l = (e >> 2) & 63;
        const int64_t row = bm * (16 * MF) + 16 * (f / NF) + (l >> 4) * 4 + (e & 3);
        const int col = bn * (16 * NF) + 16 * (f % NF) + (l & 15);
        if (row < a.m && col < a.n) put_y<T>(a, y, row, col, sum);
    }
}

// One or two rows (single nodes): every block quantises the rows into LDS by
// itself, under the loads of its first weights, and multiplies them with 16
// rows of w, k split over its eight waves.  One launch: 1 x 4096 x 4096 from
// bf16 5.8 us, against 7.9 for quantiser and product.  With a slower rounding
// two rows took 8.1 / 8.4 us and four 10.9 / 8.5, so it ends at two.
constexpr int kFewRows = 2, kFewBytes = 32768;
template <typename TX, int V>
__global__ __launch_bounds__(512) void int8_few_kernel(const TX* __restrict__ x, int64_t ldx, Int8Args a, int ldq,
                                                       void* __restrict__ y, int ycode) {
    constexpr int W = 8, kAhead = 4;
    __shared__ __attribute__((aligned(16))) signed char xq[kFewBytes];
    __shared__ int red[W][256];
    __shared__ uint32_t tops[W][kFewRows];
    __shared__ float scales[kFewRows];
    const int lane = wave_lane(), w = wave_id(), t = threadIdx.x, m = (int)a.m;
    const int r = lane & 15, kc = (lane >> 4) * 16, bn = blockIdx.x;
    const int wrow = bn * 16 + r;
    const signed char* wr = a.wq + (int64_t)(wrow < a.n ? wrow : a.n - 1) * a.ldw + kc;
    const int steps = (a.k + 63) / 64, per = (steps + W - 1) / W;
    const int first = w * per, last = (w + 1) * per < steps ? (w + 1) * per : steps;
    v4i wf[kAhead];
    auto fetch = [&](int at) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) wf[u] = load_k(wr, (at + u) * 64, at + u < last ? a.k - kc : 0);
    };
    fetch(first);
    float f[kFewRows][V];
    uint32_t top[kFewRows];
#pragma unroll
    for (int i = 0; i < kFewRows; ++i) {
        top[i] = 0;
#pragma unroll
        for (int e = 0; e < V; ++e) f[i][e] = 0.f;
        if (i < m && t * V < a.k) load_part<TX, V>(x + i * ldx + t * V, a.k - t * V, f[i]);
    }
#pragma unroll
    for (int i = 0; i < kFewRows; ++i) {
        top[i] = top_bits<V>(0u, f[i]);
        if (i < m)
            for (int j = (t + 512) * V; j < a.k; j += 512 * V) {
                float g[V];
                load_part<TX, V>(x + i * ldx + j, a.k - j, g);
                top[i] = top_bits<V>(top[i], g);
            }
        top[i] = lanes_max<64>(top[i]);
        if (lane == 0) tops[w][i] = top[i];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kFewRows; ++i) {
        if (i >= m) break;
        uint32_t b = 0;
#pragma unroll
        for (int u = 0; u < W; ++u) b = umax(b, tops[u][i]);
        const RowScale k(b);
        if (t == 0) scales[i] = k.s;
        signed char* qr = xq + i * ldq;
        if (t * V < ldq) k.put<V>(qr + t * V, f[i]);
        for (int j = (t + 512) * V; j < ldq; j += 512 * V) {
            float g[V];
#pragma unroll
            for (int e = 0; e < V; ++e) g[e] = 0.f;
            if (j < a.k) load_part<TX, V>(x + i * ldx + j, a.k - j, g);
            k.put<V>(qr + j, g);
        }
    }
    __syncthreads();
    v4i acc = {0, 0, 0, 0};
    for (int s = first; s < last; s += kAhead) {
        if (s > first) fetch(s);
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int k = (s + u) * 64 + kc;  // xq is 0 from k = a.k to ldq
            v4i xf = {0, 0, 0, 0};
            if (r < m && s + u < last && k < ldq) xf = *reinterpret_cast<const v4i*>(xq + r * ldq + k);
            acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf, wf[u], acc, 0, 0, 0);
        }
    }
    *reinterpret_cast<v4i*>(&red[w][lane * 4]) = acc;
    __syncthreads();
    const int row = (t >> 6) * 4 + (t & 3), col = bn * 16 + ((t >> 2) & 15);
    if (t < 256 && row < m && col < a.n) {
        int sum = 0;
#pragma unroll
        for (int u = 0; u < W; ++u) sum += red[u][t];
        const float b = a.bias ? load_param(a.bias, a.ptype, col) : 0.f;
        const float o = (float)sum * scales[row] * a.ws[col] + b;
        const int64_t at = row * a.ldy + col;
        if (ycode == LDS_F32)
            reinterpret_cast<float*>(y)[at] = o;
        else if (ycode == LDS_BF16)
            reinterpret_cast<bf16_t*>(y)[at] = (bf16_t)o;
        else
            reinterpret_cast<f16_t*>(y)[at] = (f16_t)o;
    }
}

typedef int v16i __attribute__((ext_vector_type(16)));

__device__ const v4i kZeroChunk = {0, 0, 0, 0};

// A BM x BN tile of y per block of WM x WN waves, k in steps of 64 bytes through a
// ring of four LDS stages filled by direct loads three steps ahead.  The
// matrix instruction is 32 x 32 x 32 with w as its first operand, so that a lane
// ends with four neighbouring columns of one row of y.
//
// A stage holds the tile's rows of 64 bytes as four 16-byte chunks; chunk c of
// row r sits at place c ^ (r / 4 % 4), so that the 16 lanes of a read phase, one
// chunk of 16 rows, meet 16 different 16-byte bank groups (no conflict counted).
//
// 8192^3: 520 us, 2115 TOP/s (the library's int8 product of that size: 544 us);
// 20000 x 4096 x 4096: 331 us, 2030 TOP/s.  Bound by power: with zeros
// in x and w the latter takes 240 us, at random values the clock is 1.8 GHz and
// the matrix units are busy 54 % of its cycles.
template <typename T, int BM, int BN, int WM, int WN, int kStages>
__global__ __launch_bounds__(64 * WM * WN) void int8_tile_kernel(Int8Args a, T* __restrict__ y) {
    constexpr int kWaves = WM * WN;
    constexpr int kStageBytes = (BM + BN) * 64;
    constexpr int kLoads = kStageBytes / 1024 / kWaves;  // direct loads per wave and stage
    constexpr int FM = BM / WM / 32, FN = BN / WN / 32;
    static_assert(kStageBytes % (1024 * kWaves) == 0 && BM % 16 == 0, "whole loads per wave");
    constexpr int kFlight = (kStages - 2) * kLoads;  // this wave's loads that may stay in flight
    static_assert(kFlight <= 63, "the load count fits the wait");
    __shared__ __attribute__((aligned(1024))) signed char smem[kStages * kStageBytes];
    const int lane = wave_lane(), w = wave_id();
    const int tm = (int)((a.m + BM - 1) / BM), tn = (a.n + BN - 1) / BN;
    // Blocks go round the eight XCDs: each takes a run of neighbouring tiles,
    // four tile rows at a time, whose operands stay in its L2.
    const int total = tm * tn, per = (total + 7) / 8;
    const int id = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (id >= total) return;
    const int band = id / (4 * tn), in_band = id - band * 4 * tn;
    const int rows_in = tm - band * 4 < 4 ? tm - band * 4 : 4;
    const int bm = band * 4 + in_band % rows_in, bn = in_band / rows_in;
    const int64_t m0 = (int64_t)bm * BM;
    const int n0 = bn * BN;

    // this lane's source of every direct load: one chunk of one row
    const signed char* src[kLoads];
    int chunk[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int u = (w * kLoads + i) * 64 + lane;  // 16-byte place in the stage
        const int r = u >> 2;
        chunk[i] = ((u & 3) ^ ((r >> 2) & 3)) * 16;
        if (r < BM) {
            const int64_t row = m0 + r;
            src[i] = a.xq + (row < a.m ? row : a.m - 1) * a.ldx + chunk[i];
        } else {
            const int row = n0 + r - BM;
            src[i] = a.wq + (int64_t)(row < a.n ? row : a.n - 1) * a.ldw + chunk[i];
        }
    }
    const int steps = (a.k + 63) / 64;
    const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) signed char*)smem;
    auto issue = [&](int t, bool tail) {
        const uint32_t to = base + (t % kStages) * kStageBytes + w * kLoads * 1024;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const signed char* p = src[i] + t * 64;
            if (tail && t * 64 + chunk[i] >= a.k) p = reinterpret_cast<const signed char*>(&kZeroChunk);
            lds_dma16(p, to + i * 1024);
        }
    };
    v16i acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0;
    const int wm = w % WM, wn = w / WM;
    const int r32 = lane & 31, half = lane >> 5;
    const int sw = (r32 >> 2) & 3;  // rows 32 apart share it
    const signed char* xs_at = smem + (wm * (BM / WM) + r32) * 64;
    const signed char* ws_at = smem + (BM + wn * (BN / WN) + r32) * 64;
    // the operands of half a step: 32 bytes of k
    auto fetch = [&](int t, int ks, v4i (&xf)[FM], v4i (&wf)[FN]) {
        const int at = (t % kStages) * kStageBytes + (((ks * 2 + half) ^ sw) * 16);
#pragma unroll
        for (int j = 0; j < FN; ++j) wf[j] = *reinterpret_cast<const v4i*>(ws_at + at + j * 2048);
#pragma unroll
        for (int i = 0; i < FM; ++i) xf[i] = *reinterpret_cast<const v4i*>(xs_at + at + i * 2048);
    };
    auto mask = [&](int t, int ks, v4i (&xf)[FM]) {
#pragma unroll
        for (int i = 0; i < FM; ++i) xf[i] = mask_k(xf[i], t * 64 + (ks * 2 + half) * 16, a.k);
    };
    auto mul = [&](const v4i (&xf)[FM], const v4i (&wf)[FN]) {
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
    };
    // every wave's loads of a step have landed and its reads of the stage that
    // is refilled next are done
    auto meet = [&](int in_flight) {
        asm volatile("" ::: "memory");
        wait_vmcnt(in_flight);
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    v4i x0[FM], w0[FN], x1[FM], w1[FN];
    for (int t = 0; t < kStages - 1 && t < steps; ++t) issue(t, t == steps - 1);
    {
        const int later = steps - 1 < kStages - 2 ? steps - 1 : kStages - 2;
        meet(later * kLoads);
    }
    if (kStages - 1 < steps) issue(kStages - 1, kStages == steps);
    fetch(0, 0, x0, w0);
    // Both halves of a step: the products of one half run while the operands of
    // the next are read; the next step's arrival is awaited in between.
    int t = 0;
    for (; t + kStages < steps - 1; ++t) {
        fetch(t, 1, x1, w1);
        __builtin_amdgcn_sched_barrier(0);
        mul(x0, w0);
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt(0x0F70 | (kFlight & 15) | (kFlight >> 4 << 14));  // vmcnt(kFlight)
        __builtin_amdgcn_s_waitcnt(0xC07F);
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        issue(t + kStages, false);
        fetch(t + 1, 0, x0, w0);
        __builtin_amdgcn_sched_barrier(0);
        mul(x1, w1);
        __builtin_amdgcn_sched_barrier(0);
    }
    for (; t < steps; ++t) {  // the last kStages + 1 steps: fewer in flight, the end of k masked
        const bool tail = t == steps - 1;
        fetch(t, 1, x1, w1);
        if (tail) mask(t, 0, x0);
        mul(x0, w0);
        if (!tail) {
            const int later = steps - 2 - t < kStages - 2 ? steps - 2 - t : kStages - 2;
            meet(later * kLoads);
            if (t + kStages < steps) issue(t + kStages, t + kStages == steps - 1);
            fetch(t + 1, 0, x0, w0);
        } else {
            mask(t, 1, x1);
        }
        mul(x1, w1);
    }
    // Out through LDS, 32 rows of the wave's 64 columns at a time, so that a store
    // writes whole lines: a lane leaves four columns of row r32 and takes VO
    // neighbouring ones.  Unit u of row r (16 bytes) sits at place u ^ (r % 16).
    static_assert(FN == 2 && kStages * kStageBytes >= kWaves * 8192, "an 8 KB region per wave");
    constexpr int VO = 16 / (int)sizeof(T), kRowLanes = 64 / VO, kRows = 64 / kRowLanes;
    signed char* region = smem + w * 8192;
    const int oc = lane % kRowLanes, orow = lane / kRowLanes;
    const int col = n0 + wn * 64 + oc * VO;
    float s[VO], b[VO];
#pragma unroll
    for (int e = 0; e < VO; ++e) {
        const int cc = col + e < a.n ? col + e : a.n - 1;
        s[e] = a.ws[cc];
        b[e] = 0.f;
    }
    if (a.bias) {
#pragma unroll
        for (int e = 0; e < VO; ++e) b[e] = load_param(a.bias, a.ptype, col + e < a.n ? col + e : a.n - 1);
    }
    // the row scales of all the lane's rows at once: one wait, not one a row
    float xs[FM * 32 / kRows];
#pragma unroll
    for (int i = 0; i < FM * 32 / kRows; ++i) {
        const int64_t row = m0 + wm * (BM / WM) + i * kRows + orow;
        xs[i] = a.xs[row < a.m ? row : a.m - 1];
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0xC07F);
    __builtin_amdgcn_s_barrier();  // every wave has read its last operands
    asm volatile("" ::: "memory");
#pragma unroll
    for (int i = 0; i < FM; ++i) {
#pragma unroll
        for (int j = 0; j < FN; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int u = 8 * j + 2 * g + half;
                *reinterpret_cast<v4i*>(region + r32 * 256 + (u ^ (r32 & 15)) * 16) =
                    v4i{acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
            }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();  // a wave's LDS operations are done in order
#pragma unroll
        for (int q = 0; q < 32 / kRows; ++q) {
            const int r = q * kRows + orow;
            const int64_t row = m0 + wm * (BM / WM) + 32 * i + r;
            if (row < a.m && col < a.n) {
                float o[VO];
#pragma unroll
                for (int h = 0; h < VO / 4; ++h) {
                    const v4i v = *reinterpret_cast<const v4i*>(region + r * 256 +
                                                                ((oc * (VO / 4) + h) ^ (r & 15)) * 16);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[4 * h + e] = (float)v[e] * xs[i * (32 / kRows) + q] * s[4 * h + e] + b[4 * h + e];
                }
                store_part<T, VO>(y + row * a.ldy + col, a.n - col, o);
            }
        }
        asm volatile("" ::: "memory");
        __builtin_amdgcn_wave_barrier();
    }
}

}  // namespace lds

using namespace lds;

namespace {

template <typename T, int MF, int NF, int W>
int launch_split(const Int8Args& a, T* y, hipStream_t st) {
    const int64_t blocks = ((a.m + 16 * MF - 1) / (16 * MF)) * ((a.n + 16 * NF - 1) / (16 * NF));
    LDS_CHECK_ARG(grid_fits(blocks, 64 * W));
    hipLaunchKernelGGL((int8_split_kernel<T, MF, NF, W>), dim3((unsigned)blocks), dim3(64 * W), 0, st, a, y);
    LDS_RETURN_LAST_ERROR();
}

template <typename T, int BM, int BN, int WM, int WN, int S>
int launch_tile(const Int8Args& a, T* y, hipStream_t st) {
    const int64_t tiles = ((a.m + BM - 1) / BM) * ((a.n + BN - 1) / BN);
    LDS_CHECK_ARG(tiles < (int64_t)1 << 30 && grid_fits(tiles + 7, 64 * WM * WN));
    const unsigned blocks = (unsigned)((tiles + 7) / 8 * 8);  // whole rounds of the eight XCDs
    hipLaunchKernelGGL((int8_tile_kernel<T, BM, BN, WM, WN, S>), dim3(blocks), dim3(64 * WM * WN), 0, st, a, y);
    LDS_RETURN_LAST_ERROR();
}

}  // namespace

extern "C" int lds_quantize_rows(const void* x, int64_t ldx, int64_t rows, int cols, int dtype, signed char* q,
                                 int64_t ldq, float* scale, void* stream) {
    LDS_CHECK_ARG(rows >= 0 && rows <= (int64_t)0x7fffffff && cols >= 0 && dtype >= LDS_F32 && dtype <= LDS_F16);
    LDS_CHECK_ARG(ldq % 16 == 0 && ldq >= cols && ldq <= (int64_t)0x7ffff000 && ldx >= cols);
    if (rows == 0) return 0;
    LDS_CHECK_ARG(scale && (cols == 0 || x) && (ldq == 0 || q) && ((uintptr_t)q & 15) == 0);
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        constexpr int V = 16 / (int)sizeof(T);
        auto go = [&](auto lanes, auto regs) {
            constexpr int G = decltype(lanes)::value, R = decltype(regs)::value, kRows = 256 / G;
            in_launches((rows + kRows - 1) / kRows, 256, [&](int64_t first, unsigned blocks) {
                const int64_t r = first * kRows;
                hipLaunchKernelGGL((quantize_rows_kernel<T, V, G, R>), dim3(blocks), dim3(256), 0, (hipStream_t)stream,
                                   (const T*)x + r * ldx, ldx, rows - r, cols, q + r * ldq, ldq, scale + r);
            });
        };
        // a row in the registers of 16 or 32 lanes, of a wave or of a block
        if (ldq <= 16 * V)
            go(IntC<16>{}, IntC<1>{});
        else if (ldq <= 32 * V)
            go(IntC<32>{}, IntC<1>{});
        else if (ldq <= 64 * V)
            go(IntC<64>{}, IntC<1>{});
        else if (ldq <= 64 * V * 4)
            go(IntC<64>{}, IntC<4>{});
        else
            go(IntC<256>{}, IntC<4>{});
        LDS_RETURN_LAST_ERROR();
    });
}

extern "C" int lds_int8_matmul(const signed char* xq, int64_t ldx, const float* xs, const signed char* wq,
                               int64_t ldw, const float* ws, const void* bias, int ptype, int64_t m, int n, int k,
                               void* y, int64_t ldy, int dtype, void* stream) {
    LDS_CHECK_ARG(m >= 0 && m <= (int64_t)0x7fffffff && n >= 0 && k >= 0 && k <= 131071);
    LDS_CHECK_ARG(dtype >= LDS_F32 && dtype <= LDS_F16 && ptype >= LDS_F32 && ptype <= LDS_F16);
    if (m == 0 || n == 0) return 0;
    LDS_CHECK_ARG(xs && ws && y && ldy >= n);
    LDS_CHECK_ARG(k == 0 || (xq && wq && ldx >= k && ldw >= k && ldx % 16 == 0 && ldw % 16 == 0 &&
                             (((uintptr_t)xq | (uintptr_t)wq) & 15) == 0));
    const Int8Args a{xq, wq, xs, ws, bias, ldx, ldw, ldy, m, n, k, ptype};
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        const hipStream_t st = (hipStream_t)stream;
        // The largest tile that gives three quarters of the 256 CUs one each; below
        // that (few rows, or few columns) k is split over a block's waves, with the
        // smallest tile that stays within 384 blocks.
        const auto tiles = [&](int bm, int bn) { return ((m + bm - 1) / bm) * (int64_t)((n + bn - 1) / bn); };
        if (k > 0) {
            if (tiles(256, 256) >= 192) return launch_tile<T, 256, 256, 2, 4, 4>(a, (T*)y, st);
            if (tiles(256, 128) >= 192) return launch_tile<T, 256, 128, 4, 2, 4>(a, (T*)y, st);
            if (tiles(128, 128) >= 192) return launch_tile<T, 128, 128, 2, 2, 4>(a, (T*)y, st);
            if (tiles(128, 64) >= 192) return launch_tile<T, 128, 64, 4, 1, 6>(a, (T*)y, st);
            if (tiles(64, 64) >= 192) return launch_tile<T, 64, 64, 2, 1, 4>(a, (T*)y, st);
        }
        if (tiles(16, 16) <= 384) return launch_split<T, 1, 1, 8>(a, (T*)y, st);
        if (tiles(32, 16) <= 384) return launch_split<T, 2, 1, 8>(a, (T*)y, st);
        if (tiles(32, 32) <= 384) return launch_split<T, 2, 2, 8>(a, (T*)y, st);
        return launch_split<T, 4, 2, 8>(a, (T*)y, st);
    });
}

extern "C" int lds_int8_linear(const void* x, int64_t ldx, int xdtype, signed char* q, int64_t ldq, float* xs,
                               const signed char* wq, int64_t ldw, const float* ws, const void* bias, int ptype,
                               int64_t m, int n, int k, void* y, int64_t ldy, int dtype, void* stream) {
    // the product's checks come first: nothing is launched by a refused call
    LDS_CHECK_ARG(m >= 0 && m <= (int64_t)0x7fffffff && n >= 0 && k >= 0 && k <= 131071);
    LDS_CHECK_ARG(dtype >= LDS_F32 && dtype <= LDS_F16 && ptype >= LDS_F32 && ptype <= LDS_F16);
    if (m == 0 || n == 0) return 0;
    LDS_CHECK_ARG(xs && ws && y && ldy >= n);
    LDS_CHECK_ARG(k == 0 || (q && wq && ldq >= k && ldw >= k && ldq % 16 == 0 && ldw % 16 == 0 &&
                             (((uintptr_t)q | (uintptr_t)wq) & 15) == 0));
    if (k > 0 && m <= kFewRows && m * ldq <= kFewBytes && grid_fits(((int64_t)n + 15) / 16, 512)) {
        LDS_CHECK_ARG(x && ldx >= k && xdtype >= LDS_F32 && xdtype <= LDS_F16);
        return with_type(xdtype, [&](auto zero) -> int {
            using TX = decltype(zero);
            constexpr int V = 16 / (int)sizeof(TX);
            const Int8Args a{nullptr, wq, nullptr, ws, bias, 0, ldw, ldy, m, n, k, ptype};
            hipLaunchKernelGGL((int8_few_kernel<TX, V>), dim3((unsigned)(((int64_t)n + 15) / 16)), dim3(512), 0,
                               (hipStream_t)stream, (const TX*)x, ldx, a, (int)ldq, y, dtype);
            LDS_RETURN_LAST_ERROR();
        });
    }
    const int e = lds_quantize_rows(x, ldx, m, k, xdtype, q, ldq, xs, stream);
    return e ? e : lds_int8_matmul(q, ldq, xs, wq, ldw, ws, bias, ptype, m, n, k, y, ldy, dtype, stream);
}
