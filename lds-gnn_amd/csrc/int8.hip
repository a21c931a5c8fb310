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

// q = x / s to the nearest integer, ties to even, of the exact quotient.  t = x · (1/s)
// is within 127 · 2^-22 of it, so only a t that close to a half is looked at again:
// there the sign of x - (q ± ½) s, one fused operation, decides.
__device__ __forceinline__ float quant_one(float x, float s, float inv) {
    const float t = x * inv;
    float q = rintf(t);
    const float d = t - q;
    if (fabsf(d) > 0.4999f) {
        const float h = q + (d < 0.f ? -0.5f : 0.5f);
        const float r = __builtin_fmaf(-h, s, x);
        q = r > 0.f ? h + 0.5f : r < 0.f ? h - 0.5f : rintf(h);
    }
    return fminf(fmaxf(q, -127.f), 127.f);
}

// One block per row: the largest |x| (as bits, so that an infinity or a NaN is
// the largest), then the row again.
template <typename T, int V>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T* __restrict__ x, int64_t ldx, int cols,
                                                            signed char* __restrict__ q, int64_t ldq,
                                                            float* __restrict__ scale) {
    __shared__ uint32_t red[4];
    const int64_t row = blockIdx.x;
    const T* xr = x + row * ldx;
    uint32_t top = 0;
    for (int j = threadIdx.x * V; j < cols; j += 256 * V) {
        float f[V];
        load_part<T, V>(xr + j, cols - j, f);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const uint32_t b = __float_as_uint(f[e]) & 0x7fffffffu;
            top = b > top ? b : top;
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const uint32_t b = __shfl_xor(top, o);
        top = b > top ? b : top;
    }
    if (wave_lane() == 0) red[wave_id()] = top;
    __syncthreads();
    for (int i = 0; i < 4; ++i) top = red[i] > top ? red[i] : top;
    const bool finite = top < 0x7f800000u;
    const float s = finite ? __uint_as_float(top) / 127.f : __uint_as_float(0x7fc00000u);
    const bool zero = !finite || s == 0.f;
    // the quotient is unchanged when both sides grow by 2^64: 1/s stays finite for
    // the smallest scales
    const float up = s < 1e-30f ? 18446744073709551616.f : 1.f;
    const float su = s * up;
    const float inv = zero ? 0.f : 1.f / su;
    if (threadIdx.x == 0) scale[row] = s;
    signed char* qr = q + row * ldq;
    for (int j = threadIdx.x * V; j < ldq; j += 256 * V) {
        float f[V];
        if (j < cols) {
            load_part<T, V>(xr + j, cols - j, f);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = 0.f;
        }
        typedef signed char cv __attribute__((ext_vector_type(V)));
        cv o;
#pragma unroll
        for (int e = 0; e < V; ++e) o[e] = zero ? (signed char)0 : (signed char)(int)quant_one(f[e] * up, su, inv);
        *reinterpret_cast<cv*>(qr + j) = o;  // ldq is a multiple of 16, V divides it
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

// A 16 MF x 16 NF tile of y per block; its four waves split k in 64-byte steps and
// meet in LDS.
template <typename T, int MF, int NF>
__global__ __launch_bounds__(256) void int8_split_kernel(Int8Args a, T* __restrict__ y) {
    __shared__ int red[4][MF * NF * 256];
    const int nt = (a.n + 16 * NF - 1) / (16 * NF);
    const int64_t bm = blockIdx.x / nt;
    const int bn = (int)(blockIdx.x - bm * nt);
    const int lane = wave_lane(), w = wave_id();
    const int r = lane & 15, kc = (lane >> 4) * 16;
    const signed char* xr[MF];
    const signed char* wr[NF];
#pragma unroll
    for (int i = 0; i < MF; ++i) {
        int64_t row = bm * (16 * MF) + 16 * i + r;
        xr[i] = a.xq + (row < a.m ? row : a.m - 1) * a.ldx;
    }
#pragma unroll
    for (int j = 0; j < NF; ++j) {
        int row = bn * (16 * NF) + 16 * j + r;
        wr[j] = a.wq + (int64_t)(row < a.n ? row : a.n - 1) * a.ldw;
    }
    v4i acc[MF][NF];
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j) acc[i][j] = v4i{0, 0, 0, 0};
    for (int k0 = w * 64; k0 < a.k; k0 += 256) {
        const int k = k0 + kc;
        v4i xf[MF], wf[NF];
#pragma unroll
        for (int i = 0; i < MF; ++i) xf[i] = load_k(xr[i], k, a.k);
#pragma unroll
        for (int j = 0; j < NF; ++j) wf[j] = load_k(wr[j], k, a.k);
        if (k0 + 64 > a.k) {
#pragma unroll
            for (int i = 0; i < MF; ++i) xf[i] = mask_k(xf[i], k, a.k);
        }
#pragma unroll
        for (int i = 0; i < MF; ++i)
#pragma unroll
            for (int j = 0; j < NF; ++j)
                acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(xf[i], wf[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < MF; ++i)
#pragma unroll
        for (int j = 0; j < NF; ++j)
            *reinterpret_cast<v4i*>(&red[w][((i * NF + j) * 64 + lane) * 4]) = acc[i][j];
    __syncthreads();
    for (int t = threadIdx.x; t < MF * NF * 256; t += 256) {
        const int f = t >> 8, l = (t >> 2) & 63, e = t & 3;
        const int64_t row = bm * (16 * MF) + 16 * (f / NF) + (l >> 4) * 4 + e;
        const int col = bn * (16 * NF) + 16 * (f % NF) + (l & 15);
        if (row < a.m && col < a.n) put_y<T>(a, y, row, col, (red[0][t] + red[1][t]) + (red[2][t] + red[3][t]));
    }
}

}  // namespace lds

using namespace lds;

extern "C" int lds_quantize_rows(const void* x, int64_t ldx, int64_t rows, int cols, int dtype, signed char* q,
                                 int64_t ldq, float* scale, void* stream) {
    LDS_CHECK_ARG(rows >= 0 && rows <= (int64_t)0x7fffffff && cols >= 0 && dtype >= LDS_F32 && dtype <= LDS_F16);
    LDS_CHECK_ARG(ldq % 16 == 0 && ldq >= cols && ldq <= (int64_t)0x7ffff000 && ldx >= cols);
    if (rows == 0) return 0;
    LDS_CHECK_ARG(scale && (cols == 0 || x) && (ldq == 0 || q) && ((uintptr_t)q & 15) == 0);
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        constexpr int V = 16 / (int)sizeof(T);
        hipLaunchKernelGGL((quantize_rows_kernel<T, V>), dim3((unsigned)rows), dim3(256), 0, (hipStream_t)stream,
                           (const T*)x, ldx, cols, q, ldq, scale);
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
    const int64_t blocks = ((m + 31) / 32) * ((n + 31) / 32);
    LDS_CHECK_ARG(blocks < (int64_t)1 << 31);
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        hipLaunchKernelGGL((int8_split_kernel<T, 2, 2>), dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a,
                           (T*)y);
        LDS_RETURN_LAST_ERROR();
    });
}
