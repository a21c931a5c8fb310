// Keyed dropout and library-level entry points (ABI version, error text).
//
// lds_dropout replaces F.dropout (src/models/gcn.py:27,29).  The mask of
// element (i, j) is a pure function of (seed, tag, counter, i, j) through the
// Philox map of common.hpp, so the backward (and the CPU oracle) regenerate it
// instead of storing it.
#include "common.hpp"
#include "vec.hpp"
#include "../../include/ldsgnn.h"

namespace lds {

// y = residual + mask(x), one thread per row quad and 16 bytes of a row: the
// quad shares its Philox calls, the four rows' loads are independent.  Rows
// start anywhere (the vectors carry the element's alignment); only a row's last
// partial vector goes element by element.  Bound by memory: 160000 x 512 bf16 with
// a residual 98 us (5.0 TB/s, the rate of a large copy), 2708 x 1433 fp32 6.4 us.
template <typename T, int V, bool RES, bool DROP>
__global__ __launch_bounds__(256) void dropout_add_kernel(const T* __restrict__ x, int64_t ldx,
                                                          const T* __restrict__ res, int64_t ldr,
                                                          T* __restrict__ y, int64_t ldy, int64_t rows, int cols,
                                                          int cvecs, int64_t total, DropKey key) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= total) return;
    int64_t rq;
    if (total <= 0xffffffffll) {
        rq = (uint32_t)t / (uint32_t)cvecs;
    } else {
        rq = t / cvecs;
    }
    const int j = (int)(t - rq * cvecs) * V;
    const int w = cols - j;
    const int64_t i0 = rq * 4;
    float v[4][V], a[4][V];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (i0 + r < rows) {
            load_part<T, V>(x + (i0 + r) * ldx + j, w, v[r]);
            if constexpr (RES) load_part<T, V>(res + (i0 + r) * ldr + j, w, a[r]);
        }
    }
    bool kept[4][V];
    if constexpr (DROP) {
        ColumnKeep<V> columns;
        columns.init(key, (uint32_t)j);
        columns.quad(key, (uint32_t)rq, kept);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        if (i0 + r >= rows) break;
#pragma unroll
        for (int e = 0; e < V; ++e) {
            float o = v[r][e] * key.scale;
            if constexpr (DROP) o = kept[r][e] ? o : 0.f;
            if constexpr (RES) o = o + a[r][e];
            v[r][e] = o;
        }
        store_part<T, V>(y + (i0 + r) * ldy + j, w, v[r]);
    }
}

}  // namespace lds

using namespace lds;

extern "C" int lds_abi_version(void) { return LDS_ABI_VERSION; }

extern "C" const char* lds_error_string(int err) {
    const char* s = hipGetErrorString((hipError_t)err);
    return s ? s : "unknown hip error";
}

extern "C" int lds_dropout_add(const void* x, int64_t ldx, const void* residual, int64_t ldr, void* y, int64_t ldy,
                               int64_t rows, int cols, int dtype, float keep_prob, float scale, uint64_t seed,
                               uint32_t tag, uint32_t counter, void* stream) {
    LDS_CHECK_ARG(rows >= 0 && cols >= 0 && dtype >= LDS_F32 && dtype <= LDS_F16);
    LDS_CHECK_ARG(rows <= (int64_t)0x7fffffff && keep_prob >= 0.f && keep_prob <= 1.f);
    if (rows == 0 || cols == 0) return 0;
    LDS_CHECK_ARG(x != nullptr && y != nullptr && ldx >= cols && ldy >= cols);
    LDS_CHECK_ARG(residual == nullptr || ldr >= cols);
    return with_type(dtype, [&](auto zero) -> int {
        using T = decltype(zero);
        constexpr int V = 16 / (int)sizeof(T);
        DropKey key;
        const bool drop = drop_key(keep_prob, scale, seed, tag, counter, &key);
        const int cvecs = (cols - 1) / V + 1;
        const int64_t total = (rows + 3) / 4 * cvecs;
        const int64_t blocks = (total + 255) / 256;
        LDS_CHECK_ARG(blocks < (int64_t)1 << 31);
        auto go = [&](auto res, auto dr) {
            hipLaunchKernelGGL((dropout_add_kernel<T, V, decltype(res)::value, decltype(dr)::value>),
                               dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, (const T*)x, ldx,
                               (const T*)residual, ldr, (T*)y, ldy, rows, cols, cvecs, total, key);
        };
        if (residual) {
            drop ? go(BoolC<true>{}, BoolC<true>{}) : go(BoolC<true>{}, BoolC<false>{});
        } else {
            drop ? go(BoolC<false>{}, BoolC<true>{}) : go(BoolC<false>{}, BoolC<false>{});
        }
        LDS_RETURN_LAST_ERROR();
    });
}

extern "C" int lds_dropout(const float* x, int ldx, float* y, int ldy, int rows, int cols,
                           float keep_prob, float scale, uint64_t seed, uint32_t tag,
                           uint32_t counter, void* stream) {
    LDS_CHECK_ARG(x != nullptr && y != nullptr && rows >= 0 && cols >= 0);
    LDS_CHECK_ARG(ldx >= cols && ldy >= cols);
    // u lies in [0, 1): a keep_prob past either end keeps all or none
    keep_prob = keep_prob >= 1.f ? 1.f : keep_prob > 0.f ? keep_prob : 0.f;
    return lds_dropout_add(x, ldx, nullptr, 0, y, ldy, rows, cols, LDS_F32, keep_prob, scale, seed, tag, counter,
                           stream);
}
