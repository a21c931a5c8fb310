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
// start anywhere (the vectors carry the element's alignment).  A row's last
// vector ends with the row, so that every load is whole; what it has in common
// with the one before is the same value in both, and both store it (`whole`),
// unless y overlaps an input: then each stores its own elements only.
// PAST: the inputs are read past the caches (launch_dropout says when).
// No lane branches before its loads, so all of them are in flight at once; with
// the last vector element by element instead, 40000 x 512 of fp16 took 28 us and
// x 511 74, now 22 and 22.  Bound by memory: 160000 x 512 bf16 with a residual
// 75 us (6.6 TB/s), 20000 x 257 fp16 8.2, 2708 x 1433 fp32 6.3.
template <typename T, int V, bool RES, bool DROP, bool PAST>
__global__ __launch_bounds__(256) void dropout_add_kernel(const T* x, int64_t ldx, const T* res, int64_t ldr,
                                                          T* y, int64_t ldy, int64_t rows, int cols, int cvecs,
                                                          int64_t total, int whole, DropKey key) {
    const int64_t t = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (t >= total) return;
    int64_t rq;
    if (total <= 0xffffffffll) {
        rq = (uint32_t)t / (uint32_t)cvecs;
    } else {
        rq = t / cvecs;
    }
    const int j0 = (int)(t - rq * cvecs) * V, j = min(j0, cols - V);
    const int64_t i0 = rq * 4;
    Raw<T, V> v[4], a[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t i = min(i0 + r, rows - 1);  // rows behind the last repeat it
        v[r] = load_raw<T, V, PAST>(x + i * ldx + j);
        if constexpr (RES) a[r] = load_raw<T, V, PAST>(res + i * ldr + j);
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
        float o[V];
#pragma unroll
        for (int e = 0; e < V; ++e) {
            o[e] = elem<T, V>(v[r], e) * key.scale;
            if constexpr (DROP) o[e] = kept[r][e] ? o[e] : 0.f;
            if constexpr (RES) o[e] = o[e] + elem<T, V>(a[r], e);
        }
        T* to = y + (i0 + r) * ldy + j;
        if (whole || j == j0) {
            store_vec<T, V>(to, o);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (j + e >= j0) to[e] = (T)o[e];
        }
    }
}

template <typename T, int V>
int launch_dropout(const T* x, int64_t ldx, const T* residual, int64_t ldr, T* y, int64_t ldy, int64_t rows, int cols,
                   bool drop, const DropKey& key, hipStream_t stream) {
    const int cvecs = (cols - 1) / V + 1;
    const int64_t total = (rows + 3) / 4 * cvecs;
    const int64_t blocks = (total + 255) / 256;
    LDS_CHECK_ARG(grid_fits(blocks, 256));
    const auto span = [&](const T* p, int64_t ld) { return ByteSpan(p, (rows - 1) * ld + cols, sizeof(T)); };
    const ByteSpan to = span(y, ldy);
    const bool whole = !to.meets(span(x, ldx)) && !(residual && to.meets(span(residual, ldr)));
    // Operands that fill the memory-side cache leave it to the result, which the
    // next call reads.  Past it and through it, in us, alone / with a multiplication
    // of the result after it: 160000 x 512 bf16 75 / 121 and 88 / 129, 130000 x 512
    // fp32 118 / 190 and 141 / 239, 200000 x 256 bf16 (307 MB) 50 / 79 and 50 / 77;
    // below the cache's size the inputs may lie in it (160000 x 256, 246 MB, read
    // past it: +1 %).
    const int64_t bytes = rows * cols * (int64_t)sizeof(T);
    const bool past = (residual ? 3 : 2) * bytes > kMemorySideCache;
    const auto go = [&](auto res, auto dr, auto ps) {
        hipLaunchKernelGGL((dropout_add_kernel<T, V, decltype(res)::value, decltype(dr)::value, decltype(ps)::value>),
                           dim3((unsigned)blocks), dim3(256), 0, stream, x, ldx, residual, ldr, y, ldy, rows, cols,
                           cvecs, total, (int)whole, key);
    };
    const auto with = [](bool b, auto&& f) { b ? f(BoolC<true>{}) : f(BoolC<false>{}); };
    with(residual != nullptr, [&](auto res) {
        with(drop, [&](auto dr) { with(past, [&](auto ps) { go(res, dr, ps); }); });
    });
    LDS_RETURN_LAST_ERROR();
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
        const auto* xs = (const T*)x;
        const auto* rs = (const T*)residual;
        if (cols < V)  // rows shorter than a vector: single columns
            return launch_dropout<T, 1>(xs, ldx, rs, ldr, (T*)y, ldy, rows, cols, drop, key, (hipStream_t)stream);
        return launch_dropout<T, V>(xs, ldx, rs, ldr, (T*)y, ldy, rows, cols, drop, key, (hipStream_t)stream);
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
