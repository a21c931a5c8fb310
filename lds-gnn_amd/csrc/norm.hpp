// Group norm with an activation, channels last: the pieces that the forward
// (norm_fwd.hip) and the backward (norm_bwd.hip) share.
//
// A thread owns V neighbouring channels, of one group (V divides the channels
// per group) or, in the parts form, across groups, and walks row quads: four
// rows whose flat indices s·n + i differ in their two low bits, the unit in
// which the keyed dropout mask is drawn.
//
// Two forms.  "Slab": a block keeps a sample's rows of a few groups in its
// registers, so that x is read once and one launch does it all.  "Parts": a
// sample's rows are cut into parts, whose sums are written, combined by a
// small launch, and used by a second pass over x.
#pragma once

#include "vec.hpp"

namespace lds {

constexpr int kNormThreads = 256;  // a block of the parts form
// Blocks of a pass of the parts form.  The sums, and the backward's passes (two
// waves a SIMD by their registers): two blocks per CU, each thread long in its
// loop behind one setup; 8 x 20000 x 256 bf16, 512 against 4096 blocks:
// statistics 17.5 / 20.8 us, backward 90 / 107.  The forward's second pass, whose
// waves are light: 36.2 us at 4096 with dropout, 38.6 at 512.
constexpr int kSumBlocks = 512;
constexpr int kApplyBlocks = 4096;
constexpr int kForwardSlabThreads = 1024;
constexpr int kBackwardSlabThreads = 512;  // x and dy: twice the registers a thread

struct NormArgs {
    int64_t samples, n, sx, ldx;
    int c, groups, cg;
    int lanes;        // vectors of a row that a block takes
    int ty;           // row quads that it takes at a time
    int chunks;       // blocks across a row
    int lpg, sub;     // vectors per group (in the chunk); chunks per group
    int span;         // vectors lie across groups (norm_plan says when)
    int whole;        // the result overlaps no input; across groups a row's last vector is stored whole (whole_store)
    int parts;        // row parts per sample
    int64_t part_q;   // row quads per part
    unsigned first;   // blocks of the launches before this one
    const void* weight;
    const void* bias;
    int ptype;
    DropKey key;
};

// What a thread works on.
struct NormPlace {
    int64_t s;            // sample
    int part, chunk;
    int tx, ty;           // vector in the chunk, first row quad of the thread in the part
    int group, c0;        // the thread's group (not across groups) and its first channel
    int skip;             // its first channels that only the vector before it stores (row end, across groups)
    bool live;
    int64_t q0, q1;       // the part's row quads (flat index / 4)
    int64_t f0, f1;       // the sample's flat rows
};

__device__ __forceinline__ NormPlace norm_place(const NormArgs& a, int v, int64_t s, int part, int chunk) {
    NormPlace p;
    p.s = s;
    p.part = part;
    p.chunk = chunk;
    p.ty = (int)((unsigned)threadIdx.x / (unsigned)a.lanes);
    p.tx = (int)threadIdx.x - p.ty * a.lanes;
    p.skip = 0;
    if (a.span) {
        const int at = p.tx * v;
        p.group = 0;
        p.c0 = at < a.c - v ? at : a.c - v;  // a row's last vector ends with the row
        p.skip = a.whole ? 0 : at - p.c0;
        p.live = p.ty < a.ty;
    } else if (a.sub == 1) {
        const int per = a.lanes / a.lpg;
        const int gi = p.tx / a.lpg;
        p.group = chunk * per + gi;
        p.c0 = p.group * a.cg + (p.tx - gi * a.lpg) * v;
        p.live = p.ty < a.ty && p.group < a.groups;
    } else {
        p.group = chunk / a.sub;
        const int at = ((chunk - p.group * a.sub) * a.lanes + p.tx) * v;
        p.c0 = p.group * a.cg + at;
        p.live = p.ty < a.ty && at < a.cg;
    }
    p.f0 = s * a.n;
    p.f1 = p.f0 + a.n;
    p.q0 = (p.f0 >> 2) + (int64_t)part * a.part_q;
    const int64_t qe = ((p.f1 - 1) >> 2) + 1;
    p.q1 = p.q0 + a.part_q < qe ? p.q0 + a.part_q : qe;
    return p;
}

__device__ __forceinline__ NormPlace norm_part_place(const NormArgs& a, int v) {
    const unsigned b = blockIdx.x + a.first, row = b / (unsigned)a.chunks;
    const unsigned s = row / (unsigned)a.parts;
    return norm_place(a, v, s, (int)(row - s * a.parts), (int)(b - row * a.chunks));
}

// A quad's rows that belong to the sample: [lo, hi) of 0..3.
struct QuadRows {
    int lo, hi;
};
__device__ __forceinline__ QuadRows quad_rows(const NormPlace& p, int64_t q) {
    QuadRows r;
    r.lo = p.f0 > 4 * q ? (int)(p.f0 - 4 * q) : 0;
    r.hi = p.f1 < 4 * q + 4 ? (int)(p.f1 - 4 * q) : 4;
    return r;
}

// The four vectors of a quad.  Rows outside the sample read its nearest row, so
// that every load is in bounds without a branch.
template <typename T, int V>
struct Quad {
    Raw<T, V> row[4];

    template <bool PAST = false>
    __device__ __forceinline__ void load(const T* base, int64_t ld, const NormPlace& p, int64_t q,
                                         const QuadRows& in) {
        const T* at = base + (4 * q - p.f0) * ld;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int k = r < in.lo ? in.lo : r >= in.hi ? in.hi - 1 : r;
            row[r] = load_raw<T, V, PAST>(at + k * ld);
        }
    }
};

// f(q, rows) for a thread's quads of a part: whole quads (all but a sample's
// first and last) with the row limits as constants.
template <typename F>
__device__ __forceinline__ void each_quad(const NormArgs& a, const NormPlace& p, F&& f) {
    for (int64_t q = p.q0 + p.ty; q < p.q1; q += a.ty) {
        if (4 * q >= p.f0 && 4 * q + 4 <= p.f1)
            f(q, QuadRows{0, 4});
        else
            f(q, quad_rows(p, q));
    }
}
// The same for passes whose arithmetic fills the registers (two waves a SIMD):
// load(q, rows) of the next quad is issued before the current one is used,
// f(quad, q, rows).
template <typename D, typename L, typename F>
__device__ __forceinline__ void each_quad_ahead(const NormArgs& a, const NormPlace& p, L&& load, F&& f) {
    const auto whole = [&](int64_t q) { return 4 * q >= p.f0 && 4 * q + 4 <= p.f1; };
    const auto fetch = [&](D& d, int64_t q) {
        if (whole(q))
            load(d, q, QuadRows{0, 4});
        else
            load(d, q, quad_rows(p, q));
    };
    int64_t q = p.q0 + p.ty;
    if (q >= p.q1) return;
    D cur, next;
    fetch(cur, q);
    for (;;) {
        const int64_t qn = q + a.ty;
        if (qn < p.q1) fetch(next, qn);
        __builtin_amdgcn_sched_barrier(0);
        if (whole(q))
            f(cur, q, QuadRows{0, 4});
        else
            f(cur, q, quad_rows(p, q));
        if (qn >= p.q1) return;
        cur = next;
        q = qn;
    }
}

template <typename F>
__device__ __forceinline__ F lane_xor(F v, int o) {
    return __shfl_xor(v, o);
}
template <>
__device__ __forceinline__ float2 lane_xor<float2>(float2 v, int o) {
    return make_float2(__shfl_xor(v.x, o), __shfl_xor(v.y, o));
}

// Σ over each group of the chunk of a value per thread (0 where the thread has
// none), in a fixed order; every thread gets its own group's sum.  red: a value
// per thread, then one per group.  Two sums in a row need no barrier between
// them if they use different `red`.
template <typename F, int NT>
__device__ __forceinline__ F group_sum(F v, const NormArgs& a, const NormPlace& p, F* red, int threads) {
    const int per = a.sub == 1 ? a.lanes / a.lpg : 1;
    if (per == 1) {  // one group: the whole block
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) v += lane_xor(v, o);
        if (threads == kWave) return v;
        if (wave_lane() == 0) red[wave_id()] = v;
        __syncthreads();
        F sum = red[0];
        for (int w = 1; w < threads / kWave; ++w) sum += red[w];
        return sum;
    }
    const int members = a.ty * a.lpg;
    int team = kWave;  // lanes per group: a power of two, no more than there are members
    while (team > 1 && team / 2 >= members) team /= 2;
    red[threadIdx.x] = v;
    __syncthreads();
    const int lane = threadIdx.x & (team - 1);
    for (int g = threadIdx.x / team; g < per; g += threads / team) {
        F sum{};
        for (int i = lane; i < members; i += team) {
            const int r = (int)((unsigned)i / (unsigned)a.lpg);
            sum += red[r * a.lanes + g * a.lpg + (i - r * a.lpg)];
        }
        for (int o = team / 2; o > 0; o >>= 1) sum += lane_xor(sum, o);
        if (lane == 0) red[NT + g] = sum;
    }
    __syncthreads();
    return red[NT + (a.sub == 1 ? p.tx / a.lpg : 0)];
}

// The masks of a slab thread's Q quads, drawn while its registers hold nothing
// else: the generator's column products and the rows together would not leave
// room for a block of 1024 threads.
template <int V, int Q>
__device__ __forceinline__ void slab_masks(const NormArgs& a, const NormPlace& p, uint32_t (&bits)[Q]) {
    ColumnKeep<V> columns;
    columns.init(a.key, (uint32_t)p.c0);
#pragma unroll
    for (int k = 0; k < Q; ++k) {
        bool kept[4][V];
        columns.quad(a.key, (uint32_t)(p.q0 + p.ty + k * a.ty), kept);
        bits[k] = pack_kept<V>(kept);
        asm volatile("" : "+v"(bits[k]));  // a word from here on, not its 4 V comparisons
        __builtin_amdgcn_sched_barrier(0);
    }
}

// v_exp_f32 and v_rcp_f32 are good to about one unit in the last place of fp32,
// below the rounding of z itself.
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
        const float s = sigmoid_f(z);  // s + z s (1 - s)
        return __builtin_fmaf(s, __builtin_fmaf(-z, s, z), s);
    }
    return 1.f;
}

// A thread's constants of its group, or (SPAN) of each channel's group.
template <int V, bool SPAN>
struct GroupValue {
    float f[SPAN ? V : 1];

    __device__ __forceinline__ float operator[](int e) const { return f[SPAN ? e : 0]; }
    // g(group) -> value
    template <typename G>
    __device__ __forceinline__ void fill(const NormArgs& a, const NormPlace& p, G&& g) {
        if constexpr (SPAN) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[e] = g((int)((unsigned)(p.c0 + e) / (unsigned)a.cg));
        } else {
            f[0] = g(p.group);
        }
    }
};

// γ rstd and β of a thread's channels: z = (x - mean) (γ rstd) + β.
template <int V>
struct NormParams {
    float rw[V], b[V];

    static __device__ __forceinline__ void values(const void* p, int code, int c0, float (&f)[V]) {
        if (code == LDS_F32)
            load_vec<float, V>(reinterpret_cast<const float*>(p) + c0, f);
        else if (code == LDS_BF16)
            load_vec<bf16_t, V>(reinterpret_cast<const bf16_t*>(p) + c0, f);
        else
            load_vec<f16_t, V>(reinterpret_cast<const f16_t*>(p) + c0, f);
    }
    __device__ __forceinline__ void load(const NormArgs& a, int c0) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
            rw[e] = 1.f;
            b[e] = 0.f;
        }
        if (a.weight) values(a.weight, a.ptype, c0, rw);
        if (a.bias) values(a.bias, a.ptype, c0, b);
    }
    template <bool SPAN>
    __device__ __forceinline__ void times(const GroupValue<V, SPAN>& rs) {
#pragma unroll
        for (int e = 0; e < V; ++e) rw[e] *= rs[e];
    }
};

// A thread's vector of a row; at a row's end across groups only what it owns.
template <typename T, int V, bool SPAN, bool PAST = false>
__device__ __forceinline__ void store_own(T* at, int skip, const float (&o)[V]) {
    if constexpr (SPAN) {
        if (skip) {
#pragma unroll
            for (int e = 0; e < V; ++e)
                if (e >= skip) at[e] = (T)o[e];
            return;
        }
    }
    store_vec<T, V, PAST>(at, o);
}

// Calls f with an integral constant for the activation / the vector width.
template <typename F>
inline int with_act(int act, F&& f) {
    if (act == LDS_ACT_NONE) return f(IntC<LDS_ACT_NONE>{});
    if (act == LDS_ACT_RELU) return f(IntC<LDS_ACT_RELU>{});
    if (act == LDS_ACT_SILU) return f(IntC<LDS_ACT_SILU>{});
    return (int)hipErrorInvalidValue;
}
template <int MAXV, typename F>
inline int with_vec(int v, bool span, F&& f) {
    if (span) return f(IntC<MAXV>{}, BoolC<true>{});
    if constexpr (MAXV >= 8)
        if (v == 8) return f(IntC<8>{}, BoolC<false>{});
    if (v == 4) return f(IntC<4>{}, BoolC<false>{});
    if (v == 2) return f(IntC<2>{}, BoolC<false>{});
    return f(IntC<1>{}, BoolC<false>{});
}

// The backward's second pass reads x and dy for the last time: past the caches, if
// a wave's vectors cover whole 128-byte lines (8 x 20000 x 256 bf16: both passes 91
// -> 79 us; with parts of lines, each fetched again, 8 x 20000 x 25 groups of 4 fp16
// 44.6 -> 49.2).  A result of more than half the memory-side cache goes past it
// too, with the forward's reads: alone / with a multiplication of the result
// after it, in us, 16 x 20000 x 256 fp32 forward 206 / 322 -> 171 / 294, backward 339 /
// 457 -> 288 / 433; bf16 (164 MB) 107 / 141 -> 86 / 142, 186 / 236 -> 144 / 218.  A
// smaller one is read from the cache afterwards: 8 x 20000 x 256 bf16 (82 MB) would
// gain 8 of 58 alone and lose 3 of 85 with what follows.
inline bool whole_lines(const void* p, int64_t samples, int64_t stride, int64_t ld, int c, int size) {
    const int64_t line = 128;
    return (uintptr_t)p % line == 0 && ld * size % line == 0 && (int64_t)c * size % line == 0 &&
           (samples == 1 || stride * size % line == 0);
}
inline bool past_caches(int64_t result_bytes) { return result_bytes > kMemorySideCache / 2; }

// What a row's last vector has in common with the one before it is the same in
// both, so both may store it (8 x 20000 x 12 groups of 5 fp16: 27.5 -> 25.8 us forward,
// 32.7 -> 30.8 backward), unless the result overlaps an input that the other
// has yet to read.
inline bool whole_store(const void* to, int64_t samples, int64_t n, int c, int size, const void* from, int64_t stride,
                        int64_t ld) {
    const ByteSpan out(to, samples * n * c, size);
    return !out.meets(ByteSpan(from, (samples > 1 ? (samples - 1) * stride : 0) + (n - 1) * ld + c, size));
}

// ... for a slab thread's quads: at most 32 values of x are held.
template <int V, typename F>
inline void with_quads(int quads, F&& f) {
    if constexpr (V <= 2)
        if (quads == 4) return f(IntC<4>{});
    if constexpr (V <= 4)
        if (quads == 2) return f(IntC<2>{});
    f(IntC<1>{});
}

// The sizes that both directions accept; false: hipErrorInvalidValue.
inline bool norm_sizes_ok(int64_t samples, int64_t n, int c, int groups) {
    if (samples < 0 || n < 0 || c < 0 || groups < 1 || c % groups) return false;
    if (samples > 0x7fffffff || n > 0x7fffffff) return false;
    return samples * n <= (int64_t)0x7fffffff;
}

inline int norm_elem(int dtype) { return dtype == LDS_F32 ? 4 : 2; }

// How a call runs: the geometry of NormArgs, the block size, the form.
struct NormPlan {
    int v;
    bool slab;
    int threads;   // slab: 64 .. slab_threads
    int quads;     // slab: row quads per thread: 1, or 2 (V <= 4), or 4 (V <= 2)
    NormArgs a;
};

// slab_threads: the largest slab block; want: blocks of a pass of the parts form.
inline NormPlan norm_plan(int64_t samples, int64_t n, int c, int groups, int dtype, int slab_threads,
                          int want = kSumBlocks) {
    NormPlan k{};
    NormArgs& a = k.a;
    const int elem = norm_elem(dtype);
    a.samples = samples;
    a.n = n;
    a.c = c;
    a.groups = groups;
    a.cg = c / groups;
    // the widest vector (<= 16 bytes) that lies in one group
    k.v = 16 / elem;
    while (k.v > 1 && a.cg % k.v) k.v /= 2;
    const int lpg = a.cg / k.v;
    const int64_t quads = (n + 2) / 4 + 1;  // a sample's quads at most, wherever its first row lies in one
    a.part_q = quads;
    a.parts = 1;
    a.sub = 1;
    a.lpg = lpg;
    const auto held = [&](int threads, int per) -> int64_t {  // quads per thread
        const int ty = threads / (per * lpg);
        return ty < 1 ? INT64_MAX : (quads + ty - 1) / ty;
    };
    // The slab form, where one block's arithmetic is short beside the two launches
    // it saves: a group of up to 32768 values of a sample (forward; half of
    // that backward).  One sample of 4000 x 8 channels a group, bf16: 10.2 us
    // against 13.2 in parts, backward 15.0 / 13.7; of 8000: 15.6 / 13.1.  And,
    // where there are more blocks than two per CU, only with whole lines to
    // read: 200 samples of 2000 x 8 groups of 8, bf16 (32 bytes of a row a
    // block): 45.0 / 34.6 us; of 1000 (64 bytes): 19.3 / 23.8.
    const int most_quads = k.v == 8 ? 1 : k.v == 4 ? 2 : 4;
    if (lpg <= slab_threads && held(slab_threads, 1) <= most_quads) {
        // As few groups a block as there are, for more blocks; more where blocks
        // abound and a row's share is under a 64-byte line or a block under 256
        // threads.
        int per = 1;
        while (per * 2 <= groups && samples * (groups / (per * 2)) >= 256 && held(slab_threads, per * 2) <= 1 &&
               (per * a.cg * elem < 64 || per * lpg * quads < 256))
            per *= 2;
        if (samples * ((groups + per - 1) / per) <= 512 || per * a.cg * elem >= 64 || per == groups) {
            k.slab = true;
            // the smallest block at which a thread holds one quad
            k.threads = 64;
            while (k.threads < slab_threads && held(k.threads, per) > 1) k.threads *= 2;
            const int64_t q = held(k.threads, per);
            k.quads = q <= 1 ? 1 : q <= 2 ? 2 : 4;
            a.lanes = per * lpg;
            a.ty = k.threads / a.lanes;
            a.chunks = (groups + per - 1) / per;
            return k;
        }
    }
    const int widest = 16 / elem;
    if (k.v == 1 && c >= widest && c <= kNormThreads * widest) {
        // Groups of an odd width: whole vectors all the same, which then lie
        // across groups, with the group's constants per channel.  16 samples of
        // 20000 x 12 groups of 5, fp16: 37.3 us against 49.4 with one channel a
        // lane, backward 49.5 / 70.0.  Groups of 12 keep four channels a lane
        // (34.4 us; 36.4 across groups), groups of 2 two (34.3; 35.3).
        k.v = widest;
        a.span = 1;
        a.lanes = (c + widest - 1) / widest;
        a.chunks = 1;
    } else if (lpg <= kNormThreads) {
        int per = kNormThreads / lpg;
        if (per > groups) per = groups;
        a.chunks = (groups + per - 1) / per;
        per = (groups + a.chunks - 1) / a.chunks;  // even chunks
        a.chunks = (groups + per - 1) / per;
        a.lanes = per * lpg;
    } else {
        a.sub = (lpg + kNormThreads - 1) / kNormThreads;
        a.lanes = (lpg + a.sub - 1) / a.sub;
        a.lpg = a.lanes;
        a.chunks = groups * a.sub;
    }
    a.ty = kNormThreads / a.lanes;
    // about `want` blocks in all, and not less than two quads to a thread
    // where there are that many
    int64_t p = want / (samples * a.chunks > 0 ? samples * a.chunks : 1);
    const int64_t most = (quads + 2 * a.ty - 1) / (2 * a.ty);
    if (p > most) p = most;
    if (p < 1) p = 1;
    a.part_q = (quads + p - 1) / p;
    a.parts = (int)((quads + a.part_q - 1) / a.part_q);
    return k;
}

// Workspace of the backward: the channel sums of every part (of every sample,
// in the slab form), then (parts) the two means of every group.
inline int64_t backward_ws(const NormArgs& a, bool slab) {
    if (slab) return a.samples == 1 ? 0 : a.samples * (int64_t)a.c * 8;
    return a.samples * a.parts * (int64_t)a.c * 8 + a.samples * a.groups * 8;
}

// f(arguments, blocks) for the launches of a pass.
template <typename F>
inline void norm_launches(NormArgs a, int64_t blocks, int threads, F&& f) {
    in_launches(blocks, threads, [&](int64_t first, unsigned count) {
        a.first = (unsigned)first;
        f(a, count);
    });
}

// Blocks of a slab launch, and a block's place in it: the blocks of a sample
// share its lines where a group is narrow, so from eight samples on a sample
// stays on one XCD (blocks go round the eight of them).
inline int64_t slab_blocks(const NormArgs& a) {
    return a.samples >= 8 ? (a.samples + 7) / 8 * 8 * a.chunks : a.samples * a.chunks;
}
__device__ __forceinline__ bool slab_place(const NormArgs& a, int64_t& s, int& chunk) {
    const unsigned b = blockIdx.x + a.first, u = a.samples >= 8 ? b >> 3 : b;
    const unsigned t = u / (unsigned)a.chunks;
    chunk = (int)(u - t * a.chunks);
    s = a.samples >= 8 ? (int64_t)t * 8 + (b & 7) : t;
    return s < a.samples;
}

}  // namespace lds
