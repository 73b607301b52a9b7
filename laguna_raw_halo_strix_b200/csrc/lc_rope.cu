// lc_rope.cu -- rotary positions of q and k: half and interleaved pairs, part
// of the head, a position per row, any row stride, f32 / f16 / bf16 in and out.
//
// Pair i of a head (rope_dim / 2 pairs) is turned by a = pos * freq[i]:
//   y1 = s (x1 cos a - x2 sin a),  y2 = s (x2 cos a + x1 sin a),
// the remaining dims are copied.  The angle of a far position needs more than
// 24 bits (pos 1e6 at freq 1 is 0.06 rad off in f32).  The product of two numbers of
// at most 31 and 24 bits has 55: it is held as a double and what that lost, and
// reduced mod 2 pi in 64 bits.  sincospif sees it as an f32, |a| <= pi, and a
// correction of first order makes up for that rounding (up to 9.4e-8 rad, half its
// square is 2^-47).  The rotation itself is f32 with one rounding to the output type.
//
// Bound by the bytes of x and y.  One CTA takes some rows (or a share of one
// row's heads when there are few): the rows' table of (cos, sin) is formed once
// in shared memory for every head, while each thread's first loads are in flight.
#include <math.h>

#include <algorithm>

#include <cuda_bf16.h>

#include "lc_internal.cuh"
#include "lc_sm100.cuh"

namespace {

constexpr int kRpThreads = 128;
// Items a thread has in flight (and loads before the table is ready): 8192 rows of
// 40 bf16 heads take 34.2 us with two in 8 CTAs an SM (4.9 TB/s), 39.8 with three in 6;
// more of narrower ones gained nothing.
constexpr int kRpItems = 2;
// CTAs an SM: narrow pieces of heads with copied dims need few registers and are bound
// by what is under way (8192 rows of 16 bf16 heads, 20 of 80 dims rotated: 24.7 us with
// 10 CTAs, 26.6 with the 9 that 53 registers leave).
constexpr int rp_ctas(bool pairs, int v, bool copies) { return !copies || v > 4 || (v == 4 && !pairs) ? 8 : v == 4 ? 9 : 10; }
constexpr uint32_t kRpMaxDim = 8192;  // a row's table of 32 KB
constexpr double kRpTurn = 0.15915494309189533577, kRpTurnLost = -9.8393383375912435e-18;  // 1 / (2 pi), its rounding

template <class T>
struct RpVec;  // 16 bytes of T
template <>
struct RpVec<float> {
    static constexpr int kN = 4;
};
template <>
struct RpVec<__half> {
    static constexpr int kN = 8;
};
template <>
struct RpVec<__nv_bfloat16> {
    static constexpr int kN = 8;
};

__device__ __forceinline__ float rp_f32(float v) { return v; }
__device__ __forceinline__ float rp_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float rp_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void rp_round(float v, float &o) { o = v; }
__device__ __forceinline__ void rp_round(float v, __half &o) { o = __float2half_rn(v); }
__device__ __forceinline__ void rp_round(float v, __nv_bfloat16 &o) { o = __float2bfloat16_rn(v); }

// N consecutive elements, as one access of N * sizeof(T) bytes where VEC.
template <class T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) RpPack {
    T v[N];
};
template <class T, int N, bool VEC>
__device__ __forceinline__ RpPack<T, N> rp_load(const T *p) {
    RpPack<T, N> r;
    if constexpr (VEC) {
        r = *reinterpret_cast<const RpPack<T, N> *>(p);
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) r.v[i] = p[i];
    }
    return r;
}
template <class T, int N, bool VEC>
__device__ __forceinline__ void rp_store(T *p, const float (&y)[N]) {
    RpPack<T, N> r;
#pragma unroll
    for (int i = 0; i < N; i++) rp_round(y[i], r.v[i]);
    if constexpr (VEC) {
        *reinterpret_cast<RpPack<T, N> *>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) p[i] = r.v[i];
    }
}

// Place of entry i in the table: items of 8 or 4 entries (64 or 32 bytes) would
// meet in the same banks, so their 16-byte pieces are rotated by the item.
template <int PER>
__device__ __forceinline__ int rp_slot(int i) {
    if (PER == 8) return i ^ ((i >> 4 & 3) << 1);
    if (PER == 4) return i ^ ((i >> 4 & 1) << 1);
    return i;
}

struct RpArgs {
    const void *x[2];   // q, k
    void *y[2];
    uint64_t ldx[2], ldy[2];  // elements between rows
    int same[2];              // y is x: dims past rope_dim stay as they are
    int n_q, n_heads;         // heads of q, of q and k together
    int head_dim, rope_dim;
    int rot, items, lanes;    // rotated items of a head, all items of a head, those side by side in a CTA
    int heads_per_cta, rows_per_cta;
    uint32_t m;
    const int32_t *pos;
    const float *freq;
    float scale;
};

// PAIRS false: an item is V dims at i and the V at i + rope_dim / 2; true: the
// V / 2 pairs of V neighbouring dims.  With COPIES, items rot.. are 2 V copied dims, V
// for the last where as many are left (a kernel of its own, for the copies' code costs
// rows that are all rotated a quarter of their speed).
template <class TI, class TO, bool PAIRS, int V, bool VEC, bool COPIES>
__global__ void __launch_bounds__(kRpThreads, rp_ctas(PAIRS, V, COPIES)) rope_kernel(const RpArgs a) {
    extern __shared__ float2 cs_rows[];  // [rows][rope_dim / 2]
    const size_t row0 = (size_t)blockIdx.x * a.rows_per_cta;
    const int rows = (int)min((size_t)a.rows_per_cta, a.m - row0);
    const int h0 = blockIdx.y * a.heads_per_cta, nh = min(a.n_heads, h0 + a.heads_per_cta) - h0;
    const int half = a.rope_dim >> 1;
    // A thread keeps its item (one of `lanes` side by side) and goes over (row, head)
    // pairs `sides` apart, rows first in steps of whole rows and rest heads.
    const int lanes = a.lanes, sides = kRpThreads / lanes, side = threadIdx.x / lanes;
    const int step_rows = sides / nh, step_heads = sides - step_rows * nh;
    auto step = [&](int &in, int &h) {
        in += step_rows, h += step_heads;
        if (h >= nh) h -= nh, in++;
    };
    int item = threadIdx.x - side * lanes;
    int in_head;  // the item's first dim (a row's heads are below 2^30 elements)
    auto take_item = [&]() { in_head = !COPIES || item < a.rot ? item * V : a.rope_dim + (item - a.rot) * (2 * V); };
    auto load = [&](int in, int h, RpPack<TI, V> &p0, RpPack<TI, V> &p1) {
        const bool k = h0 + h >= a.n_q;
        const TI *from = static_cast<const TI *>(k ? a.x[1] : a.x[0]) + (row0 + in) * (k ? a.ldx[1] : a.ldx[0]) +
                         ((h0 + h - (k ? a.n_q : 0)) * a.head_dim + in_head);
        if (COPIES && item >= a.rot && (k ? a.same[1] : a.same[0])) return;
        p0 = rp_load<TI, V, VEC>(from);
        if (COPIES && item >= a.rot) {
            if (in_head + V < a.head_dim) p1 = rp_load<TI, V, VEC>(from + V);
        } else if (!PAIRS) {
            p1 = rp_load<TI, V, VEC>(from + half);
        }
    };
    auto finish = [&](int in, int h, const RpPack<TI, V> &p0, const RpPack<TI, V> &p1) {
        const bool k = h0 + h >= a.n_q;
        TO *to = static_cast<TO *>(k ? a.y[1] : a.y[0]) + (row0 + in) * (k ? a.ldy[1] : a.ldy[0]) +
                 ((h0 + h - (k ? a.n_q : 0)) * a.head_dim + in_head);
        const float2 *cs = cs_rows + in * half;
        float o0[V], o1[V];
        if (COPIES && item >= a.rot) {
            if (k ? a.same[1] : a.same[0]) return;
#pragma unroll
            for (int i = 0; i < V; i++) o0[i] = rp_f32(p0.v[i]), o1[i] = rp_f32(p1.v[i]);
            rp_store<TO, V, VEC>(to, o0);
            if (in_head + V < a.head_dim) rp_store<TO, V, VEC>(to + V, o1);
        } else if constexpr (PAIRS) {
#pragma unroll
            for (int i = 0; i + 1 < V; i += 2) {
                const float2 c = cs[rp_slot<V / 2>((item * V + i) >> 1)];
                const float u = rp_f32(p0.v[i]), w = rp_f32(p0.v[i + 1]);
                o0[i] = u * c.x - w * c.y;
                o0[i + 1] = w * c.x + u * c.y;
            }
            rp_store<TO, V, VEC>(to, o0);
        } else {
#pragma unroll
            for (int i = 0; i < V; i++) {
                const float2 c = cs[rp_slot<V>(item * V + i)];
                const float u = rp_f32(p0.v[i]), w = rp_f32(p1.v[i]);
                o0[i] = u * c.x - w * c.y;
                o1[i] = w * c.x + u * c.y;
            }
            rp_store<TO, V, VEC>(to, o0);
            rp_store<TO, V, VEC>(to + half, o1);
        }
    };

    griddep_wait();  // the kernel before this one, whose end the launch need not wait for
    RpPack<TI, V> p0[kRpItems], p1[kRpItems];
    const int in0 = side < sides ? side / nh : rows, first_h = side - side / nh * nh;
    int in = in0, h = first_h;  // of the next load
    take_item();
#pragma unroll
    for (int j = 0; j < kRpItems; j++) {
        if (in < rows) load(in, h, p0[j], p1[j]);
        step(in, h);
    }
    if (half) {
        for (int i = threadIdx.x; i < rows * half; i += kRpThreads) {
            const int in = i / half;
            const double p = (double)a.pos[row0 + in], f = (double)a.freq[i - in * half];
            const double t = p * f, lost = fma(p, f, -t);
            const double n = t * kRpTurn;  // turns
            const double d = fma(t, kRpTurn, -n) + fma(lost, kRpTurn, t * kRpTurnLost);
            const double r = 2.0 * ((n - rint(n)) + d);  // in units of pi
            const float rf = (float)r, e = (float)(r - (double)rf) * 3.14159265f;
            float sn, cn;
            sincospif(rf, &sn, &cn);
            cs_rows[in * half + rp_slot<PAIRS ? V / 2 : V>(i - in * half)] =
                make_float2(fmaf(-sn, e, cn) * a.scale, fmaf(cn, e, sn) * a.scale);
        }
        __syncthreads();
    }
    while (true) {
        for (int fin = in0, fh = first_h; fin < rows;) {
#pragma unroll
            for (int j = 0; j < kRpItems; j++) {
                if (fin < rows) finish(fin, fh, p0[j], p1[j]);
                step(fin, fh);
            }
#pragma unroll
            for (int j = 0; j < kRpItems; j++) {
                if (in < rows) load(in, h, p0[j], p1[j]);
                step(in, h);
            }
        }
        item += lanes;  // heads of more items than threads
        if (item >= a.items) break;
        take_item();
        in = in0, h = first_h;
#pragma unroll
        for (int j = 0; j < kRpItems; j++) {
            if (in < rows) load(in, h, p0[j], p1[j]);
            step(in, h);
        }
    }
}

int type_bytes(int dtype) { return dtype == LC_F32 ? 4 : dtype == LC_F16 || dtype == LC_BF16 ? 2 : 0; }

template <class TI, class TO>
int rope_launch(lc_ctx *ctx, const RpArgs &base, uint32_t m, bool pairs) {
    constexpr int V = RpVec<TI>::kN;
    RpArgs a = base;
    const int half = a.rope_dim / 2;
    // Vectors of 16 or 8 bytes in, or of two elements, where every row, head and half starts on
    // a multiple of them (and the same element count out); single elements otherwise
    // (8192 rows of 8 + 8 bf16 heads of 80 with 20 dims rotated: 25 us in twos, 60 when
    // they went singly)
    auto fits = [&](int n) {
        bool yes = a.head_dim % n == 0 && (pairs ? a.rope_dim : half) % n == 0;
        for (int t = 0; t < 2; t++)
            if (t ? a.n_heads > a.n_q : a.n_q > 0) {
                const uintptr_t need_y = std::min<uintptr_t>(n * sizeof(TO), 16);
                yes = yes && (uintptr_t)a.x[t] % (n * sizeof(TI)) == 0 && a.ldx[t] % n == 0 &&
                      (uintptr_t)a.y[t] % need_y == 0 && a.ldy[t] % n == 0;
            }
        return yes;
    };
    const bool vec = fits(V), halves = fits(V / 2), twos = fits(2);
    const int v = vec ? V : halves ? V / 2 : twos || pairs ? 2 : 1;
    const bool q_copies = a.n_q > 0 && !a.same[0], k_copies = a.n_heads > a.n_q && !a.same[1];
    // (head_dim and rope_dim are even, so the copied dims divide by 2 as well)
    a.rot = pairs ? a.rope_dim / v : half / v;
    a.items = a.rot + ((q_copies || k_copies) ? (a.head_dim - a.rope_dim + 2 * v - 1) / (2 * v) : 0);
    if (a.items == 0) return LC_OK;
    // Few rows: a row's heads go to several CTAs, each with at least one item a
    // thread; every CTA forms the table again.  Many rows: a CTA takes as many as
    // give each thread 4 items, or until the grid is down to 4 CTAs per SM.
    const int row_items = a.n_heads * a.items;
    int splits = 1;
    if (m < 2u * ctx->num_sms) {
        const int most = std::max(1, row_items / kRpThreads);
        splits = std::min<int>(most, std::max(1, 2 * ctx->num_sms / (int)m));
    }
    a.heads_per_cta = (a.n_heads + splits - 1) / splits;
    splits = (a.n_heads + a.heads_per_cta - 1) / a.heads_per_cta;
    a.rows_per_cta = 1;
    const size_t table = (size_t)half * sizeof(float2);
    while (splits == 1 && a.rows_per_cta * row_items < 4 * kRpThreads &&
           m / (a.rows_per_cta + 1) >= 4u * ctx->num_sms && (a.rows_per_cta + 1) * table <= 32 * 1024)
        a.rows_per_cta++;
    a.m = m;
    a.lanes = std::min(a.items, kRpThreads);
    const dim3 grid((m + a.rows_per_cta - 1) / a.rows_per_cta, splits);
    const size_t smem = a.rows_per_cta * table;
    auto go = [&](auto kernel) -> int {
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(kRpThreads);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = ctx->stream;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        LC_CUDA(cudaLaunchKernelEx(&cfg, kernel, a));
        return lc_after_launch(ctx, "lc_rope");
    };
    auto width = [&](auto pair, auto copies) {
        constexpr bool P = decltype(pair)::value, C = decltype(copies)::value;
        if (vec) return go(rope_kernel<TI, TO, P, V, true, C>);
        if (halves) return go(rope_kernel<TI, TO, P, V / 2, true, C>);
        if constexpr (V / 2 > 2)
            if (twos) return go(rope_kernel<TI, TO, P, 2, true, C>);
        return go(rope_kernel<TI, TO, P, P ? 2 : 1, false, C>);
    };
    using Yes = std::true_type;
    using No = std::false_type;
    if (a.items > a.rot) return pairs ? width(Yes(), Yes()) : width(No(), Yes());
    return pairs ? width(Yes(), No()) : width(No(), No());
}

template <class TI>
int rope_out(lc_ctx *ctx, int out_dtype, const RpArgs &a, uint32_t m, bool pairs) {
    switch (out_dtype) {
    case LC_F16: return rope_launch<TI, __half>(ctx, a, m, pairs);
    case LC_BF16: return rope_launch<TI, __nv_bfloat16>(ctx, a, m, pairs);
    default: return rope_launch<TI, float>(ctx, a, m, pairs);
    }
}

}  // namespace

extern "C" int lc_rope(lc_ctx *ctx, int dtype, int out_dtype, int layout, const void *q, uint64_t ldq, void *q_out,
                       uint64_t ldq_out, uint32_t n_q_heads, const void *k, uint64_t ldk, void *k_out,
                       uint64_t ldk_out, uint32_t n_kv_heads, const int32_t *pos, const float *freq, uint32_t m,
                       uint32_t head_dim, uint32_t rope_dim, float scale) {
    LC_REQUIRE(ctx, LC_ERR_INVALID, "lc_rope: null ctx");
    const uint64_t bi = type_bytes(dtype), bo = type_bytes(out_dtype);
    LC_REQUIRE(bi && bo, LC_ERR_UNSUPPORTED, "lc_rope: types %d -> %d (LC_F32, LC_F16 and LC_BF16 only)", dtype,
               out_dtype);
    LC_REQUIRE(layout == LC_ROPE_HALF || layout == LC_ROPE_PAIRS, LC_ERR_INVALID, "lc_rope: bad layout %d", layout);
    LC_REQUIRE(head_dim > 0 && head_dim % 2 == 0, LC_ERR_INVALID, "lc_rope: head_dim %u must be even", head_dim);
    LC_REQUIRE(rope_dim % 2 == 0 && rope_dim <= head_dim, LC_ERR_INVALID,
               "lc_rope: rope_dim %u must be even and at most head_dim %u", rope_dim, head_dim);
    LC_REQUIRE(rope_dim <= kRpMaxDim, LC_ERR_UNSUPPORTED, "lc_rope: rope_dim %u above %u", rope_dim, kRpMaxDim);
    LC_REQUIRE(((uint64_t)n_q_heads + n_kv_heads) * head_dim < (1u << 30), LC_ERR_UNSUPPORTED,
               "lc_rope: rows of %u + %u heads of %u are too long", n_q_heads, n_kv_heads, head_dim);
    LC_REQUIRE(m < (1u << 31), LC_ERR_UNSUPPORTED, "lc_rope: %u rows", m);
    const uint64_t wq = (uint64_t)n_q_heads * head_dim, wk = (uint64_t)n_kv_heads * head_dim;
    if (m == 0 || wq + wk == 0) return LC_OK;
    if (!ldq) ldq = wq;
    if (!ldq_out) ldq_out = wq;
    if (!ldk) ldk = wk;
    if (!ldk_out) ldk_out = wk;
    LC_REQUIRE((!wq || (q && q_out)) && (!wk || (k && k_out)) && (!rope_dim || (pos && freq)), LC_ERR_INVALID,
               "lc_rope: null pointer");
    const uint64_t ld_max = std::max(std::max(ldq, ldq_out), std::max(ldk, ldk_out));
    LC_REQUIRE(ld_max <= ((uint64_t)1 << 60) / m, LC_ERR_INVALID, "lc_rope: row stride %llu too large",
               (unsigned long long)ld_max);
    LC_REQUIRE(ldq >= wq && ldq_out >= wq && ldk >= wk && ldk_out >= wk, LC_ERR_INVALID,
               "lc_rope: a row stride is shorter than its row");
    LC_REQUIRE((!wq || ((uintptr_t)q % bi == 0 && (uintptr_t)q_out % bo == 0)) &&
                   (!wk || ((uintptr_t)k % bi == 0 && (uintptr_t)k_out % bo == 0)) && (uintptr_t)pos % 4 == 0 &&
                   (uintptr_t)freq % 4 == 0,
               LC_ERR_INVALID, "lc_rope: a pointer is not aligned to its type");
    const bool q_same = wq && q == q_out && ldq == ldq_out && bi == bo && dtype == out_dtype;
    const bool k_same = wk && k == k_out && ldk == ldk_out && bi == bo && dtype == out_dtype;
    const bool meet = (wq && !q_same && lc_rows_meet(q, ldq * bi, wq * bi, q_out, ldq_out * bo, wq * bo, m)) ||
                      (wk && !k_same && lc_rows_meet(k, ldk * bi, wk * bi, k_out, ldk_out * bo, wk * bo, m)) ||
                      (wq && wk &&
                       (lc_rows_meet(q_out, ldq_out * bo, wq * bo, k_out, ldk_out * bo, wk * bo, m) ||
                        lc_rows_meet(q, ldq * bi, wq * bi, k_out, ldk_out * bo, wk * bo, m) ||
                        lc_rows_meet(k, ldk * bi, wk * bi, q_out, ldq_out * bo, wq * bo, m)));
    LC_REQUIRE(!meet, LC_ERR_INVALID, "lc_rope: an output overlaps another tensor (only y = x in place is possible)");
    const LcRows outs[2] = {{q_out, ldq_out * bo, wq * bo, m}, {k_out, ldk_out * bo, wk * bo, m}};
    if (rope_dim)
        for (const LcRows &y : outs)
            LC_REQUIRE(!lc_rows_meet({pos, 0, 4ull * m, 1}, y) && !lc_rows_meet({freq, 0, 2ull * rope_dim, 1}, y),
                       LC_ERR_INVALID, "lc_rope: an output overlaps pos or freq");
    RpArgs a = {};
    a.x[0] = q, a.x[1] = k, a.y[0] = q_out, a.y[1] = k_out;
    a.ldx[0] = ldq, a.ldx[1] = ldk, a.ldy[0] = ldq_out, a.ldy[1] = ldk_out;
    a.same[0] = q_same, a.same[1] = k_same;
    a.n_q = (int)n_q_heads, a.n_heads = (int)(n_q_heads + n_kv_heads);
    a.head_dim = (int)head_dim, a.rope_dim = (int)rope_dim;
    a.pos = pos, a.freq = freq, a.scale = scale;
    const bool pairs = layout == LC_ROPE_PAIRS;
    if (int s = lc_use_device(ctx)) return s;
    switch (dtype) {
    case LC_F16: return rope_out<__half>(ctx, out_dtype, a, m, pairs);
    case LC_BF16: return rope_out<__nv_bfloat16>(ctx, out_dtype, a, m, pairs);
    default: return rope_out<float>(ctx, out_dtype, a, m, pairs);
    }
}

extern "C" int lc_rope_freq_scaled(float *freq, uint32_t rope_dim, float base, int kind, float factor,
                                   uint32_t orig_ctx, float beta_fast, float beta_slow, float *scale) {
    LC_REQUIRE(scale && (freq || rope_dim < 2), LC_ERR_INVALID, "lc_rope_freq_scaled: null out");
    LC_REQUIRE(rope_dim % 2 == 0, LC_ERR_INVALID, "lc_rope_freq_scaled: rope_dim %u must be even", rope_dim);
    LC_REQUIRE(base > 1.f && base < INFINITY, LC_ERR_INVALID, "lc_rope_freq_scaled: base %g must be above 1", base);
    LC_REQUIRE(kind >= LC_ROPE_SCALE_NONE && kind <= LC_ROPE_SCALE_YARN, LC_ERR_INVALID,
               "lc_rope_freq_scaled: bad kind %d", kind);
    LC_REQUIRE(kind == LC_ROPE_SCALE_NONE || (factor >= 1.f && factor < INFINITY), LC_ERR_INVALID,
               "lc_rope_freq_scaled: factor %g must be at least 1", factor);
    LC_REQUIRE(kind != LC_ROPE_SCALE_NTK || rope_dim > 2, LC_ERR_INVALID,
               "lc_rope_freq_scaled: the NTK base needs rope_dim above 2");
    LC_REQUIRE(kind != LC_ROPE_SCALE_YARN || (orig_ctx > 0 && beta_slow > 0.f && beta_fast >= beta_slow &&
                                              beta_fast < INFINITY),
               LC_ERR_INVALID, "lc_rope_freq_scaled: YaRN needs orig_ctx > 0 and beta_fast >= beta_slow > 0");
    *scale = 1.f;
    const double d = rope_dim, b = base, f = factor;
    const double used = kind == LC_ROPE_SCALE_NTK ? b * pow(f, d / (d - 2)) : b;
    // YaRN: the pair whose wavelength fits `beta` times into the original context
    double low = 0, high = 0;
    if (kind == LC_ROPE_SCALE_YARN) {
        auto pair_of = [&](double beta) { return d * log(orig_ctx / (beta * 2 * M_PI)) / (2 * log(b)); };
        low = std::max(floor(pair_of(beta_fast)), 0.0);
        high = std::min(ceil(pair_of(beta_slow)), d - 1);
        *scale = (float)(0.1 * log(f) + 1);
    }
    for (uint32_t i = 0; i < rope_dim / 2; i++) {
        double w = pow(used, -2.0 * i / d);
        if (kind == LC_ROPE_SCALE_LINEAR) w /= f;
        if (kind == LC_ROPE_SCALE_YARN) {
            const double t = std::min(1.0, std::max(0.0, (i - low) / std::max(high - low, 1e-3)));
            w = w * (1 - t) + w / f * t;  // t = 0: short wavelengths, as they are
        }
        freq[i] = (float)w;
    }
    return LC_OK;
}
