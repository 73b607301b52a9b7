// lc_logits.cu -- penalties for repeated tokens, biases and grammar masks on
// logits, with the row's argmax key.
//
// For token j of a row (r, f, p its repetition, frequency and presence
// penalties, c_j how often the row generated j):
//   x = logit;  seen in the row's history: x = x > 0 ? x / r : x * r
//   c_j > 0:    x = (x - f * c_j) - p
//   biased:     x = x + bias (the last of the row's entries for j)
//   masked:     x = -inf
// each operation rounded once, in this order, so that equal inputs give equal
// bits whatever the launch shape.
//
// Bound by reading and writing the logits once.  The history and the bias list
// are scattered: a CTA owns a slice of the vocabulary and counts the row's tokens
// that fall into it in shared memory (integer adds, and a maximum over list
// positions for biases: no order changes a result), then streams the slice.  In
// the stream a warp works its touched tokens out one per lane at a time: there are
// a few dozen in 8192, so most warps meet one, and few lanes two.
// A row is one cluster of CTAs, so the row's key is reduced over distributed
// shared memory and the whole call is one launch without a workspace.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "lc_internal.cuh"
#include "lc_sm100.cuh"

namespace {

constexpr int kLgThreads = 512;
constexpr int kLgVecs = 4;
constexpr int kLgHold = 8;  // 4096 tokens of a row's history
constexpr int kLgSlice = kLgThreads * 4 * kLgVecs;  // 8192 tokens counted at a time
constexpr uint32_t kLgListMax = 0x7FFF0000u;  // list positions + kLgHold * kLgThreads stay int32
constexpr uint32_t kSeen = 0x80000000u;  // of a counter: in the history (low bits: generated count)

struct LgArgs {
    const float *x;
    float *y;
    uint64_t ldx, ldy;
    uint32_t n, row_offset, part;  // part: tokens of a CTA of the cluster, a multiple of 128
    lc_logits_rules r;
    uint64_t *keys;
    int vec_x, vec_y;  // rows 16-byte aligned
};

__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t v;
    asm("mov.u32 %0, %%cluster_nctaid.x;\n" : "=r"(v));
    return v;
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t v;
    asm("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(v));
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.aligned;\nbarrier.cluster.wait.aligned;\n" ::: "memory");
}
// Store to the same shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ void cluster_store(uint64_t *p, uint32_t rank, uint64_t v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(at), "l"(v) : "memory");
}

__device__ __forceinline__ int clamp_index(int v, int lo, int hi) { return min(max(v, lo), hi); }

// One token after the penalties, the bias entry s - 1 (0: none) and the mask bit.
struct LgRow {
    float rep, freq, pres;
    const float *bias;
    __device__ __forceinline__ float operator()(float v, uint32_t c, uint32_t s) const {
        if (c) {
            v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
            c &= ~kSeen;
            if (c) v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)c)), pres);
        }
        return s ? __fadd_rn(v, bias[s - 1]) : v;
    }
};

__global__ void __launch_bounds__(kLgThreads, 2) logits_kernel(const __grid_constant__ LgArgs a) {
    extern __shared__ __align__(16) uint32_t lg_smem[];
    __shared__ long long best_warp[kLgThreads / 32];
    __shared__ uint64_t best_cta[16];
    uint32_t *cnt = lg_smem;              // [kLgSlice]
    uint32_t *slot = lg_smem + kLgSlice;  // [kLgSlice], only with a bias list: 1 + list position
    const uint32_t cl = cluster_size(), rank = cluster_rank();
    const uint32_t row = blockIdx.x / cl;
    const float *x = a.x + (size_t)row * a.ldx;
    float *y = a.y ? a.y + (size_t)row * a.ldy : nullptr;
    const lc_logits_rules &r = a.r;
    const uint32_t p0 = min(a.n, rank * a.part), p1 = min(a.n, p0 + a.part);

    // A thread's share of a slice: kLgVecs pieces of 4 tokens, kLgThreads * 4 apart.
    // A piece of the next slice is requested where the last one's has been written,
    // so that it arrives while the lists are counted.
    float4 v[kLgVecs];
    auto load = [&](int u, uint32_t s0) {
        const uint32_t i = s0 + (threadIdx.x + u * kLgThreads) * 4;
        if (a.vec_x && i + 4 <= p1) {
            v[u] = __ldcs(reinterpret_cast<const float4 *>(x + i));
        } else {
            v[u].x = i < p1 ? x[i] : 0.f;
            v[u].y = i + 1 < p1 ? x[i + 1] : 0.f;
            v[u].z = i + 2 < p1 ? x[i + 2] : 0.f;
            v[u].w = i + 3 < p1 ? x[i + 3] : 0.f;
        }
    };
#pragma unroll
    for (int u = 0; u < kLgVecs; u++) load(u, p0);

    // the row's lists; indexes from the device are held inside the arrays
    int h0 = 0, h1 = 0, g0 = 0, b0 = 0, b1 = 0;
    if (r.hist_start) {
        h0 = clamp_index(r.hist_start[row], 0, (int)r.hist_len);
        h1 = clamp_index(r.hist_start[row + 1], h0, (int)r.hist_len);
        g0 = r.gen_start ? r.gen_start[row] : h0;
    }
    if (r.bias_start) {
        b0 = clamp_index(r.bias_start[row], 0, (int)r.bias_len);
        b1 = clamp_index(r.bias_start[row + 1], b0, (int)r.bias_len);
    }
    const uint32_t *mask = nullptr;
    if (r.mask) {
        const int mr = r.mask_row ? r.mask_row[row] : (int)row;
        if (mr >= 0 && (uint32_t)mr < r.n_masks) mask = r.mask + (size_t)mr * r.mask_ld;
    }
    const LgRow rules = {r.repetition ? r.repetition[row] : 1.f, r.frequency ? r.frequency[row] : 0.f,
                         r.presence ? r.presence[row] : 0.f, r.bias + b0};
    const bool listed = h1 > h0 || b1 > b0, biased = b1 > b0;

    // best (value order of lc_pack_key: the bits as a signed integer; token)
    int best_ord = INT_MIN;
    uint32_t best_j = 0;
    bool any = false;
    // The first kLgHold tokens of a thread's share of the history, and its first bias
    // token, stay in registers for every slice (~0: none).
    uint32_t held[kLgHold], held_bias = ~0u;
#pragma unroll
    for (int u = 0; u < kLgHold; u++) {
        const int i = h0 + (int)threadIdx.x + u * kLgThreads;
        held[u] = i < h1 ? (uint32_t)r.hist[i] : ~0u;
    }
    if (b0 + (int)threadIdx.x < b1) held_bias = (uint32_t)r.bias_tok[b0 + threadIdx.x];
    if (listed) {
#pragma unroll
        for (int u = 0; u < kLgVecs; u++) {
            const uint32_t i = (threadIdx.x + u * kLgThreads) * 4;
            *reinterpret_cast<uint4 *>(cnt + i) = make_uint4(0, 0, 0, 0);
            if (biased) *reinterpret_cast<uint4 *>(slot + i) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
    }
    for (uint32_t s0 = p0; s0 < p1; s0 += kLgSlice) {
        const uint32_t len = min((uint32_t)kLgSlice, p1 - s0);
        if (listed) {
            // tokens outside [first, first + len) wrap past len
            const uint32_t first = a.row_offset + s0;
            auto count = [&](uint32_t token, int i) {
                const uint32_t t = token - first;
                if (t >= len) return;
                if (i >= g0)
                    atomicAdd(cnt + t, 1u);
                else
                    atomicOr(cnt + t, kSeen);
            };
#pragma unroll
            for (int u = 0; u < kLgHold; u++) count(held[u], h0 + (int)threadIdx.x + u * kLgThreads);
#pragma unroll 4
            for (int i = h0 + (int)threadIdx.x + kLgHold * kLgThreads; i < h1; i += kLgThreads)
                count((uint32_t)r.hist[i], i);
            if (biased) {
                auto enter = [&](uint32_t token, uint32_t place) {
                    const uint32_t t = token - first;
                    if (t < len) atomicMax(slot + t, place);
                };
                enter(held_bias, threadIdx.x + 1u);
                for (int i = b0 + (int)threadIdx.x + kLgThreads; i < b1; i += kLgThreads)
                    enter((uint32_t)r.bias_tok[i], (uint32_t)(i - b0) + 1u);
            }
            __syncthreads();
        }
#pragma unroll
        for (int u = 0; u < kLgVecs; u++) {
            const uint32_t i = (threadIdx.x + u * kLgThreads) * 4, j = s0 + i;
            if (i >= len) break;
            float e[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
            if (listed) {  // what was counted is cleared for the next slice
                uint4 c = *reinterpret_cast<const uint4 *>(cnt + i), s = make_uint4(0, 0, 0, 0);
                if (c.x | c.y | c.z | c.w) *reinterpret_cast<uint4 *>(cnt + i) = s;
                if (biased) {
                    const uint4 t = *reinterpret_cast<const uint4 *>(slot + i);
                    if (t.x | t.y | t.z | t.w) *reinterpret_cast<uint4 *>(slot + i) = s;
                    s = t;
                }
                uint32_t left = (c.x | s.x ? 1u : 0u) | (c.y | s.y ? 2u : 0u) | (c.z | s.z ? 4u : 0u) |
                                (c.w | s.w ? 8u : 0u);
#pragma unroll 1
                while (left) {
                    const uint32_t bit = left & (0u - left);
                    left ^= bit;
                    const float x = bit == 1 ? e[0] : bit == 2 ? e[1] : bit == 4 ? e[2] : e[3];
                    const uint32_t n = bit == 1 ? c.x : bit == 2 ? c.y : bit == 4 ? c.z : c.w;
                    const uint32_t b = bit == 1 ? s.x : bit == 2 ? s.y : bit == 4 ? s.z : s.w;
                    const float w = rules(x, n, b);
                    e[0] = bit == 1 ? w : e[0], e[1] = bit == 2 ? w : e[1];
                    e[2] = bit == 4 ? w : e[2], e[3] = bit == 8 ? w : e[3];
                }
            }
            if (s0 + kLgSlice < p1) load(u, s0 + kLgSlice);
            if (mask) {
                const uint32_t g = a.row_offset + j;  // 4 bits that may end in the next word, if that exists
                const uint32_t lo = mask[g >> 5], hi = (g & 31) > 28 && i + 32 - (g & 31) < len ? mask[(g >> 5) + 1] : 0u;
                const uint32_t bits = __funnelshift_r(lo, hi, g & 31);
#pragma unroll
                for (int q = 0; q < 4; q++)
                    if (!(bits >> q & 1)) e[q] = -INFINITY;
            }
#pragma unroll
            for (int q = 0; q < 4; q++) {
                const int b = __float_as_int(e[q]), ord = b ^ ((b >> 31) & 0x7FFFFFFF);
                if (ord >= best_ord && i + q < len) best_ord = ord, best_j = j + q, any = true;
            }
            if (y) {
                if (a.vec_y && i + 4 <= len) {
                    __stcs(reinterpret_cast<float4 *>(y + j), make_float4(e[0], e[1], e[2], e[3]));
                } else {
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        if (i + q < len) y[j + q] = e[q];
                }
            }
        }
        if (listed) __syncthreads();  // the counters are read before the next slice clears them
    }
    if (!a.keys) return;  // uniform over the cluster
    // (order, global token) as the signed key of lc_pack_key
    long long best = any ? (long long)(((uint64_t)(uint32_t)best_ord << 32) | (a.row_offset + best_j)) : LLONG_MIN;
#pragma unroll
    for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if ((threadIdx.x & 31) == 0) best_warp[threadIdx.x >> 5] = best;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kLgThreads / 32; w++) best = max(best, best_warp[w]);
        cluster_store(best_cta + rank, 0, (uint64_t)best);
    }
    __syncwarp();
    cluster_sync();
    if (rank == 0 && threadIdx.x == 0) {
        for (uint32_t c = 0; c < cl; c++) best = max(best, (long long)best_cta[c]);
        a.keys[row] = (uint64_t)best;
    }
}

}  // namespace

extern "C" int lc_logits_process(lc_ctx *ctx, const float *logits, uint64_t ld, float *out, uint64_t ld_out,
                                 uint32_t m, uint32_t n, uint32_t row_offset, const lc_logits_rules *rules,
                                 uint64_t *keys) {
    LC_REQUIRE(ctx, LC_ERR_INVALID, "lc_logits_process: null ctx");
    if (m == 0) return LC_OK;
    LC_REQUIRE(logits && rules && (out || keys), LC_ERR_INVALID, "lc_logits_process: null pointer");
    LC_REQUIRE(n > 0 && n <= (1u << 30), LC_ERR_INVALID, "lc_logits_process: n %u not in 1..2^30", n);
    LC_REQUIRE(row_offset <= 0x7FFFFFFFu - n, LC_ERR_INVALID,
               "lc_logits_process: tokens %u .. + %u do not fit an int32", row_offset, n);
    LC_REQUIRE(m <= (1u << 24), LC_ERR_UNSUPPORTED, "lc_logits_process: %u rows", m);
    const lc_logits_rules &r = *rules;
    LC_REQUIRE(r.hist_len <= kLgListMax && r.bias_len <= kLgListMax, LC_ERR_UNSUPPORTED,
               "lc_logits_process: token lists above %u entries", kLgListMax);
    LC_REQUIRE((!r.hist_len || r.hist) && (!r.hist || r.hist_start), LC_ERR_INVALID,
               "lc_logits_process: hist and hist_start go together");
    LC_REQUIRE((!r.bias_len || (r.bias_tok && r.bias)) && (!r.bias_tok || r.bias_start), LC_ERR_INVALID,
               "lc_logits_process: bias_tok, bias and bias_start go together");
    const uint64_t words = ((uint64_t)row_offset + n + 31) / 32;
    LC_REQUIRE(!r.mask || r.mask_ld >= words, LC_ERR_INVALID,
               "lc_logits_process: masks of %llu words do not reach token %llu", (unsigned long long)r.mask_ld,
               (unsigned long long)row_offset + n);
    LC_REQUIRE(!r.mask || r.mask_row || r.n_masks >= m, LC_ERR_INVALID,
               "lc_logits_process: %u masks for %u rows and no mask_row", r.n_masks, m);
    LC_REQUIRE(!r.mask || r.mask_ld <= (1ull << 40), LC_ERR_INVALID, "lc_logits_process: mask stride too large");
    if (!ld) ld = n;
    if (!ld_out) ld_out = n;
    LC_REQUIRE(ld >= n && (!out || ld_out >= n), LC_ERR_INVALID, "lc_logits_process: a row stride is shorter than n");
    LC_REQUIRE(ld <= (1ull << 58) / m && ld_out <= (1ull << 58) / m, LC_ERR_INVALID,
               "lc_logits_process: row stride too large");
    LC_REQUIRE((((uintptr_t)logits | (uintptr_t)out | (uintptr_t)r.hist | (uintptr_t)r.hist_start |
                 (uintptr_t)r.gen_start | (uintptr_t)r.repetition | (uintptr_t)r.frequency | (uintptr_t)r.presence |
                 (uintptr_t)r.bias_tok | (uintptr_t)r.bias | (uintptr_t)r.bias_start | (uintptr_t)r.mask |
                 (uintptr_t)r.mask_row) & 3) == 0 && ((uintptr_t)keys & 7) == 0,
               LC_ERR_INVALID, "lc_logits_process: a pointer is not aligned to its type");
    LC_REQUIRE(!out || (out == logits && ld == ld_out) ||
                   !lc_rows_meet(logits, ld * 4, n * 4ull, out, ld_out * 4, n * 4ull, m),
               LC_ERR_INVALID, "lc_logits_process: out overlaps logits (only out = logits in place is possible)");
    if (int s = lc_use_device(ctx)) return s;
    LgArgs a = {};
    a.x = logits, a.y = out, a.ldx = ld, a.ldy = ld_out, a.n = n, a.row_offset = row_offset, a.r = r, a.keys = keys;
    a.vec_x = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    a.vec_y = ((uintptr_t)out & 15) == 0 && ld_out % 4 == 0;
    // CTAs of a row's cluster: 4, more where few rows leave SMs idle (one row of 128256
    // tokens is a slice a CTA with 16; 256 rows take 100 us with 4, 110 with 8, 132 with
    // 16); each with at least 2048 tokens
    uint32_t cl = m * 16 <= 2u * ctx->num_sms ? 16 : m * 8 <= 2u * ctx->num_sms ? 8 : 4;
    while (cl > 1 && n / cl < 2048) cl /= 2;
    static std::atomic<uint64_t> wide{0};  // devices (below 64) on which the size is allowed already
    if (cl > 8 && (ctx->device > 63 || !(wide.load() >> ctx->device & 1))) {
        LC_CUDA(cudaFuncSetAttribute(logits_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        if (ctx->device < 64) wide |= 1ull << ctx->device;
    }
    a.part = ((n + cl - 1) / cl + 127) / 128 * 128;
    const size_t smem = (size_t)kLgSlice * (r.bias_len ? 8 : 4);
    if (int s = lc_set_smem_attr((const void *)logits_kernel, smem)) return s;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(m * cl);
    cfg.blockDim = dim3(kLgThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = ctx->stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    LC_CUDA(cudaLaunchKernelEx(&cfg, logits_kernel, (const LgArgs)a));
    return lc_after_launch(ctx, "lc_logits_process");
}
