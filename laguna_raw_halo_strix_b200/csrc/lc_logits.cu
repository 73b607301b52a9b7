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
// are scattered: a CTA owns slices of the vocabulary and counts the row's tokens
// that fall into one in shared memory (integer adds, and a maximum over list
// positions for biases: no order changes a result).  A row is one cluster of CTAs,
// so the row's key is reduced over distributed shared memory and a call is one
// launch without a workspace.
//
// Few rows (logits_row_kernel): a slice a CTA, which counts, then streams it with
// the touched tokens worked out by the lanes that hold them: the fewest steps that
// wait for one another.  Many rows (logits_kernel): clusters go from row to row.
// In a CTA four warps are a slice ahead of the eight that stream: they gather the
// touched tokens, a few dozen, and leave the bits that change in their logits,
// which the stream applies with an exclusive or.  Its loads of the next slice, over
// the ends of rows too, never wait for lists.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "lc_internal.cuh"
#include "lc_sm100.cuh"

namespace {

constexpr int kLgThreads = 256, kLgListThreads = 128;  // logits_kernel: stream, then list warps
constexpr int kLgAll = kLgThreads + kLgListThreads;
constexpr int kLgRowThreads = 512;  // logits_row_kernel
constexpr int kLgVecs = 4;          // a stream thread's pieces of 4 tokens in a slice
constexpr uint32_t kLgSlice = kLgThreads * 4 * kLgVecs, kLgRowSlice = kLgRowThreads * 4 * kLgVecs;
constexpr int kLgMine = 4096;       // tokens of the history kept for a CTA,
constexpr int kLgGroups = 32;       // in at most that many groups of slices
constexpr int kLgRowCost = 2000;    // what a row costs besides its tokens, in tokens
// counts stay below kBiased, list positions + 8 threads' strides int32
constexpr uint32_t kLgListMax = 0x3FFF0000u;
// Of a counter: in the history before the generated tokens; in the bias list
// (the low 30 bits are the generated count).
constexpr uint32_t kSeen = 0x80000000u, kBiased = 0x40000000u;

struct LgArgs {
    const float *x;
    float *y;
    uint64_t ldx, ldy;
    uint32_t m, n, row_offset, cl, clusters;
    uint32_t part;  // tokens of a CTA of the cluster, a multiple of 128
    uint32_t group_shift, group_room;
    lc_logits_rules r;
    uint64_t *keys;
    unsigned *status;
    int vec_x, vec_y;  // rows 16-byte aligned
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t v;
    asm volatile("mov.u32 %0, %%cluster_ctarank;\n" : "=r"(v));
    return v;
}
// A barrier over the cluster in two halves (writes before the first are seen after
// the second).
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.aligned;\n" ::: "memory"); }
// Store to the same shared variable of CTA `rank` of the cluster.
__device__ __forceinline__ void cluster_store(long long *p, uint32_t rank, long long v) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(at) : "r"(smem_addr(p)), "r"(rank));
    asm volatile("st.shared::cluster.u64 [%0], %1;\n" ::"r"(at), "l"(v) : "memory");
}

__device__ __forceinline__ int clamp_index(int v, int lo, int hi) { return min(max(v, lo), hi); }

__device__ __forceinline__ void lg_list_sync() { asm volatile("bar.sync 1, %0;\n" ::"n"(kLgListThreads) : "memory"); }

// 4 tokens from x on, `left` of them inside the row (0 behind it).
__device__ __forceinline__ float4 lg_load(const float *x, int left, int vec) {
    if (vec && left >= 4) return __ldcs(reinterpret_cast<const float4 *>(x));
    return make_float4(left > 0 ? x[0] : 0.f, left > 1 ? x[1] : 0.f, left > 2 ? x[2] : 0.f, left > 3 ? x[3] : 0.f);
}
__device__ __forceinline__ void lg_store(float *y, int left, int vec, const uint32_t (&e)[4]) {
    if (vec && left >= 4) {
        __stcs(reinterpret_cast<uint4 *>(y), make_uint4(e[0], e[1], e[2], e[3]));
        return;
    }
#pragma unroll
    for (int q = 0; q < 4; q++)
        if (left > q) y[q] = __uint_as_float(e[q]);
}
// The masks.  A warp holds the words of its 4 x 128 tokens of a slice, lanes 8 u ..
// 8 u + 4 those of piece u (a row_offset may have them end in a fifth word).
static_assert(kLgVecs == 4);
__device__ __forceinline__ int lg_mask(const LgArgs &a, uint32_t row) {  // its row's mask, or -1
    const lc_logits_rules &r = a.r;
    if (!r.mask || row >= a.m) return -1;
    const int mr = r.mask_row ? r.mask_row[row] : (int)row;
    return mr >= 0 && (uint32_t)mr < r.n_masks ? mr : -1;
}
// warp0: the warp's first token of the slice; step: tokens between its pieces.
__device__ __forceinline__ uint32_t lg_mask_words(const LgArgs &a, int mask, uint32_t warp0, uint32_t step,
                                                  uint32_t p1, uint32_t lane) {
    const uint32_t at = warp0 + (lane >> 3) * step, w = ((a.row_offset + at) >> 5) + (lane & 7);
    return at < p1 && w <= (a.row_offset + p1 - 1) >> 5 ? a.r.mask[(size_t)mask * a.r.mask_ld + w] : 0u;
}
// The bits of token j on, of a piece u whose first token in the warp is piece0.
__device__ __forceinline__ uint32_t lg_mask_bits(const LgArgs &a, uint32_t words, int u, uint32_t piece0, uint32_t j) {
    const uint32_t g = a.row_offset + j, src = u * 8 + ((g >> 5) - ((a.row_offset + piece0) >> 5));
    return __funnelshift_r(__shfl_sync(~0u, words, src), __shfl_sync(~0u, words, src + 1), g & 31);
}
// The best token: value order of lc_pack_key (the bits as a signed integer), then
// the later token.
struct LgBest {
    int ord = INT_MIN;
    uint32_t j = 0;
    // 4 tokens from j0 on, `left` of them inside the row: the others become the
    // lowest of the order, 0xFFFFFFFF.
    __device__ __forceinline__ void take(uint32_t (&e)[4], uint32_t j0, int left) {
        if (left < 4) {
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (left <= q) e[q] = ~0u;
        }
        int o[4];
#pragma unroll
        for (int q = 0; q < 4; q++) o[q] = (int)e[q] ^ (((int)e[q] >> 31) & 0x7FFFFFFF);
        const uint32_t j01 = j0 + (o[1] >= o[0]), j23 = j0 + 2 + (o[3] >= o[2]);
        const int o01 = max(o[0], o[1]), o23 = max(o[2], o[3]), top = max(o01, o23);
        j = top >= ord ? (o23 >= o01 ? j23 : j01) : j;
        ord = max(ord, top);
    }
    // (order, global token) as the signed key of lc_pack_key, the warp's highest.  A
    // token behind the row is the best only where all of it is the lowest too, which
    // makes its last token the best.
    __device__ __forceinline__ long long key(const LgArgs &a) const {
        long long best = (long long)((uint64_t)(uint32_t)ord << 32 | (a.row_offset + min(j, a.n - 1)));
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
        return best;
    }
};

// A row's numbers, one a thread: starts and ends of its lists, then its penalties.
constexpr int kLgNumbers = 8;
__device__ __forceinline__ int lg_number(const lc_logits_rules &r, uint32_t row, int which) {
    switch (which) {
    case 0: return r.hist_start ? r.hist_start[row] : 0;
    case 1: return r.hist_start ? r.hist_start[row + 1] : 0;
    case 2: return r.hist_start && r.gen_start ? r.gen_start[row] : INT_MIN;
    case 3: return r.bias_start ? r.bias_start[row] : 0;
    case 4: return r.bias_start ? r.bias_start[row + 1] : 0;
    case 5: return __float_as_int(r.repetition ? r.repetition[row] : 1.f);
    case 6: return __float_as_int(r.frequency ? r.frequency[row] : 0.f);
    default: return __float_as_int(r.presence ? r.presence[row] : 0.f);
    }
}
// The lists, held inside their arrays, and the rules.
struct LgLists {
    int h0, h1, g0, b0, b1;
    float rep, freq, pres;
    __device__ __forceinline__ LgLists(const lc_logits_rules &r, const int *number) {
        h0 = clamp_index(number[0], 0, (int)r.hist_len);
        h1 = clamp_index(number[1], h0, (int)r.hist_len);
        g0 = number[2];  // INT_MIN: all were generated
        b0 = clamp_index(number[3], 0, (int)r.bias_len);
        b1 = clamp_index(number[4], b0, (int)r.bias_len);
        rep = __int_as_float(number[5]), freq = __int_as_float(number[6]), pres = __int_as_float(number[7]);
    }
    // A token of the history after the penalties; c: its counter.
    __device__ __forceinline__ float penalised(float v, uint32_t c) const {
        v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
        const uint32_t made = c & ~(kSeen | kBiased);
        return made ? __fsub_rn(__fsub_rn(v, __fmul_rn(freq, (float)made)), pres) : v;
    }
};

// What the list threads of a CTA share.
struct LgShared {
    // The row's history in the CTA's part: token - p0, times 2, + 1 if generated, those
    // of 2^group_shift slices together, up to group_room.
    uint32_t *mine;     // [kLgMine]
    uint16_t *touched;  // [kLgSlice]
    uint32_t *slot;     // [kLgSlice], only with a bias list: 1 + list position; all 0 between slices
    uint32_t *n_mine;   // [kLgGroups]; of a group above group_room the history is read again for each slice
};

// Thread `tid` of `threads` collects the row's history in the CTA's part (n_mine 0
// before, to be complete at the next barrier).
template <int kThreads>
__device__ __forceinline__ void lg_collect(const LgArgs &a, const LgLists &l, uint32_t p0, uint32_t p1,
                                           const LgShared &sh, int tid) {
    for (int base = l.h0 + tid; base < l.h1; base += 8 * kThreads) {  // 8 loads in flight
        uint32_t t[8];
#pragma unroll
        for (int u = 0; u < 8; u++) {
            const int i = base + u * kThreads;
            t[u] = i < l.h1 ? (uint32_t)a.r.hist[i] - (a.row_offset + p0) : ~0u;
        }
#pragma unroll
        for (int u = 0; u < 8; u++)
            if (t[u] < p1 - p0) {
                const uint32_t g = t[u] / kLgSlice >> a.group_shift, k = atomicAdd(sh.n_mine + g, 1u);
                if (k < a.group_room) sh.mine[g * a.group_room + k] = t[u] << 1 | (base + u * kThreads >= l.g0);
            }
    }
}

// The touched tokens of the slice [s0, s0 + len) of row x, the `from`-th on of the
// CTA's part: cnt (all 0 before) holds the bits that change in their logits after it.
// By the list threads; bias0: token of the row's bias entry `tid`, if there is one.
__device__ __forceinline__ void lg_touch(const LgArgs &a, const LgLists &l, const float *x, uint32_t s0, uint32_t len,
                                         uint32_t from, uint32_t bias0, const LgShared &sh, uint32_t *cnt,
                                         uint32_t *n_touched, int tid) {
    const lc_logits_rules &r = a.r;
    const uint32_t first = a.row_offset + s0;  // tokens outside [first, first + len) wrap past len
    auto enter = [&](uint32_t t, uint32_t old) {
        if (old == 0) sh.touched[atomicAdd(n_touched, 1u)] = (uint16_t)t;
    };
    auto count = [&](uint32_t t, bool made) {
        if (t < len) enter(t, made ? atomicAdd(cnt + t, 1u) : atomicOr(cnt + t, kSeen));
    };
    const uint32_t g = from / kLgSlice >> a.group_shift, n_mine = sh.n_mine[g];
    if (n_mine <= a.group_room) {
        const uint32_t *mine = sh.mine + g * a.group_room;
        for (uint32_t i = tid; i < n_mine; i += kLgListThreads) count((mine[i] >> 1) - from, mine[i] & 1);
    } else {
        for (int i = l.h0 + tid; i < l.h1; i += kLgListThreads) count((uint32_t)r.hist[i] - first, i >= l.g0);
    }
    auto bias = [&](uint32_t t, int i) {
        if (t < len) {
            atomicMax(sh.slot + t, (uint32_t)(i - l.b0) + 1u);
            enter(t, atomicOr(cnt + t, kBiased));
        }
    };
    if (l.b0 + tid < l.b1) bias(bias0 - first, l.b0 + tid);
    for (int i = l.b0 + tid + kLgListThreads; i < l.b1; i += kLgListThreads) bias((uint32_t)r.bias_tok[i] - first, i);
    lg_list_sync();
    const uint32_t nt = *n_touched;
    for (uint32_t k = tid; k < nt; k += kLgListThreads) {
        const uint32_t t = sh.touched[k], c = cnt[t];
        const float old = x[s0 + t];
        float v = old;
        if (c & ~kBiased) v = l.penalised(v, c);
        if (c & kBiased) {
            v = __fadd_rn(v, r.bias[l.b0 + sh.slot[t] - 1]);
            sh.slot[t] = 0;
        }
        cnt[t] = __float_as_uint(v) ^ __float_as_uint(old);
    }
}

// Rows by the CTAs of a cluster, a part of each a CTA.  Three CTAs an SM keep 48 KB of
// loads under way, which the 56 registers allow as long as none are spilled: shared
// memory leaves so little L1 that a spilled one comes back from L2 (three words took 256
// rows of 128256 in an earlier form from 94 to 158 us).  Without lists those rows take
// 49 us, 5.4 TB/s; what lists add, to 74 us with up to 4096 tokens of history, 100 biases
// and masks a row (77 with 300), is the list warps' time where a slice of theirs takes
// longer than the stream's.  Tokens that are not spread over the vocabulary cost more: 99
// us where most have low ids, for a slice whose group has no room counts the whole history.
__global__ void __launch_bounds__(kLgAll, 3) logits_kernel(const __grid_constant__ LgArgs a) {
    extern __shared__ __align__(16) uint32_t lg_smem[];
    __shared__ long long best_of[2][16 * kLgThreads / 32];  // of rank 0, by the row's parity
    __shared__ uint32_t n_touched[2], n_mine[kLgGroups];
    __shared__ int number[2][kLgNumbers];  // by the row's parity
    __shared__ volatile int gave_up;
    __shared__ uint64_t full[2], empty[2];  // the counters of a slice's parity
    uint32_t *cnt = lg_smem;                // [2][kLgSlice], by the slice's parity
    LgShared sh;
    sh.mine = cnt + 2 * kLgSlice, sh.touched = reinterpret_cast<uint16_t *>(sh.mine + kLgMine);
    sh.slot = sh.mine + kLgMine + kLgSlice / 2, sh.n_mine = n_mine;
    const uint32_t clusters = a.clusters;
    const lc_logits_rules &r = a.r;
    const uint32_t p0 = min(a.n, cluster_rank() * a.part), p1 = min(a.n, p0 + a.part);
    const uint32_t slices = (p1 - p0 + kLgSlice - 1) / kLgSlice;
    const int tid = threadIdx.x;
    const uint32_t lane = tid & 31;
    const bool stream = tid < kLgThreads, lists = r.hist_len || r.bias_len;
    uint32_t row = blockIdx.x / a.cl;  // the cluster's rows: `clusters` apart
    griddep_wait();  // the kernel before this one, whose end the launch need not wait for
    if (a.keys) cluster_arrive();      // that all its CTAs run, before the first store to another one

    // A stream thread's share of a slice: kLgVecs pieces of 4 tokens, kLgThreads * 4
    // apart.  A piece of the next slice (the next row's first after the last) is
    // requested where the last one's has been written.
    constexpr int kStep = kLgThreads * 4;
    float4 v[kLgVecs];
    const float *xt = a.x + (size_t)row * a.ldx + p0 + tid * 4;
    int left = (int)(p1 - p0) - tid * 4;  // tokens from the thread's first of the slice being loaded
    const uint32_t warp_at = (tid & ~31) * 4;
    int mask = -1;
    uint32_t words = 0;
    if (stream) {
#pragma unroll
        for (int u = 0; u < kLgVecs; u++) v[u] = lg_load(xt + u * kStep, left - u * kStep, a.vec_x);
        mask = lg_mask(a, row);
        if (mask >= 0) words = lg_mask_words(a, mask, p0 + warp_at, kStep, p1, lane);
    }
    auto bias_at = [&](const LgLists &l, int i) { return l.b0 + i < l.b1 ? (uint32_t)r.bias_tok[l.b0 + i] : 0u; };
    if (lists) {
        if (tid < kLgNumbers) number[0][tid] = lg_number(r, row, tid);
        for (uint32_t i = tid * 4; i < 2 * kLgSlice; i += kLgAll * 4)
            *reinterpret_cast<uint4 *>(cnt + i) = make_uint4(0, 0, 0, 0);
        if (r.bias_len)
            for (uint32_t i = tid * 4; i < kLgSlice; i += kLgAll * 4)
                *reinterpret_cast<uint4 *>(sh.slot + i) = make_uint4(0, 0, 0, 0);
        if (tid < 2) n_touched[tid] = 0;
        if (tid < kLgGroups) n_mine[tid] = 0;
        if (tid == 2) gave_up = 0;
        if (tid == 3) {
            for (int b = 0; b < 2; b++) mbar_init(full + b, kLgListThreads / 32), mbar_init(empty + b, kLgThreads / 32);
            mbar_init_fence();
        }
        __syncthreads();
        lg_collect<kLgAll>(a, LgLists(r, number[0]), p0, p1, sh, tid);  // the first row's, by every thread
        __syncthreads();
    }

    // A bounded wait; once one has given up (the launch is reported as failed), the
    // CTA's others give up at once.
    auto wait = [&](uint64_t *bar, uint32_t parity) {
        for (uint32_t i = 0; !mbar_test(bar, parity); i++)
            if (i > kWaitSpins || gave_up) {
                gave_up = 1;
                atomicOr(a.status, LC_DEV_WAIT_TIMEOUT);
                break;
            }
    };
    uint32_t k = 0;  // slices before this one, over the rows: its counters are those of k's parity
    uint32_t turn = 0;  // rows before this one
    if (!stream) {
        for (; row < a.m; row += clusters, turn++) {
            const bool more = row + clusters < a.m;
            if (lists) {
                const float *x = a.x + (size_t)row * a.ldx;
                const int at = tid - kLgThreads;
                if (turn) {
                    lg_list_sync();  // the last row's tokens are no longer read
                    if (at < kLgGroups) n_mine[at] = 0;
                    lg_list_sync();
                    lg_collect<kLgListThreads>(a, LgLists(r, number[turn & 1]), p0, p1, sh, at);
                }
                const uint32_t bias0 = bias_at(LgLists(r, number[turn & 1]), at);
                int next = 0;
                if (more && at < kLgNumbers) next = lg_number(r, row + clusters, at);
                for (uint32_t s = 0; s < slices; s++, k++) {
                    const uint32_t b = k & 1, s0 = p0 + s * kLgSlice;
                    if (k >= 2) wait(empty + b, (k - 2) >> 1 & 1);
                    if (at == 0) n_touched[b] = 0;  // last used two slices ago
                    lg_list_sync();
                    lg_touch(a, LgLists(r, number[turn & 1]), x, s0, min(kLgSlice, p1 - s0), s0 - p0, bias0, sh,
                             cnt + b * kLgSlice, n_touched + b, at);
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full + b);
                }
                if (at < kLgNumbers) number[(turn + 1) & 1][at] = next;
            }
            if (a.keys) {
                __syncwarp();
                cluster_wait();
                cluster_arrive();
            }
        }
        if (a.keys) cluster_wait();
        return;
    }
    auto write_key = [&](uint32_t row, uint32_t parity) {  // by the first warp of rank 0
        long long best = LLONG_MIN;
        for (uint32_t i = lane; i < a.cl * (kLgThreads / 32); i += 32) best = max(best, best_of[parity][i]);
#pragma unroll
        for (int o = 16; o; o >>= 1) best = max(best, __shfl_xor_sync(~0u, best, o));
        if (lane == 0) a.keys[row] = (uint64_t)best;
    };
    for (; row < a.m; row += clusters, turn++) {
        const bool more_rows = row + clusters < a.m;
        LgBest best;
        for (uint32_t s0 = p0; s0 < p1; s0 += kLgSlice, k++) {
            const int here = (int)(p1 - s0) - tid * 4;
            const bool more = s0 + kLgSlice < p1 || more_rows, masked = mask >= 0;
            const uint32_t held = words;
            if (s0 + kLgSlice < p1) {
                xt += kLgSlice, left -= kLgSlice;
                if (mask >= 0) words = lg_mask_words(a, mask, s0 + kLgSlice + warp_at, kStep, p1, lane);
            } else if (more_rows) {
                xt = a.x + (size_t)(row + clusters) * a.ldx + p0 + tid * 4, left = (int)(p1 - p0) - tid * 4;
                mask = lg_mask(a, row + clusters);
                if (mask >= 0) words = lg_mask_words(a, mask, p0 + warp_at, kStep, p1, lane);
            }
            if (lists) wait(full + (k & 1), k >> 1 & 1);
            float *yt = a.y + (size_t)row * a.ldy + s0 + tid * 4;
            uint32_t *changed = cnt + (k & 1) * kLgSlice + tid * 4;
#pragma unroll
            for (int u = 0; u < kLgVecs; u++) {
                const uint32_t j = s0 + tid * 4 + u * kStep;
                uint32_t bits = 0;
                if (masked) bits = lg_mask_bits(a, held, u, s0 + warp_at + u * kStep, j);
                uint32_t e[4] = {__float_as_uint(v[u].x), __float_as_uint(v[u].y), __float_as_uint(v[u].z),
                                 __float_as_uint(v[u].w)};
                if (lists) {
                    const uint4 c = *reinterpret_cast<const uint4 *>(changed + u * kStep);
                    e[0] ^= c.x, e[1] ^= c.y, e[2] ^= c.z, e[3] ^= c.w;
                    if (c.x | c.y | c.z | c.w)  // cleared for the slice after next
                        *reinterpret_cast<uint4 *>(changed + u * kStep) = make_uint4(0, 0, 0, 0);
                }
                if (more) v[u] = lg_load(xt + u * kStep, left - u * kStep, a.vec_x);
                if (masked) {
#pragma unroll
                    for (int q = 0; q < 4; q++)
                        if (!(bits >> q & 1)) e[q] = 0xFF800000u;  // -inf
                }
                best.take(e, j, here - u * kStep);
                if (a.y) lg_store(yt + u * kStep, here - u * kStep, a.vec_y, e);
            }
            if (lists) {
                __syncwarp();
                if (lane == 0) mbar_arrive(empty + (k & 1));
            }
        }
        if (!a.keys) continue;
        const long long key = best.key(a);
        // Rank 0 takes the warps' keys of a row up one row later, so that nobody waits
        // for the slowest: the wait is for the row before.
        cluster_wait();
        if (turn && cluster_rank() == 0 && tid < 32) write_key(row - clusters, (turn - 1) & 1);
        if (lane == 0)
            cluster_store(&best_of[turn & 1][cluster_rank() * (kLgThreads / 32) + (tid >> 5)], 0, key);
        __syncwarp();
        cluster_arrive();
    }
    if (!a.keys) return;
    cluster_wait();
    if (cluster_rank() == 0 && tid < 32) write_key(row - clusters, (turn - 1) & 1);
}

// One row a cluster, one slice a CTA (a.part <= kLgRowSlice).
__global__ void __launch_bounds__(kLgRowThreads, 2) logits_row_kernel(const __grid_constant__ LgArgs a) {
    extern __shared__ __align__(16) uint32_t lg_smem[];
    __shared__ long long best_of[16 * kLgRowThreads / 32];  // of rank 0
    __shared__ int number[kLgNumbers];
    uint32_t *cnt = lg_smem;                 // [kLgRowSlice]
    uint32_t *slot = lg_smem + kLgRowSlice;  // [kLgRowSlice], only with a bias list: 1 + list position
    const lc_logits_rules &r = a.r;
    const uint32_t row = blockIdx.x / a.cl, rank = cluster_rank();
    const uint32_t p0 = min(a.n, rank * a.part), len = min(a.n - p0, a.part);
    const int tid = threadIdx.x;
    const uint32_t lane = tid & 31, warp_at = (tid & ~31) * 4;
    griddep_wait();  // the kernel before this one, whose end the launch need not wait for
    if (a.keys) cluster_arrive();  // that all its CTAs run, before the first store to another one

    constexpr int kStep = kLgRowThreads * 4;
    const int left = (int)len - tid * 4;
    const bool lists = r.hist_len || r.bias_len;
    if (lists && tid < kLgNumbers) number[tid] = lg_number(r, row, tid);
    const float *xt = a.x + (size_t)row * a.ldx + p0 + tid * 4;
    float4 v[kLgVecs];
#pragma unroll
    for (int u = 0; u < kLgVecs; u++) v[u] = lg_load(xt + u * kStep, left - u * kStep, a.vec_x);
    const int mask = lg_mask(a, row);
    uint32_t words = 0;
    if (mask >= 0) words = lg_mask_words(a, mask, p0 + warp_at, kStep, p0 + len, lane);
    if (lists) {
        for (uint32_t i = tid * 4; i < (r.bias_len ? 2 : 1) * kLgRowSlice; i += kLgRowThreads * 4)
            *reinterpret_cast<uint4 *>(cnt + i) = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    const LgLists l(r, number);
    const bool biased = lists && l.b1 > l.b0, listed = lists && (l.h1 > l.h0 || biased);
    if (listed) {
        const uint32_t first = a.row_offset + p0;  // tokens outside [first, first + len) wrap past len
        for (int base = l.h0 + tid; base < l.h1; base += 8 * kLgRowThreads) {  // 8 loads in flight
            uint32_t t[8];
#pragma unroll
            for (int u = 0; u < 8; u++) {
                const int i = base + u * kLgRowThreads;
                t[u] = i < l.h1 ? (uint32_t)r.hist[i] - first : ~0u;
            }
#pragma unroll
            for (int u = 0; u < 8; u++) {
                if (t[u] >= len) continue;
                if (base + u * kLgRowThreads >= l.g0)
                    atomicAdd(cnt + t[u], 1u);
                else
                    atomicOr(cnt + t[u], kSeen);
            }
        }
        for (int i = l.b0 + tid; i < l.b1; i += kLgRowThreads) {
            const uint32_t t = (uint32_t)r.bias_tok[i] - first;
            if (t < len) atomicMax(slot + t, (uint32_t)(i - l.b0) + 1u);
        }
        __syncthreads();
    }
    LgBest best;
    float *yt = a.y + (size_t)row * a.ldy + p0 + tid * 4;
#pragma unroll
    for (int u = 0; u < kLgVecs; u++) {
        const uint32_t at = tid * 4 + u * kStep, j = p0 + at;
        uint32_t e[4] = {__float_as_uint(v[u].x), __float_as_uint(v[u].y), __float_as_uint(v[u].z),
                         __float_as_uint(v[u].w)};
        if (listed) {
            uint4 c = *reinterpret_cast<const uint4 *>(cnt + at), s = make_uint4(0, 0, 0, 0);
            if (biased) s = *reinterpret_cast<const uint4 *>(slot + at);
            uint32_t todo = (c.x | s.x ? 1u : 0u) | (c.y | s.y ? 2u : 0u) | (c.z | s.z ? 4u : 0u) |
                            (c.w | s.w ? 8u : 0u);
#pragma unroll 1
            while (todo) {  // one per lane at a time: few lanes have two
                const uint32_t bit = todo & (0u - todo);
                todo ^= bit;
                float w = __uint_as_float(bit == 1 ? e[0] : bit == 2 ? e[1] : bit == 4 ? e[2] : e[3]);
                const uint32_t n = bit == 1 ? c.x : bit == 2 ? c.y : bit == 4 ? c.z : c.w;
                const uint32_t b = bit == 1 ? s.x : bit == 2 ? s.y : bit == 4 ? s.z : s.w;
                if (n) w = l.penalised(w, n);
                if (b) w = __fadd_rn(w, r.bias[l.b0 + b - 1]);
                const uint32_t o = __float_as_uint(w);
                e[0] = bit == 1 ? o : e[0], e[1] = bit == 2 ? o : e[1];
                e[2] = bit == 4 ? o : e[2], e[3] = bit == 8 ? o : e[3];
            }
        }
        if (mask >= 0) {
            const uint32_t bits = lg_mask_bits(a, words, u, p0 + warp_at + u * kStep, j);
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (!(bits >> q & 1)) e[q] = 0xFF800000u;  // -inf
        }
        best.take(e, j, left - u * kStep);
        if (a.y) lg_store(yt + u * kStep, left - u * kStep, a.vec_y, e);
    }
    if (!a.keys) return;  // uniform over the cluster
    const long long key = best.key(a);
    cluster_wait();
    if (lane == 0)
        cluster_store(&best_of[rank * (kLgRowThreads / 32) + (tid >> 5)], 0, key);
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (rank == 0 && tid < 32) {
        long long top = LLONG_MIN;
        for (uint32_t i = lane; i < a.cl * (kLgRowThreads / 32); i += 32) top = max(top, best_of[i]);
#pragma unroll
        for (int o = 16; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
        if (lane == 0) a.keys[row] = (uint64_t)top;
    }
}

// What a launch of clusters of `cl` CTAs says (attr: its two attributes).
cudaLaunchConfig_t lg_config(int threads, size_t smem, uint32_t cl, cudaLaunchAttribute *attr) {
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cl;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cl);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return cfg;
}

// Clusters of `cl` CTAs of a kernel (0: logits_kernel, 1: logits_row_kernel) that the
// device runs at a time, with the most shared memory that it takes.
int lg_resident(lc_ctx *ctx, int kernel, uint32_t cl, int *clusters) {
    static std::atomic<int> known[64][2][17];  // by device: 1 + the answer
    std::atomic<int> *at = ctx->device < 64 ? &known[ctx->device][kernel][cl] : nullptr;
    if (at && at->load()) {
        *clusters = at->load() - 1;
        return LC_OK;
    }
    const void *f = kernel ? (const void *)logits_row_kernel : (const void *)logits_kernel;
    const size_t smem = kernel ? kLgRowSlice * 8 : kLgSlice * 14 + kLgMine * 4;
    LC_CUDA(cudaFuncSetAttribute(f, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
    if (int s = lc_set_smem_attr(f, smem)) return s;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = lg_config(kernel ? kLgRowThreads : kLgAll, smem, cl, attr);
    cfg.numAttrs = 1;
    LC_CUDA(cudaOccupancyMaxActiveClusters(clusters, f, &cfg));
    if (at) at->store(1 + *clusters);
    return LC_OK;
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
    const LcRows key_span = {keys, 0, keys ? 8ull * m : 0, 1}, out_rows = {out, ld_out * 4, out ? n * 4ull : 0, m};
    LC_REQUIRE(!lc_rows_meet(key_span, {logits, ld * 4, n * 4ull, m}) && !lc_rows_meet(key_span, out_rows),
               LC_ERR_INVALID, "lc_logits_process: keys overlap the logits");
    const struct {
        const void *at;
        uint64_t entries;
    } read[] = {{r.hist, r.hist_len}, {r.hist_start, m + 1ull}, {r.gen_start, m}, {r.repetition, m}, {r.frequency, m},
                {r.presence, m}, {r.bias_tok, r.bias_len}, {r.bias, r.bias_len}, {r.bias_start, m + 1ull},
                {r.mask_row, m}};
    for (const auto &l : read) {
        const LcRows span = {l.at, 0, l.at ? 4 * l.entries : 0, 1};
        LC_REQUIRE(!lc_rows_meet(span, out_rows) && !lc_rows_meet(span, key_span), LC_ERR_INVALID,
                   "lc_logits_process: an output overlaps a list");
    }
    const LcRows masks = {r.mask, r.mask_ld * 4, r.mask ? words * 4 : 0, r.n_masks};
    LC_REQUIRE(!lc_rows_meet(masks, out_rows) && !lc_rows_meet(masks, key_span), LC_ERR_INVALID,
               "lc_logits_process: an output overlaps the masks");
    if (int s = lc_use_device(ctx)) return s;
    LgArgs a = {};
    a.x = logits, a.y = out, a.ldx = ld, a.ldy = ld_out, a.m = m, a.n = n, a.row_offset = row_offset;
    a.r = r, a.keys = keys, a.status = ctx->dev_status;
    a.vec_x = ((uintptr_t)logits & 15) == 0 && ld % 4 == 0;
    a.vec_y = ((uintptr_t)out & 15) == 0 && ld_out % 4 == 0;
    // Few rows, a slice a CTA and all at a time, as many CTAs a row as that allows but
    // at least 4096 tokens each (one row of 128256: 7.9 us against 11.5 in the other
    // kernel, 37 of 50021: 9.1 against 12.8; with clusters that wait for others to end
    // 15.0; 16 rows of 32000 with 2048 each 7.4 us, with 4096 7.2).  16 slices end at 131072
    // tokens: one row of 151936 goes the other way, in 11.7 us.  Rows of one slice
    // with a history above an eighth of it too, which all of the CTA's threads count then
    // (512 rows of 4495 with 2000 tokens: 20 against 37; with 50 tokens on 3000, 41 against 24).
    const bool long_lists = r.hist_len > (uint64_t)m * n / 8;
    uint32_t cl = 1, clusters = 1;
    bool few = false;
    if ((n + 15) / 16 <= kLgRowSlice) {
        cl = 16;
        while (cl > 1 && n / cl < 4096) cl--;
        for (; (n + cl - 1) / cl <= kLgRowSlice; cl--) {
            int at_a_time = 0;
            if (int s = lg_resident(ctx, 1, cl, &at_a_time)) return s;
            few = m <= (uint32_t)at_a_time || (cl == 1 && long_lists);
            if (few || cl == 1) break;
        }
    }
    // Many: the CTAs of a cluster with which they end first.  Clusters of c take
    // ceil(m / clusters at a time) rows, each n / c tokens and what a row costs (256
    // rows of 128256: 74 us with the 3 that this gives, 79 with 5, 81 with 8).
    if (!few) {
        uint64_t least = ~0ull;
        for (uint32_t c = 1; c <= 16 && (c == 1 || n / c >= 2048); c++) {
            int at_a_time = 0;
            if (int s = lg_resident(ctx, 0, c, &at_a_time)) return s;
            if (at_a_time < 1) continue;
            const uint64_t rounds = (m + at_a_time - 1) / at_a_time, time = rounds * (n / c + kLgRowCost);
            if (time < least) least = time, cl = c, clusters = std::min<uint32_t>(m, at_a_time);
        }
        LC_REQUIRE(least != ~0ull, LC_ERR_UNSUPPORTED, "lc_logits_process: the device holds no CTA of the kernel");
    }
    a.part = ((n + cl - 1) / cl + 127) / 128 * 128;
    a.cl = cl, a.clusters = few ? m : clusters;
    const uint32_t slices = (a.part + kLgSlice - 1) / kLgSlice;
    while ((slices - 1) >> a.group_shift >= kLgGroups) a.group_shift++;
    a.group_room = kLgMine / (((slices - 1) >> a.group_shift) + 1);
    const bool lists = r.hist_len || r.bias_len;
    const size_t smem = !lists ? 0
                        : few  ? kLgRowSlice * (r.bias_len ? 8 : 4)
                               : kLgSlice * (r.bias_len ? 14 : 10) + kLgMine * 4;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t cfg = lg_config(few ? kLgRowThreads : kLgAll, smem, cl, attr);
    cfg.gridDim = dim3(a.clusters * cl);
    cfg.stream = ctx->stream;
    LC_CUDA(cudaLaunchKernelEx(&cfg, few ? logits_row_kernel : logits_kernel, (const LgArgs)a));
    return lc_after_launch(ctx, "lc_logits_process");
}
