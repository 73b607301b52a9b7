// lc_prefix_attn.cu -- attention of a batch of sequences that share the K/V rows
// of a prefix and have rows of their own behind it.
//
// out_r = sum_j w_j v_j / sum_j w_j,  w_j = exp(scale q_r . k_j), j over the
// prefix and the row's visible own keys.  The softmax of the joined axis splits
// into partial states (m, l, O) that merge exactly, so the prefix is computed
// once for the query rows of the whole batch (every sequence and every query
// head of a KV head are rows of one matrix product against it), the own parts
// per sequence, and a small kernel merges.
//
// A work item is up to 128 query rows of one KV head (whole tokens) against a
// range of the virtual key axis [prefix | own rows of its sequence].  Per tile
// of 64 keys
//   S = Q K^T   tcgen05, Q and K K-major in shared memory, S in TMEM 0..127
//   P           softmax warps, one thread a row and half tile, written over S as
//               16-bit pairs (for f32 outputs with one or two planes more of what
//               the rounding lost)
//   O += P V    tcgen05, P from TMEM, V read MN-major as it lies in memory
// Q, K and V come by TMA.  Roles: warps 0-7 softmax, 8 loads of Q and K and the
// hand-out of work, 9 loads of V, 10 issues S, 11 issues O.  K, V and S have two
// stages: the next tile's scores are formed while the softmax warps work on this
// one's, so that these, the longest link, do not wait (with one stage of 128 keys
// a tile's products and softmax alternated; now 890 TFLOP/s with 4 prompts of 512 tokens on
// 4096 f16 keys, 133 us, and 930 with one of 2048 on 32768).  Two CTAs share an
// SM (256 TMEM columns and 100 KB each).  CTAs stay for several items: the next
// one's Q and K are loaded while the last one's values and results are worked on.
#include <float.h>
#include <math.h>

#include <algorithm>

#include <cuda_bf16.h>

#include "lc_internal.cuh"
#include "lc_sm100.cuh"

namespace {

constexpr int kPaRows = 128, kPaKeys = 64;
constexpr int kPaLoadWarp = 8, kPaValueWarp = 9, kPaScoreWarp = 10, kPaMmaWarp = 11;  // 0..7 softmax
constexpr int kPaThreads = 384;
constexpr int kPaHalf = kPaKeys / 2;           // keys of a softmax warp, and of the smaller TMA copy
constexpr uint32_t kPaPlane = kPaRows * 128;   // 128 rows of Q x 64 16-bit elements (one swizzle span)
constexpr uint32_t kPaKvPlane = kPaKeys * 128;  // the same of K or V
constexpr uint32_t kPaColS = 0, kPaColO = 128, kPaTmemCols = 256;
constexpr int64_t kPaMaxItems = 1 << 22;
constexpr uint32_t kPaMaxLen = 0x3FFFF000u;  // prefix_len + own_cap: ranges of the key axis stay int32

// Shared memory: Q, then two stages of K and of V, in HD / 64 planes each; barriers.
template <int HD>
struct PaSmem {
    static constexpr uint32_t kTile = HD / 64 * kPaKvPlane;
    static constexpr uint32_t kQ = 0, kK = HD / 64 * kPaPlane, kV = kK + 2 * kTile, kBar = kV + 2 * kTile;
    // kRed: maxima [2][kPaRows], sums [2][kPaRows]
    static constexpr uint32_t kSched = kBar + 128, kJobs = kSched + 48, kRed = kJobs + 128;
    static constexpr uint32_t kBytes = kRed + 4 * kPaRows * 4 + 1024;  // + slack to 1024-align the base
};

// Division of numbers below 2^31 by a divisor known at launch, as a product with
// ceil(2^63 / d).
struct PaDiv {
    uint64_t inv;
    int d;
    __device__ __forceinline__ int operator()(int &rest) const {  // rest <- rest % d; the quotient
        const int q = (int)__umul64hi((uint64_t)rest << 1, inv);
        rest -= q * d;
        return q;
    }
};

struct PaArgs {
    const void *q;
    void *out;
    uint64_t ldq, ldo;
    int rows, n_q, n_kv, group;
    uint32_t group_inv;  // ceil(2^16 / group): r * group_inv >> 16 is r / group for r < 128
    int tile_toks, box_toks;  // tokens of a row tile and of one TMA copy of Q
    int prefix_len, own_cap, n_seqs;
    const int32_t *own_len, *seq_start;
    float scale_log2;  // scale * log2(e)
    int causal;
    // plan: items 0 .. prefix_items - 1 take the prefix for rows of all
    // sequences, the rest rows of one sequence over [seq_from, end) of the
    // virtual axis
    int prefix_items, row_tiles, prefix_keys;
    int prefix_splits, seq_splits, seq_keys, seq_from, seq_lanes;
    int seq_base;  // n_kv * n_seqs * seq_lanes
    PaDiv by_rest, by_heads, by_seqs, by_tiles;  // seq_base - direct, n_kv, n_seqs, row_tiles
    // The first `direct` sequence items run over the whole axis and write out (their
    // rows' first state says so: l = -1); merge: the others leave states
    int direct, merge;
    int merge_ways;  // warps that share the states of 32 rows and 8 dims: 1 or 4
    // partial states of row r = token * group + head within the group: O
    // unnormalised as [split][KV head][r / 32][HD / 4][r % 32][4] (32 rows' 16-byte
    // pieces side by side: the lanes of a warp hold neighbouring rows), and (m in
    // log2 units, l) as [split][KV head][r]
    float *o_part;
    float2 *ml_part;
    int row_blocks;     // 32-row blocks of a KV head
    unsigned *status;
};

// K/V copies: [half a tile or a whole one][prefix or own][K or V], as
// [sequence][row][element] (one sequence for the prefix); Q as [token][head][element].
struct PaMaps {
    CUtensorMap kv[2][2][2], q;
};

// Tokens first .. first + count - 1 (rows r = token within the tile * group +
// head within the group) of one KV head against prefix keys [p0, p1) and keys
// [o0, o1) of sequence seq.
struct PaJob {
    int n;  // tiles; -1: no more jobs
    int direct;
    int first, count, p0, p1, o0, o1, seq, hk, split;
    int pos0;  // own position of token t is pos0 + t
    __device__ __forceinline__ int prefix_tiles() const { return (p1 - p0 + kPaKeys - 1) / kPaKeys; }
    // tile i: first key, keys, own or prefix
    __device__ __forceinline__ void tile(int i, int &key, int &nk, bool &own) const {
        const int np = prefix_tiles();
        own = i >= np;
        key = own ? o0 + (i - np) * kPaKeys : p0 + i * kPaKeys;
        nk = min(kPaKeys, (own ? o1 : p1) - key);
    }
};

// Token of row r < 128 of a tile, within the tile.
__device__ __forceinline__ int pa_token(const PaArgs &a, int r) { return (int)((uint32_t)r * a.group_inv >> 16); }

struct PaItem {
    int direct, hk, split, t, t_step;  // token tiles at t, t + t_step, .. below count
    int start, count, len, seq, v0, v1;
};

// Item i in two steps: the first ends in loads whose values only the second looks
// at, so that they can be under way while the last item's copies are waited for.
__device__ __forceinline__ PaItem pa_item_begin(const PaArgs &a, int i) {
    PaItem t;
    const bool prefix = i < a.prefix_items;
    if (!prefix) i -= a.prefix_items;
    // sequence items: the direct ones, then the splits of the rest
    t.direct = !prefix && i < a.direct;
    int sp = 0;
    if (!prefix && !t.direct) {
        i -= a.direct;
        sp = a.by_rest(i);
        i += a.direct;
    }
    int hk = i;
    i = a.by_heads(hk);
    t.hk = hk;
    if (prefix) {
        int tile = i;
        t.split = a.by_tiles(tile);
        t.t = tile * a.tile_toks;
        t.seq = -1;
        t.start = 0, t.count = a.rows, t.len = 0;
    } else {
        int seq = i;
        t.t = a.by_seqs(seq) * a.tile_toks;
        t.seq = seq;
        t.split = a.prefix_splits + sp;
        t.start = a.seq_start[seq];
        t.count = a.seq_start[seq + 1];
        t.len = a.own_len ? a.own_len[seq] : 0;
    }
    return t;
}
__device__ __forceinline__ void pa_item_finish(const PaArgs &a, PaItem &t) {
    if (t.seq < 0) {
        t.t_step = 1 << 30;
        t.v0 = t.split * a.prefix_keys;
        t.v1 = min(a.prefix_len, t.v0 + a.prefix_keys);
    } else {
        t.t_step = a.seq_lanes * a.tile_toks;
        // values from the device are held inside the arrays
        t.start = min(max(t.start, 0), a.rows);
        t.count = min(max(t.count, t.start), a.rows) - t.start;
        t.len = min(max(t.len, 0), a.own_cap);
        t.v0 = a.seq_from + (t.split - a.prefix_splits) * a.seq_keys;
        t.v1 = a.prefix_len + a.own_cap;
        if (!t.direct) t.v1 = min(t.v1, t.v0 + a.seq_keys);
    }
}

__device__ __forceinline__ PaJob pa_job(const PaArgs &a, const PaItem &t, int at) {
    PaJob j;
    j.first = t.start + at;
    j.count = min(a.tile_toks, t.count - at);
    j.pos0 = t.len - t.count - t.start;
    j.p0 = min(t.v0, a.prefix_len), j.p1 = min(t.v1, a.prefix_len);
    j.o0 = max(t.v0, a.prefix_len) - a.prefix_len;
    j.o1 = min(max(t.v1, a.prefix_len) - a.prefix_len, t.len);
    if (a.causal) j.o1 = min(j.o1, j.pos0 + j.first + j.count);  // the last token's reach
    j.o1 = max(j.o1, j.o0);
    j.n = j.prefix_tiles() + (j.o1 - j.o0 + kPaKeys - 1) / kPaKeys;
    j.seq = t.seq, j.hk = t.hk, j.split = t.split, j.direct = t.direct;
    return j;
}

// A bounded wait that, once it has given up, is not repeated: the launch is
// reported as failed, so what follows only has to end.
struct PaWait {
    unsigned *status;
    bool ok = true;
    __device__ __forceinline__ void operator()(uint64_t *bar, uint32_t parity) {
        if (!ok) return;
        uint32_t left;
        asm volatile(
            "{\n .reg .pred p;\n mov.u32 %0, %3;\n"
            "AGAIN: mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n"
            " sub.u32 %0, %0, 1;\n setp.ne.u32 p, %0, 0;\n @p bra AGAIN;\nDONE:\n}\n"
            : "=&r"(left)
            : "r"(smem_addr(bar)), "r"(parity), "n"(kWaitSpins)
            : "memory");
        if (left == 0) {
            ok = false;
            atomicOr(status, LC_DEV_WAIT_TIMEOUT);
        }
    }
};

// The two warps of a lane quarter meet (named barriers 1..4; the id an immediate),
// the second form telling all 64 threads whether any of them said `yes`.
__device__ __forceinline__ void pa_meet(int quarter) {
    switch (quarter) {
    case 0: asm volatile("bar.sync 1, 64;\n" ::: "memory"); break;
    case 1: asm volatile("bar.sync 2, 64;\n" ::: "memory"); break;
    case 2: asm volatile("bar.sync 3, 64;\n" ::: "memory"); break;
    default: asm volatile("bar.sync 4, 64;\n" ::: "memory"); break;
    }
}
__device__ __forceinline__ bool pa_meet_any(int quarter, bool yes) {
    uint32_t any;
#define LC_MEET(ID)                                                                                      \
    asm volatile("{\n .reg .pred p, q;\n setp.ne.u32 p, %1, 0;\n bar.red.or.pred q, " #ID               \
                 ", 64, p;\n selp.u32 %0, 1, 0, q;\n}\n"                                                \
                 : "=r"(any)                                                                             \
                 : "r"((uint32_t)yes)                                                                    \
                 : "memory")
    switch (quarter) {
    case 0: LC_MEET(1); break;
    case 1: LC_MEET(2); break;
    case 2: LC_MEET(3); break;
    default: LC_MEET(4); break;
    }
#undef LC_MEET
    return any != 0;
}

// Items beyond a CTA's own: a resident CTA takes over CTAs of the grid that have
// not been launched (cluster launch control), so long and short items even out
// without a counter in memory.  Asked for one item ahead, by the load thread; an
// answer holds the taken CTA's index, or that none was left.
struct PaSched {
    unsigned char *at;  // answer, then a barrier
    uint32_t got = 0;
    __device__ __forceinline__ uint64_t *bar() { return reinterpret_cast<uint64_t *>(at + 16); }
    __device__ __forceinline__ void ask() {
        mbar_expect_tx(bar(), 16);
        asm volatile(
            "clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];\n" ::"r"(
                smem_addr(at)),
            "r"(smem_addr(bar()))
            : "memory");
    }
    __device__ __forceinline__ int next(PaWait &wait) {  // the next item, -1 if there is none
        wait(bar(), got++ & 1);
        if (!wait.ok) return -1;
        int w;
        asm volatile(
            "{\n .reg .b128 h;\n .reg .pred p;\n mov.u32 %0, -1;\n ld.shared.b128 h, [%1];\n"
            " clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\n"
            " @p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, h;\n}\n"
            : "=&r"(w)
            : "r"(smem_addr(at))
            : "memory");
        fence_proxy_async_smem();  // read before the next answer is written there
        return w;
    }
};

// Jobs in shared memory, from the load thread to the other warps: two slots, each
// filled once and released by the softmax warps and those of V and the products.
struct PaJobs {
    PaJob *slot;
    uint64_t *bar;  // full[2], empty[2]
    uint32_t k = 0;
    __device__ __forceinline__ void put(PaWait &wait, const PaJob &j) {
        if (k >= 2) wait(bar + 2 + (k & 1), ((k >> 1) - 1) & 1);
        if (!wait.ok) return;
        slot[k & 1] = j;
        mbar_arrive(bar + (k & 1));
        k++;
    }
    __device__ __forceinline__ const PaJob &get(PaWait &wait) {  // a whole warp: its lanes agree on wait.ok
        wait(bar + (k & 1), (k >> 1) & 1);
        wait.ok = __all_sync(0xffffffffu, wait.ok);
        return slot[k & 1];
    }
    __device__ __forceinline__ void release(int lane) {
        __syncwarp();
        if (lane == 0) mbar_arrive(bar + 2 + (k & 1));
        k++;
    }
};

__device__ __forceinline__ void tma_load_3d_plain(uint32_t dst, const CUtensorMap *tm, int x, int y, int z,
                                                  uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], "
        "[%5];\n" ::"r"(dst),
        "l"(tm), "r"(x), "r"(y), "r"(z), "r"(bar)
        : "memory");
}

// MN-major operand with the 128-byte swizzle: 64 MN elements (128 bytes) a row,
// one row per K, groups of 8 K 1024 bytes apart (SBO), the next 64 MN elements
// `mn_stride` bytes on (LBO).
__device__ __forceinline__ uint64_t pa_desc_mn(uint32_t saddr, uint32_t mn_stride) {
    uint64_t d = 0;
    d |= (uint64_t)((saddr >> 4) & 0x3FFFu);
    d |= (uint64_t)((mn_stride >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)(1024u >> 4) << 32;
    d |= (uint64_t)1u << 46;
    d |= (uint64_t)2u << 61;
    return d;
}

template <class T>
__host__ __device__ constexpr uint32_t pa_idesc(int n, bool b_mn) {
    constexpr uint32_t bf = sizeof(T) == 2 && !std::is_same<T, __half>::value ? 1u : 0u;
    return umma_idesc_f16(128, n) | (bf << 7) | (bf << 10) | (b_mn ? 1u << 16 : 0u);
}

// 32 consecutive TMEM columns of this thread's lane (complete after tmem_ld_wait).
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,"
        "%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];\n"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 32; i++) v[i] = __uint_as_float(r[i]);
}

__device__ __forceinline__ void tmem_ld8(uint32_t taddr, float (&v)[8]) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float (&v)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(taddr),
                 "r"(__float_as_uint(v[0])), "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])),
                 "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])), "r"(__float_as_uint(v[5])),
                 "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
                 : "memory");
}
__device__ __forceinline__ float2 fadd2(float2 a, float2 b) {
    float2 d;
    asm("{\n .reg .b64 ra, rb, rd;\n mov.b64 ra, {%2, %3};\n mov.b64 rb, {%4, %5};\n"
        " add.rn.f32x2 rd, ra, rb;\n mov.b64 {%0, %1}, rd;\n}\n"
        : "=f"(d.x), "=f"(d.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

// 2^x to about 2 ulp, 0 below the normal range.
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// (a, b) as a pair of T, and what that lost.
template <class T>
__device__ __forceinline__ uint32_t pa_pack(float a, float b, float &la, float &lb);
template <>
__device__ __forceinline__ uint32_t pa_pack<__half>(float a, float b, float &la, float &lb) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const float2 d = fadd2(make_float2(a, b), make_float2(-f.x, -f.y));
    la = d.x, lb = d.y;
    return *reinterpret_cast<const uint32_t *>(&h);
}
template <>
__device__ __forceinline__ uint32_t pa_pack<__nv_bfloat16>(float a, float b, float &la, float &lb) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    const float2 d = fadd2(make_float2(a, b), make_float2(-f.x, -f.y));
    la = d.x, lb = d.y;
    return *reinterpret_cast<const uint32_t *>(&h);
}

// 4 consecutive outputs.
__device__ __forceinline__ void pa_store4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
template <class T>
__device__ __forceinline__ void pa_store4(T *p, float4 v) {
    float l;
    uint2 u;
    u.x = pa_pack<T>(v.x, v.y, l, l), u.y = pa_pack<T>(v.z, v.w, l, l);
    *reinterpret_cast<uint2 *>(p) = u;
}

__device__ __forceinline__ void pa_store16(float *p, const float (&v)[16]) {
#pragma unroll
    for (int e = 0; e < 16; e += 4) pa_store4(p + e, make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]));
}
template <class T>
__device__ __forceinline__ void pa_store16(T *p, const float (&v)[16]) {
    float l;
#pragma unroll
    for (int e = 0; e < 16; e += 8)
        *reinterpret_cast<uint4 *>(p + e) =
            make_uint4(pa_pack<T>(v[e], v[e + 1], l, l), pa_pack<T>(v[e + 2], v[e + 3], l, l),
                       pa_pack<T>(v[e + 4], v[e + 5], l, l), pa_pack<T>(v[e + 6], v[e + 7], l, l));
}

template <class T, class TO, int HD>
__global__ void __launch_bounds__(kPaThreads, 2)
    prefix_attn_kernel(const __grid_constant__ PaMaps maps, const __grid_constant__ PaArgs a) {
    using L = PaSmem<HD>;
    // Planes of P: 1, or for f32 outputs as many as hold 22 bits or more (of f16 weights
    // above 2^-10 of the row's largest; below, to 2^-32 of that one)
    constexpr int kPlanes = !std::is_same<TO, float>::value ? 1 : std::is_same<T, __half>::value ? 2 : 3;
    // The reference of a row's weights lies 2^kShift below its maximum.  The planes of f16
    // weights end at its subnormals' spacing, 2^-24: with weights about 2^7 (below 2^15,
    // see where the reference moves) that is 2^-31 of the largest (f32 outputs of 300 rows
    // with a first key 14 nats above 5299 others: 2.5e-6 off, 1.8e-5 with weights about 1;
    // no difference in time).  bf16 has the exponents of f32.
    constexpr float kShift = std::is_same<T, __half>::value ? 7.f : 0.f;
    // TMEM columns of S: two stages of 64; a warp's planes of 16 columns overwrite its
    // own 32 scores, and the third, where there is one, takes the second stage's place
    constexpr int kStages = kPlanes < 3 ? 2 : 1;
    // Tiles whose products are summed in TMEM.  The tensor cores' f32 sums drop what lies
    // below the last bit, always downwards, so for f32 outputs O is added to a sum in
    // memory after that many (998 rows of 8/8 heads of 128 on 5884 + 431 bf16 keys: 9.6e-7
    // off and 131 us; with an item's tiles in one sum 5.2e-6 and 113 us)
    constexpr int kRun = kPlanes > 1 ? 4 : 1 << 30;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    unsigned char *smem = smem_raw + ((1024u - (smem_addr(smem_raw) & 1023u)) & 1023u);
    uint64_t *bar = reinterpret_cast<uint64_t *>(smem + L::kBar);
    // two of each, for the tiles of either parity
    uint64_t *k_full = bar, *v_full = bar + 2, *s_full = bar + 4, *p_ready = bar + 6, *pv_done = bar + 8;
    uint32_t *tslot = reinterpret_cast<uint32_t *>(bar + 14);
    const uint32_t sbase = smem_addr(smem);
    PaSched sched{smem + L::kSched};
    PaJobs jobs{reinterpret_cast<PaJob *>(smem + L::kJobs), bar + 10};
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

    PaItem next;
    if (threadIdx.x == 32 * kPaLoadWarp) prefetch_tensormap(&maps.q);
    if (threadIdx.x == 0) {
        mbar_init(sched.bar(), 1);
        for (int k = 0; k < 2; k++) {
            mbar_init(k_full + k, 1);
            mbar_init(v_full + k, 1);
            mbar_init(s_full + k, 1);
            mbar_init(p_ready + k, 8);
            mbar_init(pv_done + k, 1);
            mbar_init(jobs.bar + k, 1);
            mbar_init(jobs.bar + 2 + k, 11);
        }
        mbar_init_fence();
    }
    // The kernel before this one, whose end the launch and the lines above need not wait for.
    // Its CTAs may still have to allocate their TMEM: nothing is held of that before.
    griddep_wait();
    if (threadIdx.x == 32 * kPaLoadWarp) next = pa_item_begin(a, blockIdx.x);
    if (warp == kPaMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(tslot)),
                     "r"(kPaTmemCols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        tc_fence_before();
    }
    __syncthreads();
    tc_fence_after();
    const uint32_t tbase = *tslot;
    PaWait wait{a.status};
    // Tile `it` counts on through the CTA's jobs; its stage is it & 1, and each barrier
    // of that stage completes once for it: the phase (it >> 1) & 1.
    uint32_t it = 0;
    auto tile_done = [&](uint64_t *b, uint32_t t) { wait(b + (t & 1), (t >> 1) & 1); };
    auto load_rows = [&](uint32_t slot, const PaJob &j, int key, int nk, bool own, int kv, uint64_t *b, uint32_t more) {
        const bool full = nk > kPaHalf;
        mbar_expect_tx(b, (full ? kPaKeys : kPaHalf) * HD * 2 + more);
#pragma unroll
        for (int c = 0; c < HD / 64; c++)
            tma_load_3d_plain(sbase + slot + c * kPaKvPlane, &maps.kv[full][own][kv], j.hk * HD + 64 * c, key,
                              own ? j.seq : 0, smem_addr(b));
    };

    if (warp == kPaLoadWarp) {  // ---- work, Q and K
        if (lane == 0) {
            while (true) {
                pa_item_finish(a, next);
                bool asked = false;
#pragma unroll 1
                for (int at = next.t; at < next.count && wait.ok; at += next.t_step) {
                    const PaJob j = pa_job(a, next, at);
                    if (j.n == 0 && !j.direct && j.count * a.group <= 32) {  // nothing visible: the states here
                        const size_t blk = (size_t)(j.split * a.n_kv + j.hk) * a.row_blocks;
                        for (int r = 0; r < j.count * a.group; r++)
                            a.ml_part[blk * 32 + j.first * a.group + r] = make_float2(-INFINITY, 0.f);
                        continue;
                    }
                    jobs.put(wait, j);
#pragma unroll 1
                    for (int i = 0; i < j.n && wait.ok; i++, it++) {
                        // The next item is asked for four tiles before this one's end (not sooner:
                        // an item taken early would wait behind this one while other CTAs run dry).
                        if (!asked && i >= j.n - 4 && at + next.t_step >= next.count) sched.ask(), asked = true;
                        int key, nk;
                        bool own;
                        j.tile(i, key, nk, own);
                        // K's stage is free once the scores of two tiles ago are formed, Q's place
                        // once the last job's all are
                        if (it >= 2) tile_done(s_full, it - 2);
                        uint32_t q_bytes = 0;
                        if (i == 0) {
                            if (it) tile_done(s_full, it - 1);
                            if (!wait.ok) break;
                            const int qb = (j.count + a.box_toks - 1) / a.box_toks, q_rows = a.box_toks * a.group;
                            q_bytes = qb * q_rows * HD * 2;
#pragma unroll 1
                            for (int r = 0; r < qb; r++)
#pragma unroll
                                for (int c = 0; c < HD / 64; c++)
                                    tma_load_3d_plain(sbase + L::kQ + c * kPaPlane + r * q_rows * 128, &maps.q, 64 * c,
                                                      j.hk * a.group, j.first + r * a.box_toks,
                                                      smem_addr(k_full + (it & 1)));
                        }
                        if (!wait.ok) break;
                        load_rows(L::kK + (it & 1) * L::kTile, j, key, nk, own, 0, k_full + (it & 1), q_bytes);
                    }
                }
                if (!asked) sched.ask();
                const int w = sched.next(wait);
                if (w < 0) break;
                next = pa_item_begin(a, w);
            }
            // Nothing is left to take over: the merge kernel may be scheduled once every CTA is
            // here (not from the start: its waiting CTAs kept SMs from this kernel's)
            griddep_launch_dependents();
            PaJob last = {};
            last.n = -1;
            jobs.put(wait, last);
            if (!wait.ok) {  // copies of this CTA still in flight, and the last answer
                for (uint32_t t = it > 2 ? it - 2 : 0; t <= it; t++) mbar_wait(k_full + (t & 1), (t >> 1) & 1);
                mbar_wait(sched.bar(), (sched.got - 1) & 1);
            }
        }
    } else if (warp == kPaValueWarp) {  // ---- V
#pragma unroll 1
        while (wait.ok) {
            const PaJob &j = jobs.get(wait);
            const int n = wait.ok ? j.n : -1;
            if (n < 0) break;
            if (lane == 0) {
#pragma unroll 1
                for (int i = 0; i < n && wait.ok; i++) {
                    const uint32_t t = it + i;
                    int key, nk;
                    bool own;
                    j.tile(i, key, nk, own);
                    if (t >= 2) tile_done(pv_done, t - 2);
                    if (wait.ok) load_rows(L::kV + (t & 1) * L::kTile, j, key, nk, own, 1, v_full + (t & 1), 0);
                }
            }
            it += n;
            wait.ok = __all_sync(0xffffffffu, wait.ok);
            if (wait.ok) jobs.release(lane);
        }
        if (lane == 0 && !wait.ok)
            for (uint32_t t = it > 2 ? it - 2 : 0; t <= it; t++) mbar_wait(v_full + (t & 1), (t >> 1) & 1);
    } else if (warp == kPaScoreWarp) {  // ---- scores
#pragma unroll 1
        while (wait.ok) {
            const PaJob &j = jobs.get(wait);
            const int n = wait.ok ? j.n : -1;
            if (n < 0) break;
#pragma unroll 1
            for (int i = 0; i < n && wait.ok; i++, it++) {
                // S's stage is free once the products with the weights that took its place are done
                if (it >= kStages) tile_done(pv_done, it - kStages);
                tile_done(k_full, it);
                wait.ok = __all_sync(0xffffffffu, wait.ok);
                tc_fence_after();
                // unrolled: a product runs 50 cycles, and a loop around one takes 88 to issue it
                if (lane == 0 && wait.ok) {
                    const uint64_t qd = umma_desc_sw128(sbase + L::kQ);
                    const uint64_t kd = umma_desc_sw128(sbase + L::kK + (it & 1) * L::kTile);
                    const uint32_t d = tbase + kPaColS + (it & (kStages - 1)) * kPaKeys;
#pragma unroll
                    for (int s = 0; s < HD / 16; s++)
                        umma_f16_ss(d, qd + (((s >> 2) * kPaPlane + (s & 3) * 32) >> 4),
                                    kd + (((s >> 2) * kPaKvPlane + (s & 3) * 32) >> 4), pa_idesc<T>(kPaKeys, false),
                                    s ? 1u : 0u);
                    umma_commit(s_full + (it & 1));
                }
                __syncwarp();
            }
            if (wait.ok) jobs.release(lane);
        }
        if (!wait.ok)  // products still under way
            for (uint32_t t = it > 2 ? it - 2 : 0; t < it; t++) mbar_wait(s_full + (t & 1), (t >> 1) & 1);
    } else if (warp == kPaMmaWarp) {  // ---- values
#pragma unroll 1
        while (wait.ok) {
            const PaJob &j = jobs.get(wait);
            const int n = wait.ok ? j.n : -1;
            if (n < 0) break;
#pragma unroll 1
            for (int i = 0; i < n && wait.ok; i++, it++) {
                int key, nk;
                bool own;
                j.tile(i, key, nk, own);
                tile_done(v_full, it);
                // keys of the tile's last 16-key step that do not exist: their P is 0,
                // and 0 times whatever lies there must not be NaN
                const uint32_t v_at = L::kV + (it & 1) * L::kTile;
                const int steps = (nk + 15) >> 4, gone = steps * 16 - nk;
                if (gone && wait.ok) {
#pragma unroll 1
                    for (int e = lane; e < gone * (HD / 8); e += 32) {
                        const int row = nk + e / (HD / 8), ch = e % (HD / 8);
                        *reinterpret_cast<uint4 *>(smem + v_at + (ch >> 3) * kPaKvPlane + row * 128 + (ch & 7) * 16) =
                            make_uint4(0, 0, 0, 0);
                    }
                    fence_proxy_async_smem();
                    __syncwarp();
                }
                tile_done(p_ready, it);
                wait.ok = __all_sync(0xffffffffu, wait.ok);
                if (!wait.ok) break;
                tc_fence_after();
                if (lane == 0) {
                    const uint64_t vd = pa_desc_mn(sbase + v_at, HD > 64 ? kPaKvPlane : 1024u);
                    const uint32_t ps = tbase + kPaColS + (it & (kStages - 1)) * kPaKeys;
                    auto step = [&](int s) {
                        const uint32_t p = ps + (s >> 1) * 32 + (s & 1) * 8;
                        const uint64_t v = vd + ((s * 2048) >> 4);
                        constexpr uint32_t id = pa_idesc<T>(HD, true);
                        umma_f16_ts(tbase + kPaColO, p, v, id, (i % kRun | s) ? 1u : 0u);
                        if constexpr (kPlanes > 1) umma_f16_ts(tbase + kPaColO, p + 16, v, id, 1u);
                        if constexpr (kPlanes > 2)
                            umma_f16_ts(tbase + kPaColO, tbase + kPaColS + 64 + 8 * s, v, id, 1u);
                    };
                    if (steps == 4) {
#pragma unroll
                        for (int s = 0; s < 4; s++) step(s);
                    } else {
#pragma unroll 1
                        for (int s = 0; s < steps; s++) step(s);
                    }
                    umma_commit(pv_done + (it & 1));
                }
                __syncwarp();
            }
            jobs.release(lane);
        }
        if (!wait.ok)  // products still under way
            for (uint32_t t = it > 2 ? it - 2 : 0; t < it; t++) mbar_wait(pv_done + (t & 1), (t >> 1) & 1);
    } else {  // ---- softmax
        // Row = TMEM lane; the two warps of a lane quarter take half of a tile's keys, and of
        // O's columns, each.  Thread pairs meet at a barrier of their two warps to agree
        // on a row's maximum.
        const int quarter = warp & 3, half = warp >> 2, row = 32 * quarter + lane;
        const uint32_t lanes = (uint32_t)(32 * quarter) << 16;
        const uint32_t ts = tbase + lanes + kPaColS, to = tbase + lanes + kPaColO + half * (HD / 2);
        float *mine = reinterpret_cast<float *>(smem + L::kRed) + half * kPaRows + row;
        const float *other = reinterpret_cast<float *>(smem + L::kRed) + (half ^ 1) * kPaRows + row;
#pragma unroll 1
        while (true) {
            const PaJob &j = jobs.get(wait);
            // a warp that gave up takes its partner along, which would wait for it
            if (pa_meet_any(quarter, !wait.ok || j.n < 0)) break;
            const int n = j.n;
            {
                const bool busy = 32 * quarter < j.count * a.group;
                float m_ref = -INFINITY;
                float2 l = make_float2(0.f, 0.f);
                // O so far, in the place of the row's state, with the maximum m_run
                float m_run = -INFINITY;
                bool run = false;
                auto state_at = [&]() {  // the row's half of its state: 4 columns are 128 floats on
                    const int gq = j.first * a.group + row;
                    const size_t blk = (size_t)(j.split * a.n_kv + j.hk) * a.row_blocks + (gq >> 5);
                    return a.o_part + blk * (32 * HD) + (gq & 31) * 4 + half * (HD * 16);
                };
                auto out_at = [&]() {  // the row's half of its result
                    const int gq = j.first * a.group + row, tok = j.first + pa_token(a, row);
                    return static_cast<TO *>(a.out) + (size_t)tok * a.ldo +
                           (size_t)(j.hk * a.group + gq - tok * a.group) * HD + half * (HD / 2);
                };
                auto add_run = [&](const float *p, float (&o)[16]) {  // 16 columns of it to those of TMEM
                    const float f = m_run == m_ref ? 1.f : exp2_fast(m_run - m_ref);
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 b = *reinterpret_cast<const float4 *>(p + e * 32);
                        o[e] += b.x * f, o[e + 1] += b.y * f, o[e + 2] += b.z * f, o[e + 3] += b.w * f;
                    }
                };
#pragma unroll 1
                for (int i = 0; i < n; i++, it++) {
                    int key, nk;
                    bool own;
                    j.tile(i, key, nk, own);
                    tile_done(s_full, it);
                    __syncwarp();
                    if (busy) {
                        const uint32_t st = ts + (it & (kStages - 1)) * kPaKeys + kPaHalf * half;
                        tc_fence_after();
                        if (kPlanes > 1 && i && i % kRun == 0) {
                            tile_done(pv_done, it - 1);
                            __syncwarp();
                            tc_fence_after();
                            const bool real = row < j.count * a.group;
                            float *part = state_at();
#pragma unroll 1
                            for (int c = 0; c < HD / 2; c += 16, part += 16 * 32) {
                                float o[16];
                                tmem_ld16(to + c, o);
                                tmem_ld_wait();
                                tmem_regs_ready(o);
                                if (real) {
                                    if (run) add_run(part, o);
#pragma unroll
                                    for (int e = 0; e < 16; e += 4)
                                        pa_store4(part + e * 32, make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]));
                                }
                                __syncwarp();
                            }
                            m_run = m_ref, run = true;
                        }
                        // keys [0, lim) of this half are visible to the row
                        int lim = nk;
                        if (own && a.causal)
                            lim = min(max(j.pos0 + j.first + pa_token(a, row) + 1 - key, 0), nk);
                        lim -= kPaHalf * half;
                        float x[kPaHalf];
                        tmem_ld32(st, x);
                        tmem_ld_wait();
                        tmem_regs_ready(x);
                        if (__any_sync(0xffffffffu, lim < kPaHalf)) {
#pragma unroll
                            for (int e = 0; e < kPaHalf; e++)
                                if (e >= lim) x[e] = -INFINITY;
                        }
                        float t0 = x[0], t1 = x[1], t2 = x[2], t3 = x[3];
#pragma unroll
                        for (int e = 4; e < kPaHalf; e += 4) {
                            t0 = fmaxf(t0, x[e]), t1 = fmaxf(t1, x[e + 1]);
                            t2 = fmaxf(t2, x[e + 2]), t3 = fmaxf(t3, x[e + 3]);
                        }
                        const float top = fmaxf(fmaxf(t0, t1), fmaxf(t2, t3)) * a.scale_log2;
                        // The reference moves, and O is rescaled, only when a score is more than
                        // 2^8 above the last maximum: weights up to 2^(8 + kShift) are as exact,
                        // and fit f16
                        if (pa_meet_any(quarter, i == 0 || top > m_ref + (8.f + kShift))) {
                            *mine = top;
                            pa_meet(quarter);
                            const float m_new = fmaxf(m_ref, fmaxf(top, *other) - kShift);
                            const float f = m_new == m_ref ? 1.f : exp2_fast(m_ref - m_new);
                            if (i % kRun) {
                                tile_done(pv_done, it - 1);
                                __syncwarp();
                                tc_fence_after();
#pragma unroll 1
                                for (int c = 0; c < HD / 16; c++) {
                                    float o[8];
                                    tmem_ld8(to + 8 * c, o);
                                    tmem_ld_wait();
                                    tmem_regs_ready(o);
#pragma unroll
                                    for (int e = 0; e < 8; e++) o[e] *= f;
                                    tmem_st8(to + 8 * c, o);
                                }
                            }
                            l.x *= f, l.y *= f;
                            m_ref = m_new;
                        }
                        const float neg = m_ref == -INFINITY ? 0.f : -m_ref;
                        const float2 sc = make_float2(a.scale_log2, a.scale_log2), ng = make_float2(neg, neg);
                        // P as pairs over the first half of the warp's own scores, what the rounding
                        // lost over the second, and what that lost in the other stage
                        if (nk > kPaHalf * half) {  // the products stop at nk
                            uint32_t p[kPlanes][16];
#pragma unroll
                            for (int e = 0; e < 16; e++) {
                                const float2 t = ffma2(make_float2(x[2 * e], x[2 * e + 1]), sc, ng);
                                float2 w = make_float2(exp2_fast(t.x), exp2_fast(t.y));
                                l = fadd2(l, w);
#pragma unroll
                                for (int k = 0; k < kPlanes; k++) p[k][e] = pa_pack<T>(w.x, w.y, w.x, w.y);
                            }
                            tmem_st16(st, p[0]);
                            if constexpr (kPlanes > 1) tmem_st16(st + 16, p[1]);
                            if constexpr (kPlanes > 2) tmem_st16(ts + 64 + 16 * half, p[2]);
                        }
                        tmem_st_wait();
                        tc_fence_before();
                        __syncwarp();
                    }
                    if (lane == 0) mbar_arrive(p_ready + (it & 1));
                }
                if (busy) {
                    mine[2 * kPaRows] = l.x + l.y;
                    pa_meet(quarter);
                    const float sum = l.x + l.y + other[2 * kPaRows];
                    const bool real = row < j.count * a.group;
                    if (n) {
                        tile_done(pv_done, it - 1);
                        __syncwarp();
                        tc_fence_after();
                    }
                    const size_t blk = (size_t)(j.split * a.n_kv + j.hk) * a.row_blocks;
                    float2 *ml = a.ml_part + blk * 32 + j.first * a.group + row;
                    if (j.direct) {
                        if (real && half == 0 && a.merge) *ml = make_float2(0.f, -1.f);
                        const bool none = n == 0 || sum == 0.f;  // no visible key: 0
                        const float f = none ? 0.f : 1.f / sum;
                        const float *part = kPlanes > 1 && run ? state_at() : nullptr;
                        TO *out = out_at();
#pragma unroll 1
                        for (int c = 0; c < HD / 2; c += 16, out += 16, part += 16 * 32) {
                            float o[16];
                            tmem_ld16(to + c, o);  // without a tile whatever is there, and not used
                            tmem_ld_wait();
                            tmem_regs_ready(o);
                            if (real) {
                                if (kPlanes > 1 && run) add_run(part, o);
#pragma unroll
                                for (int e = 0; e < 16; e++) o[e] = none ? 0.f : o[e] * f;
                                pa_store16(out, o);
                            }
                            __syncwarp();
                        }
                    } else {
                        if (real && half == 0) *ml = make_float2(m_ref, sum);
                        float *part = state_at();
#pragma unroll 1
                        for (int c = 0; c < HD / 2 && n; c += 16, part += 16 * 32) {
                            float o[16];
                            tmem_ld16(to + c, o);
                            tmem_ld_wait();
                            tmem_regs_ready(o);
                            if (real) {
                                if (kPlanes > 1 && run) add_run(part, o);
#pragma unroll
                                for (int e = 0; e < 16; e += 4)
                                    pa_store4(part + e * 32, make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]));
                            }
                            __syncwarp();
                        }
                    }
                    tc_fence_before();  // O has been read before the next job's products overwrite it
                }
            }
            jobs.release(lane);
        }
    }
    __syncthreads();
    if (warp == kPaMmaWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tbase), "r"(kPaTmemCols)
                     : "memory");
    }
}

// out = sum_s 2^(m_s - M) O_s / sum_s 2^(m_s - M) l_s over the splits that saw a
// key, 0 if none did.  One warp per 32 rows of a KV head and 8 dims, a lane per
// row: the states' pieces are read 512 bytes at a time, 8 splits in flight; or the four
// warps of a block, a share of the splits each.
// Rows outside [seq_start[0], seq_start[n_seqs]) belong to no sequence and stay
// as they are.
template <class TO, int HD>
__global__ void __launch_bounds__(128) prefix_attn_merge_kernel(const __grid_constant__ PaArgs a) {
    constexpr int kPer = HD / 8, kBatch = 8;  // warps of a block of rows; splits in flight
    griddep_wait();  // the partial states
    __shared__ float shares[3][10][32];
    const int ways = a.merge_ways, way = threadIdx.x / 32 & (ways - 1);
    const int w = (blockIdx.x * 4 + (threadIdx.x >> 5)) / ways, lane = threadIdx.x & 31;
    const int piece = w % kPer, blk = w / kPer % a.row_blocks, hk = w / kPer / a.row_blocks;
    const int gq = blk * 32 + lane, tok = gq / a.group;
    if (hk >= a.n_kv || gq >= a.rows * a.group) return;
    const int first = a.seq_start[0], last = a.seq_start[a.n_seqs];  // (looked at below, with the states)
    const int splits = a.prefix_splits + a.seq_splits;
    const size_t stride = (size_t)a.n_kv * a.row_blocks;  // blocks of a split
    const size_t at = (size_t)hk * a.row_blocks + blk;
    const float2 *ml = a.ml_part + at * 32 + lane;
    const float4 *op = reinterpret_cast<const float4 *>(a.o_part + at * (32 * HD)) + piece * 64 + lane;
    // rows written already (without direct items not worth a round trip of its own)
    if (a.direct && ml[0].y < 0.f) return;
    // a batch's (m, l) and pieces in one round trip; the sums move to its maximum
    float M = -INFINITY, sum = 0.f, o[8] = {};
    const int share = (splits + ways - 1) / ways, end = min(splits, (way + 1) * share);
#pragma unroll 1
    for (int s0 = way * share; s0 < end; s0 += kBatch) {
        float2 st[kBatch];
        float4 x[kBatch][2];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            const size_t s = min(s0 + u, splits - 1);
            st[u] = ml[s * stride * 32];
            x[u][0] = op[s * stride * (8 * HD)];
            x[u][1] = op[s * stride * (8 * HD) + 32];
        }
        if (tok < first || tok >= last) return;  // of no sequence
        float top = M;
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            if (s0 + u >= end) st[u].y = 0.f;
            if (st[u].y != 0.f) top = fmaxf(top, st[u].x);
        }
        if (top > M) {
            const float f = exp2f(M - top);
            sum *= f;
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] *= f;
            M = top;
        }
#pragma unroll
        for (int u = 0; u < kBatch; u++)
            if (st[u].y != 0.f) {  // O of a state that saw no key may be unwritten
                const float f = exp2f(st[u].x - M);
                sum += st[u].y * f;
                o[0] += x[u][0].x * f, o[1] += x[u][0].y * f, o[2] += x[u][0].z * f, o[3] += x[u][0].w * f;
                o[4] += x[u][1].x * f, o[5] += x[u][1].y * f, o[6] += x[u][1].z * f, o[7] += x[u][1].w * f;
            }
    }
    if (tok < first || tok >= last) return;
    if (ways > 1) {
        if (way) {
            float *to = &shares[way - 1][0][lane];
            to[0] = M, to[32] = sum;
#pragma unroll
            for (int e = 0; e < 8; e++) to[(2 + e) * 32] = o[e];
        }
        __syncthreads();
        if (way) return;
        float top = M;
        for (int k = 0; k < ways - 1; k++) top = fmaxf(top, shares[k][0][lane]);
        const float f = sum != 0.f ? exp2f(M - top) : 0.f;
        sum *= f;
#pragma unroll
        for (int e = 0; e < 8; e++) o[e] *= f;
        for (int k = 0; k < ways - 1; k++) {
            const float *from = &shares[k][0][lane];
            if (from[32] == 0.f) continue;
            const float g = exp2f(from[0] - top);
            sum += from[32] * g;
#pragma unroll
            for (int e = 0; e < 8; e++) o[e] += from[(2 + e) * 32] * g;
        }
    }
    const float f = sum != 0.f ? 1.f / sum : 0.f;
    TO *out = static_cast<TO *>(a.out) + (size_t)tok * a.ldo + (size_t)(hk * a.group + gq - tok * a.group) * HD +
              8 * piece;
    pa_store4(out, make_float4(o[0] * f, o[1] * f, o[2] * f, o[3] * f));
    pa_store4(out + 4, make_float4(o[4] * f, o[5] * f, o[6] * f, o[7] * f));
}

// A tensor of dims[0] contiguous elements and strides ld[] (elements) of the
// outer dims, copied in boxes of 64 elements x box1 (x box2) in the 128-byte
// swizzle; what lies past an end reads as zero.
int pa_map(CUtensorMap *tm, const void *p, int dtype, const uint64_t (&dims)[3], const uint64_t (&ld)[2],
           uint32_t box1, uint32_t box2) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = nullptr;
    if (int s = lc_tensor_map_encoder(&enc)) return s;
    cuuint64_t d[3] = {dims[0], dims[1], dims[2]}, strides[2] = {ld[0] * 2, ld[1] * 2};
    cuuint32_t box[3] = {64, box1, box2}, es[3] = {1, 1, 1};
    const CUresult r =
        enc(tm, dtype == LC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3,
            const_cast<void *>(p), d, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    LC_REQUIRE(r == CUDA_SUCCESS, LC_ERR_CUDA, "lc_prefix_attn: cuTensorMapEncodeTiled failed (%d)", (int)r);
    return LC_OK;
}

int div_up(int64_t a, int64_t b) { return (int)((a + b - 1) / b); }

// How the work is cut into items.
void pa_plan(PaArgs &a, int num_sms, int hd, int planes) {
    const int slots = 2 * num_sms;  // CTAs resident at once
    const int64_t R = (int64_t)a.rows * a.group;
    // Tokens of a row tile: as many as fit 128 rows in whole copies of Q, which hold
    // about 32 rows and, where several make a tile, a multiple of 8 rows (the swizzle's
    // period)
    int unit = 1;
    while (unit * a.group % 8) unit *= 2;
    if (unit * a.group > kPaRows) {
        a.box_toks = a.tile_toks = kPaRows / a.group;
    } else {
        a.box_toks = unit * std::max(1, 32 / (unit * a.group));
        a.tile_toks = kPaRows / (a.box_toks * a.group) * a.box_toks;
    }
    const int tiles_all = div_up(a.rows, a.tile_toks), tiles_avg = div_up(div_up(a.rows, a.n_seqs), a.tile_toks);
    // row tiles of a sequence that run side by side (a longer one goes round again)
    a.seq_lanes = a.n_seqs == 1 ? tiles_all : std::min(tiles_all, tiles_avg > 1 ? 2 * tiles_avg : 1);
    // Splits of the key axis for `base` items of `tiles` tiles: the fewest rounds of tiles
    // over the resident CTAs (about 1 us a tile, 0.6 more for a further plane, and 2 us an
    // item), against writing and reading the states (8 bytes a picosecond), the merge's
    // launch and its round trips, 8 states each (one row of 4 heads on 10581 keys: 25 us
    // without that last part, 14 with).
    const double tile_us = 1.0 + 0.6 * (planes - 1);
    const double state_us = 2.0 * a.n_kv * div_up(R, 32) * 32 * (hd * 4 + 8) / 8e6;
    // Few rows leave warps to share their states (4 x 2 rows on 16487 keys: 15.8 us in one
    // warp, 11.0 in four); more rows fill the merge's warps by themselves (64 sequences of 32
    // heads on 8192: 47.7 us, with four 48.7).
    const bool shared_merge = a.n_kv * div_up(R, 32) * (hd / 8) <= 2 * slots;
    const double split_us = state_us + (shared_merge ? 0.03 : 0.09);
    auto splits_for = [&](int64_t base, int tiles, bool merged_anyway) {
        int best = 1;
        double best_us = 1e30;
        for (int n = 1; n <= std::min(tiles, 256); n++) {
            const int per = div_up(tiles, n);
            if (n > 1 && div_up(tiles, n - 1) == per) continue;  // the same cut with an empty split more
            const double us = (per * tile_us + 2) * div_up(base * n, slots) +
                              (n > 1 || merged_anyway ? n * split_us + 4 : 0);
            if (us < best_us) best = n, best_us = us;
        }
        return best;
    };
    // A sequence whose rows fill tiles by themselves gains nothing from sharing
    // the prefix with others: its items run over [prefix | own] in one go.
    const bool joint = a.prefix_len == 0 || a.n_seqs == 1 || R >= (int64_t)kPaRows * a.n_seqs;
    a.prefix_items = 0, a.prefix_splits = 0, a.row_tiles = 1, a.prefix_keys = kPaKeys;
    a.seq_from = joint ? 0 : a.prefix_len;
    if (!joint) {
        a.row_tiles = tiles_all;
        const int base = a.n_kv * a.row_tiles, tiles = div_up(a.prefix_len, kPaKeys);
        const int per = div_up(tiles, splits_for(base, tiles, true));
        a.prefix_keys = per * kPaKeys;
        a.prefix_splits = div_up(tiles, per);
        a.prefix_items = base * a.prefix_splits;
    }
    const int tiles = div_up(a.prefix_len + a.own_cap - a.seq_from, kPaKeys);
    a.seq_base = a.n_kv * a.n_seqs * a.seq_lanes;
    a.seq_splits = 0, a.seq_keys = kPaKeys, a.direct = 0;
    if (tiles) {
        int per;
        const int64_t real = (int64_t)a.n_kv * tiles_all;  // about so many items have rows
        if (!joint) {
            // Own parts differ in length: items of at most 8 tiles keep one long sequence from
            // being the launch's tail, unless there are many sequences to even out.
            per = div_up(tiles, splits_for(a.seq_base, tiles, true));
            if (a.seq_base < 16 * slots) per = std::min(per, 8);
        } else if (real < slots) {
            per = div_up(tiles, splits_for(real, tiles, false));
            if (per == tiles) a.direct = a.seq_base;
        } else {
            // Items over the whole axis write out directly.  Where they are little more than one
            // round of the resident CTAs, those left over for the second are split to fill it, in
            // pieces of 16 tiles or more (4 prompts of 512 tokens on 4096: 140 -> 132 us; 8 of
            // 256 on 2048, split finer, 85 -> 90).  Later rounds are even enough by themselves (16 of
            // 300 on 1000, with the rest split: 90 -> 112 us).
            const int rest = (int)(real - slots);
            const int n = real < slots * 3 / 2 ? std::min(tiles / 16, 3 * slots / (2 * std::max(rest, 1))) : 1;
            per = div_up(tiles, std::max(n, 1));
            a.direct = per == tiles ? a.seq_base : std::min<int64_t>(a.seq_base, slots);
        }
        a.seq_keys = per * kPaKeys;
        a.seq_splits = a.direct == a.seq_base ? 1 : div_up(tiles, per);
    }
    a.merge = a.direct < a.seq_base || !tiles;
    a.merge_ways = shared_merge && a.prefix_splits + a.seq_splits > 8 ? 4 : 1;
    auto div = [](int d) { return PaDiv{((1ull << 63) + d - 1) / d, d}; };
    a.by_rest = div(std::max(1, a.seq_base - a.direct));
    a.by_heads = div(a.n_kv), a.by_seqs = div(a.n_seqs), a.by_tiles = div(a.row_tiles);
}

template <class T, class TO, int HD>
int pa_launch(lc_ctx *ctx, const PaArgs &a, int items, const PaMaps &maps) {
    auto kernel = prefix_attn_kernel<T, TO, HD>;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.stream = ctx->stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (items) {
        if (int s = lc_set_smem_attr((const void *)kernel, PaSmem<HD>::kBytes)) return s;
        cfg.gridDim = dim3(items);
        cfg.blockDim = dim3(kPaThreads);
        cfg.dynamicSmemBytes = PaSmem<HD>::kBytes;
        LC_CUDA(cudaLaunchKernelEx(&cfg, kernel, maps, a));
    }
    if (a.merge) {
        cfg.gridDim = dim3(div_up((int64_t)a.n_kv * a.row_blocks * (HD / 8) * a.merge_ways, 4));
        cfg.blockDim = dim3(128);
        cfg.dynamicSmemBytes = 0;
        LC_CUDA(cudaLaunchKernelEx(&cfg, prefix_attn_merge_kernel<TO, HD>, a));
    }
    return lc_after_launch(ctx, "lc_prefix_attn");
}

template <class T>
int pa_types(lc_ctx *ctx, int out_dtype, uint32_t hd, const PaArgs &a, int items, const PaMaps &maps) {
    if (out_dtype == LC_F32)
        return hd == 128 ? pa_launch<T, float, 128>(ctx, a, items, maps) : pa_launch<T, float, 64>(ctx, a, items, maps);
    return hd == 128 ? pa_launch<T, T, 128>(ctx, a, items, maps) : pa_launch<T, T, 64>(ctx, a, items, maps);
}

}  // namespace

extern "C" int lc_prefix_attn(lc_ctx *ctx, int dtype, int out_dtype, const void *q, uint64_t ldq,
                              const lc_prefix_kv *kv, void *out, uint64_t ldo, uint32_t rows, uint32_t n_q_heads,
                              uint32_t n_kv_heads, uint32_t head_dim, float scale, uint32_t causal) {
    LC_REQUIRE(ctx, LC_ERR_INVALID, "lc_prefix_attn: null ctx");
    LC_REQUIRE(dtype == LC_F16 || dtype == LC_BF16, LC_ERR_UNSUPPORTED,
               "lc_prefix_attn: type %d (q, k and v are LC_F16 or LC_BF16)", dtype);
    LC_REQUIRE(out_dtype == dtype || out_dtype == LC_F32, LC_ERR_UNSUPPORTED,
               "lc_prefix_attn: output type %d (the input's or LC_F32)", out_dtype);
    LC_REQUIRE(head_dim == 64 || head_dim == 128, LC_ERR_UNSUPPORTED, "lc_prefix_attn: head_dim %u (64 or 128)",
               head_dim);
    LC_REQUIRE(n_kv_heads > 0 && n_q_heads % n_kv_heads == 0, LC_ERR_UNSUPPORTED,
               "lc_prefix_attn: n_q_heads %u must be a multiple of n_kv_heads %u", n_q_heads, n_kv_heads);
    LC_REQUIRE(n_q_heads / n_kv_heads <= (uint32_t)kPaRows, LC_ERR_UNSUPPORTED,
               "lc_prefix_attn: %u query heads to a KV head (at most %d)", n_q_heads / n_kv_heads, kPaRows);
    const float scale_log2 = scale * 1.44269504088896340736f;
    LC_REQUIRE(scale >= FLT_MIN && scale_log2 < INFINITY, LC_ERR_INVALID,
               "lc_prefix_attn: scale %g must be a positive normal number", scale);
    if (rows == 0 || n_q_heads == 0) return LC_OK;
    LC_REQUIRE(kv, LC_ERR_INVALID, "lc_prefix_attn: null kv");
    if (kv->n_seqs == 0) return LC_OK;
    LC_REQUIRE(q && out && kv->seq_start && (!kv->prefix_len || (kv->k_prefix && kv->v_prefix)) &&
                   (!kv->own_cap || (kv->k_own && kv->v_own && kv->own_len)),
               LC_ERR_INVALID, "lc_prefix_attn: null pointer");
    LC_REQUIRE(kv->n_seqs <= (1u << 20), LC_ERR_UNSUPPORTED, "lc_prefix_attn: %u sequences", kv->n_seqs);
    const uint64_t wq = (uint64_t)n_q_heads * head_dim, wk = (uint64_t)n_kv_heads * head_dim;
    LC_REQUIRE((uint64_t)rows * n_q_heads <= (1u << 29) && wq < (1u << 24), LC_ERR_UNSUPPORTED,
               "lc_prefix_attn: %u rows of %u heads", rows, n_q_heads);
    LC_REQUIRE((uint64_t)n_kv_heads * (rows + 2ull * kv->n_seqs) <= (1u << 29), LC_ERR_UNSUPPORTED,
               "lc_prefix_attn: %u sequences of %u KV heads", kv->n_seqs, n_kv_heads);
    LC_REQUIRE((uint64_t)kv->prefix_len + kv->own_cap <= kPaMaxLen, LC_ERR_UNSUPPORTED,
               "lc_prefix_attn: %u + %u keys", kv->prefix_len, kv->own_cap);
    if (!ldq) ldq = wq;
    if (!ldo) ldo = wq;
    const uint64_t ldp = kv->ld_prefix ? kv->ld_prefix : wk, ldw = kv->ld_own ? kv->ld_own : wk;
    const uint64_t seq_ld = kv->own_stride ? kv->own_stride : ldw * kv->own_cap;
    LC_REQUIRE(ldq >= wq && ldo >= wq && ldp >= wk && ldw >= wk, LC_ERR_INVALID,
               "lc_prefix_attn: a row stride is shorter than its row");
    LC_REQUIRE(!kv->own_cap || kv->n_seqs == 1 || seq_ld >= (kv->own_cap - 1) * ldw + wk, LC_ERR_INVALID,
               "lc_prefix_attn: own_stride is shorter than own_cap rows");
    // strides of a tensor map are below 2^40 bytes
    LC_REQUIRE(ldq < (1ull << 38) && ldo < (1ull << 38) && ldp < (1ull << 38) && ldw < (1ull << 38) &&
                   seq_ld < (1ull << 39),
               LC_ERR_INVALID, "lc_prefix_attn: stride too large");
    const uint64_t out_vec = out_dtype == LC_F32 ? 4 : 8;
    LC_REQUIRE((((uintptr_t)q | (uintptr_t)out) & 15) == 0 && ldq % 8 == 0 && ldo % out_vec == 0 &&
                   (!kv->prefix_len ||
                    ((((uintptr_t)kv->k_prefix | (uintptr_t)kv->v_prefix) & 15) == 0 && ldp % 8 == 0)) &&
                   (!kv->own_cap || ((((uintptr_t)kv->k_own | (uintptr_t)kv->v_own) & 15) == 0 && ldw % 8 == 0 &&
                                     seq_ld % 8 == 0)) &&
                   (((uintptr_t)kv->seq_start | (uintptr_t)kv->own_len) & 3) == 0,
               LC_ERR_INVALID, "lc_prefix_attn: rows must start on 16-byte boundaries");
    const uint64_t bo = out_dtype == LC_F32 ? 4 : 2;
    const LcRows out_rows = {out, ldo * bo, wq * bo, rows};
    LC_REQUIRE(!lc_rows_meet(q, ldq * 2, wq * 2, out, ldo * bo, wq * bo, rows), LC_ERR_INVALID,
               "lc_prefix_attn: out overlaps q");
    for (const void *p : {kv->k_prefix, kv->v_prefix})
        LC_REQUIRE(!lc_rows_meet({p, ldp * 2, wk * 2, kv->prefix_len}, out_rows), LC_ERR_INVALID,
                   "lc_prefix_attn: out overlaps the prefix");
    for (const void *p : {kv->k_own, kv->v_own}) {
        // the sequences' extents against out's, then (columns of one buffer) row by row
        const uint64_t extent = kv->own_cap ? ((kv->own_cap - 1) * ldw + wk) * 2 : 0;
        if (!lc_rows_meet({p, seq_ld * 2, extent, kv->n_seqs}, {out, 0, (rows - 1) * ldo * bo + wq * bo, 1})) continue;
        for (uint32_t i = 0; i < kv->n_seqs; i++)
            LC_REQUIRE(!lc_rows_meet({(const char *)p + i * seq_ld * 2, ldw * 2, wk * 2, kv->own_cap}, out_rows),
                       LC_ERR_INVALID, "lc_prefix_attn: out overlaps the own rows of sequence %u", i);
    }
    LC_REQUIRE(!lc_rows_meet({kv->seq_start, 0, 4 * (kv->n_seqs + 1ull), 1}, out_rows) &&
                   (!kv->own_cap || !lc_rows_meet({kv->own_len, 0, 4ull * kv->n_seqs, 1}, out_rows)),
               LC_ERR_INVALID, "lc_prefix_attn: out overlaps lengths or starts");
    if (int s = lc_use_device(ctx)) return s;

    PaArgs a = {};
    a.q = q, a.out = out, a.ldq = ldq, a.ldo = ldo;
    a.rows = (int)rows, a.n_q = (int)n_q_heads, a.n_kv = (int)n_kv_heads, a.group = a.n_q / a.n_kv;
    a.prefix_len = (int)kv->prefix_len, a.own_cap = (int)kv->own_cap, a.n_seqs = (int)kv->n_seqs;
    a.own_len = kv->own_cap ? kv->own_len : nullptr, a.seq_start = kv->seq_start;
    a.group_inv = (65536 + a.group - 1) / a.group;
    a.scale_log2 = scale_log2;
    a.causal = causal != 0;
    a.status = ctx->dev_status;
    pa_plan(a, ctx->num_sms, (int)head_dim, out_dtype != LC_F32 ? 1 : dtype == LC_F16 ? 2 : 3);
    const int64_t items = a.prefix_items + a.direct + (int64_t)(a.seq_base - a.direct) * a.seq_splits;
    // (a CTA that skips empty items must not keep its other warps waiting past their bound)
    LC_REQUIRE(items <= kPaMaxItems, LC_ERR_UNSUPPORTED, "lc_prefix_attn: %lld work items", (long long)items);
    if (a.merge || out_dtype == LC_F32) {  // (items that write out sum long rows there too)
        a.row_blocks = div_up((int64_t)rows * a.group, 32);
        const size_t states = (size_t)(a.prefix_splits + a.seq_splits) * a.n_kv * a.row_blocks * 32;
        void *scr = nullptr;
        if (int s = lc_scratch_here(ctx, states * (head_dim * 4 + 8) + 256, &scr)) return s;
        a.ml_part = (float2 *)scr;
        a.o_part = (float *)((char *)scr + ((states * 8 + 255) & ~(size_t)255));
    }
    PaMaps maps = {};
    for (int full = 0; full < 2; full++) {
        const uint32_t box = full ? kPaKeys : kPaHalf;
        if (a.prefix_len) {
            const uint64_t dims[3] = {wk, kv->prefix_len, 1}, ld[2] = {ldp, ldp};
            if (int s = pa_map(&maps.kv[full][0][0], kv->k_prefix, dtype, dims, ld, box, 1)) return s;
            if (int s = pa_map(&maps.kv[full][0][1], kv->v_prefix, dtype, dims, ld, box, 1)) return s;
        }
        if (a.own_cap) {
            const uint64_t dims[3] = {wk, kv->own_cap, kv->n_seqs}, ld[2] = {ldw, seq_ld};
            if (int s = pa_map(&maps.kv[full][1][0], kv->k_own, dtype, dims, ld, box, 1)) return s;
            if (int s = pa_map(&maps.kv[full][1][1], kv->v_own, dtype, dims, ld, box, 1)) return s;
        }
    }
    {  // a box of Q is the heads of a group for box_toks tokens, in row order
        const uint64_t dims[3] = {head_dim, n_q_heads, rows}, ld[2] = {head_dim, ldq};
        if (int s = pa_map(&maps.q, q, dtype, dims, ld, a.group, a.box_toks)) return s;
    }
    const int status = dtype == LC_F16 ? pa_types<__half>(ctx, out_dtype, head_dim, a, (int)items, maps)
                                       : pa_types<__nv_bfloat16>(ctx, out_dtype, head_dim, a, (int)items, maps);
    if (status == LC_OK) ctx->stream_scratch->called = true;
    return status;
}
