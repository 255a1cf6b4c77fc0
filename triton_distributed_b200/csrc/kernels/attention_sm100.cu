// Attention of many query rows over a paged KV cache on the tcgen05 tensor cores: prefill of a ragged batch (causal, with an
// optional sliding window and first tokens that stay visible), and the keys that all sequences of a decode batch share.
//
//   out[r] = sum_j p[r, j] v[j],  p[r, j] = exp(s[r, j] - lse[r]),  s = cap(scale q k^T),  lse[r] = log sum_j exp(s[r, j])
//   over the keys j that row r sees: j <= pos(r) and (j > pos(r) - window or j < sinks)
//
// A tile is 128 rows of one kv head: the G query heads that share it for 128 / G tokens, so that a key is read once for all of
// them. A CTA goes over its keys 64 at a time with the running maximum and sum of a softmax:
//   S = Q K^T in TMEM (128 x 64 fp32), a thread per row turns it into P = exp2(S - m) in 16 bits, in place of S in TMEM, and
//   O += P V takes P from TMEM and V as it lies in the cache (its N dimension contiguous).
// Two such chains ("streams") run in one CTA: two row tiles over the same keys where there are enough rows, else one row tile over every
// other block of keys, joined at the end (one stream with head_dim 256, whose O fills TMEM). Each stream has two S, so that the
// tensor cores work on the next block's S and the last one's O while its threads are in a softmax.
// Warps: 4 per stream for the softmax, one per stream that issues MMAs, kLoaders that copy K and V into a ring of tiles in the 128-byte-swizzled
// layout the MMAs read: by TMA, a box per page (or 64 rows of it) and 64 head dimensions, where the page is a multiple of 8 rows and the
// whole block is seen; by 16-byte cp.async else (pages of any size; rows that nobody sees are not read and become zeros).
// Few rows over many keys are split along the keys; the partial results meet in attention_merge_kernel, or in the decode kernel.
//
// P is rounded to the inputs' 16 bits (relative 2^-8; 2^-11 in fp16, whose numbers end at 2^-24: smaller P are multiples of that), S, O,
// maximum and sum are fp32. The maximum that is subtracted is raised only when it has grown by more than 2^8 (kRaise): O is read, scaled and
// written back a few times per row instead of once per block, and the largest P, which is 1 otherwise, is rounded like the others. Raised at once /
// by this rule: 2048 tokens 186 / 160 us, error against 64 bits 2.3e-3 both; 16384 tokens 2347 / 1921; ragged prompts in fp16 315 / 271, 2.5e-4 /
// 2.6e-4; prefix of 32768 keys 95 / 88, 2.3e-3 / 2.4e-3.
// A product that lies below the accumulator's 24 bits is cut by the tensor cores, as in any sum in fp32, and fp16's P below 2^-25 are zero: beside
// one key that weighs 2^24 times as much as each of n others in its chain, up to n 2^-25 of the result is lost (131072 keys alike, 2^-25 each:
// 3.9e-3; a P lifted by 2^7 to keep fp16's small ones was no better and lost more to the cut, 2.0e-3 where it is 0 without, at 2^-20).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cstring>
#include <mutex>
#include <string>

#include "../device/ptx.cuh"
#include "../device/signal.cuh"
#include "../device/soft_cap.cuh"
#include "../include/tdist.h"
#include "../runtime/host_common.h"

namespace tdist {
namespace attention {

constexpr int kKernelAttention = 9;
constexpr int kRows = 128;      // rows of a tile: the MMA's M
constexpr int kKeys = 64;       // keys of a block
constexpr int kLoaders = 2;     // warps that copy K and V
constexpr float kRaise = 8.f;   // log2 of how far scores may exceed the maximum that is subtracted

struct alignas(64) Params {
    CUtensorMap tm_k, tm_v;  // 64 x 1 x box_rows x 1 of (head_dim, Hkv, page, blocks); box_rows > 0
    const void* q;           // rows of D values, strides below
    const void* k_cache;     // [blocks, page, Hkv, D]
    const void* v_cache;
    const int* block_table;  // [B, max_blocks]; shared: [max_blocks]
    const int* q_starts;     // [B + 1]; shared: nullptr
    const int* kv_lens;      // [B]; shared: [1]
    void* out;               // T [tokens, Hq, D], where one part holds the result
    float* part_o;           // fp32 [splits][tokens * Hq][D], normalised
    float* part_lse;         // fp32 [splits][tokens * Hq], natural log
    long long q_token, q_head, stride_head;   // in elements
    uint32_t unit_block, unit_token;          // strides of the cache in units of 2^unit_shift elements
    int unit_shift, box_rows;                 // box_rows 0: no TMA
    int tokens, B, Hq, Hkv, G, page_size, page_shift, max_blocks, blocks, splits;
    int tile_tokens;         // tokens of a row tile: 128 / G
    int shared;              // 1: every query token sees all kv_lens[0] keys
    int window, sinks;       // window 0x7fffffff: none
    float scale_log2, soft_cap;   // |scale| x log2 e
    uint32_t q_and, q_xor;   // sign of the scale, applied to q (0 / 0: scale 0)
    WaitCtx wctx;
};

template <int D>
struct Shape {
    static constexpr int STREAMS = D <= 128 ? 2 : 1;
    static constexpr int TILE = kKeys * D * 2;            // bytes of a K or V block
    static constexpr int QTILE = kRows * D * 2;
    static constexpr int CHUNKS = D / 64;                 // 128-byte columns of a tile
    static constexpr int AREA = D == 64 ? 160 * 1024 : 224 * 1024;
    static constexpr int SOFT = 128 * STREAMS;            // softmax threads
    static constexpr int THREADS = SOFT + 32 * STREAMS + 32 * kLoaders;
    static constexpr uint32_t O_COL = 256;                // TMEM columns: S / P of stream s at s * 128 (+ 64), O at O_COL + s * D
};
template <int D, int QT>
constexpr int stages() {
    return (Shape<D>::AREA - QT * Shape<D>::QTILE) / Shape<D>::TILE;
}
constexpr int kMaxStages = 18;
constexpr int kBars = 2 * kMaxStages + 14;   // full, empty, S, P, O, Q, go

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int src_bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
// arrives on `bar` once all cp.async that this thread has issued are complete
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// D (TMEM) (+)= A (TMEM: a row per lane, two 16-bit values per column) x B (shared memory)
__device__ __forceinline__ void umma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
        "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// 32 lanes x 16 columns: thread t of the warp writes columns [col, col + 16) of TMEM lane (lane_base + t)
__device__ __forceinline__ void tmem_st_32x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(taddr)
        : "memory");
}
// the same, 8 columns
__device__ __forceinline__ void tmem_st_32x8(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float lo, float hi) { return pack_f16x2(lo, hi); }

// ---- two fp32 values at a time
__device__ __forceinline__ uint64_t pair(float lo, float hi) {
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi));
    return v;
}
__device__ __forceinline__ void unpair(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// P = 2^(s scale - m) for 32 scores, packed, and their sum. (Some of the exponentials as a polynomial on the FMA pipe, to relieve the
// special-function unit with its 8 clocks per warp: of 16 pairs 2 to 6, in stages between the others or not: no faster, 16384 tokens 1864 us
// without, 1897 to 1974 with them.)
template <typename T>
__device__ __forceinline__ void exponentials(const uint32_t (&s)[32], uint64_t scale2, uint64_t minus2, uint32_t (&pk)[16], uint64_t (&sum2)[2]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float a, b;
        unpair(fma2(pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), scale2, minus2), a, b);
        a = exp2f(a);
        b = exp2f(b);
        sum2[i & 1] = add2(sum2[i & 1], pair(a, b));
        pk[i] = pack2<T>(a, b);
    }
}

// out tanh(in s) where |in s| <= kCapSmall, by the polynomial. (The exponential and the quotient it does without cost 16 clocks of the
// special-function unit per warp, twice what the softmax's own exponential does.) The coefficients hold the powers of `in` up to the ninth (FOLDED):
// within fp32's range for `in` in [2^-12, 2^12] and `in` x `out` in [2^-23, 2^23]. Other caps multiply the score by `in` first, in a kernel of its
// own (for all caps: 7 ragged prompts with heads of 64 284 us instead of 271; 2 x 1024 tokens, cap 1000, 170 us, by the way of large scores 475).
__host__ __device__ inline bool foldable(float in, float scale) {
    return in >= 1.f / 4096.f && in <= 4096.f && scale >= 1.f / 8388608.f && scale <= 8388608.f;
}
enum Capped { kUncapped, kFolded, kUnfolded };
struct Cap {
    float c[5], in;
};
template <bool FOLDED>
__device__ __forceinline__ Cap cap_polynomial(float in, float scale) {   // scale: out * in
    const float u = FOLDED ? in * in : 1.f;
    Cap k;
    k.in = FOLDED ? 1.f : fmaxf(in, 1e-37f);   // above zero for masked scores, which are -inf
    float f = scale;
    k.c[0] = kCapC0 * f;
    k.c[1] = kCapC1 * (f *= u);
    k.c[2] = kCapC2 * (f *= u);
    k.c[3] = kCapC3 * (f *= u);
    k.c[4] = kCapC4 * (f *= u);
    return k;
}
template <bool FOLDED>
__device__ __forceinline__ float cap_score(float s, const Cap& k) {   // -inf stays -inf
    const float z = FOLDED ? s : s * k.in, u = z * z;
    return fmaf(fmaf(fmaf(fmaf(u, k.c[4], k.c[3]), u, k.c[2]), u, k.c[1]), u, k.c[0]) * s;
}
// P = 2^(cap(s) - m): as above. The maximum is known before the cap is taken, as the cap keeps the order, so that one pair's polynomial runs
// under another's exponentials.
template <typename T, bool FOLDED>
__device__ __forceinline__ void capped_exponentials(const uint32_t (&s)[32], const Cap& k, uint64_t minus2, uint32_t (&pk)[16], uint64_t (&sum2)[2]) {
    auto both = [&](int i) { return pair(k.c[i], k.c[i]); };
    const uint64_t c0 = both(0), c1 = both(1), c2 = both(2), c3 = both(3), c4 = both(4), in2 = pair(k.in, k.in);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const uint64_t x = pair(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), z = FOLDED ? x : mul2(x, in2), u = mul2(z, z);
        float a, b;
        unpair(fma2(fma2(fma2(fma2(fma2(u, c4, c3), u, c2), u, c1), u, c0), x, minus2), a, b);
        a = exp2f(a);
        b = exp2f(b);
        sum2[i & 1] = add2(sum2[i & 1], pair(a, b));
        pk[i] = pack2<T>(a, b);
    }
}

// What a CTA works on: sequence b, its query tokens [i0, i0 + QT * tile_tokens) of n, the split and the blocks of keys.
struct Work {
    int b, i0, n, q0, kvh, split;
    int first;      // position of token i0
    int hi, lo;     // keys [lo, hi) and [0, s_end) are seen by some row
    int s_end;
    int n_sink, m0; // blocks 0 .. n_sink - 1, then m0 ..
    int c0, nt;     // of these, the split's
};

template <int D, int QT>
__device__ __forceinline__ bool find_work(const Params& p, Work& w) {
    constexpr int KT = kKeys;
    const int lane = static_cast<int>(threadIdx.x) & 31;
    w.split = static_cast<int>(blockIdx.x) % p.splits;
    w.kvh = static_cast<int>(blockIdx.x) / p.splits % p.Hkv;
    int tile = static_cast<int>(blockIdx.x) / p.splits / p.Hkv;
    const int per = QT * p.tile_tokens;
    const long long table_keys = static_cast<long long>(p.max_blocks) * p.page_size;
    int kv = 0;
    if (p.shared) {
        w.b = 0;
        w.q0 = 0;
        w.n = p.tokens;
        w.i0 = tile * per;
        kv = p.kv_lens[0];
    } else {
        // 32 sequences at a time: the one whose tiles hold number `tile`
        int b = -1;
        for (int b0 = 0; b0 < p.B; b0 += 32) {
            int start = 0, n = 0, keys = 0;
            if (b0 + lane < p.B) {
                keys = p.kv_lens[b0 + lane];
                start = min(max(p.q_starts[b0 + lane], 0), p.tokens);
                n = max(min(p.q_starts[b0 + lane + 1], p.tokens) - start, 0);
            }
            const int mine = (n + per - 1) / per;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, tile < upto);
            if (hit != 0) {
                const int src = __ffs(hit) - 1;
                b = b0 + src;
                w.q0 = __shfl_sync(0xffffffffu, start, src);
                w.n = __shfl_sync(0xffffffffu, n, src);
                kv = __shfl_sync(0xffffffffu, keys, src);
                // the last tokens, which see the most keys, first
                w.i0 = (__shfl_sync(0xffffffffu, upto, src) - 1 - tile) * per;
                break;
            }
            tile -= __shfl_sync(0xffffffffu, upto, 31);
        }
        if (b < 0) return false;
        w.b = b;
    }
    kv = kv < 0 ? 0 : (kv > table_keys ? static_cast<int>(table_keys) : kv);
    const int rows_end = min(w.n, w.i0 + per);
    if (p.shared) {
        w.first = kv - 1;
        w.lo = w.s_end = 0;
        w.hi = kv;
    } else {
        w.first = kv - w.n + w.i0;
        w.hi = max(0, kv - w.n + rows_end);
        w.lo = min(p.window > w.first ? 0 : w.first - p.window + 1, w.hi);   // (the first position may lie before the first key)
        w.s_end = min(p.sinks, w.lo);
    }
    w.n_sink = (w.s_end + KT - 1) / KT;
    w.m0 = max(w.lo / KT, w.n_sink);
    const int total = w.hi > 0 ? w.n_sink + max(0, (w.hi + KT - 1) / KT - w.m0) : 0;
    const int each = (total + p.splits - 1) / p.splits;
    w.c0 = min(total, w.split * each);
    w.nt = min(total, w.c0 + each) - w.c0;
    return true;
}

// QT: row tiles of the CTA. Two: a stream each, all blocks of keys. One: the streams take turns at the blocks. CAP: with a soft cap (a kernel of
// its own: with both in one, 16384 tokens without a cap 1890 to 1940 us, by itself 1710 to 1820).
template <typename T, int D, int QT, Capped CAP>
__global__ void __launch_bounds__(Shape<D>::THREADS, 1) attention_kernel(const __grid_constant__ Params p) {
    using S = Shape<D>;
    constexpr bool CAPPED = CAP != kUncapped, FOLDED = CAP == kFolded;
    constexpr int KT = kKeys, NSTR = S::STREAMS, NST = stages<D, QT>(), CH = D / 8;
    static_assert(NST >= 2 && NST <= kMaxStages, "a tile is released only once the one after it has arrived");
    static_assert(QT == 1 || NSTR == 2, "two row tiles need two streams");
    constexpr int LOOK = QT == 2 ? 2 : 2 * NSTR;   // K blocks ahead of the first V block: two S per stream
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::AREA);
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + kBars);
    const uint32_t q_smem = smem_u32(smem), ring = q_smem + QT * S::QTILE;
    const uint32_t bars_u32 = smem_u32(bars);
    auto bar_full = [&](int s) { return bars_u32 + 8u * s; };
    auto bar_empty = [&](int s) { return bars_u32 + 8u * (kMaxStages + s); };
    auto bar_s = [&](int s, int b) { return bars_u32 + 8u * (2 * kMaxStages + 2 * s + b); };        // S is complete
    auto bar_p = [&](int s, int b) { return bars_u32 + 8u * (2 * kMaxStages + 4 + 2 * s + b); };    // P is in its place
    auto bar_o = [&](int s, int b) { return bars_u32 + 8u * (2 * kMaxStages + 8 + 2 * s + b); };    // O has taken it in
    const uint32_t bar_q = bars_u32 + 8u * (2 * kMaxStages + 12), bar_go = bars_u32 + 8u * (2 * kMaxStages + 13);
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;

    if (tid == 0) {
        for (int s = 0; s < NST; ++s) {
            mbar_init(bar_full(s), 32 * kLoaders);
            mbar_init(bar_empty(s), QT);   // streams that take it in
        }
        for (int s = 0; s < 2; ++s) {
            for (int b = 0; b < 2; ++b) {
                mbar_init(bar_s(s, b), 1);
                mbar_init(bar_p(s, b), 128);
                mbar_init(bar_o(s, b), 1);
            }
        }
        mbar_init(bar_q, S::SOFT);
        mbar_init(bar_go, 1);
        fence_mbar_init();
    }
    if (warp == S::SOFT / 32) {
        tmem_alloc<1>(smem_u32(tmem_slot), 512);
        tmem_relinquish<1>();
    }
    pdl_wait_and_release();
    Work w = {};
    const bool live = find_work<D, QT>(p, w);   // its loads under the others' set-up
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    const int nt = live ? w.nt : 0;
    auto block_start = [&](int j) {   // first key of the split's j-th block
        const int i = w.c0 + j;
        return (i < w.n_sink ? i : w.m0 + i - w.n_sink) * KT;
    };
    // Blocks of which every key is seen by some row come by TMA: the split's [tma0, tma1)
    int tma0 = 0, tma1 = 0;
    if (p.box_rows > 0 && nt > 0) {
        tma0 = max(0, w.n_sink + max(w.m0, (w.lo + KT - 1) / KT) - w.m0 - w.c0);
        tma1 = min(nt, w.n_sink + w.hi / KT - w.m0 - w.c0);
    }
    auto by_tma = [&](int j) { return j >= tma0 && j < tma1; };
    // The ring's items in the order in which the loaders bring them: LOOK blocks of K, then V and K in turn, the last of V.
    const int look = min(LOOK, nt);
    auto item_v = [&](int j) { return j < nt - look ? look + 2 * j : nt + j; };
    auto item_k = [&](int j) { return j < look ? j : look + 2 * (j - look) + 1; };

    if (warp >= S::SOFT / 32 + NSTR) {
        // ---------------------------------------------------------------- loaders
        constexpr int RW = KT / kLoaders, RL = RW / 32, RPI = 32 / CH;   // cp.async: rows of a warp, of a lane's lookups, of an instruction
        const int loader = warp - S::SOFT / 32 - NSTR, r0 = loader * RW;
        const int* table = p.block_table + static_cast<size_t>(live ? w.b : 0) * p.max_blocks;
        const int lrow = lane / CH, lch = lane % CH;
        const T* kl = static_cast<const T*>(p.k_cache) + static_cast<size_t>(w.kvh) * p.stride_head + lch * 8;
        const T* vl = static_cast<const T*>(p.v_cache) + static_cast<size_t>(w.kvh) * p.stride_head + lch * 8;
        const uint32_t lane_dst = static_cast<uint32_t>((lch >> 3) * (KT * 128));
        const int items = 2 * nt;
        // TMA: the loaders take a block's groups of box_rows rows in turn (the first one all of a block in one page), a box per 64 columns of a group
        const int box_rows = p.box_rows;
        auto block_of = [&](int n, bool& is_k) {
            const int m = n - look, pairs = 2 * (nt - look);
            is_k = n < look || (m < pairs && (m & 1));
            return n < look ? n : (m < pairs ? (m >> 1) + (is_k ? look : 0) : m - (nt - look));
        };
        auto page_of = [&](int t, int& in_page) {
            const int in_table = p.page_shift >= 0 ? t >> p.page_shift : t / p.page_size;
            in_page = t - in_table * p.page_size;
            return table[in_table];
        };
        constexpr uint32_t kUnseen = 0xffffffffu;
        struct Item {
            int t0, page, in_page;   // TMA: of the lane's group of box_rows rows
            bool is_k, whole;
            uint32_t off[RL];        // cp.async: the lane's rows in the cache, in units; kUnseen: nobody sees the key
        };
        auto lookup = [&](int n, Item& x) {
            if (n >= items) return;
            const int j = block_of(n, x.is_k);
            x.t0 = block_start(j);
            x.whole = by_tma(j);
            if (x.whole) {
                if (lane * box_rows < KT) x.page = page_of(x.t0 + lane * box_rows, x.in_page);
            } else {
#pragma unroll
                for (int r = 0; r < RL; ++r) {
                    const int t = x.t0 + r0 + lane + 32 * r;
                    x.off[r] = kUnseen;
                    if (t < w.s_end || (t >= w.lo && t < w.hi)) {
                        int in_page;
                        const int page = page_of(t, in_page);
                        if (static_cast<unsigned>(page) < static_cast<unsigned>(p.blocks)) x.off[r] = static_cast<uint32_t>(page) * p.unit_block + static_cast<uint32_t>(in_page) * p.unit_token;
                    }
                }
            }
        };
        Item next;
        lookup(0, next);
        for (int n = 0; n < items; ++n) {
            const Item x = next;
            lookup(n + 1, next);
            const int slot = n % NST;
            mbar_wait(bar_empty(slot), ((n / NST) & 1u) ^ 1u, p.wctx, 1);
            const uint32_t dst = ring + static_cast<uint32_t>(slot) * S::TILE;
            if (x.whole) {
                if (loader == 0 && lane == 0) mbar_expect_tx(bar_full(slot), S::TILE);
                else mbar_arrive(bar_full(slot));
                const CUtensorMap* map = x.is_k ? &p.tm_k : &p.tm_v;
                for (int r = loader; r * box_rows < KT; r += kLoaders) {
                    const int page = __shfl_sync(0xffffffffu, x.page, r), in_page = __shfl_sync(0xffffffffu, x.in_page, r);
                    if (elect_one()) {
#pragma unroll
                        for (int c = 0; c < S::CHUNKS; ++c)
                            tma_load_4d(dst + c * (KT * 128) + r * box_rows * 128, map, bar_full(slot), c * 64, w.kvh, in_page, page);
                    }
                }
                __syncwarp();
            } else {
                const T* src = x.is_k ? kl : vl;
#pragma unroll
                for (int j = 0; j < RW / RPI; ++j) {
                    const int row = j * RPI + lrow, at = r0 + row;
                    const uint32_t o = __shfl_sync(0xffffffffu, x.off[j * RPI / 32], row & 31);
                    const bool seen = o != kUnseen;
                    cp_async16(dst + lane_dst + static_cast<uint32_t>(at * 128 + (((lch & 7) ^ (at & 7)) << 4)),
                               src + (seen ? static_cast<size_t>(o) << p.unit_shift : 0), seen ? 16 : 0);
                }
                cp_async_arrive(bar_full(slot));
            }
        }
    } else if (warp >= S::SOFT / 32) {
        // ---------------------------------------------------------------- MMA issue, a warp per stream: one's waits under the other's products
        const int stream = warp - S::SOFT / 32;
        const bool leader = elect_one();   // the whole warp goes along, so that descriptors stay in uniform registers
        const uint32_t fmt = sizeof(T) == 2 && __is_same(T, __half) ? 0u : 1u;
        const uint32_t idesc_s = umma_idesc(fmt, fmt, kRows, KT);
        const uint32_t idesc_o = umma_idesc(fmt, fmt, kRows, D) | kIdescBNMajor;
        const uint32_t qb = q_smem + (QT == 2 ? stream : 0) * S::QTILE, s_col = tmem + stream * 128, o_col = tmem + S::O_COL + stream * D;
        const int my_blocks = QT == 2 ? nt : (nt - stream + NSTR - 1) / NSTR;
        auto block = [&](int it) { return QT == 2 ? it : it * NSTR + stream; };   // number of the stream's `it`-th block
        auto arrived = [&](int item, int j) {
            mbar_wait(bar_full(item % NST), (item / NST) & 1u, p.wctx, 2);
            if (!by_tma(j)) fence_proxy_async_smem();   // what cp.async wrote, to the MMAs' proxy
            tc_fence_after();
        };
        auto qk = [&](int it) {
            const int j = block(it), item = item_k(j), slot = item % NST, buf = it & 1;
            arrived(item, j);
            const uint32_t kb = ring + static_cast<uint32_t>(slot) * S::TILE;
            if (leader) {
#pragma unroll
                for (int c = 0; c < S::CHUNKS; ++c) {
                    const uint64_t a = umma_desc_k_sw128(qb + c * (kRows * 128)), b = umma_desc_k_sw128(kb + c * (KT * 128));
#pragma unroll
                    for (int k = 0; k < 4; ++k) umma_bf16<1>(s_col + buf * 64, a + 2 * k, b + 2 * k, idesc_s, (c | k) != 0 ? 1u : 0u);
                }
                umma_commit(bar_s(stream, buf));
                umma_commit(bar_empty(slot));
            }
            __syncwarp();
        };
        if (my_blocks > 0) {
            mbar_wait(bar_q, 0, p.wctx, 3);
            // half a block behind the other stream, so that one's exponentials run beside the other's loads and maxima (a barrier of one phase: that
            // of the other's P may be two phases further by the time this warp looks)
            if (stream == 1) mbar_wait(bar_go, 0, p.wctx, 9);
            for (int it = 0; it < min(2, my_blocks); ++it) qk(it);
            for (int it = 0; it < my_blocks; ++it) {
                const int j = block(it), item = item_v(j), slot = item % NST, buf = it & 1;
                arrived(item, j);
                const uint64_t b = umma_desc_mn_sw128(ring + static_cast<uint32_t>(slot) * S::TILE, KT * 128);
                mbar_wait(bar_p(stream, buf), (it >> 1) & 1u, p.wctx, 4);
                if (NSTR == 2 && stream == 0 && it == 0 && lane == 0) mbar_arrive(bar_go);
                tc_fence_after();
                if (leader) {
#pragma unroll
                    for (int k = 0; k < KT / 16; ++k) umma_ts(o_col, s_col + buf * 64 + 8 * k, b + 128 * k, idesc_o, it > 0 || k != 0 ? 1u : 0u);
                    umma_commit(bar_o(stream, buf));
                    umma_commit(bar_empty(slot));
                }
                __syncwarp();
                if (it + 2 < my_blocks) {
                    // this P has been taken in: the next S but one takes its columns
                    mbar_wait(bar_o(stream, buf), (it >> 1) & 1u, p.wctx, 5);
                    tc_fence_after();
                    qk(it + 2);
                }
            }
        }
    } else {
        // ---------------------------------------------------------------- softmax: a thread per row
        const int stream = warp >> 2, row = tid & 127;
        const int q_tile = QT == 2 ? stream : 0;
        if (live) {
            // Q into shared memory, zeros for rows without a token
            constexpr int UNITS = QT * kRows * CH / S::SOFT, AHEAD = UNITS < 8 ? UNITS : 8;   // 16 bytes each; loads of a thread under way at once
            static_assert(UNITS % AHEAD == 0 && S::SOFT % CH == 0, "a thread keeps its place in a row");
            const int c = tid % CH;
            const T* q = static_cast<const T*>(p.q) + static_cast<long long>(w.q0 + w.i0) * p.q_token + static_cast<long long>(w.kvh * p.G) * p.q_head + c * 8;
#pragma unroll 1
            for (int u0 = 0; u0 < UNITS; u0 += AHEAD) {
                uint4 v[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int r = tid / CH + (u0 + u) * (S::SOFT / CH), rt = r & (kRows - 1), t = rt / p.G, tok = r / kRows * p.tile_tokens + t;
                    v[u] = make_uint4(0u, 0u, 0u, 0u);
                    if (t < p.tile_tokens && w.i0 + tok < w.n) v[u] = ld_v4(q + static_cast<long long>(tok) * p.q_token + static_cast<long long>(rt - t * p.G) * p.q_head);
                }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int r = tid / CH + (u0 + u) * (S::SOFT / CH), rt = r & (kRows - 1);
                    v[u].x = (v[u].x & p.q_and) ^ p.q_xor;
                    v[u].y = (v[u].y & p.q_and) ^ p.q_xor;
                    v[u].z = (v[u].z & p.q_and) ^ p.q_xor;
                    v[u].w = (v[u].w & p.q_and) ^ p.q_xor;
                    *reinterpret_cast<uint4*>(smem + r / kRows * S::QTILE + (c >> 3) * (kRows * 128) + rt * 128 + (((c & 7) ^ (rt & 7)) << 4)) = v[u];
                }
            }
            fence_proxy_async_smem();
        }
        mbar_arrive(bar_q);
        if (!p.shared) {
            // tokens of no sequence, before the first one's and behind the last one's: zeros (LSE -inf), spread over the CTAs of a kv head and split
            const int lead = min(max(p.q_starts[0], 0), p.tokens), tail = max(min(p.q_starts[p.B], p.tokens), lead);
            const int per_tile = p.splits * p.Hkv, n = lead + p.tokens - tail;
            for (int i = static_cast<int>(blockIdx.x) / per_tile; i < n; i += static_cast<int>(gridDim.x) / per_tile) {
                const size_t first = static_cast<size_t>(i < lead ? i : tail + i - lead) * p.Hq + static_cast<size_t>(w.kvh) * p.G;
                const size_t rows = static_cast<size_t>(p.tokens) * p.Hq;
                uint4* dst = p.part_o != nullptr ? reinterpret_cast<uint4*>(p.part_o + (w.split * rows + first) * D)
                                                 : reinterpret_cast<uint4*>(static_cast<T*>(p.out) + first * D);
                const int units = p.G * D / (p.part_o != nullptr ? 4 : 8);
                for (int u = tid; u < units; u += S::SOFT) dst[u] = make_uint4(0u, 0u, 0u, 0u);
                if (p.part_o != nullptr && tid < p.G) p.part_lse[w.split * rows + first + tid] = -CUDART_INF_F;
            }
        }

        const int t_in = row / p.G;
        const int tok = w.i0 + q_tile * p.tile_tokens + t_in;
        const bool mine = live && t_in < p.tile_tokens && tok < w.n;
        // rows of a tile see up to first .. last, and from first - window + 1 .. last - window + 1 on
        const int tile_first = p.shared ? w.first : w.first + q_tile * p.tile_tokens;
        const int tile_last = p.shared ? w.first : min(tile_first + p.tile_tokens - 1, w.first - w.i0 + w.n - 1);
        const int pos = p.shared ? w.first : tile_first + t_in;
        // the keys up to these are out of the window: of this row, of the tile's last one
        const int below = p.window > pos ? -1 : pos - p.window, tile_below = p.window > tile_last ? -1 : tile_last - p.window;
        const float sl2 = CAPPED ? 1.f : p.scale_log2;
        // cap_out tanh(cap_in s): the cap in the exponent's domain; scores up to cap_small by a polynomial
        const float cap_out = p.soft_cap * 1.4426950408889634f, cap_in = CAPPED ? p.scale_log2 / cap_out : 0.f;
        const float cap_small = p.scale_log2 >= 1e-30f ? kCapSmall / cap_in : -1.f;   // (the coefficients must not be zero either)
        const Cap cap = cap_polynomial<FOLDED>(cap_in, p.scale_log2);
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
        const uint32_t s_at = tmem + lanes + stream * 128, o_at = tmem + lanes + S::O_COL + stream * D;
        const int my_blocks = QT == 2 ? nt : (nt - stream + NSTR - 1) / NSTR;
        float m_ref = -CUDART_INF_F, l_run = 0.f;
        for (int it = 0; it < my_blocks; ++it) {
            const int t0 = block_start(QT == 2 ? it : it * NSTR + stream);
            const int buf = it & 1;
            const uint32_t at = s_at + buf * 64;
            const bool edge = !(t0 + KT - 1 <= tile_first && (t0 > tile_below || t0 + KT <= p.sinks));   // some row does not see all
            mbar_wait(bar_s(stream, buf), (it >> 1) & 1u, p.wctx, 6);
            tc_fence_after();
            uint32_t s[2][32];
            tmem_ld_32x32(at, s[0]);
            tmem_ld_32x32(at + 32, s[1]);
            tmem_ld_wait();
            bool small = false;   // the cap is yet to be taken, by its polynomial
            if constexpr (CAPPED) {
                float big[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) big[i & 3] = fmaxf(big[i & 3], fabsf(__uint_as_float(s[c][i])));
                small = __all_sync(0xffffffffu, fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) <= cap_small);
                if (!small) {
                    // Score by score, the small ones beside large ones too. Eight columns at a time through TMEM: unrolled, it would crowd the
                    // loop out of the instruction cache.
#pragma unroll 1
                    for (int c = 0; c < 64; c += 8) {
                        uint32_t e[8];
                        tmem_ld_32x8(at + c, e);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; ++i)
                            e[i] = __float_as_uint(p.soft_cap > kCapNear ? soft_cap(__uint_as_float(e[i]) * p.scale_log2, __uint_as_float(e[i]) * cap_in, cap_out)
                                                                         : soft_cap_far(__uint_as_float(e[i]) * cap_in, cap_out));
                        tmem_st_32x8(at + c, e);
                    }
                    tmem_st_wait();
                    tmem_ld_32x32(at, s[0]);
                    tmem_ld_32x32(at + 32, s[1]);
                    tmem_ld_wait();
                }
            }
            if (edge) {
                const int hi = pos - t0, lo = below - t0, sink = p.sinks - t0;
#pragma unroll
                for (int c = 0; c < 2; ++c)
#pragma unroll
                    for (int i = 0; i < 32; ++i) {
                        const int j = 32 * c + i;
                        if (!(j <= hi && (j > lo || j < sink))) s[c][i] = 0xff800000u;
                    }
            }
            float mx[4] = {-CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F, -CUDART_INF_F};
#pragma unroll
            for (int c = 0; c < 2; ++c)
#pragma unroll
                for (int i = 0; i < 32; i += 2) mx[(i >> 1) & 3] = max3(mx[(i >> 1) & 3], __uint_as_float(s[c][i]), __uint_as_float(s[c][i + 1]));
            const float raw = fmaxf(max3(mx[0], mx[1], mx[2]), mx[3]), top = small ? cap_score<FOLDED>(raw, cap) : raw * sl2;
            if (it == 0) {
                m_ref = top;
            } else if (__any_sync(0xffffffffu, top > m_ref + kRaise)) {
                const float m_new = fmaxf(m_ref, top);
                const float alpha = m_new == m_ref ? 1.f : exp2f(m_ref - m_new);
                m_ref = m_new;
                l_run *= alpha;
                mbar_wait(bar_o(stream, buf ^ 1), ((it - 1) >> 1) & 1u, p.wctx, 7);
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 16) {
                    uint32_t o[16];
                    tmem_ld_32x16(o_at + c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                    tmem_st_32x16(o_at + c, o);
                }
            }
            const float m_use = m_ref == -CUDART_INF_F ? 0.f : m_ref;
            const uint64_t scale2 = pair(sl2, sl2), minus2 = pair(-m_use, -m_use);
            uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                uint32_t pk[16];
                if (small) capped_exponentials<T, FOLDED>(s[c], cap, minus2, pk, sum2);
                else exponentials<T>(s[c], scale2, minus2, pk, sum2);
                tmem_st_32x16(at + 16 * c, pk);
            }
            tmem_st_wait();
            tc_fence_before();
            mbar_arrive(bar_p(stream, buf));
            float sum_lo, sum_hi;
            unpair(add2(sum2[0], sum2[1]), sum_lo, sum_hi);
            l_run += sum_lo + sum_hi;
        }
        if (my_blocks > 0) {
            // The last two products may both be under way or both be done. A barrier only tells its phases' parity, hence one for each S: the phase
            // before the last product's is over, as the last S came after it.
            mbar_wait(bar_o(stream, (my_blocks - 1) & 1), ((my_blocks - 1) >> 1) & 1u, p.wctx, 8);
            tc_fence_after();
        }

        // ---- one row tile, two streams: the second's result to the first through shared memory (every MMA is done with it)
        float* ex = reinterpret_cast<float*>(smem);   // [D + 2][128]
        float f0 = 1.f, f1 = 0.f;
        if constexpr (QT == 1 && NSTR == 2) {
            named_barrier(1, S::SOFT);
            if (stream == 1) {
                ex[D * 128 + row] = m_ref;
                ex[(D + 1) * 128 + row] = l_run;
#pragma unroll 1
                for (int c = 0; c < D && my_blocks > 0; c += 32) {
                    uint32_t o[32];
                    tmem_ld_32x32(o_at + c, o);
                    tmem_ld_wait();
#pragma unroll
                    for (int i = 0; i < 32; ++i) ex[(c + i) * 128 + row] = __uint_as_float(o[i]);
                }
            }
            named_barrier(1, S::SOFT);
            const float m1 = ex[D * 128 + row], l1 = ex[(D + 1) * 128 + row];
            const float m = fmaxf(m_ref, m1), mu = m == -CUDART_INF_F ? 0.f : m;
            f0 = exp2f(m_ref - mu);
            f1 = exp2f(m1 - mu);
            l_run = l_run * f0 + l1 * f1;
            m_ref = m;
        }
        if (QT == 2 || stream == 0) {
            const float inv = l_run > 0.f ? 1.f / l_run : (l_run == l_run ? 0.f : l_run);   // NaN stays NaN
            const size_t out_row = static_cast<size_t>(w.q0 + tok) * p.Hq + static_cast<size_t>(w.kvh) * p.G + (row - t_in * p.G);
            const size_t rows = static_cast<size_t>(p.tokens) * p.Hq;
            const bool other = QT == 1 && NSTR == 2 && nt > 1;
            if (p.part_o != nullptr && mine)
                p.part_lse[w.split * rows + out_row] = l_run > 0.f ? m_ref * 0.6931471805599453f + logf(l_run) : (l_run == l_run ? -CUDART_INF_F : l_run);
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                uint32_t o[32];
                if (my_blocks > 0) {   // alike in the whole warp
                    tmem_ld_32x32(o_at + c, o);
                    tmem_ld_wait();
                }
                float v[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    v[i] = my_blocks > 0 ? __uint_as_float(o[i]) * f0 : 0.f;
                    if (other) v[i] += ex[(c + i) * 128 + row] * f1;
                    v[i] *= inv;
                }
                if (!mine) continue;
                if (p.part_o != nullptr) {
                    float* dst = p.part_o + (w.split * rows + out_row) * D + c;
#pragma unroll
                    for (int i = 0; i < 32; i += 8)   // a sector at a time
                        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst + i), "f"(v[i]), "f"(v[i + 1]), "f"(v[i + 2]),
                                     "f"(v[i + 3]), "f"(v[i + 4]), "f"(v[i + 5]), "f"(v[i + 6]), "f"(v[i + 7])
                                     : "memory");
                } else {
                    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(p.out) + out_row * D + c);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        dst[i] = make_uint4(pack2<T>(v[8 * i], v[8 * i + 1]), pack2<T>(v[8 * i + 2], v[8 * i + 3]),
                                            pack2<T>(v[8 * i + 4], v[8 * i + 5]), pack2<T>(v[8 * i + 6], v[8 * i + 7]));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == S::SOFT / 32) {
        tc_fence_after();
        tmem_dealloc<1>(tmem, 512);
    }
}

// out[row] = sum over the parts of exp(lse[part, row] - lse[row]) o[part, row]: D / 4 threads per row
template <typename T, int D>
__global__ void __launch_bounds__(128) attention_merge_kernel(const float* part_o, const float* part_lse, int parts, int rows, T* out) {
    pdl_wait_and_release();
    const int per = 128 / (D / 4);
    const long long row = static_cast<long long>(blockIdx.x) * per + threadIdx.x / (D / 4);
    const int c = static_cast<int>(threadIdx.x) % (D / 4) * 4;
    if (row >= rows) return;
    float mm = -CUDART_INF_F;
    for (int i = 0; i < parts; ++i) mm = fmaxf(mm, part_lse[static_cast<size_t>(i) * rows + row]);
    const float mu = mm == -CUDART_INF_F ? 0.f : mm;
    float sum = 0.f;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
        const float f = __expf(part_lse[static_cast<size_t>(i) * rows + row] - mu);
        const float4 v = *reinterpret_cast<const float4*>(part_o + (static_cast<size_t>(i) * rows + row) * D + c);
        sum += f;
        acc.x += f * v.x;
        acc.y += f * v.y;
        acc.z += f * v.z;
        acc.w += f * v.w;
    }
    const float inv = sum > 0.f ? 1.f / sum : (sum == sum ? 0.f : sum);
    *reinterpret_cast<uint2*>(out + row * D + c) = make_uint2(pack2<T>(acc.x * inv, acc.y * inv), pack2<T>(acc.z * inv, acc.w * inv));
}

}  // namespace attention
}  // namespace tdist

using namespace tdist;
using tdist_host::fail;

namespace {

template <typename T, int D, int QT, attention::Capped CAP>
int launch_attention(const attention::Params& p, long long grid, cudaStream_t stream) {
    using S = attention::Shape<D>;
    constexpr int smem = S::AREA + 1024 + attention::kBars * 8 + 16;
    static bool done[64] = {};
    static std::mutex setup_lock;
    int dev = 0;
    TDIST_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(TDIST_EINVAL, "attention: device ordinal out of range");
    {
        std::lock_guard<std::mutex> guard(setup_lock);
        if (!done[dev]) {
            TDIST_CUDA_OK(cudaFuncSetAttribute(attention::attention_kernel<T, D, QT, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
            done[dev] = true;
        }
    }
    TDIST_CUDA_OK(tdist_host::launch_pdl(attention::attention_kernel<T, D, QT, CAP>, dim3(static_cast<unsigned>(grid)), S::THREADS, smem, stream, p));
    return 0;
}

template <typename T, int D, attention::Capped CAP>
int run_attention(const TdistAttentionArgs* a, attention::Params& p) {
    cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    const long long per = static_cast<long long>(a->row_tiles) * p.tile_tokens;
    // a sequence's last tile may be short: at most one more per sequence than the tokens fill
    const long long tiles = p.shared ? (p.tokens + per - 1) / per : p.tokens / per + (p.B < p.tokens ? p.B : p.tokens);
    const long long grid = tiles * p.Hkv * p.splits;
    if (grid > 0x7fffffffLL) return fail(TDIST_ELIMIT, "attention: tiles * Hkv * splits exceeds the grid limit");
    int rc;
    if constexpr (D <= 128)
        rc = a->row_tiles == 2 ? launch_attention<T, D, 2, CAP>(p, grid, stream) : launch_attention<T, D, 1, CAP>(p, grid, stream);
    else
        rc = launch_attention<T, D, 1, CAP>(p, grid, stream);
    if (rc != 0 || p.splits == 1 || a->out == nullptr) return rc;
    const long long rows = static_cast<long long>(p.tokens) * p.Hq, per_cta = 128 / (D / 4);
    TDIST_CUDA_OK(tdist_host::launch_pdl(attention::attention_merge_kernel<T, D>, dim3(static_cast<unsigned>((rows + per_cta - 1) / per_cta)), 128, 0,
                                         stream, p.part_o, p.part_lse, p.splits, static_cast<int>(rows), static_cast<T*>(a->out)));
    return 0;
}

template <typename T, attention::Capped CAP>
int by_head_dim(const TdistAttentionArgs* a, attention::Params& p) {
    if (a->head_dim == 64) return run_attention<T, 64, CAP>(a, p);
    if (a->head_dim == 128) return run_attention<T, 128, CAP>(a, p);
    return run_attention<T, 256, CAP>(a, p);
}
template <typename T>
int by_head_dim(const TdistAttentionArgs* a, attention::Params& p) {
    using namespace attention;
    if (!(p.soft_cap > 0.f)) return by_head_dim<T, kUncapped>(a, p);
    return foldable(p.scale_log2 / (p.soft_cap * 1.4426950408889634f), p.scale_log2) ? by_head_dim<T, kFolded>(a, p) : by_head_dim<T, kUnfolded>(a, p);
}

int attention_impl(const TdistAttentionArgs* a) {
    if (a == nullptr) return fail(TDIST_EINVAL, "attention: null args");
    if (a->tokens < 1 || a->B < 1 || a->Hq < 1 || a->Hkv < 1 || a->Hq % a->Hkv) return fail(TDIST_EINVAL, "attention: bad token or head counts");
    if (a->Hq / a->Hkv > attention::kRows) return fail(TDIST_ELIMIT, "attention: at most 128 query heads per kv head");
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return fail(TDIST_EINVAL, "attention: head_dim must be 64, 128 or 256");
    if (a->page_size < 1 || a->max_blocks < 1 || a->blocks < 1) return fail(TDIST_EINVAL, "attention: page_size, max_blocks and blocks must be at least 1");
    if ((a->stride_token | a->stride_block | a->stride_head | a->q_token | a->q_head) % 8) return fail(TDIST_EINVAL, "attention: strides must be multiples of 8 elements");
    if ((reinterpret_cast<uintptr_t>(a->q) | reinterpret_cast<uintptr_t>(a->k_cache) | reinterpret_cast<uintptr_t>(a->v_cache) |
         reinterpret_cast<uintptr_t>(a->out)) % 16 || reinterpret_cast<uintptr_t>(a->part_o) % 32)
        return fail(TDIST_EINVAL, "attention: q, caches and output must be 16-byte aligned, partials 32-byte");
    if (a->splits < 1 || a->splits > 256) return fail(TDIST_EINVAL, "attention: splits must be in [1, 256]");
    if (a->row_tiles < 1 || a->row_tiles > 2 || (a->row_tiles == 2 && a->head_dim > 128)) return fail(TDIST_EINVAL, "attention: bad row_tiles");
    if (a->window < 1 || a->sinks < 0) return fail(TDIST_EINVAL, "attention: the window must be at least 1, sinks not negative");
    if (static_cast<long long>(a->tokens) * a->Hq > 0x7fffffffLL) return fail(TDIST_ELIMIT, "attention: tokens * Hq exceeds 2^31 - 1");
    const bool parts = a->splits > 1 || a->out == nullptr;
    if (!a->q || !a->k_cache || !a->v_cache || !a->block_table || !a->kv_lens || (!a->shared && !a->q_starts) || (parts && (!a->part_o || !a->part_lse)))
        return fail(TDIST_EINVAL, "attention: null pointer");
    if (!(a->soft_cap >= 0.f)) return fail(TDIST_EINVAL, "attention: soft_cap must not be negative");
    attention::Params p;
    memset(&p, 0, sizeof(p));
    p.q = a->q;
    p.k_cache = a->k_cache;
    p.v_cache = a->v_cache;
    p.block_table = static_cast<const int*>(a->block_table);
    p.q_starts = static_cast<const int*>(a->q_starts);
    p.kv_lens = static_cast<const int*>(a->kv_lens);
    p.out = a->out;
    p.part_o = parts ? static_cast<float*>(a->part_o) : nullptr;
    p.part_lse = static_cast<float*>(a->part_lse);
    p.q_token = a->q_token;
    p.q_head = a->q_head;
    p.stride_head = a->stride_head;
    // offsets of a key in the cache as 32-bit numbers of the largest unit that divides both strides (at least 16 bytes: 64 GB per cache)
    const long long strides = a->stride_block | a->stride_token;
    p.unit_shift = strides == 0 ? 3 : __builtin_ctzll(static_cast<unsigned long long>(strides));
    if (p.unit_shift > 16) p.unit_shift = 16;
    const long long units = (a->stride_block >> p.unit_shift) * (a->blocks - 1LL) + (a->stride_token >> p.unit_shift) * (a->page_size - 1LL);
    if (a->stride_block < 0 || a->stride_token < 0 || a->stride_head < 0 || units >= 0xffffffffLL) return fail(TDIST_ELIMIT, "attention: cache strides negative or beyond 2^32 units");
    p.unit_block = static_cast<uint32_t>(a->stride_block >> p.unit_shift);
    p.unit_token = static_cast<uint32_t>(a->stride_token >> p.unit_shift);
    p.tokens = a->tokens;
    p.B = a->B;
    p.Hq = a->Hq;
    p.Hkv = a->Hkv;
    p.G = a->Hq / a->Hkv;
    p.page_size = a->page_size;
    p.page_shift = (a->page_size & (a->page_size - 1)) == 0 ? __builtin_ctz(static_cast<unsigned>(a->page_size)) : -1;
    p.max_blocks = a->max_blocks;
    p.blocks = a->blocks;
    p.splits = a->splits;
    p.tile_tokens = attention::kRows / p.G;
    p.shared = a->shared;
    p.window = a->shared ? 0x7fffffff : a->window;
    p.sinks = a->shared ? 0 : a->sinks;
    p.scale_log2 = (a->scale < 0.f ? -a->scale : a->scale) * 1.4426950408889634f;
    p.soft_cap = a->soft_cap;
    // a scale of zero: scores of zero, through q (the kernel's factor stays positive, so that masked scores stay -inf)
    p.q_and = a->scale == 0.f ? 0u : 0xffffffffu;
    p.q_xor = a->scale < 0.f ? 0x80008000u : 0u;
    if (a->scale == 0.f) p.scale_log2 = 1.f;
    // TMA: boxes of as many rows as divide both a page and a block of keys, at least the swizzle's eight
    int rows = a->page_size & -a->page_size;
    if (rows > attention::kKeys) rows = attention::kKeys;
    if (rows >= 8 && a->stride_token > 0 && a->stride_block > 0 && a->stride_head > 0) {
        const uint64_t dims[4] = {static_cast<uint64_t>(a->head_dim), static_cast<uint64_t>(a->Hkv), static_cast<uint64_t>(a->page_size), static_cast<uint64_t>(a->blocks)};
        const uint64_t bytes[3] = {static_cast<uint64_t>(a->stride_head) * 2, static_cast<uint64_t>(a->stride_token) * 2, static_cast<uint64_t>(a->stride_block) * 2};
        const uint32_t box[4] = {64, 1, static_cast<uint32_t>(rows), 1};
        const CUtensorMapDataType type = a->dtype == TDIST_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
        int rc = tdist_host::encode_tmap(&p.tm_k, type, 2, 4, a->k_cache, dims, bytes, box, tdist_host::Swizzle::B128, false);
        if (rc == 0) rc = tdist_host::encode_tmap(&p.tm_v, type, 2, 4, a->v_cache, dims, bytes, box, tdist_host::Swizzle::B128, false);
        if (rc != 0) return rc;
        p.box_rows = rows;
    }
    p.wctx.status = static_cast<Status*>(a->status);
    p.wctx.timeout_ns = a->timeout_ns;
    p.wctx.kernel_id = attention::kKernelAttention;
    if (a->dtype == TDIST_BF16) return by_head_dim<__nv_bfloat16>(a, p);
    if (a->dtype == TDIST_F16) return by_head_dim<__half>(a, p);
    return fail(TDIST_EINVAL, "attention: dtype must be bf16 or fp16");
}

}  // namespace

extern "C" int tdist_attention(const TdistAttentionArgs* a) { return attention_impl(a); }
