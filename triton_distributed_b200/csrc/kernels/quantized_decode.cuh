// Decode attention over a paged KV cache in 8 or 4 bits (format: quantized_cache.cu), one query token per sequence.
//
//   s_j = scale q . k_j, k_j = ks_j c_j             4 bits: k_j = step_jg c_j + least_jg in every group g of 64 dimensions
//   o   = sum_j p_j vs_j c'_j / sum_j p_j           p_j = exp(s_j - max)
//
// The rows are never dequantised: the scales are applied where they are one number per key, to the score (4 bits: to a group's part of it, and
// least_jg times the sum of q over the group is added), and to the weight p_j vs_j, with the sum of p_j least_jg kept beside the product.
//
// K. Codes are 8-bit operands of the integer MMA (m16n8k32, u8 x s8) as they lie in memory, 4-bit ones after two logic instructions
// per eight. A query is brought to 16 bits for it, times the power of two that takes its largest element to 2^14 and above, as a high and a low byte
// with a product each: the sums are exact, the second continues from 256 times the first, and 128 times the sum of q takes the codes' offset off. (As fp16 operands the codes of a tile cost 64
// instructions, and the kernel was bound by its issue slots: 567 per tile of 16 x 128, 32 x 16384 keys of 8 kv heads 148 us.)
// Elements down to 2^-6 of the largest are exact in bf16 (2^-3 in fp16), smaller ones off by up to max |q| / 32640, and a score by that times the sum of
// their |k_d| scale. (With 32512 / max |q| every element was rounded, and above 2^126, where a fast quotient is zero, the query was lost.)
//
// V. Codes become fp16, exactly, two tokens per register. The weights p_j vs_j of a head (4 bits: p_j step_jg of a head and group) are held in units of a power of two
// that follows the largest of them so far: 2^-5 of it or less where it is set, down again as the maximum of the scores rises. So they stay below 2^15 whatever the values' magnitude, and
// rounded to fp16 one is off by 2^-11 of itself, or by 2^-25 of a unit, 2^-30 of the largest (one below 2^-126 is zero). In units of the largest scale, which may be one
// of a key that weighs nothing, a value 2^25 times the others took the others' weights away; looking at weights and factors costs heads of 256 2 %, 4 bits with fp16 results 2 %.
// For fp16 results what that rounding left is a second weight (without it errors of 3.0e-4 of a result where its own rounding is 2.1e-4). 4-bit codes are taken as c - 8 with least + 8 step, so that the sums stay small.
//
// As in the plain decode tokens are the 16 rows of the MMA and query heads its 8 columns (two tiles of them above 8 heads per kv head):
// S^T = K Q^T, O^T = V^T P^T, P transposed by movmatrix, and every warp streams tiles of 16 tokens through a cp.async ring of its own.
// The sum over a row's dimensions may run in any order, the output's dimensions may be dealt to the MMA's rows in any order and so may the
// tokens, so all three are chosen by what a wide load from shared memory gives: of 64 dimensions of a key, the four lanes of a quad take 16 neighbouring
// ones each, and of a value's each eighth lane an eighth. Not by TMA: a box of 16 rows of one head costs it some 5 clocks a row and SM, whatever the rows' width
// (16 x 16384 keys of 8 kv heads of 128, loads alone: 4 bits 75 us, these copies 55; 8 bits 93 and 88). Not straight into registers: too few bytes under
// way, warps waited for memory half of their time.
//
// Work. A segment is the keys of one (sequence, kv head, tile of query heads), cut into tiles of 16 tokens. Either a segment has `splits` CTAs, up to 8, a
// cluster that exchanges slices of the sums (CTA r adds up the r-th slice of all parts); or, where there are many short ones, a small CTA of two or four
// warps each; or the machine is filled once by groups of CTAs, one
// for each segment of a sequence, and every group takes an equal share of all sequences' tiles in a row, from the lengths on the device: pieces
// of sequences, of which the first and the last may be shared with other groups. Those leave their sums in a workspace, and a second kernel
// adds them up. (The heads of a key lie side by side in memory, so they are read side by side: with shares dealt out head by head 4-bit rows of 64 bytes were
// read from HBM twice, and 16 x 16384 keys took 107 us in 8 bits.) The copies run on from one piece to the next: while a piece's sums meet,
// the next one's first tiles are under way. No counters: nothing has to be zero before a call, and calls share nothing.
//
// Measured, heads of 128, 8 of kv, 4 query heads each, 16 x 16384 keys: 8 bits 92 us, 6.0 TB/s of codes and scales, HBM. 4 bits 91 us where HBM would take
// 46: a chain of dependent steps per tile (loads from shared memory, unpacking, integer MMAs, scales, exponentials, transposes, fp16 MMAs) in three warps per scheduler. No unit is full:
// 426 instructions per tile of 16 tokens, issue slots 61 % busy, the integer pipe 53 %, the tensor pipe 27 %, 1.2 warps ready per cycle at 1.77 GHz. One
// sequence of 4096 keys, 8 bits: 9.7 us (10.5 where L2 has lost the inputs), a chain of latencies: length, page, codes, merge.

#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <atomic>
#include <cstring>
#include <string>

#include "../device/ptx.cuh"
#include "../device/soft_cap.cuh"
#include "../include/tdist.h"
#include "../runtime/host_common.h"

namespace tdist {
namespace qdecode {

constexpr int TOK = 16;          // tokens of a tile
constexpr int MAX_CLUSTER = 8;
// The maximum that weights are relative to is raised, and the sums scaled, when two weights of a lane come to more than 2^8 (4 bits, 524288 keys 162.7 us, 166.4
// where more than 2 raises it). Before the first score it is fp32's lowest number.
constexpr float kMostPair = 256.f, kNoScore = -3.4028234663852886e38f;
constexpr float kLog2e = 1.4426950408889634f;
// A product of codes is multiplied by the query's factor before the key's scale, so that a huge key beside a small query stays in fp32; a factor outside 2^-60 .. 2^60
// is taken in two steps, the other one behind the key's scale.
constexpr float kFactor = 1152921504606846976.f;
// Units of weights: powers of two from 2^-110, far below the least scale there is, to 2^123, as biased exponents. A new one is at least 2^-5 and more
// than 2^-6 of the largest weighted scale, which is looked for among products with 2^-20.
constexpr int kLeastExponent = 17, kMostExponent = 250, kTopExponent = 20 - 5;
constexpr float kLeastUnit = 7.703719777548943e-34f, kTopScale = 9.5367431640625e-07f;   // 2^-110, 2^-20

struct Params {
    const void* q;                 // [B, Hq, D]
    const uint8_t *k, *v;
    const char *ks, *vs;
    const int *table, *lens;
    float* part;                   // shares: [CTAs][2][8 NH][D + 2]: sums, maximum, sum of weights of a CTA's first and last piece
    int4* info;                    // shares: [CTAs]: the segment that this CTA's first piece goes on with (see merge_kernel)
    void* out;
    long long code_block, code_token, code_head, scale_block, scale_head, scale_token;   // bytes
    int B, shares;                 // shares: groups of CTAs that share all tiles equally, 0: `splits` CTAs per segment
    int Hq, Hkv, head_tiles, page_size, page_shift, max_blocks, blocks, splits, window, sinks, table_keys;
    float scale, soft_cap;
    uint32_t page_mul;             // not PAGED: t / page_size = (t page_mul) >> page_shift for t < 2^31
};

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t a) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
    return r;
}
__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same from c0 (rows of a register pair's first column) and c1
__device__ __forceinline__ void mma_u8s8_from(int (&d)[4], int c0, int c1, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %10, %11};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c0), "r"(c1));
}
// Codes as operands of the fp16 MMA, exactly. A byte n under the exponent of 1024 is 1024 + n, from which 1152 is taken. A nibble n alone is the subnormal n 2^-24,
// and in the upper nibble of a byte n 2^-20: rows of the MMA that take those are off by 16 until the end, and the offset of 8 is taken off by a product of its
// own with the same weights, one MMA for four subtractions (when it was brought in: 64 ragged sequences to 16384 keys of 8 kv heads 193 us, 210 with subtractions; 8 bits, whose
// weights are two numbers in fp16 and would need two such products, 16 x 16384 keys 98 and 94). The sums stay small either way; with the offset
// in them until the end, their roundings come to 1.5e-3 of a flat result over 524288 keys.
constexpr uint32_t kMagic = 0x64006400u;
constexpr uint32_t kLowBytes = 0x7150u, kHighBytes = 0x7352u;   // bytes 0, 1 / 2, 3 of a word, each under a 0x64
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t w, uint32_t sel) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(__byte_perm(w, kMagic, sel)), "r"(0x64806480u));
    return r;
}
__device__ __forceinline__ uint32_t low_nibbles(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t high_nibbles(uint32_t w) { return w & 0x00f000f0u; }
constexpr uint32_t kLowOffset = 0x80088008u, kHighOffset = 0x80808080u;   // -8 2^-24, -8 2^-20
// of a power of two whose inverse is a normal number too
__device__ __forceinline__ float one_over(float power) { return __uint_as_float((254u << 23) - __float_as_uint(power)); }
__device__ __forceinline__ uint32_t pack_bytes(int a, int b, int c, int d) {
    return __byte_perm(__byte_perm(static_cast<uint32_t>(a), static_cast<uint32_t>(b), 0x0040u), __byte_perm(static_cast<uint32_t>(c), static_cast<uint32_t>(d), 0x0040u), 0x5410u);
}

__device__ __forceinline__ uint32_t ldg32(const void* p) {
    uint32_t v;
    asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
template <int W>
struct Words { uint32_t w[W]; };
// W words from p, aligned to their size (W up to 4) or to 16 bytes
template <int W>
__device__ __forceinline__ Words<W> load_words(const void* p) {
    Words<W> r;
    if constexpr (W == 1) {
        r.w[0] = ldg32(p);
    } else if constexpr (W == 2) {
        asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "l"(p));
    } else {
#pragma unroll
        for (int i = 0; i < W / 4; ++i)
            asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(r.w[4 * i]), "=r"(r.w[4 * i + 1]), "=r"(r.w[4 * i + 2]), "=r"(r.w[4 * i + 3])
                         : "l"(static_cast<const char*>(p) + 16 * i));
    }
    return r;
}

// A tile in shared memory: 16 rows of K codes, 16 of V codes, the rows' scales. The 16-byte chunks of a row are swizzled with its number (rows
// of 256 bytes as two halves of 128), and the MMA's rows are tokens in an order that makes
// the loads below free of bank conflicts but for two of K's in twos (4 bits, heads of 64 and 256): a key's load takes two rows whose tokens differ in
// bit 0, or four whose tokens differ in bits 0 and 2, and a value's four columns whose tokens differ in bits 0 and 2, and in bits 1 and 2.
template <int BITS, int D>
struct Shape {
    static constexpr int NG = BITS == 8 ? 1 : D / 64;      // scales of a row
    static constexpr int KC = D / 64;                      // 64-dimension chunks of a key
    static constexpr int KW = BITS == 8 ? 4 : 2;           // words of a chunk and lane
    // values: VC chunks, of each of which a lane holds an eighth of the dimensions in VW words
    static constexpr int VC = BITS == 4 ? D / 64 : (D == 256 ? 2 : 1);
    static constexpr int VD = D / VC / 8;                  // dimensions of a chunk and lane
    static constexpr int VW = VD * BITS / 32;
    static constexpr int VB = D * BITS / 8 / VC;           // bytes of a chunk
    static constexpr int MT = D / 16;                      // MMAs of a tile
    static constexpr int ROW = D * BITS / 8;               // bytes of a row
    static constexpr int BOX = ROW < 128 ? ROW : 128;      // bytes of a row that lie together
    static constexpr int SB = 4 * NG;                      // bytes of its scales
    static constexpr int TILE = TOK * ROW;                 // K; V behind it
    static constexpr int SCALES = TOK * SB;                // K's; V's behind them
    static constexpr int STAGE = 2 * TILE + 2 * SCALES;

    static __device__ __forceinline__ uint32_t at(int t, int byte) {
        const int chunk = (byte & (BOX - 1)) >> 4;
        const int swizzled = BOX == 32 ? chunk ^ ((t >> 2) & 1) : (BOX == 64 ? chunk ^ ((t >> 1) & 3) : chunk ^ (t & 7));
        return static_cast<uint32_t>((byte / BOX) * (TOK * BOX) + t * BOX + swizzled * 16 + (byte & 15));
    }
    // the 16 dimensions of 64-dimension chunk j that lane c of a quad holds: 8 bits 16 neighbouring codes, 4 bits 8 bytes of a group
    static __device__ __forceinline__ int k_byte(int j, int c) {
        return BITS == 4 ? j * 32 + c * 8 : (D == 64 ? c * 16 : ((j >> 1) * 8 + 2 * c + (j & 1)) * 16);
    }
};
// token that row r of the MMA is
__device__ __forceinline__ int token_of(int r) { return static_cast<int>((0x76234510u >> (4 * (r & 7))) & 7u) + (r & 8); }

// O and what belongs to it, per warp, in shared memory: heads [8 NH] rows of D + 4 floats
__host__ __device__ constexpr int o_pitch(int d) { return d + 4; }

template <int W>
__device__ __forceinline__ Words<W> lds_words(uint32_t at) {
    Words<W> r;
    if constexpr (W == 1) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(r.w[0]) : "r"(at));
    else if constexpr (W == 2) asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(r.w[0]), "=r"(r.w[1]) : "r"(at));
    else asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3]) : "r"(at));
    return r;
}
// `none`: zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool none) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tcp.async.cg.shared.global [%0], [%1], 16, p;\n\t}" ::"r"(dst), "l"(src),
                 "r"(static_cast<uint32_t>(none))
                 : "memory");
}
template <int N>
__device__ __forceinline__ void copy_small(uint32_t dst, const void* src, bool none) {
    if constexpr (N == 16) copy16(dst, src, none);
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %2, 0;\n\tcp.async.ca.shared.global [%0], [%1], %3, p;\n\t}" ::"r"(dst), "l"(src),
                     "r"(static_cast<uint32_t>(none)), "n"(N)
                     : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory behind the rings: buffers in which the warps' sums meet, q, then a cluster's slices or the shares' lengths and prefix sums.
constexpr int MAX_SHARED = 511;   // sequences of a call that is dealt out in shares
// CTAs per SM and their warps: two of six, which then have up to 168 registers per thread, or one of eight where a thread needs more. SMALL: as many
// warps in three or two times as many CTAs, each of which has all keys of a segment.
__host__ __device__ constexpr bool wide_of(int d, int nh) { return d == 256 || nh == 2; }
__host__ __device__ constexpr int ctas_per_sm(int d, int nh, bool small) { return wide_of(d, nh) ? (small ? 2 : 1) : (small ? 6 : 2); }
__host__ __device__ constexpr int warps_of(int d, int nh, bool small) { return wide_of(d, nh) ? (small ? 4 : 8) : (small ? 2 : 6); }
__host__ __device__ constexpr int buffers_of(int d, int nh, bool small) { return wide_of(d, nh) && d != 256 && !small ? 4 : 2; }
// (SMALL: the sums meet in the rings' places, and there are neither slices nor lengths)
__host__ __device__ constexpr int sums_bytes(int d, int nh, bool small) { return small ? 0 : buffers_of(d, nh, small) * 8 * nh * o_pitch(d) * 4; }
__host__ __device__ constexpr int last_bytes(int d, int nh, bool small) {
    return small ? 0 : ((8 * nh * d + 4 * MAX_CLUSTER) * 4 > 8 * (MAX_SHARED + 1) ? (8 * nh * d + 4 * MAX_CLUSTER) * 4 : 8 * (MAX_SHARED + 1));
}
__host__ __device__ constexpr int behind_rings(int d, int nh, bool small) { return sums_bytes(d, nh, small) + 16 * nh * d + last_bytes(d, nh, small); }
// tiles that a warp's ring has room for, 8 at most: of 228 KB per SM, 1 KB per CTA the system's and 2 KB for static shared memory
__host__ __device__ constexpr int stages_of(int stage, int d, int nh, bool small) {
    const int each = (228 * 1024 / ctas_per_sm(d, nh, small) - 3 * 1024 - behind_rings(d, nh, small)) / stage / warps_of(d, nh, small);
    return each < 8 ? each : 8;
}

// A sequence's keys as tiles: those of the first `first` tokens, then those from the window's first token on (a tile's first token is a multiple of 16)
struct Keys {
    int n, lo, first, sink_tiles, t_lo, tiles;
    __device__ __forceinline__ int first_token(int i) const { return (i < sink_tiles ? i : i - sink_tiles + t_lo) * TOK; }
};
__device__ __forceinline__ Keys keys_of(const Params& p, int length) {
    Keys k;
    k.n = min(max(length, 0), p.table_keys);
    k.lo = max(0, k.n - p.window);
    k.first = min(p.sinks, k.lo);
    k.sink_tiles = (k.first + TOK - 1) / TOK;
    k.t_lo = k.lo / TOK;
    k.tiles = k.sink_tiles + (k.n + TOK - 1) / TOK - k.t_lo;
    return k;
}

// Tiles i0 .. i1 - 1 of sequence b
struct Piece {
    int b, i0, i1;
};
// The pieces of this CTA, one after the other
struct Pieces {
    const uint32_t* prefix;   // shares: tiles of the sequences before b; nullptr: one piece
    uint32_t at, end;         // tiles of this CTA; one piece: whether it is still to come
    int b, i0, i1;

    __device__ __forceinline__ bool next(Piece& x) {
        if (at >= end) return false;
        if (prefix == nullptr) {
            x = Piece{b, i0, i1};
            at = end;
            return true;
        }
        while (prefix[b + 1] <= at) ++b;
        x.b = b;
        x.i0 = static_cast<int>(at - prefix[b]);
        const uint32_t take = min(prefix[b + 1] - at, end - at);
        x.i1 = x.i0 + static_cast<int>(take);
        at += take;
        return true;
    }
};

template <int BITS, int D, int NH, bool PAGED, bool F16, bool SMALL>
__global__ void __launch_bounds__(32 * warps_of(D, NH, SMALL), ctas_per_sm(D, NH, SMALL)) decode_kernel(const __grid_constant__ Params p) {
    using S = Shape<BITS, D>;
    constexpr int WARPS = warps_of(D, NH, SMALL), THREADS = 32 * WARPS, BUFS = buffers_of(D, NH, SMALL);
    constexpr int HEADS = 8 * NH, OP = o_pitch(D), STAGES = stages_of(S::STAGE, D, NH, SMALL);
    static_assert(!SMALL || WARPS * STAGES * S::STAGE >= BUFS * HEADS * OP * 4, "the sums meet in the rings");
    static_assert(STAGES >= 3, "two tiles ahead at least");
    extern __shared__ __align__(128) uint8_t smem[];
    // rings [WARPS][STAGES][STAGE], the sums' buffers, q as bytes [2][HEADS][D], a cluster's slices or lengths and prefix sums
    float* sums_s = reinterpret_cast<float*>(smem + (SMALL ? 0 : WARPS * STAGES * S::STAGE));   // [BUFS][HEADS][OP]
    uint8_t* q_s = smem + WARPS * STAGES * S::STAGE + sums_bytes(D, NH, SMALL);
    uint8_t* last_s = q_s + 2 * HEADS * D;
    __shared__ float m_s[BUFS][HEADS], l_s[BUFS][HEADS];
    __shared__ float factor_s[HEADS], far_s[HEADS], qsum_s[HEADS][S::NG];
    __shared__ int bias_s[HEADS];
    __shared__ float part_m[MAX_CLUSTER][HEADS], part_l[MAX_CLUSTER][HEADS];
    __shared__ uint32_t scan_s[WARPS];
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = static_cast<int>(threadIdx.x) & 31;
    const int g = lane >> 2, c = lane & 3;
    const bool in_cluster = !SMALL && p.shares == 0 && p.splits > 1, in_shares = !SMALL && p.shares > 0;
    if (in_cluster) cluster_arrive();                       // waited for before the first store into another CTA
    pdl_wait_and_release();

    const int G = p.Hq / p.Hkv;
    const int split = in_cluster ? static_cast<int>(blockIdx.x) % p.splits : 0;
    Pieces pieces;
    pieces.prefix = nullptr;
    const int per_b = p.Hkv * p.head_tiles;                 // segments of a sequence
    const int group = static_cast<int>(blockIdx.x) / (in_shares ? per_b : p.splits);   // shares: this CTA's group; otherwise its segment
    const int of_b = in_shares ? static_cast<int>(blockIdx.x) % per_b : group % per_b;
    const int kvh = of_b / p.head_tiles, tile_of_heads = of_b % p.head_tiles;
    const int heads = min(HEADS, G - tile_of_heads * HEADS);
    const int head_of_b = kvh * G + tile_of_heads * HEADS;
    if (in_shares) {
        uint32_t* prefix = reinterpret_cast<uint32_t*>(last_s);
        int* lens = reinterpret_cast<int*>(last_s) + MAX_SHARED + 1;
        uint32_t carry = 0;
        for (int b0 = 0; b0 < p.B; b0 += THREADS) {
            const int b = b0 + static_cast<int>(threadIdx.x);
            const int length = b < p.B ? p.lens[b] : 0;
            if (b < p.B) lens[b] = length;
            uint32_t sum = static_cast<uint32_t>(keys_of(p, length).tiles);
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t v = __shfl_up_sync(0xffffffffu, sum, o);
                sum += lane >= o ? v : 0u;
            }
            if (lane == 31) scan_s[warp] = sum;
            __syncthreads();
            uint32_t all = 0;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                if (w == warp) sum += carry + all;
                all += scan_s[w];
            }
            if (b < p.B) prefix[b + 1] = sum;
            carry += all;
            __syncthreads();
        }
        if (threadIdx.x == 0) prefix[0] = 0;
        __syncthreads();
        const uint32_t total = carry, groups = min(static_cast<uint32_t>(p.shares), total);   // all tiles, the groups that have some
        auto first_of = [&](uint32_t of) { return static_cast<uint32_t>(static_cast<uint64_t>(of) * total / groups); };
        auto group_of = [&](uint32_t tile) { return static_cast<uint32_t>(((static_cast<uint64_t>(tile) + 1) * groups - 1) / total); };
        const uint32_t mine = static_cast<uint32_t>(group);
        pieces.b = 0;
        pieces.at = pieces.end = 0;
        if (mine < groups) {
            pieces.at = first_of(mine);
            pieces.end = first_of(mine + 1);
            int lo = 0, hi = p.B;   // the sequence of the first tile: the last one that starts at it or before (those without tiles start where the next does)
            while (hi - lo > 1) {
                const int m = (lo + hi) >> 1;
                if (prefix[m] <= pieces.at) lo = m;
                else hi = m;
            }
            pieces.b = lo;
        }
        pieces.prefix = prefix;
        if (threadIdx.x == 0) {
            // for the second kernel: head 0 and heads of the segment that goes on here, where its first sums are, the last CTA that has some
            int4 info = make_int4(-1, 0, 0, 0);
            if (mine < groups && pieces.at > prefix[pieces.b]) {
                const uint32_t start = prefix[pieces.b], g0 = group_of(start), g1 = group_of(prefix[pieces.b + 1] - 1);
                if (mine == g0 + 1)   // (the sequence is that group's first piece or its last)
                    info = make_int4(pieces.b * p.Hq + head_of_b, heads, static_cast<int>(2 * (g0 * per_b + of_b) + (first_of(g0) == start ? 0 : 1)), static_cast<int>(g1 * per_b + of_b));
            }
            p.info[blockIdx.x] = info;
        }
        // sequences without keys
        for (int b = static_cast<int>(blockIdx.x); b < p.B; b += static_cast<int>(gridDim.x))
            if (prefix[b + 1] == prefix[b])
                for (int i = static_cast<int>(threadIdx.x); i < p.Hq * D / 2; i += THREADS) static_cast<uint32_t*>(p.out)[static_cast<size_t>(b) * (p.Hq * D / 2) + i] = 0u;
    } else {
        pieces.b = group / per_b;
        const int tiles = keys_of(p, p.lens[pieces.b]).tiles, per = (tiles + p.splits - 1) / p.splits;
        pieces.i0 = min(split * per, tiles);
        pieces.i1 = min((split + 1) * per, tiles);
        pieces.at = 0;
        pieces.end = 1;
    }
    auto keys_in = [&](int b) { return keys_of(p, in_shares ? reinterpret_cast<const int*>(last_s)[MAX_SHARED + 1 + b] : p.lens[b]); };

    // ---- The copies. A cursor goes over this warp's tiles of all pieces, STAGES - 1 of them ahead of the sums. PAGED (pages of 16, 32, 64 .. tokens): a tile lies
    // in one page, every lane knows where. Otherwise lane r and r + 16 look token r up and tell the others. -1: not seen; rows that are
    // not seen, or whose page the cache does not have, are zeros.
    constexpr int CHUNKS = S::ROW / 16, ROWS = 32 / CHUNKS;   // a warp copies ROWS rows at once, 16 bytes a lane
    const int lrow = lane / CHUNKS, lchunk = lane % CHUNKS, my_token = lane & 15;
    const uint32_t ring = smem_u32(smem) + static_cast<uint32_t>(warp * STAGES * S::STAGE);
    uint32_t dst_at[TOK / ROWS];
#pragma unroll
    for (int j = 0; j < TOK / ROWS; ++j) dst_at[j] = S::at(j * ROWS + lrow, lchunk * 16);
    const uint32_t code_token = static_cast<uint32_t>(p.code_token);   // PAGED: strides fit 32 bits
    const uint64_t code_rows = static_cast<uint64_t>(code_token) * ROWS;
    auto in_table = [&](int t) {
        return PAGED ? t >> p.page_shift : static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(t)) * p.page_mul) >> p.page_shift);
    };
    Pieces coming = pieces;
    Keys c_keys = keys_of(p, 0);
    const int* c_table = p.table;
    const uint8_t* c_k = p.k + kvh * p.code_head + lchunk * 16 + (PAGED ? lrow * p.code_token : 0);
    const uint8_t* c_v = p.v + kvh * p.code_head + lchunk * 16 + (PAGED ? lrow * p.code_token : 0);
    const ptrdiff_t v_from_k = static_cast<ptrdiff_t>(reinterpret_cast<uintptr_t>(c_v) - reinterpret_cast<uintptr_t>(c_k));   // (an instruction less than two sums)
    // lanes 0..15 copy the scales of the keys, 16..31 of the values
    const char* c_s = (lane < 16 ? p.ks : p.vs) + kvh * p.scale_head + (PAGED ? my_token * p.scale_token : 0);
    // A run: tiles whose tokens follow one another (the first keys, or the window's). Tiles left of it, the next one's first token (not PAGED: this lane's),
    // the last one's, the next one's page; whether there are no more
    int c_left = 0, c_t = 0, c_last = 0, c_page = -1;
    int c_i = 0, c_end = 0, c_turn = 0;   // the piece's next tile behind the run, its end
    bool c_done = false;
    auto page_of = [&]() {
        const bool seen = !c_done && (PAGED || c_t < c_keys.first || (c_t >= c_keys.lo && c_t < c_keys.n));
        return seen ? static_cast<int>(ldg32(c_table + in_table(c_t))) : -1;
    };
    auto new_run = [&]() {
        while (c_i >= c_end) {
            Piece x;
            if (!coming.next(x)) {
                // nothing from here on: what is "copied" are zeros
                c_left = 0x7fffffff;
                c_last = c_t;
                c_page = -1;
                c_done = true;
                return;
            }
            c_keys = keys_in(x.b);
            c_table = p.table + static_cast<size_t>(x.b) * p.max_blocks;
            c_i = x.i0 + (warp + WARPS - c_turn) % WARPS;
            c_end = x.i1;
            c_turn = (c_turn + x.i1 - x.i0) % WARPS;
        }
        const int stop = c_i < c_keys.sink_tiles ? min(c_keys.sink_tiles, c_end) : c_end;
        c_left = (stop - c_i + WARPS - 1) / WARPS;
        c_t = c_keys.first_token(c_i) + (PAGED ? 0 : my_token);
        c_last = c_t + (c_left - 1) * (WARPS * TOK);
        c_i += c_left * WARPS;
        c_page = page_of();
    };
    auto copy_next = [&](uint32_t to) {
        if (c_left == 0) new_run();
        const bool live = static_cast<unsigned>(c_page) < static_cast<unsigned>(p.blocks);
        const uint32_t from = live ? static_cast<uint32_t>(c_page) : 0u;
        if (PAGED) {
            const uint32_t row = static_cast<uint32_t>(c_t) & static_cast<uint32_t>(p.page_size - 1);
            const uint64_t off = static_cast<uint64_t>(from) * static_cast<uint32_t>(p.code_block) + static_cast<uint64_t>(row) * code_token;
            const uint8_t *k = c_k + off, *v = k + v_from_k;
#pragma unroll
            for (int j = 0; j < TOK / ROWS; ++j) {
                copy16(to + dst_at[j], k, !live);
                copy16(to + dst_at[j] + S::TILE, v, !live);
                k += code_rows;
                v += code_rows;
            }
            copy_small<S::SB>(to + 2 * S::TILE + lane * S::SB, c_s + (static_cast<uint64_t>(from) * static_cast<uint32_t>(p.scale_block) + row * static_cast<uint32_t>(p.scale_token)), !live);
        } else {
            const int row = c_t - in_table(c_t) * p.page_size;
            const long long off = live ? from * p.code_block + row * p.code_token : 0;
#pragma unroll
            for (int j = 0; j < TOK / ROWS; ++j) {
                const long long at = __shfl_sync(0xffffffffu, off, j * ROWS + lrow);
                const bool none = !__shfl_sync(0xffffffffu, static_cast<int>(live), j * ROWS + lrow);
                copy16(to + dst_at[j], c_k + at, none);
                copy16(to + dst_at[j] + S::TILE, c_v + at, none);
            }
            copy_small<S::SB>(to + 2 * S::TILE + lane * S::SB, c_s + (live ? from * p.scale_block + row * p.scale_token : 0), !live);
        }
        copy_commit();
        --c_left;
        c_t = c_t < c_last ? c_t + WARPS * TOK : c_last;   // (no further than a token whose page the table has)
        c_page = page_of();
    };
#pragma unroll 1
    for (int a = 0; a < STAGES - 1; ++a) copy_next(ring + a * S::STAGE);

    // what this lane reads of a tile: tokens of rows g and g + 8 of the MMA (keys and scales), of columns 2 c, 2 c + 1, 2 c + 8, 2 c + 9 (values)
    const int t_row = token_of(g);
    uint32_t k_at[S::KC], v_at[2][S::VC];
#pragma unroll
    for (int j = 0; j < S::KC; ++j) k_at[j] = S::at(t_row, S::k_byte(j, c));
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < S::VC; ++j) v_at[r][j] = S::TILE + S::at(token_of(2 * c + r), j * S::VB + g * (S::VB / 8));   // tokens 8 further on: 8 rows
    const float cap_inv = p.soft_cap > 0.f ? 1.f / p.soft_cap : 0.f;
    constexpr bool FINE = F16;   // weights as two fp16 numbers, what the first one's rounding leaves in the second
    uint32_t stage = ring, free_stage = ring + (STAGES - 1) * S::STAGE;
    int turn = 0;            // the warp that has a piece's first tile: tiles go round the warps from piece to piece
    bool first_piece = true;
    Piece x;
    while (pieces.next(x)) {
    const Keys keys = keys_in(x.b);
    const size_t head0 = static_cast<size_t>(x.b) * p.Hq + head_of_b;
    const int i0 = x.i0 + (warp + WARPS - turn) % WARPS, i1 = x.i1;
    // tiles that are seen whole
    const int whole0 = keys.sink_tiles - keys.t_lo + (keys.lo + TOK - 1) / TOK;
    const unsigned whole = static_cast<unsigned>(max(0, keys.sink_tiles - keys.t_lo + keys.n / TOK - whole0));

    // ---- q to 16 bits, a warp per head: the high and the low bytes in the order in which the codes' registers have their dimensions
    for (int head = warp; head < HEADS; head += WARPS) {
        constexpr int E = D / 32;                // dimensions of a lane
        float f[E];
        const bool there = head < heads;
        {
            const Words<E / 2> w = load_words<E / 2>(static_cast<const char*>(p.q) + (head0 + (there ? head : 0)) * (D * 2) + lane * (E * 2));
#pragma unroll
            for (int e = 0; e < E / 2; ++e) {
                if (F16) {
                    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w.w[e]));
                    f[2 * e] = t.x;
                    f[2 * e + 1] = t.y;
                } else {
                    f[2 * e] = __uint_as_float(w.w[e] << 16);
                    f[2 * e + 1] = __uint_as_float(w.w[e] & 0xffff0000u);
                }
            }
        }
        uint32_t top = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
        top = __reduce_max_sync(0xffffffffu, top);
        // magnitudes below 2^-100 count as that; a query with a NaN or an infinity has a factor of NaN, and so has its result. The power of two by
        // which the largest element comes to 2^14 .. 32639 (two signed bytes' largest): from 32640, whose upper eight bits are ones, half of it
        const bool good = top < 0x7f800000u;
        const uint32_t e_most = (max(good ? top : 0u, 27u << 23) + 0x10000u) >> 23;
        const float mul = there && good ? __uint_as_float((268u - e_most) << 23) : 0.f;
        int sum = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int v = __float2int_rn(f[e] * mul);
            const int hi = (v + 128) >> 8, d = lane * E + e;
            const int at = BITS == 8 ? d : (d & ~7) + (d & 1) * 4 + ((d >> 1) & 3);
            q_s[head * D + at] = static_cast<uint8_t>(hi);
            q_s[(HEADS + head) * D + at] = static_cast<uint8_t>(v - 256 * hi);
            sum += v;
        }
        constexpr int PER = 32 / S::NG;          // lanes of a group (8 bits: all)
#pragma unroll
        for (int o = 1; o < PER; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane % PER == 0) qsum_s[head][lane / PER] = static_cast<float>(sum);
        if (lane == 0) {
            bias_s[head] = BITS == 8 ? sum * -128 : 0;
            // the factor, or as much of it as lies in kFactor's range, and the rest
            const float power = __uint_as_float((e_most - 14u) << 23), scale = p.scale * (p.soft_cap > 0.f ? 1.f : kLog2e), both = power * scale;
            const bool near = fabsf(both) >= 1.f / kFactor && fabsf(both) <= kFactor;
            const float part = fminf(fmaxf(power, 1.f / kFactor), kFactor);
            factor_s[head] = !good ? __uint_as_float(0x7fffffffu) : (near ? both : part);
            far_s[head] = near ? 1.f : power / part * scale;
        }
    }
    __syncthreads();

    // ---- q as the second operand: column g of the MMA is head 8 h + g
    uint32_t qf[NH][S::KC][4][2];  // high and low bytes of four dimensions
    float factor[NH][2];           // of heads 8 h + 2 c + {0, 1}: what turns a product of codes, times the key's scale, into a score in units of log2
    bool more = p.soft_cap > 0.f;  // whether that is not all
    int bias[NH][2];               // 8 bits: -128 times the sum of the 16-bit q
    float qsum[NH][2][S::NG];      // 4 bits: that sum over a group, times the factor
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
        for (int j = 0; j < S::KC; ++j)
#pragma unroll
            for (int part = 0; part < 2; ++part) {
                const uint4 w = *reinterpret_cast<const uint4*>(q_s + (part * HEADS + 8 * h + g) * D + (BITS == 8 ? 1 : 2) * S::k_byte(j, c));
                qf[h][j][0][part] = w.x;
                qf[h][j][1][part] = w.y;
                qf[h][j][2][part] = w.z;
                qf[h][j][3][part] = w.w;
            }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            factor[h][r] = factor_s[8 * h + 2 * c + r];
            bias[h][r] = bias_s[8 * h + 2 * c + r];
#pragma unroll
            for (int k = 0; k < S::NG; ++k) qsum[h][r][k] = qsum_s[8 * h + 2 * c + r][k] * factor[h][r];
            more |= far_s[8 * h + 2 * c + r] != 1.f;
        }
    }

    // ---- sums: O^T in units of `unit` (a power of two), columns are heads 8 h + 2 c + {0, 1}
    float o[NH][S::MT][4];
    float m_run[NH][2], l_run[NH][2];   // weights are relative to 2^m_run, which is raised late
    float low[NH][2][S::NG];       // 4 bits: sum of p (least + 8 step), of this lane's tokens
    float inv_unit[NH][2][S::NG];  // 1 / unit
    float seconds[NH][2][S::NG];   // 4 bits, FINE: sum of the second weights, in units, of this lane's tokens
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
        for (int j = 0; j < S::MT; ++j) o[h][j][0] = o[h][j][1] = o[h][j][2] = o[h][j][3] = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            m_run[h][r] = kNoScore;
            l_run[h][r] = 0.f;
#pragma unroll
            for (int k = 0; k < S::NG; ++k) {
                low[h][r][k] = seconds[h][r][k] = 0.f;
                inv_unit[h][r][k] = one_over(kLeastUnit);
            }
        }
    }

    for (int i = i0; i < i1; i += WARPS) {
        copy_wait<STAGES - 2>();
        __syncwarp();   // the tile is here, and the place of the one before it is free
        copy_next(free_stage);
        const uint32_t scales = stage + 2 * S::TILE + static_cast<uint32_t>(t_row * S::SB);
        // ---- S^T = K Q^T, a sum per group of dimensions and byte of q
        float s[NH][4];
        Words<S::KW> kw[2][S::KC];
        Words<S::NG> kscale[2], vscale[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int j = 0; j < S::KC; ++j) kw[r][j] = lds_words<S::KW>(stage + k_at[j] + r * (8 * S::BOX));
            kscale[r] = lds_words<S::NG>(scales + r * (8 * S::SB));
            vscale[r] = lds_words<S::NG>(scales + S::SCALES + r * (8 * S::SB));
        }
        int acc[NH][S::NG][4], acc_low[NH][S::NG][4];
        uint32_t ka[S::KC][4][2];    // [chunk][register][token]
#pragma unroll
        for (int j = 0; j < S::KC; ++j)
#pragma unroll
            for (int r = 0; r < 2; ++r)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    ka[j][k][r] = BITS == 8 ? kw[r][j].w[k % S::KW] : (kw[r][j].w[(k >> 1) % S::KW] >> (4 * (k & 1))) & 0x0f0f0f0fu;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int k = 0; k < S::NG; ++k) {
#pragma unroll
                for (int j = k * (S::KC / S::NG); j < (k + 1) * (S::KC / S::NG); ++j)
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const uint32_t a0 = ka[j][2 * m][0], a1 = ka[j][2 * m][1], a2 = ka[j][2 * m + 1][0], a3 = ka[j][2 * m + 1][1];
                        if (m == 0 && j == k * (S::KC / S::NG)) {
                            mma_u8s8_from(acc[h][k], 0, 0, a0, a1, a2, a3, qf[h][j][0][0], qf[h][j][1][0]);
                            mma_u8s8_from(acc_low[h][k], bias[h][0], bias[h][1], a0, a1, a2, a3, qf[h][j][0][1], qf[h][j][1][1]);
                        } else {
                            mma_u8s8(acc[h][k], a0, a1, a2, a3, qf[h][j][2 * m][0], qf[h][j][2 * m + 1][0]);
                            mma_u8s8(acc_low[h][k], a0, a1, a2, a3, qf[h][j][2 * m][1], qf[h][j][2 * m + 1][1]);
                        }
                    }
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[h][k][e] = acc[h][k][e] * 256 + acc_low[h][k][e];
            }
        // ---- scales, cap; masks at the ends of what is seen
        bool higher = false;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = e >> 1;
                if (BITS == 8) {
                    s[h][e] = static_cast<float>(acc[h][0][e]) * factor[h][e & 1] * __uint_as_float(kscale[r].w[0]);
                } else {
                    s[h][e] = 0.f;
#pragma unroll
                    for (int k = 0; k < S::NG; ++k)
                        s[h][e] += __uint_as_float(kscale[r].w[k] << 16) * (static_cast<float>(acc[h][k][e]) * factor[h][e & 1]) + __uint_as_float(kscale[r].w[k] & 0xffff0000u) * qsum[h][e & 1][k];
                }
            }
        if (more) {
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[h][e] *= far_s[8 * h + 2 * c + (e & 1)];
                    if (p.soft_cap > 0.f) s[h][e] = soft_cap(s[h][e] * kLog2e, s[h][e] * cap_inv, p.soft_cap * kLog2e);
                }
        }
        // ---- the values' scales
        float vmul[2][S::NG], vleast[2][S::NG];
        if (static_cast<unsigned>(i - whole0) >= whole) {
            const int t0 = keys.first_token(i);
            const bool sink = i < keys.sink_tiles;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int t = t0 + t_row + 8 * r;
                const bool seen = sink ? t < keys.first : t >= keys.lo && t < keys.n;
#pragma unroll
                for (int h = 0; h < NH; ++h)
#pragma unroll
                    for (int e = 0; e < 2; ++e) s[h][2 * r + e] = seen ? s[h][2 * r + e] : -CUDART_INF_F;
#pragma unroll
                for (int k = 0; k < S::NG; ++k) vscale[r].w[k] = seen ? vscale[r].w[k] : 0;
            }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int k = 0; k < S::NG; ++k) {
                vmul[r][k] = __uint_as_float(BITS == 8 ? vscale[r].w[k] : vscale[r].w[k] << 16);
                if (BITS == 4) vleast[r][k] = fmaf(8.f, vmul[r][k], __uint_as_float(vscale[r].w[k] & 0xffff0000u));
            }
        // ---- P^T times the scales, in units, as the second operand: tokens in pairs per lane, heads over lane / 4
        float pr[NH][4], pair[NH][2], rest[NH][2][S::NG];
        uint32_t pb[NH][S::NG][2], pl[NH][S::NG][2];
        __half2 all;             // a sum of weights that is at least the largest
        auto weights = [&]() {
            all = __half2half2(__ushort_as_half(0));
#pragma unroll
            for (int h = 0; h < NH; ++h) {
#pragma unroll
                for (int e = 0; e < 4; ++e) pr[h][e] = exp2f(s[h][e] - m_run[h][e & 1]);
#pragma unroll
                for (int r = 0; r < 2; ++r) pair[h][r] = pr[h][r] + pr[h][2 + r];
#pragma unroll
                for (int k = 0; k < S::NG; ++k) {
                    const float w0 = pr[h][0] * vmul[0][k] * inv_unit[h][0][k], w1 = pr[h][1] * vmul[0][k] * inv_unit[h][1][k];
                    const float w2 = pr[h][2] * vmul[1][k] * inv_unit[h][0][k], w3 = pr[h][3] * vmul[1][k] * inv_unit[h][1][k];
                    const uint32_t a = pack_f16x2(w0, w1), bb = pack_f16x2(w2, w3);
                    all = __hadd2(__hadd2(all, *reinterpret_cast<const __half2*>(&a)), *reinterpret_cast<const __half2*>(&bb));
                    pb[h][k][0] = movmatrix_trans(a);
                    pb[h][k][1] = movmatrix_trans(bb);
                    if (FINE) {
                        const float2 ra = __half22float2(*reinterpret_cast<const __half2*>(&a)), rb = __half22float2(*reinterpret_cast<const __half2*>(&bb));
                        const float l0 = w0 - ra.x, l1 = w1 - ra.y, l2 = w2 - rb.x, l3 = w3 - rb.y;
                        pl[h][k][0] = movmatrix_trans(pack_f16x2(l0, l1));
                        pl[h][k][1] = movmatrix_trans(pack_f16x2(l2, l3));
                        rest[h][0][k] = l0 + l2;
                        rest[h][1][k] = l1 + l3;
                    }
                }
            }
        };
        weights();
        Words<S::VW> vw[4][S::VC];
        auto load_values = [&]() {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < S::VC; ++j) vw[r][j] = lds_words<S::VW>(stage + v_at[r & 1][j] + (r >> 1) * (8 * S::BOX));
        };
        if (D != 256) load_values();   // (heads of 256 have no registers to hold them over the branch: 64 x 8000 keys in 4 bits 54.4 us, 52.3 behind it)
        bool again = !__hblt2(all, __half2half2(__ushort_as_half(0x7800)));   // 2^15 and above, infinities and NaN
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int r = 0; r < 2; ++r) again |= pair[h][r] > kMostPair;
        if (__any_sync(0xffffffffu, again)) {
            float alpha[NH][2];
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float mx = fmaxf(s[h][r], s[h][2 + r]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    mx = fmaxf(m_run[h][r], mx);
                    alpha[h][r] = exp2f(m_run[h][r] - mx);
                    m_run[h][r] = mx;
                    l_run[h][r] *= alpha[h][r];
                }
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    const float p0 = exp2f(s[h][r] - m_run[h][r]), p1 = exp2f(s[h][2 + r] - m_run[h][r]);
#pragma unroll
                    for (int k = 0; k < S::NG; ++k) {
                        float top = fmaxf(p0 * (vmul[0][k] * kTopScale), p1 * (vmul[1][k] * kTopScale));   // (not beyond fp32)
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 16));
                        const int e_alpha = static_cast<int>(__float_as_uint(alpha[h][r]) >> 23), e_old = 254 - static_cast<int>(__float_as_uint(inv_unit[h][r][k]) >> 23);
                        const int e_new = min(max(max(static_cast<int>(__float_as_uint(top) >> 23) + kTopExponent, e_old + e_alpha - 127), kLeastExponent), kMostExponent);
                        inv_unit[h][r][k] = __uint_as_float(static_cast<uint32_t>(254 - e_new) << 23);
                        const int e_both = e_alpha + e_old - e_new;   // alpha times the old unit over the new one: below 2
                        low[h][r][k] *= alpha[h][r];
                        const float both = e_alpha > 0 && e_both > 0 ? __uint_as_float((__float_as_uint(alpha[h][r]) & 0x7fffffu) | static_cast<uint32_t>(e_both) << 23) : 0.f;
                        seconds[h][r][k] *= both;
#pragma unroll
                        for (int j = k * (S::MT / S::NG); j < (k + 1) * (S::MT / S::NG); ++j) {
                            o[h][j][r] *= both;
                            o[h][j][2 + r] *= both;
                        }
                    }
                }
            weights();
        }
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                l_run[h][r] += pair[h][r];
                if (BITS == 4) {
#pragma unroll
                    for (int k = 0; k < S::NG; ++k) {
                        low[h][r][k] += pr[h][r] * vleast[0][k] + pr[h][2 + r] * vleast[1][k];
                        if (FINE) seconds[h][r][k] += rest[h][r][k];
                    }
                }
            }
        if (D == 256) load_values();
        // ---- O^T += V^T P^T: row g of MMA m is dimension 2 m of the lane's, row g + 8 the one after it
        if (BITS == 4) {
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int m = 0; m < S::MT; ++m) {
                    const int k = min(m / (S::VD / 2), S::NG - 1);
                    mma_f16(o[h][m], kLowOffset, kHighOffset, kLowOffset, kHighOffset, pb[h][k][0], pb[h][k][1]);
                }
        }
#pragma unroll
        for (int j = 0; j < S::VC; ++j) {
            constexpr int last = S::NG - 1;
#pragma unroll
            for (int w = 0; w < S::VW; ++w) {
                const uint32_t w0 = vw[0][j].w[w], w1 = vw[1][j].w[w], w2 = vw[2][j].w[w], w3 = vw[3][j].w[w];
                if (BITS == 8) {
                    // bytes of two tokens side by side
                    const uint32_t a01 = __byte_perm(w0, w1, 0x5140u), a23 = __byte_perm(w0, w1, 0x7362u);
                    const uint32_t b01 = __byte_perm(w2, w3, 0x5140u), b23 = __byte_perm(w2, w3, 0x7362u);
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        const uint32_t a = m ? a23 : a01, bb = m ? b23 : b01;
                        const uint32_t x0 = bytes_to_half2(a, kLowBytes), x1 = bytes_to_half2(a, kHighBytes);
                        const uint32_t x2 = bytes_to_half2(bb, kLowBytes), x3 = bytes_to_half2(bb, kHighBytes);
#pragma unroll
                        for (int h = 0; h < NH; ++h) {
                            mma_f16(o[h][j * (S::VD / 2) + w * 2 + m], x0, x1, x2, x3, pb[h][min(j, last)][0], pb[h][min(j, last)][1]);
                            if (FINE) mma_f16(o[h][j * (S::VD / 2) + w * 2 + m], x0, x1, x2, x3, pl[h][min(j, last)][0], pl[h][min(j, last)][1]);
                        }
                    }
                } else {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        // four codes of each of two tokens
                        const uint32_t a = __byte_perm(w0, w1, half ? 0x7632u : 0x5410u), bb = __byte_perm(w2, w3, half ? 0x7632u : 0x5410u);
#pragma unroll
                        for (int m = 0; m < 2; ++m) {
                            const uint32_t x0 = low_nibbles(a >> (8 * m)), x1 = high_nibbles(a >> (8 * m));
                            const uint32_t x2 = low_nibbles(bb >> (8 * m)), x3 = high_nibbles(bb >> (8 * m));
#pragma unroll
                            for (int h = 0; h < NH; ++h) {
                                mma_f16(o[h][j * (S::VD / 2) + w * 4 + half * 2 + m], x0, x1, x2, x3, pb[h][min(j, last)][0], pb[h][min(j, last)][1]);
                                if (FINE) mma_f16(o[h][j * (S::VD / 2) + w * 4 + half * 2 + m], x0, x1, x2, x3, pl[h][min(j, last)][0], pl[h][min(j, last)][1]);
                            }
                        }
                    }
                }
            }
        }
        free_stage = stage;
        stage = stage + S::STAGE == ring + STAGES * S::STAGE ? ring : stage + S::STAGE;
    }
    turn = (turn + x.i1 - x.i0) % WARPS;

    // ---- the warps' sums, in the values' units
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            l_run[h][r] += __shfl_xor_sync(0xffffffffu, l_run[h][r], 4);
            l_run[h][r] += __shfl_xor_sync(0xffffffffu, l_run[h][r], 8);
            l_run[h][r] += __shfl_xor_sync(0xffffffffu, l_run[h][r], 16);
#pragma unroll
            for (int j = 0; j < S::VC; ++j) {
                float add = 0.f;
                if (BITS == 4) {
                    add = low[h][r][min(j, S::NG - 1)];
                    if (FINE) add -= 8.f * one_over(inv_unit[h][r][min(j, S::NG - 1)]) * seconds[h][r][min(j, S::NG - 1)];   // the offset of the codes that they were multiplied by
                    add += __shfl_xor_sync(0xffffffffu, add, 4);
                    add += __shfl_xor_sync(0xffffffffu, add, 8);
                    add += __shfl_xor_sync(0xffffffffu, add, 16);
                }
#pragma unroll
                for (int k = 0; k < S::VD / 2; ++k) {
                    const int m = j * (S::VD / 2) + k;
                    const float unit = one_over(inv_unit[h][r][m / (S::MT / S::NG)]);
                    if (BITS == 4) {
                        o[h][m][r] *= 16777216.f;   // 2^24
                        o[h][m][2 + r] *= 1048576.f;
                    }
                    o[h][m][r] = o[h][m][r] * unit + add;
                    o[h][m][2 + r] = o[h][m][2 + r] * unit + add;
                }
            }
        }
    // they meet two and two: warps 4 .. give theirs to 0 .., 2 and 3 to 0 and 1, 1 to 0
    auto give = [&](int buf) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int head = 8 * h + 2 * c + r;
                if (head >= heads) continue;
                if (g == 0) {
                    m_s[buf][head] = m_run[h][r];
                    l_s[buf][head] = l_run[h][r];
                }
                float* dst = sums_s + (buf * HEADS + head) * OP + g * S::VD;
#pragma unroll
                for (int m = 0; m < S::MT; ++m)
                    *reinterpret_cast<float2*>(dst + (m / (S::VD / 2)) * (D / S::VC) + 2 * (m % (S::VD / 2))) = make_float2(o[h][m][r], o[h][m][2 + r]);
            }
    };
    auto take = [&](int buf) {
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int head = 8 * h + 2 * c + r;
                if (head >= heads) continue;
                const float m_other = m_s[buf][head], m = fmaxf(m_run[h][r], m_other);
                const float fa = exp2f(m_run[h][r] - m), fb = exp2f(m_other - m);
                l_run[h][r] = l_run[h][r] * fa + l_s[buf][head] * fb;
                m_run[h][r] = m;
                const float* src = sums_s + (buf * HEADS + head) * OP + g * S::VD;
#pragma unroll
                for (int k = 0; k < S::MT; ++k) {
                    const float2 v = *reinterpret_cast<const float2*>(src + (k / (S::VD / 2)) * (D / S::VC) + 2 * (k % (S::VD / 2)));
                    o[h][k][r] = o[h][k][r] * fa + v.x * fb;
                    o[h][k][2 + r] = o[h][k][2 + r] * fa + v.y * fb;
                }
            }
    };
    if (SMALL) {
        copy_wait<0>();   // (zeros, behind the last tile)
        __syncthreads();
    }
#pragma unroll
    for (int from = 4; from < WARPS; from += BUFS) {
        if (warp >= from && warp < from + BUFS) give(warp - from);
        __syncthreads();
        if (warp >= from - 4 && warp < from - 4 + BUFS && warp + 4 < WARPS) take(warp - (from - 4));
        __syncthreads();
    }
    if (WARPS > 2) {
        if (warp == 2 || warp == 3) give(warp - 2);
        __syncthreads();
        if (warp < 2) take(warp);
        __syncwarp();   // warp 1: all lanes have read what its first ones overwrite
    }
    if (warp == 1) give(1);
    __syncthreads();
    if (warp == 0) {
        take(1);
        give(0);
    }
    __syncthreads();

    const int total = heads * D;
    if (in_cluster) {
        // ---- the parts' sums go to their slice's owner, relative to the part's maximum
        cluster_wait();   // every CTA of the cluster runs
        const int slice = ((total + p.splits - 1) / p.splits + 3) & ~3;
        float* slice_s = reinterpret_cast<float*>(last_s);   // [splits][slice]
        for (int idx = static_cast<int>(threadIdx.x); idx < total; idx += THREADS) {
            const int head = idx / D, d = idx % D, owner = idx / slice;
            st_shared_cluster_f32(mapa_u32(smem_u32(slice_s + split * slice + (idx - owner * slice)), static_cast<uint32_t>(owner)), sums_s[head * OP + d]);
        }
        for (int idx = static_cast<int>(threadIdx.x); idx < heads * p.splits; idx += THREADS) {
            const int head = idx % heads;
            const uint32_t to = static_cast<uint32_t>(idx / heads);
            st_shared_cluster_f32(mapa_u32(smem_u32(&part_m[split][head]), to), m_s[0][head]);
            st_shared_cluster_f32(mapa_u32(smem_u32(&part_l[split][head]), to), l_s[0][head]);
        }
        cluster_arrive();
        cluster_wait();
        const int base = split * slice, mine = min(slice, total - base);
        for (int idx = static_cast<int>(threadIdx.x) * 2; idx < mine; idx += THREADS * 2) {   // (D and slices are even)
            const int head = (base + idx) / D;
            float m = kNoScore;
            for (int s2 = 0; s2 < p.splits; ++s2) m = fmaxf(m, part_m[s2][head]);
            float l = 0.f, a0 = 0.f, a1 = 0.f;
            for (int s2 = 0; s2 < p.splits; ++s2) {
                const float f = exp2f(part_m[s2][head] - m);
                l += part_l[s2][head] * f;
                const float2 v = *reinterpret_cast<const float2*>(slice_s + s2 * slice + idx);
                a0 += v.x * f;
                a1 += v.y * f;
            }
            // a sum of weights that is not positive: no keys (zeros), or a NaN among the scores
            const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
            const uint32_t w = F16 ? pack_f16x2(a0 * inv, a1 * inv) : pack_bf16x2(a0 * inv, a1 * inv);
            *reinterpret_cast<uint32_t*>(static_cast<char*>(p.out) + (head0 * D + base + idx) * 2) = w;
        }
    } else if (in_shares && (x.i0 > 0 || x.i1 < keys.tiles)) {
        float* dst = p.part + (2 * static_cast<size_t>(blockIdx.x) + (first_piece ? 0 : 1)) * (HEADS * (D + 2));
        for (int idx = static_cast<int>(threadIdx.x); idx < total; idx += THREADS) dst[idx / D * (D + 2) + idx % D] = sums_s[idx / D * OP + idx % D];
        if (threadIdx.x < heads) {
            dst[threadIdx.x * (D + 2) + D] = m_s[0][threadIdx.x];
            dst[threadIdx.x * (D + 2) + D + 1] = l_s[0][threadIdx.x];
        }
    } else {
        for (int idx = static_cast<int>(threadIdx.x) * 2; idx < total; idx += THREADS * 2) {
            const int head = idx / D;
            const float l = l_s[0][head], inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
            const float a0 = sums_s[head * OP + idx % D], a1 = sums_s[head * OP + idx % D + 1];
            const uint32_t w = F16 ? pack_f16x2(a0 * inv, a1 * inv) : pack_bf16x2(a0 * inv, a1 * inv);
            *reinterpret_cast<uint32_t*>(static_cast<char*>(p.out) + (head0 * D + idx) * 2) = w;
        }
    }
    first_piece = false;
    }
}

template <int BITS, int D, int NH, bool PAGED, bool F16, bool SMALL>
int launch(const Params& p, int grid, cudaStream_t stream) {
    const int cluster = p.shares == 0 ? p.splits : 1;
    using S = Shape<BITS, D>;
    constexpr int smem = warps_of(D, NH, SMALL) * stages_of(S::STAGE, D, NH, SMALL) * S::STAGE + behind_rings(D, NH, SMALL);
    const auto fn = decode_kernel<BITS, D, NH, PAGED, F16, SMALL>;
    static std::atomic<bool> opted_in[64];   // (for each instance of this template)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64 || !opted_in[dev]) {
        TDIST_CUDA_OK(cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
        if (dev >= 0 && dev < 64) opted_in[dev] = true;
    }
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(32 * warps_of(D, NH, SMALL));
    cfg.dynamicSmemBytes = static_cast<size_t>(smem);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0] = tdist_host::pdl_attribute();
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 1 ? 2 : 1;
    TDIST_CUDA_OK(cudaLaunchKernelEx(&cfg, fn, p));
    return 0;
}

template <int BITS, int D, int NH, bool F16>
int launch_way(const Params& p, bool paged, bool small, int grid, cudaStream_t stream) {
    if (small) return paged ? launch<BITS, D, NH, true, F16, true>(p, grid, stream) : launch<BITS, D, NH, false, F16, true>(p, grid, stream);
    return paged ? launch<BITS, D, NH, true, F16, false>(p, grid, stream) : launch<BITS, D, NH, false, F16, false>(p, grid, stream);
}

template <int BITS, bool F16>
int launch_shape(const Params& p, int head_dim, int nh, bool paged, bool small, int grid, cudaStream_t stream) {
    // heads of 256 take one tile of query heads: two would need more registers than there are
    if (head_dim == 256) return launch_way<BITS, 256, 1, F16>(p, paged, small, grid, stream);
    if (nh == 2) return head_dim == 64 ? launch_way<BITS, 64, 2, F16>(p, paged, small, grid, stream) : launch_way<BITS, 128, 2, F16>(p, paged, small, grid, stream);
    return head_dim == 64 ? launch_way<BITS, 64, 1, F16>(p, paged, small, grid, stream) : launch_way<BITS, 128, 1, F16>(p, paged, small, grid, stream);
}

template <int BITS>
int launch_bits(const Params& p, int head_dim, int nh, bool paged, bool f16, bool small, int grid, cudaStream_t stream) {
    return f16 ? launch_shape<BITS, true>(p, head_dim, nh, paged, small, grid, stream) : launch_shape<BITS, false>(p, head_dim, nh, paged, small, grid, stream);
}

// (compiled in quantized_decode_8bit.cu and quantized_decode_4bit.cu)
extern template int launch_bits<8>(const Params&, int, int, bool, bool, bool, int, cudaStream_t);
extern template int launch_bits<4>(const Params&, int, int, bool, bool, bool, int, cudaStream_t);

}  // namespace qdecode
}  // namespace tdist
