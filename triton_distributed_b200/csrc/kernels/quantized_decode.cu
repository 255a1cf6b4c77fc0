// Decode attention over a paged KV cache in 8 or 4 bits (format: quantized_cache.cu), one query token per sequence.
//
//   s_j = scale q . k_j, k_j = ks_j c_j             4 bits: k_j = step_jg c_j + least_jg in every group g of 64 dimensions
//   o   = sum_j p_j vs_j c'_j / sum_j p_j           p_j = exp(s_j - max)
//
// The rows are never dequantised: the scales are applied where they are one number per key, to the score (4 bits: to a group's part of it, and
// least_jg times the sum of q over the group is added), and to the weight p_j vs_j, with the sum of p_j least_jg kept beside the product.
//
// K. Codes are 8-bit operands of the integer MMA (m16n8k32, u8 x s8) as they lie in memory, 4-bit ones after two logic instructions
// per eight. A query is brought to 16 bits for it, rint(q 32512 / max |q|), as a high and a low byte with a product each: the sums are exact, the second
// continues from 256 times the first, and 128 times the sum of q takes the codes' offset off. (As fp16 operands the codes of a tile cost 64
// instructions, and the kernel was bound by its issue slots: 567 per tile of 16 x 128, 32 x 16384 keys of 8 kv heads 148 us.)
// A score is off by up to 2^-17 max |q| sum |k_d|: a 16-bit query against bf16's 8 bits.
//
// V. Codes become fp16, exactly, two tokens per register. Weights are divided by a power of two above all vs_j so far, so that p_j vs_j / S lies
// in [0, 1] whatever the values' magnitude: rounded to fp16 it is off by 2^-12 of itself, or 2^-25 of the largest. 4-bit codes are taken as
// c - 8 with least + 8 step, so that the sums stay small.
//
// As in the plain decode tokens are the 16 rows of the MMA and query heads its 8 columns (two tiles of them above 8 heads per kv head):
// S^T = K Q^T, O^T = V^T P^T, P transposed by movmatrix, and every warp streams tiles of 16 tokens through a cp.async ring of its own.
// The sum over a row's dimensions may run in any order, the output's dimensions may be dealt to the MMA's rows in any order and so may the
// tokens, so all three are chosen by what a wide load from shared memory gives: of 64 dimensions of a key, the four lanes of a quad take 16 neighbouring
// ones each, and of a value's each eighth lane an eighth. (Loads straight into registers, each as soon as the registers are free: too few bytes under
// way, warps waited for memory half of their time.)
//
// A CTA is 8 warps of one (sequence, kv head, part of the keys); tiles of 16 tokens go round the warps. Warps meet in shared memory;
// up to 8 parts are a cluster that exchanges slices of the sums (CTA r adds up the r-th slice of all parts); more parts go through a
// workspace and a second kernel. No counters: nothing has to be zero before a call, and calls share nothing.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cstring>
#include <string>

#include "../device/ptx.cuh"
#include "../device/signal.cuh"
#include "../device/soft_cap.cuh"
#include "../include/tdist.h"
#include "../runtime/host_common.h"

namespace tdist {
namespace qdecode {

constexpr int WARPS = 8, THREADS = WARPS * 32;
// warps that compute: where tiles come by TMA, one warp loads for the others
__host__ __device__ constexpr int consumers(bool paged) { return paged ? WARPS - 1 : WARPS; }
constexpr int TOK = 16;          // tokens of a tile
constexpr int MAX_CLUSTER = 8;
constexpr int kKernelQuantDecode = 13;
// Scores may pass the maximum that weights are relative to by this much (in powers of two) before it is raised and the sums are scaled: a weight
// times its scale's share of the unit is rounded to fp16 whatever its size, and 2^8 is far below fp16's largest.
constexpr float kSlack = 8.f;
constexpr float kLog2e = 1.4426950408889634f;

struct Params {
    CUtensorMap tm_k, tm_v;        // PAGED: codes as bytes {ROW, Hkv, page, blocks}, box {BOX, 1, 16, 1}
    CUtensorMap tm_ks, tm_vs;      // scales as words {page NG, Hkv, blocks}, box {16 NG, 1, 1}
    const void* q;                 // [B, Hq, D]
    const uint8_t *k, *v;
    const char *ks, *vs;
    const int *table, *lens;
    float* part;                   // [B * Hq][splits][D + 2]: sums, maximum, sum of weights (more than MAX_CLUSTER parts)
    void* out;
    long long code_block, code_token, code_head, scale_block, scale_head, scale_token;   // bytes
    int Hq, Hkv, head_tiles, page_size, page_shift, max_blocks, blocks, splits, window, sinks, table_keys, is_f16;
    float scale, soft_cap;
    uint32_t page_mul;             // t / page_size = (t page_mul) >> page_shift for t < 2^31
    WaitCtx wctx;
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
__device__ __forceinline__ uint32_t hsub2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
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
// A byte or nibble n under the exponent of 1024 is the fp16 number 1024 + n; in the upper nibble of a byte, 1024 + 16 n.
constexpr uint32_t kMagic = 0x64006400u;
constexpr uint32_t kLowBytes = 0x7150u, kHighBytes = 0x7352u;   // bytes 0, 1 / 2, 3 of a word, each under a 0x64
__device__ __forceinline__ uint32_t bytes_to_half2(uint32_t w, uint32_t sel) { return hsub2(__byte_perm(w, kMagic, sel), 0x64806480u); }   // - 1152
__device__ __forceinline__ uint32_t low_nibbles(uint32_t w) { return hsub2((w & 0x000f000fu) | kMagic, 0x64086408u); }                     // - 1032: n - 8
// 16 (n - 8): the rows of the MMA that take it are off by that factor until the end (a multiply-add here has two constants to keep in registers)
__device__ __forceinline__ uint32_t high_nibbles(uint32_t w) { return hsub2((w & 0x00f000f0u) | kMagic, 0x64806480u); }                     // - 1152
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

// A tile in shared memory: 16 rows of K codes, 16 of V codes, and apart from them the rows' scales. The 16-byte chunks of a row lie as a TMA load with the
// swizzle of the row's width leaves them (rows of 256 bytes as two halves of 128), and the MMA's rows are tokens in an order that makes
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
    static constexpr int SCALES = TOK * SB < 128 ? 128 : TOK * SB;   // K's, on 128 bytes as TMA wants them; V's behind them
    static constexpr int STAGE = 2 * TILE + 2 * SCALES;    // bytes of a place in the ring
    static constexpr int LOADED = 2 * TILE + 2 * TOK * SB;

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

// CTAs per SM, and tiles that the rings of a CTA have room for in 206 KB per SM: at most 8 per warp, and as many for each. (A place belongs to one
// warp: only a warp that has waited for a place's earlier tiles itself can tell by a barrier's parity that the next one is there.)
__host__ __device__ constexpr int ctas_per_sm(int d, int nh) { return d == 256 || nh == 2 ? 1 : 2; }
__host__ __device__ constexpr int places_of(int stage, int d, int nh, bool paged) {
    const int each = 206 * 1024 / ctas_per_sm(d, nh) / stage / consumers(paged);
    return (each < 8 ? each : 8) * consumers(paged);
}

template <int BITS, int D, int NH, bool PAGED>
__global__ void __launch_bounds__(THREADS, ctas_per_sm(D, NH)) decode_kernel(const __grid_constant__ Params p) {
    using S = Shape<BITS, D>;
    constexpr int HEADS = 8 * NH, OP = o_pitch(D), CW = consumers(PAGED);
    constexpr int PLACES = places_of(S::STAGE, D, NH, PAGED), STAGES = PLACES / CW;   // of all rings; of a warp's own
    static_assert(STAGES >= 3 && PLACES * S::STAGE >= CW * HEADS * OP * 4, "the warps' sums reuse the ring");
    extern __shared__ uint8_t smem_raw[];
    // [PLACES] K and V codes, [PLACES] scales, the cluster's slices
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    float* o_s = reinterpret_cast<float*>(smem);            // [CW][HEADS][OP], when the rings are done
    __shared__ uint64_t bars[2][PAGED ? PLACES : 1];       // PAGED: a tile's bytes are there; its place is free
    __shared__ float m_s[CW][HEADS], l_s[CW][HEADS];
    __shared__ float part_m[MAX_CLUSTER][HEADS], part_l[MAX_CLUSTER][HEADS];
    const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x) >> 5, 0), lane = static_cast<int>(threadIdx.x) & 31;
    const int g = lane >> 2, c = lane & 3;
    const bool in_cluster = p.splits > 1 && p.splits <= MAX_CLUSTER;
    if (in_cluster) cluster_arrive();                       // waited for before the first store into another CTA
    if (PAGED) {
        if (threadIdx.x < PLACES) {
            mbar_init(smem_u32(&bars[0][threadIdx.x]), 1);
            mbar_init(smem_u32(&bars[1][threadIdx.x]), 1);
            fence_mbar_init();
        }
        __syncthreads();
    }
    pdl_wait_and_release();

    int x = static_cast<int>(blockIdx.x);
    const int split = x % p.splits;
    x /= p.splits;
    const int tile_of_heads = x % p.head_tiles;
    x /= p.head_tiles;
    const int kvh = x % p.Hkv, b = x / p.Hkv;
    const int G = p.Hq / p.Hkv;
    const int heads = min(HEADS, G - tile_of_heads * HEADS);
    const size_t head0 = static_cast<size_t>(b) * p.Hq + kvh * G + tile_of_heads * HEADS;

    // ---- the keys: tiles of the first `first` tokens, then those from the window's first token on (a tile's first token is a multiple of 16)
    const int n = min(max(p.lens[b], 0), p.table_keys);
    const int lo = max(0, n - p.window);
    const int first = min(p.sinks, lo);
    const int sink_tiles = (first + TOK - 1) / TOK;
    const int t_lo = lo / TOK;
    const int tiles = sink_tiles + (n + TOK - 1) / TOK - t_lo;
    const int per = (tiles + p.splits - 1) / p.splits;
    const int first_tile = min(split * per, tiles), i0 = first_tile + warp, i1 = min((split + 1) * per, tiles);

    const int* table = p.table + static_cast<size_t>(b) * p.max_blocks;
    auto first_token = [&](int i) { return (i < sink_tiles ? i : i - sink_tiles + t_lo) * TOK; };
    auto in_table = [&](int t) { return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(t)) * p.page_mul) >> p.page_shift); };
    auto codes_at = [&](int place) { return smem_u32(smem) + static_cast<uint32_t>(place * 2 * S::TILE); };
    auto scales_at = [&](int place) { return smem_u32(smem) + static_cast<uint32_t>(PLACES * 2 * S::TILE + place * 2 * S::SCALES); };

    if (PAGED && warp == CW) {
        // ---- the loading warp: a lane looks up the page of one of the next 32 tiles, then tile after tile is sent on its way. A page that the
        // cache does not have is out of the tensor map's bounds and reads as zeros.
        auto lookup = [&](int i) { return i < i1 ? static_cast<int>(ldg32(table + in_table(first_token(i)))) : 0; };
        int place = 0;
        uint32_t parity = 1;
        int pages = lookup(first_tile + lane);
        for (int base = first_tile; base < i1; base += 32) {
            const int now = pages, row = first_token(base + lane) - in_table(first_token(base + lane)) * p.page_size;
            pages = lookup(base + 32 + lane);
            const int count = min(32, i1 - base);
            for (int j = 0; j < count; ++j) {
                const int page_j = __shfl_sync(0xffffffffu, now, j), row_j = __shfl_sync(0xffffffffu, row, j);
                mbar_wait(smem_u32(&bars[1][place]), parity, p.wctx, 2);
                if (elect_one()) {
                    const uint32_t bar = smem_u32(&bars[0][place]), codes = codes_at(place), scales = scales_at(place);
                    mbar_expect_tx(bar, S::LOADED);
                    tma_load_4d(codes, &p.tm_k, bar, 0, kvh, row_j, page_j);
                    if (S::ROW > S::BOX) tma_load_4d(codes + TOK * S::BOX, &p.tm_k, bar, S::BOX, kvh, row_j, page_j);
                    tma_load_3d(scales, &p.tm_ks, bar, row_j * S::NG, kvh, page_j);
                    tma_load_4d(codes + S::TILE, &p.tm_v, bar, 0, kvh, row_j, page_j);
                    if (S::ROW > S::BOX) tma_load_4d(codes + S::TILE + TOK * S::BOX, &p.tm_v, bar, S::BOX, kvh, row_j, page_j);
                    tma_load_3d(scales + S::SCALES, &p.tm_vs, bar, row_j * S::NG, kvh, page_j);
                }
                __syncwarp();
                if (++place == PLACES) {
                    place = 0;
                    parity ^= 1u;
                }
            }
        }
    } else {
    // ---- not PAGED (pages of other sizes, scales with strides): every warp copies its own tiles, 16 bytes of a row per lane. A lane looks up token
    // lane % 16; -1: not seen. Rows that are not seen, or whose page the cache does not have, are zeros.
    const int my_token = lane & 15;
    auto lookup = [&](int i) {
        const int t = first_token(i) + my_token;
        return i < i1 && (i < sink_tiles ? t < first : t >= lo && t < n) ? static_cast<int>(ldg32(table + in_table(t))) : -1;
    };
    constexpr int CHUNKS = S::ROW / 16, ROWS = 32 / CHUNKS;   // rows that a warp copies at once
    const int lrow = lane / CHUNKS, lchunk = lane % CHUNKS;
    const uint8_t* k_lane = p.k + kvh * p.code_head + lchunk * 16;
    const uint8_t* v_lane = p.v + kvh * p.code_head + lchunk * 16;
    const char* s_lane = (lane < 16 ? p.ks : p.vs) + kvh * p.scale_head;   // lanes 0..15 copy the scales of the keys, 16..31 of the values
    auto issue = [&](int i, int page, int place) {
        const int t = first_token(i) + my_token;
        const int row = t - in_table(t) * p.page_size;
        const bool live = static_cast<unsigned>(page) < static_cast<unsigned>(p.blocks);
        const long long from = live ? page : 0;
        const long long off = from * p.code_block + row * p.code_token, soff = from * p.scale_block + row * p.scale_token;
        const uint32_t codes = codes_at(place);
#pragma unroll
        for (int j = 0; j < TOK / ROWS; ++j) {
            const int r = j * ROWS + lrow;
            const long long at = __shfl_sync(0xffffffffu, off, r);
            const bool none = !__shfl_sync(0xffffffffu, static_cast<int>(live), r);
            const uint32_t dst = codes + S::at(r, lchunk * 16);
            copy16(dst, k_lane + at, none);
            copy16(dst + S::TILE, v_lane + at, none);
        }
        copy_small<S::SB>(scales_at(place) + (lane >> 4) * S::SCALES + my_token * S::SB, s_lane + soff, !live);
    };
    int page = -1;
    if (!PAGED) {
        page = lookup(i0);
#pragma unroll
        for (int a = 0; a < STAGES - 1; ++a) {
            const int i = i0 + a * WARPS, now = page;
            page = lookup(i + WARPS);
            if (i < i1) issue(i, now, warp * STAGES + a);
            copy_commit();
        }
    }

    // ---- q as the second operand: column g of the MMA is head 8 h + g, its dimensions 16 c .. 16 c + 15 of every 64 are this lane's
    uint32_t qf[NH][S::KC][4][2];  // high and low bytes of four dimensions
    float factor[NH][2];           // of heads 8 h + 2 c + {0, 1}: what turns a product of codes into a score in units of log2
    int bias[NH][2];               // 8 bits: -128 times the sum of the 16-bit q
    float qsum[NH][2][S::NG];      // 4 bits: that sum over a group
#pragma unroll
    for (int h = 0; h < NH; ++h) {
        const int head = 8 * h + g;
        const char* src = static_cast<const char*>(p.q) + (head0 + (head < heads ? head : 0)) * (D * 2);
        float f[S::KC][16];
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < S::KC; ++j) {
            // the dimensions whose codes lie in this lane's bytes of chunk j
            const Words<8> w = load_words<8>(src + (BITS == 8 ? 2 : 4) * S::k_byte(j, c));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if (p.is_f16) {
                    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w.w[e]));
                    f[j][2 * e] = t.x;
                    f[j][2 * e + 1] = t.y;
                } else {
                    f[j][2 * e] = __uint_as_float(w.w[e] << 16);
                    f[j][2 * e + 1] = __uint_as_float(w.w[e] & 0xffff0000u);
                }
                top = max(top, max(__float_as_uint(f[j][2 * e]) & 0x7fffffffu, __float_as_uint(f[j][2 * e + 1]) & 0x7fffffffu));
            }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // magnitudes below 2^-100 count as that; a query with a NaN or an infinity has a factor of NaN, and so has its result
        const bool good = top < 0x7f800000u;
        const float most = fmaxf(good ? __uint_as_float(top) : 1.f, 7.888609052210118e-31f);
        const float mul = head < heads && good ? 32512.f / most : 0.f;
        int sum = 0;
#pragma unroll
        for (int j = 0; j < S::KC; ++j) {
            int part = 0, hi[16], low8[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
                const int v = max(-32512, min(32512, __float2int_rn(f[j][k] * mul)));
                hi[k] = (v + 128) >> 8;
                low8[k] = v - 256 * hi[k];
                part += v;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                // four codes of a register of the first operand
                const int d = BITS == 8 ? 4 * k : 8 * (k >> 1) + (k & 1), e = BITS == 8 ? 1 : 2;
                qf[h][j][k][0] = pack_bytes(hi[d], hi[d + e], hi[d + 2 * e], hi[d + 3 * e]);
                qf[h][j][k][1] = pack_bytes(low8[d], low8[d + e], low8[d + 2 * e], low8[d + 3 * e]);
            }
            part += __shfl_xor_sync(0xffffffffu, part, 1);
            part += __shfl_xor_sync(0xffffffffu, part, 2);
            sum += part;
            if (BITS == 4) {
#pragma unroll
                for (int r = 0; r < 2; ++r) qsum[h][r][j] = static_cast<float>(__shfl_sync(0xffffffffu, part, (2 * c + r) * 4));
            }
        }
        const float down = good ? most * (1.f / 32512.f) * p.scale : __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            factor[h][r] = __shfl_sync(0xffffffffu, down, (2 * c + r) * 4) * (p.soft_cap > 0.f ? 1.f : kLog2e);
            bias[h][r] = BITS == 8 ? __shfl_sync(0xffffffffu, sum, (2 * c + r) * 4) * -128 : 0;
        }
    }

    // ---- sums: O^T in units of `unit` (a power of two), columns are heads 8 h + 2 c + {0, 1}
    float o[NH][S::MT][4];
    float limit[NH][2], m_use[NH][2], l_run[NH][2];   // weights are relative to 2^m_use; it is raised when a score passes `limit`
    float low[NH][2][S::NG];       // 4 bits: sum of p least, of this lane's tokens
    float unit = 0.f, inv_unit = 0.f;
#pragma unroll
    for (int h = 0; h < NH; ++h) {
#pragma unroll
        for (int j = 0; j < S::MT; ++j) o[h][j][0] = o[h][j][1] = o[h][j][2] = o[h][j][3] = 0.f;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            limit[h][r] = -CUDART_INF_F;
            m_use[h][r] = l_run[h][r] = 0.f;
#pragma unroll
            for (int k = 0; k < S::NG; ++k) low[h][r][k] = 0.f;
        }
    }
    const float cap_inv = p.soft_cap > 0.f ? 1.f / p.soft_cap : 0.f;

    // what this lane reads of a tile: tokens of rows g and g + 8 of the MMA (keys and scales), of columns 2 c, 2 c + 1, 2 c + 8, 2 c + 9 (values)
    const int t_row = token_of(g);
    uint32_t k_at[S::KC], v_at[2][S::VC];
#pragma unroll
    for (int j = 0; j < S::KC; ++j) k_at[j] = S::at(t_row, S::k_byte(j, c));
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int j = 0; j < S::VC; ++j) v_at[r][j] = S::TILE + S::at(token_of(2 * c + r), j * S::VB + g * (S::VB / 8));   // tokens 8 further on: 8 rows
    int place = PAGED ? warp : warp * STAGES, free_place = warp * STAGES + STAGES - 1;
    uint32_t parity = 0;
    for (int i = i0; i < i1; i += CW) {
        if (PAGED) {
            mbar_wait(smem_u32(&bars[0][place]), parity, p.wctx, 1);
        } else {
            copy_wait<STAGES - 2>();
            __syncwarp();   // the tile is here, and the place of the one before it is free
            const int ahead = i + (STAGES - 1) * WARPS, now = page;
            page = lookup(ahead + WARPS);
            if (ahead < i1) issue(ahead, now, free_place);
            copy_commit();
        }
        const uint32_t stage = codes_at(place), scales = scales_at(place) + static_cast<uint32_t>(t_row * S::SB);
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
        const int t0 = first_token(i);
        const bool sink = i < sink_tiles, edge = sink || t0 < lo || t0 + TOK > n;
        bool higher = false;
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int r = e >> 1;
                float v = 0.f;
                if (BITS == 8) {
                    v = static_cast<float>(acc[h][0][e]) * __uint_as_float(kscale[r].w[0]);
                } else {
#pragma unroll
                    for (int k = 0; k < S::NG; ++k)
                        v += __uint_as_float(kscale[r].w[k] << 16) * static_cast<float>(acc[h][k][e]) + __uint_as_float(kscale[r].w[k] & 0xffff0000u) * qsum[h][e & 1][k];
                }
                s[h][e] = v * factor[h][e & 1];
            }
        if (p.soft_cap > 0.f) {
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int e = 0; e < 4; ++e) s[h][e] = soft_cap(s[h][e] * kLog2e, s[h][e] * cap_inv, p.soft_cap * kLog2e);
        }
        // ---- the values' scales, as weights in units of `unit`
        float vmul[2][S::NG], vleast[2][S::NG];
        float most = 0.f;
        if (edge) {
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const int t = t0 + t_row + 8 * r;
                const bool seen = sink ? t < first : t >= lo && t < n;
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
                most = fmaxf(most, vmul[r][k]);
            }
#pragma unroll
        for (int h = 0; h < NH; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) higher |= s[h][e] > limit[h][e & 1];
        higher |= most > unit;
        if (__any_sync(0xffffffffu, higher)) {
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
            most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
            float shrink = 1.f;
            if (most > unit) {
                // the next power of two, whose inverse is a normal number too
                const uint32_t e = min((__float_as_uint(most) >> 23) + 1u, 250u);
                const float up = __uint_as_float(e << 23);
                shrink = unit / up;
                unit = up;
                inv_unit = __uint_as_float((254u - e) << 23);
            }
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    float mx = fmaxf(s[h][r], s[h][2 + r]);
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float m_old = limit[h][r] == -CUDART_INF_F ? -CUDART_INF_F : m_use[h][r], m_new = fmaxf(m_old, mx);
                    m_use[h][r] = m_new == -CUDART_INF_F ? 0.f : m_new;
                    limit[h][r] = m_new + kSlack;
                    const float alpha = exp2f(m_old - m_use[h][r]);
                    l_run[h][r] *= alpha;
#pragma unroll
                    for (int k = 0; k < S::NG; ++k) low[h][r][k] *= alpha;
                    const float both = alpha * shrink;
#pragma unroll
                    for (int j = 0; j < S::MT; ++j) {
                        o[h][j][r] *= both;
                        o[h][j][2 + r] *= both;
                    }
                }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int k = 0; k < S::NG; ++k) vmul[r][k] *= inv_unit;
        // ---- P^T times the scales as the second operand: tokens in pairs per lane, heads over lane / 4
        uint32_t pb[NH][S::NG][2];
#pragma unroll
        for (int h = 0; h < NH; ++h) {
            const float p0 = exp2f(s[h][0] - m_use[h][0]), p1 = exp2f(s[h][1] - m_use[h][1]);
            const float p2 = exp2f(s[h][2] - m_use[h][0]), p3 = exp2f(s[h][3] - m_use[h][1]);
            l_run[h][0] += p0 + p2;
            l_run[h][1] += p1 + p3;
#pragma unroll
            for (int k = 0; k < S::NG; ++k) {
                if (BITS == 4) {
                    low[h][0][k] += p0 * vleast[0][k] + p2 * vleast[1][k];
                    low[h][1][k] += p1 * vleast[0][k] + p3 * vleast[1][k];
                }
                pb[h][k][0] = movmatrix_trans(pack_f16x2(p0 * vmul[0][k], p1 * vmul[0][k]));
                pb[h][k][1] = movmatrix_trans(pack_f16x2(p2 * vmul[1][k], p3 * vmul[1][k]));
            }
        }
        // ---- O^T += V^T P^T: row g of MMA m is dimension 2 m of the lane's, row g + 8 the one after it
        Words<S::VW> vw[4][S::VC];
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int j = 0; j < S::VC; ++j) vw[r][j] = lds_words<S::VW>(stage + v_at[r & 1][j] + (r >> 1) * (8 * S::BOX));
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
                        for (int h = 0; h < NH; ++h) mma_f16(o[h][j * (S::VD / 2) + w * 2 + m], x0, x1, x2, x3, pb[h][min(j, last)][0], pb[h][min(j, last)][1]);
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
                            for (int h = 0; h < NH; ++h)
                                mma_f16(o[h][j * (S::VD / 2) + w * 4 + half * 2 + m], x0, x1, x2, x3, pb[h][min(j, last)][0], pb[h][min(j, last)][1]);
                        }
                    }
                }
            }
        }
        if (PAGED) {
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bars[1][place]));
            place += CW;
            if (place >= PLACES) {
                place -= PLACES;
                parity ^= 1u;
            }
        } else {
            free_place = place;
            if (++place == warp * STAGES + STAGES) place = warp * STAGES;
        }
    }
    if (!PAGED) copy_wait<0>();
    // the rings are done once every warp is here: the sums take their place
    named_barrier(1, CW * 32);

    // ---- the warps meet in shared memory
#pragma unroll
    for (int h = 0; h < NH; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int head = 8 * h + 2 * c + r;
            float l = l_run[h][r];
            l += __shfl_xor_sync(0xffffffffu, l, 4);
            l += __shfl_xor_sync(0xffffffffu, l, 8);
            l += __shfl_xor_sync(0xffffffffu, l, 16);
            if (g == 0) {
                m_s[warp][head] = limit[h][r] == -CUDART_INF_F ? -CUDART_INF_F : m_use[h][r];
                l_s[warp][head] = l;
            }
            float* dst = o_s + (warp * HEADS + head) * OP;
#pragma unroll
            for (int j = 0; j < S::VC; ++j) {
                float add = 0.f;
                if (BITS == 4) {
                    add = low[h][r][min(j, S::NG - 1)];
                    add += __shfl_xor_sync(0xffffffffu, add, 4);
                    add += __shfl_xor_sync(0xffffffffu, add, 8);
                    add += __shfl_xor_sync(0xffffffffu, add, 16);
                }
#pragma unroll
                for (int k = 0; k < S::VD / 2; ++k) {
                    const int m = j * (S::VD / 2) + k;
                    *reinterpret_cast<float2*>(dst + j * (D / S::VC) + g * S::VD + 2 * k) =
                        make_float2(o[h][m][r] * unit + add, o[h][m][2 + r] * (BITS == 8 ? unit : unit * 0.0625f) + add);
                }
            }
        }
    }
    __syncthreads();
    if (in_cluster) cluster_wait();   // every CTA of the cluster runs

    // A part's sums go to the slice's owner (the CTA itself without a cluster), relative to the part's maximum
    const int total = heads * D;
    const int slices = in_cluster ? p.splits : 1;
    const int slice = ((total + slices - 1) / slices + 3) & ~3;
    float* slice_s = reinterpret_cast<float*>(smem + PLACES * S::STAGE);   // [splits][slice]
    const bool to_workspace = p.splits > MAX_CLUSTER;
    for (int idx = static_cast<int>(threadIdx.x); idx < total; idx += THREADS) {
        const int head = idx / D, d = idx % D;
        float m = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < CW; ++w) m = fmaxf(m, m_s[w][head]);
        const float mu = m == -CUDART_INF_F ? 0.f : m;
        float l = 0.f, sum = 0.f;
#pragma unroll
        for (int w = 0; w < CW; ++w) {
            const float f = exp2f(m_s[w][head] - mu);
            l += l_s[w][head] * f;
            sum += o_s[(w * HEADS + head) * OP + d] * f;
        }
        if (to_workspace) {
            float* dst = p.part + ((head0 + head) * p.splits + split) * (D + 2);
            dst[d] = sum;
            if (d == 0) {
                dst[D] = m;
                dst[D + 1] = l;
            }
        } else {
            const int owner = idx / slice;
            float* at = slice_s + split * slice + (idx - owner * slice);
            if (in_cluster) st_shared_cluster_f32(mapa_u32(smem_u32(at), static_cast<uint32_t>(owner)), sum);
            else *at = sum;
            if (d == 0) {
                for (int o2 = 0; o2 < slices; ++o2) {
                    if (in_cluster) {
                        st_shared_cluster_f32(mapa_u32(smem_u32(&part_m[split][head]), static_cast<uint32_t>(o2)), m);
                        st_shared_cluster_f32(mapa_u32(smem_u32(&part_l[split][head]), static_cast<uint32_t>(o2)), l);
                    } else {
                        part_m[0][head] = m;
                        part_l[0][head] = l;
                    }
                }
            }
        }
    }
    if (to_workspace) return;
    if (in_cluster) {
        cluster_arrive();
        cluster_wait();
    } else {
        __syncthreads();
    }
    const int base = in_cluster ? split * slice : 0;
    const int mine = min(slice, total - base);
    for (int idx = static_cast<int>(threadIdx.x) * 2; idx < mine; idx += THREADS * 2) {   // (D and slices are even)
        const int head = (base + idx) / D;
        float m = -CUDART_INF_F;
        for (int s2 = 0; s2 < slices; ++s2) m = fmaxf(m, part_m[s2][head]);
        const float mu = m == -CUDART_INF_F ? 0.f : m;
        float l = 0.f, a0 = 0.f, a1 = 0.f;
        for (int s2 = 0; s2 < slices; ++s2) {
            const float f = exp2f(part_m[s2][head] - mu);
            l += part_l[s2][head] * f;
            const float2 v = *reinterpret_cast<const float2*>(slice_s + s2 * slice + idx);
            a0 += v.x * f;
            a1 += v.y * f;
        }
        // a sum of weights that is not positive: no keys (zeros), or a NaN among the scores
        const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
        const uint32_t w = p.is_f16 ? pack_f16x2(a0 * inv, a1 * inv) : pack_bf16x2(a0 * inv, a1 * inv);
        *reinterpret_cast<uint32_t*>(static_cast<char*>(p.out) + (head0 * D + base + idx) * 2) = w;
    }
}

// The parts of a head, from the workspace: a CTA per head, a thread per two dimensions.
__global__ void __launch_bounds__(128) merge_kernel(const float* part, int splits, int D, int is_f16, void* out) {
    __shared__ float f_s[512];
    __shared__ float l_s;
    pdl_wait_and_release();
    const size_t head = blockIdx.x;
    const float* src = part + head * splits * (D + 2);
    const int lane = static_cast<int>(threadIdx.x) & 31;
    if (threadIdx.x < 32) {
        float m = -CUDART_INF_F;
        for (int s = lane; s < splits; s += 32) m = fmaxf(m, src[s * (D + 2) + D]);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float mu = m == -CUDART_INF_F ? 0.f : m;
        float l = 0.f;
        for (int s = lane; s < splits; s += 32) {
            const float f = exp2f(src[s * (D + 2) + D] - mu);
            f_s[s] = f;
            l += f * src[s * (D + 2) + D + 1];
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (lane == 0) l_s = l;
    }
    __syncthreads();
    const float l = l_s;
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    const int d = static_cast<int>(threadIdx.x) * 2;
    if (d >= D) return;
    float a0 = 0.f, a1 = 0.f;
#pragma unroll 8
    for (int s = 0; s < splits; ++s) {
        const float2 v = *reinterpret_cast<const float2*>(src + s * (D + 2) + d);
        a0 += v.x * f_s[s];
        a1 += v.y * f_s[s];
    }
    const uint32_t w = is_f16 ? pack_f16x2(a0 * inv, a1 * inv) : pack_bf16x2(a0 * inv, a1 * inv);
    *reinterpret_cast<uint32_t*>(static_cast<char*>(out) + (head * D + d) * 2) = w;
}

template <int BITS, int D, int NH, bool PAGED>
int launch(const Params& p, int grid, cudaStream_t stream) {
    const int cluster = p.splits > 1 && p.splits <= MAX_CLUSTER ? p.splits : 1;
    // slices: a part's share of 8 NH heads, rounded up to 4 floats
    using S = Shape<BITS, D>;
    const int smem = 1024 + places_of(S::STAGE, D, NH, PAGED) * S::STAGE + (8 * NH * D + 4 * MAX_CLUSTER) * 4;
    const auto fn = decode_kernel<BITS, D, NH, PAGED>;
    TDIST_CUDA_OK(cudaFuncSetAttribute(reinterpret_cast<const void*>(fn), cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(grid));
    cfg.blockDim = dim3(THREADS);
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

template <int BITS, int D>
int launch_heads(const Params& p, int nh, bool paged, int grid, cudaStream_t stream) {
    // heads of 256 take one tile of query heads: two would need more registers than there are
    if constexpr (D != 256) {
        if (nh == 2) return paged ? launch<BITS, D, 2, true>(p, grid, stream) : launch<BITS, D, 2, false>(p, grid, stream);
    }
    return paged ? launch<BITS, D, 1, true>(p, grid, stream) : launch<BITS, D, 1, false>(p, grid, stream);
}

template <int BITS>
int launch_dim(const Params& p, int head_dim, int nh, bool paged, int grid, cudaStream_t stream) {
    return head_dim == 64 ? launch_heads<BITS, 64>(p, nh, paged, grid, stream)
                          : (head_dim == 128 ? launch_heads<BITS, 128>(p, nh, paged, grid, stream) : launch_heads<BITS, 256>(p, nh, paged, grid, stream));
}

}  // namespace qdecode
}  // namespace tdist

using namespace tdist;
using tdist_host::fail;

extern "C" int tdist_quant_decode(const TdistQuantDecodeArgs* a) {
    using namespace tdist::qdecode;
    const TdistQuantCacheArgs& c = a->cache;
    if (c.bits != 8 && c.bits != 4) return fail(TDIST_EINVAL, "quantised decode: 8 or 4 bits");
    if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256) return fail(TDIST_EINVAL, "quantised decode: head_dim must be 64, 128 or 256");
    if (c.Hkv < 1 || a->Hq < 1 || a->Hq % c.Hkv || c.page_size < 1 || c.B < 0 || c.blocks < 0 || c.max_blocks < 0)
        return fail(TDIST_EINVAL, "quantised decode: bad shape");
    if (c.dtype != TDIST_BF16 && c.dtype != TDIST_F16) return fail(TDIST_EINVAL, "quantised decode: q must be bf16 or fp16");
    if (a->splits < 1 || a->splits > TDIST_QUANT_DECODE_SPLITS || (a->splits > MAX_CLUSTER && a->part == nullptr))
        return fail(TDIST_EINVAL, "quantised decode: parts");
    if (a->window < 1 || a->sinks < 0 || !(a->soft_cap >= 0.f)) return fail(TDIST_EINVAL, "quantised decode: window, sinks or soft cap");
    const uintptr_t code_align = reinterpret_cast<uintptr_t>(c.k_codes) | reinterpret_cast<uintptr_t>(c.v_codes) |
                                 static_cast<uintptr_t>(c.code_block | c.code_token | c.code_head);
    const uintptr_t scale_align = reinterpret_cast<uintptr_t>(c.k_scales) | reinterpret_cast<uintptr_t>(c.v_scales) |
                                  static_cast<uintptr_t>(c.scale_block | c.scale_head | c.scale_token);
    if ((code_align & 15) || (scale_align & (c.bits == 8 ? 3 : c.head_dim / 16 - 1)))
        return fail(TDIST_EINVAL, "quantised decode: codes must lie on 16 bytes, a row's scales on their size");
    if ((reinterpret_cast<uintptr_t>(a->q) & 15) || (reinterpret_cast<uintptr_t>(a->out) & 3))
        return fail(TDIST_EINVAL, "quantised decode: q must lie on 16 bytes, out on 4");
    if (c.B == 0) return 0;
    if (c.blocks == 0) {   // every page reads as zeros, and there is no place to read instead
        TDIST_CUDA_OK(cudaMemsetAsync(a->out, 0, static_cast<size_t>(c.B) * a->Hq * c.head_dim * 2, static_cast<cudaStream_t>(c.stream)));
        return 0;
    }
    Params p;
    memset(&p, 0, sizeof(p));
    p.q = a->q;
    p.k = static_cast<const uint8_t*>(c.k_codes);
    p.v = static_cast<const uint8_t*>(c.v_codes);
    p.ks = static_cast<const char*>(c.k_scales);
    p.vs = static_cast<const char*>(c.v_scales);
    p.table = static_cast<const int*>(c.table);
    p.lens = static_cast<const int*>(c.lens);
    p.part = static_cast<float*>(a->part);
    p.out = a->out;
    p.code_block = c.code_block;
    p.code_token = c.code_token;
    p.code_head = c.code_head;
    p.scale_block = c.scale_block;
    p.scale_head = c.scale_head;
    p.scale_token = c.scale_token;
    p.Hq = a->Hq;
    p.Hkv = c.Hkv;
    const int G = a->Hq / c.Hkv;
    const int nh = G > 8 && c.head_dim != 256 ? 2 : 1;
    p.head_tiles = (G + 8 * nh - 1) / (8 * nh);
    p.page_size = c.page_size;
    // with 2^l >= page_size the multiplier ceil(2^(31 + l) / page_size) is off by less than one, so t < 2^31 times it by less than 2^31 <= 2^(31 + l) / page_size
    int l = 0;
    while ((1ll << l) < c.page_size) ++l;
    p.page_shift = 31 + l;
    p.page_mul = static_cast<uint32_t>(((1ull << (31 + l)) + static_cast<uint64_t>(c.page_size) - 1) / static_cast<uint64_t>(c.page_size));
    p.max_blocks = c.max_blocks;
    p.blocks = c.blocks;
    p.splits = a->splits;
    p.window = a->window;
    p.sinks = a->sinks;
    const long long keys = static_cast<long long>(c.max_blocks) * c.page_size;
    p.table_keys = static_cast<int>(keys < 0x7fffffc0ll ? keys : 0x7fffffc0ll);
    p.is_f16 = c.dtype == TDIST_F16;
    p.scale = a->scale;
    p.soft_cap = a->soft_cap;
    const long long grid = static_cast<long long>(c.B) * c.Hkv * p.head_tiles * a->splits;
    if (grid > 0x7fffffffll) return fail(TDIST_EINVAL, "quantised decode: too many sequences");
    p.wctx.status = static_cast<Status*>(a->status);
    p.wctx.timeout_ns = a->timeout_ns;
    p.wctx.kernel_id = kKernelQuantDecode;
    // pages of whole tiles whose rows' scales lie side by side are loaded by TMA
    const int groups = c.bits == 8 ? 1 : c.head_dim / 64, row_bytes = c.head_dim * c.bits / 8;
    const bool paged = c.page_size % TOK == 0 && c.scale_token == 4 * groups &&
                       ((reinterpret_cast<uintptr_t>(c.k_scales) | reinterpret_cast<uintptr_t>(c.v_scales) | static_cast<uintptr_t>(c.scale_block | c.scale_head)) & 15) == 0;
    if (paged) {
        const uint32_t box_bytes = static_cast<uint32_t>(row_bytes < 128 ? row_bytes : 128);
        const tdist_host::Swizzle sw = box_bytes == 128 ? tdist_host::Swizzle::B128 : (box_bytes == 64 ? tdist_host::Swizzle::B64 : tdist_host::Swizzle::B32);
        const uint64_t dims[4] = {static_cast<uint64_t>(row_bytes), static_cast<uint64_t>(c.Hkv), static_cast<uint64_t>(c.page_size), static_cast<uint64_t>(c.blocks)};
        const uint64_t strides[3] = {static_cast<uint64_t>(c.code_head), static_cast<uint64_t>(c.code_token), static_cast<uint64_t>(c.code_block)};
        const uint32_t box[4] = {box_bytes, 1, TOK, 1};
        const uint64_t sdims[3] = {static_cast<uint64_t>(c.page_size) * groups, static_cast<uint64_t>(c.Hkv), static_cast<uint64_t>(c.blocks)};
        const uint64_t sstrides[2] = {static_cast<uint64_t>(c.scale_head), static_cast<uint64_t>(c.scale_block)};
        const uint32_t sbox[3] = {static_cast<uint32_t>(TOK * groups), 1, 1};
        int rc;
        if ((rc = tdist_host::encode_tmap(&p.tm_k, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 4, c.k_codes, dims, strides, box, sw))) return rc;
        if ((rc = tdist_host::encode_tmap(&p.tm_v, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, 4, c.v_codes, dims, strides, box, sw))) return rc;
        if ((rc = tdist_host::encode_tmap(&p.tm_ks, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, 3, c.k_scales, sdims, sstrides, sbox, tdist_host::Swizzle::None))) return rc;
        if ((rc = tdist_host::encode_tmap(&p.tm_vs, CU_TENSOR_MAP_DATA_TYPE_UINT32, 4, 3, c.v_scales, sdims, sstrides, sbox, tdist_host::Swizzle::None))) return rc;
    }
    const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
    const int rc = c.bits == 8 ? launch_dim<8>(p, c.head_dim, nh, paged, static_cast<int>(grid), stream)
                               : launch_dim<4>(p, c.head_dim, nh, paged, static_cast<int>(grid), stream);
    if (rc) return rc;
    if (a->splits > MAX_CLUSTER)
        TDIST_CUDA_OK(tdist_host::launch_pdl(merge_kernel, dim3(static_cast<unsigned>(c.B * a->Hq)), 128, 0, stream, p.part, a->splits, c.head_dim,
                                             p.is_f16, a->out));
    return 0;
}
