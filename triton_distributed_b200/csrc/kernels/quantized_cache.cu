// A paged KV cache in 8 or 4 bits: rows of new keys and values quantised into their places, and sequences read back as rows.
//
//   8 bits   a = max(max |x|, 2^-100), scale = a / 127 (fp32), code = 128 + rint(x (127 / a)); value = (code - 128) scale
//   4 bits   per 64 values: least = min rounded down to bf16, step = max((max - least) / 15, 2^-100) rounded up to bf16,
//            code = rint((x - least) (1 / step)) in [0, 15]; value = least + step code. Two codes per byte, the even index low.
// A row (group of 64) that holds a NaN or an infinity gets a scale (step, least) of NaN and reads as NaN: codes are always numbers.
// The roundings to bf16 go outwards, so that the 16 steps cover the group whatever its offset; a pair of fp16 would overflow where
// bf16 rows do not, one of fp32 would make 5 bits of 4.5.
// Quotients and products are IEEE's (this file is compiled without fast math): the same codes as the statement in torch.
//
// Bound by bytes. A lane takes 16 values (32 bytes) of a k row and of the v row beside it when writing, 16 codes of each of two places when reading:
// four loads of each lane under way at once. Quotients of places by heads and page sizes go by a multiplication, rounding by
// the addition of 1.5 2^23, whose low byte is the code. (8 values a lane when writing: 24 us for 16.8 below.)
//
// Measured, 8 kv heads of 128, bf16 (at HBM's copy rate): 16384 tokens written in 8 bits 16.9 us (15.5), in 4 22.1 (13.1); 131072 keys read
// back from 8 bits 131 us (124), from 4 122 (105). Writing 4 bits is bound by instructions (issue slots 81 % busy, the integer pipe 73 %): a largest magnitude, a minimum and a
// maximum per 64 values, each with two shuffles, and per code a subtraction, a product and its half of a byte. Reading 4 bits waits for memory (7 of 14 stalls per
// instruction; issue slots 61 %), some thousand keys for a chain of latencies: search, length, page, codes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstring>
#include <string>

#include "../device/ptx.cuh"
#include "../include/tdist.h"
#include "../runtime/host_common.h"

namespace tdist {
namespace qcache {

constexpr int THREADS = 256;
constexpr float kLeast = 7.888609052210118e-31f;   // 2^-100
constexpr int MAX_ROWS = 32;                       // rows of a reading CTA

struct Params {
    const char* x[2];      // write: k, v
    char* out[2];          // read: k, v
    uint8_t* codes[2];
    char* scales[2];
    const int* slots;      // write
    const int *starts, *lens, *table;   // read
    long long x_token[2], x_head[2];    // bytes
    long long code_block, code_token, code_head, scale_block, scale_head, scale_token;   // bytes
    long long rows;        // write: tokens; read: rows of the output
    int B, Hkv, blocks, page_size, max_blocks, is_f16, rows_per_cta;
    uint32_t head_mul, page_mul;   // n / Hkv = (n head_mul) >> head_shift for n < 2^31, the same for page_size
    int head_shift, page_shift;
};

__device__ __forceinline__ uint32_t quotient(uint32_t n, uint32_t mul, int shift) { return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift); }

// the largest bf16 that is not above x (x finite), as its 16 bits
__device__ __forceinline__ uint32_t bf16_down(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u >> 16) + ((u >> 31) && (u & 0xffffu) ? 1u : 0u);
}

// pairs of 16-bit numbers
template <bool F16>
struct Pair {
    static __device__ __forceinline__ float low(uint32_t w) { return F16 ? __low2float(*reinterpret_cast<const __half2*>(&w)) : __uint_as_float(w << 16); }
    static __device__ __forceinline__ float high(uint32_t w) { return F16 ? __high2float(*reinterpret_cast<const __half2*>(&w)) : __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t least(uint32_t a, uint32_t b) {
        if (F16) {
            const __half2 r = __hmin2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
            return *reinterpret_cast<const uint32_t*>(&r);
        }
        const __nv_bfloat162 r = __hmin2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    static __device__ __forceinline__ uint32_t most(uint32_t a, uint32_t b) {
        if (F16) {
            const __half2 r = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
            return *reinterpret_cast<const uint32_t*>(&r);
        }
        const __nv_bfloat162 r = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
};

// LANES lanes hold a row, 16 values each: what a row costs once (its place, the scale's quotients, the exchange between its lanes) counts as much as its
// values (8 per lane: 16384 tokens of 8 heads of 128 24.2 us in 8 bits, 33.6 in 4). Magnitudes are compared as 16-bit integers, whose order is the numbers'.
template <int BITS, int D, bool F16>
__global__ void __launch_bounds__(THREADS) write_kernel(const Params p) {
    using P = Pair<F16>;
    constexpr int LANES = D / 16, GROUP = BITS == 8 ? LANES : 4;   // lanes that share a scale
    const uint32_t item = static_cast<uint32_t>((static_cast<uint64_t>(blockIdx.x) * THREADS + threadIdx.x) / LANES);
    const int l = static_cast<int>(threadIdx.x) % LANES;
    pdl_wait_and_release();
    const long long t = quotient(item, p.head_mul, p.head_shift);
    const int h = static_cast<int>(item - static_cast<uint32_t>(t) * p.Hkv);
    const bool live = t < p.rows;
    const int slot = live ? p.slots[t] : -1;
    uint32_t w[2][8];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint4 v = live ? ld_v4(p.x[i] + t * p.x_token[i] + h * p.x_head[i] + l * 32 + j * 16) : make_uint4(0u, 0u, 0u, 0u);
            w[i][4 * j] = v.x;
            w[i][4 * j + 1] = v.y;
            w[i][4 * j + 2] = v.z;
            w[i][4 * j + 3] = v.w;
        }
    const int page = slot < 0 ? 0 : static_cast<int>(quotient(static_cast<uint32_t>(slot), p.page_mul, p.page_shift));
    const int row = slot - page * p.page_size;
    const bool kept = slot >= 0 && page < p.blocks;
    bool again[2] = {false, false};
    float bases[2], invs[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        uint32_t top = 0, lo2 = w[i][0], hi2 = w[i][0];
#pragma unroll
        for (int j = 0; j < 4; ++j) top = __vimax3_u16x2(top, w[i][2 * j] & 0x7fff7fffu, w[i][2 * j + 1] & 0x7fff7fffu);
        top = max(top & 0xffffu, top >> 16);
        if (BITS == 4) {
#pragma unroll
            for (int j = 1; j < 8; ++j) {
                lo2 = P::least(lo2, w[i][j]);
                hi2 = P::most(hi2, w[i][j]);
            }
        }
#pragma unroll
        for (int o = 1; o < GROUP; o <<= 1) {
            top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (BITS == 4) {
                lo2 = P::least(lo2, __shfl_xor_sync(0xffffffffu, lo2, o));
                hi2 = P::most(hi2, __shfl_xor_sync(0xffffffffu, hi2, o));
            }
        }
        const bool good = top < (F16 ? 0x7c00u : 0x7f80u);
        uint8_t* dst = p.codes[i] + page * p.code_block + row * p.code_token + h * p.code_head;
        char* sdst = p.scales[i] + page * p.scale_block + h * p.scale_head + row * p.scale_token;
        if (BITS == 8) {
            const float a = good ? fmaxf(P::low(top), kLeast) : 1.f;
            const float inv = __fdiv_rn(127.f, a);
            uint32_t o[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // 1.5 2^23 + 128 + the code: the low byte is what is stored
                const uint32_t b0 = __float_as_uint(__fadd_rn(__fmul_rn(P::low(w[i][2 * j]), inv), 12583040.f)), b1 = __float_as_uint(__fadd_rn(__fmul_rn(P::high(w[i][2 * j]), inv), 12583040.f));
                const uint32_t b2 = __float_as_uint(__fadd_rn(__fmul_rn(P::low(w[i][2 * j + 1]), inv), 12583040.f)), b3 = __float_as_uint(__fadd_rn(__fmul_rn(P::high(w[i][2 * j + 1]), inv), 12583040.f));
                o[j] = good ? __byte_perm(__byte_perm(b0, b1, 0x0040), __byte_perm(b2, b3, 0x0040), 0x5410) : 0x80808080u;
            }
            if (kept) {
                *reinterpret_cast<uint4*>(dst + l * 16) = make_uint4(o[0], o[1], o[2], o[3]);
                if (l == 0) *reinterpret_cast<float*>(sdst) = good ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fffffffu);
            }
        } else {
            const float lo = fminf(P::low(lo2), P::high(lo2)), hi = fmaxf(P::low(hi2), P::high(hi2));
            const uint32_t least = bf16_down(lo);
            const float base = __uint_as_float(least << 16);
            const float range = __fsub_rn(hi, base);
            const bool halved = !F16 && range > 3.4028234663852886e38f;   // a range beyond fp32's largest: differences of halves
            const float part = __fdiv_rn(halved ? __fsub_rn(0.5f * hi, 0.5f * base) : range, 15.f), wide = halved ? 2.f * part : fmaxf(part, kLeast);
            const uint32_t step = bf16_down(-wide) & 0x7fffu;   // up: down of the negative
            const float inv = __fdiv_rn(1.f, __uint_as_float(step << 16));
            uint32_t o[2] = {0u, 0u};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float c0 = fminf(15.f, fmaxf(0.f, __fmul_rn(__fsub_rn(P::low(w[i][j]), base), inv))), c1 = fminf(15.f, fmaxf(0.f, __fmul_rn(__fsub_rn(P::high(w[i][j]), base), inv)));
                const uint32_t pair = (__float_as_uint(__fadd_rn(c0, 12582912.f)) & 15u) | (__float_as_uint(__fadd_rn(c1, 12582912.f)) & 15u) << 4;
                o[j >> 2] |= pair << (8 * (j & 3));
            }
            if (kept) {
                *reinterpret_cast<uint2*>(dst + l * 8) = good ? make_uint2(o[0], o[1]) : make_uint2(0u, 0u);
                if ((l & 3) == 0) *reinterpret_cast<uint32_t*>(sdst + (l >> 2) * 4) = good ? step | (least << 16) : 0x7fff7fffu;
                again[i] = halved && good;
                bases[i] = base;
                invs[i] = inv;
            }
        }
    }
    if (BITS == 4 && (again[0] || again[1])) {   // the codes once more, from the values as they were read: a rare case, behind both rows so that their work stays side by side
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (!again[i]) continue;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(p.x[i] + t * p.x_token[i] + h * p.x_head[i] + l * 32);
            uint8_t* dst = p.codes[i] + page * p.code_block + row * p.code_token + h * p.code_head + l * 8;
#pragma unroll 1
            for (int j = 0; j < 8; ++j) {
                const float c0 = fminf(15.f, __fmul_rn(__fsub_rn(0.5f * P::low(src[j]), 0.5f * bases[i]), 2.f * invs[i])), c1 = fminf(15.f, __fmul_rn(__fsub_rn(0.5f * P::high(src[j]), 0.5f * bases[i]), 2.f * invs[i]));
                dst[j] = static_cast<uint8_t>((__float_as_uint(__fadd_rn(c0, 12582912.f)) & 15u) | (__float_as_uint(__fadd_rn(c1, 12582912.f)) & 15u) << 4);
            }
        }
    }
}

// 16 values of a row
template <int BITS>
__device__ __forceinline__ void values16(const uint4& codes, float scale, float least, float (&f)[16]) {
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        if (BITS == 8) f[j] = (static_cast<float>((w[j >> 2] >> (8 * (j & 3))) & 255u) - 128.f) * scale;
        else f[j] = fmaf(static_cast<float>((w[j >> 3] >> (4 * (j & 7))) & 15u), scale, least);   // the product is exact
    }
}

// 4 bits: a value beyond the largest number of the type by no more than half a step, as rounding to a code and the pair's rounding outwards leave it of one that was not
// beyond, is that number: stored once more, over the infinity. In halves: 15 steps above the least value may lie beyond fp32.
__device__ __forceinline__ void store_within(uint16_t* dst, uint32_t w0, uint32_t w1, float scale, float least, bool is_f16) {
    const float most = is_f16 ? 32752.f : 1.69476569462576775e38f;
    if (!(fmaxf(fmaf(7.5f, scale, 0.5f * least), -0.5f * least) > most)) return;   // (NaN too)
#pragma unroll 1
    for (int j = 0; j < 16; ++j) {
        const float half = fmaf(static_cast<float>(((j < 8 ? w0 : w1) >> (4 * (j & 7))) & 15u), 0.5f * scale, 0.5f * least);
        if (fabsf(half) > most && fabsf(half) - 0.25f * scale <= most) dst[j] = static_cast<uint16_t>((is_f16 ? 0x7bffu : 0x7f7fu) | (half < 0.f ? 0x8000u : 0u));
    }
}

// A CTA takes `rows_per_cta` rows of the output: first a thread per row looks its place up, then LANES lanes read a (row, head)'s k and v.
template <int BITS, int D>
__global__ void __launch_bounds__(THREADS, 4) read_kernel(const Params p) {
    constexpr int LANES = D / 16;
    __shared__ int page_s[MAX_ROWS], row_s[MAX_ROWS];
    pdl_wait_and_release();
    const long long r0 = static_cast<long long>(blockIdx.x) * p.rows_per_cta;
    const int n = static_cast<int>(min(static_cast<long long>(p.rows_per_cta), p.rows - r0));
    if (static_cast<int>(threadIdx.x) < n) {
        const int r = static_cast<int>(r0) + static_cast<int>(threadIdx.x);
        // the last sequence that starts at r or before (of those without rows, the last: the one behind them is r's)
        int a = 0, b = p.B;
        while (a < b) {
            const int m = (a + b) >> 1;
            if (p.starts[m] <= r) a = m + 1;
            else b = m;
        }
        int page = -1, row = 0;
        // (a sequence that starts before row 0 has none: rows count from 0, and r less its start might pass 31 bits)
        const int start = a > 0 ? p.starts[a - 1] : -1;
        if (start >= 0 && r < p.starts[a]) {
            const int j = r - start;
            const int in_table = static_cast<int>(quotient(static_cast<uint32_t>(j), p.page_mul, p.page_shift));
            if (j < min(p.lens[a - 1], 0x7fffffc0) && in_table < p.max_blocks) {
                page = p.table[static_cast<long long>(a - 1) * p.max_blocks + in_table];
                row = j - in_table * p.page_size;
                if (page < 0 || page >= p.blocks) page = -1;
            }
        }
        page_s[threadIdx.x] = page;
        row_s[threadIdx.x] = row;
    }
    __syncthreads();
    const int l = static_cast<int>(threadIdx.x) % LANES;
    const int items = n * p.Hkv;
    constexpr int STEP = THREADS / LANES, AT_ONCE = 2;
    for (int first = static_cast<int>(threadIdx.x) / LANES; first < items; first += STEP * AT_ONCE) {
        uint4 codes[AT_ONCE][2];
        float scale[AT_ONCE][2], least[AT_ONCE][2];
        bool there[AT_ONCE];
        int r[AT_ONCE], h[AT_ONCE];
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            const int item = first + u * STEP;
            r[u] = static_cast<int>(quotient(static_cast<uint32_t>(item), p.head_mul, p.head_shift));
            h[u] = item - r[u] * p.Hkv;
            const int page = item < items ? page_s[r[u]] : -1;
            there[u] = page >= 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                codes[u][i] = make_uint4(0u, 0u, 0u, 0u);
                scale[u][i] = least[u][i] = 0.f;
                if (!there[u]) continue;
                const int row = row_s[r[u]];
                const uint8_t* src = p.codes[i] + page * p.code_block + row * p.code_token + h[u] * p.code_head;
                const char* ssrc = p.scales[i] + page * p.scale_block + h[u] * p.scale_head + row * p.scale_token;
                if (BITS == 8) {
                    codes[u][i] = ld_v4(src + l * 16);
                    scale[u][i] = *reinterpret_cast<const float*>(ssrc);
                } else {
                    const uint2 w = *reinterpret_cast<const uint2*>(src + l * 8);
                    codes[u][i].x = w.x;
                    codes[u][i].y = w.y;
                    const uint32_t pair = *reinterpret_cast<const uint32_t*>(ssrc + (l >> 2) * 4);
                    scale[u][i] = __uint_as_float(pair << 16);
                    least[u][i] = __uint_as_float(pair & 0xffff0000u);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
            if (first + u * STEP >= items) break;
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                float f[16];
                values16<BITS>(codes[u][i], scale[u][i], least[u][i], f);
                uint32_t o[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    o[j] = p.is_f16 ? pack_f16x2(f[2 * j], f[2 * j + 1]) : pack_bf16x2(f[2 * j], f[2 * j + 1]);
                    if (!there[u]) o[j] = 0u;   // (codes of 0 would be -128 times 0: a negative zero)
                }
                uint4* dst = reinterpret_cast<uint4*>(p.out[i] + ((r0 + r[u]) * p.Hkv + h[u]) * (D * 2ll) + l * 32);
                dst[0] = make_uint4(o[0], o[1], o[2], o[3]);
                dst[1] = make_uint4(o[4], o[5], o[6], o[7]);
                if (BITS == 4 && there[u]) store_within(reinterpret_cast<uint16_t*>(dst), codes[u][i].x, codes[u][i].y, scale[u][i], least[u][i], p.is_f16);
            }
        }
    }
}

static void multiplier(int n, uint32_t* mul, int* shift) {
    // with 2^l >= n the multiplier ceil(2^(31 + l) / n) is off by less than one, so its product with a number below 2^31 by less than 2^31
    int l = 0;
    while ((1ll << l) < n) ++l;
    *shift = 31 + l;
    *mul = static_cast<uint32_t>(((1ull << (31 + l)) + static_cast<uint64_t>(n) - 1) / static_cast<uint64_t>(n));
}

static int fill(const TdistQuantCacheArgs* a, Params& p) {
    if (a->bits != 8 && a->bits != 4) return tdist_host::fail(TDIST_EINVAL, "quantised cache: 8 or 4 bits");
    if (a->head_dim != 64 && a->head_dim != 128 && a->head_dim != 256) return tdist_host::fail(TDIST_EINVAL, "quantised cache: head_dim must be 64, 128 or 256");
    if (a->Hkv < 1 || a->page_size < 1 || a->blocks < 0) return tdist_host::fail(TDIST_EINVAL, "quantised cache: bad shape");
    if (a->dtype != TDIST_BF16 && a->dtype != TDIST_F16) return tdist_host::fail(TDIST_EINVAL, "quantised cache: rows must be bf16 or fp16");
    memset(&p, 0, sizeof(p));
    p.codes[0] = static_cast<uint8_t*>(a->k_codes);
    p.codes[1] = static_cast<uint8_t*>(a->v_codes);
    p.scales[0] = static_cast<char*>(a->k_scales);
    p.scales[1] = static_cast<char*>(a->v_scales);
    p.code_block = a->code_block;
    p.code_token = a->code_token;
    p.code_head = a->code_head;
    p.scale_block = a->scale_block;
    p.scale_head = a->scale_head;
    p.scale_token = a->scale_token;
    p.B = a->B;
    p.Hkv = a->Hkv;
    p.blocks = a->blocks;
    p.page_size = a->page_size;
    p.max_blocks = a->max_blocks;
    p.is_f16 = a->dtype == TDIST_F16;
    p.rows = a->rows;
    multiplier(a->Hkv, &p.head_mul, &p.head_shift);
    multiplier(a->page_size, &p.page_mul, &p.page_shift);
    const uintptr_t code_align = reinterpret_cast<uintptr_t>(a->k_codes) | reinterpret_cast<uintptr_t>(a->v_codes) |
                                 static_cast<uintptr_t>(a->code_block | a->code_token | a->code_head);
    const uintptr_t scale_align = reinterpret_cast<uintptr_t>(a->k_scales) | reinterpret_cast<uintptr_t>(a->v_scales) |
                                  static_cast<uintptr_t>(a->scale_block | a->scale_head | a->scale_token);
    if ((code_align & 15) || (scale_align & (a->bits == 8 ? 3 : a->head_dim / 16 - 1)))
        return tdist_host::fail(TDIST_EINVAL, "quantised cache: codes must lie on 16 bytes, a row's scales on their size");
    return 0;
}

}  // namespace qcache
}  // namespace tdist

using namespace tdist;
using tdist_host::fail;

namespace {
template <int BITS, int D>
cudaError_t write_rows(bool f16, dim3 grid, cudaStream_t stream, const qcache::Params& p) {
    return f16 ? tdist_host::launch_pdl(qcache::write_kernel<BITS, D, true>, grid, qcache::THREADS, 0, stream, p)
               : tdist_host::launch_pdl(qcache::write_kernel<BITS, D, false>, grid, qcache::THREADS, 0, stream, p);
}
template <int BITS, int D>
cudaError_t read_rows(dim3 grid, cudaStream_t stream, const qcache::Params& p) {
    return tdist_host::launch_pdl(qcache::read_kernel<BITS, D>, grid, qcache::THREADS, 0, stream, p);
}
}  // namespace

extern "C" int tdist_quant_cache_write(const TdistQuantCacheArgs* a) {
    qcache::Params p;
    int rc = qcache::fill(a, p);
    if (rc) return rc;
    if (a->rows <= 0 || a->blocks == 0) return 0;
    p.x[0] = static_cast<const char*>(a->k);
    p.x[1] = static_cast<const char*>(a->v);
    p.x_token[0] = a->k_token;
    p.x_head[0] = a->k_head;
    p.x_token[1] = a->v_token;
    p.x_head[1] = a->v_head;
    p.slots = static_cast<const int*>(a->slots);
    if ((reinterpret_cast<uintptr_t>(a->k) | reinterpret_cast<uintptr_t>(a->v) | static_cast<uintptr_t>(a->k_token | a->k_head | a->v_token | a->v_head)) & 15)
        return fail(TDIST_EINVAL, "quantised cache: rows must lie on 16 bytes");
    const long long lanes = a->head_dim / 16, threads = a->rows * a->Hkv * lanes;
    const long long grid = (threads + qcache::THREADS - 1) / qcache::THREADS;
    if (a->rows * a->Hkv > 0x7ffffff0ll) return fail(TDIST_EINVAL, "quantised cache: too many rows in one call");
    const dim3 blocks(static_cast<unsigned>(grid));
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    const bool f16 = a->dtype == TDIST_F16;
    cudaError_t e;
    if (a->bits == 8)
        e = (a->head_dim == 64 ? write_rows<8, 64>(f16, blocks, stream, p) : (a->head_dim == 128 ? write_rows<8, 128>(f16, blocks, stream, p) : write_rows<8, 256>(f16, blocks, stream, p)));
    else
        e = (a->head_dim == 64 ? write_rows<4, 64>(f16, blocks, stream, p) : (a->head_dim == 128 ? write_rows<4, 128>(f16, blocks, stream, p) : write_rows<4, 256>(f16, blocks, stream, p)));
    TDIST_CUDA_OK(e);
    return 0;
}

extern "C" int tdist_quant_cache_read(const TdistQuantCacheArgs* a) {
    qcache::Params p;
    int rc = qcache::fill(a, p);
    if (rc) return rc;
    if (a->rows <= 0) return 0;
    if (a->rows > 0x7fffffffll || a->B < 0 || a->max_blocks < 0) return fail(TDIST_EINVAL, "quantised cache: bad shape");
    p.out[0] = static_cast<char*>(a->k_out);
    p.out[1] = static_cast<char*>(a->v_out);
    if ((reinterpret_cast<uintptr_t>(a->k_out) | reinterpret_cast<uintptr_t>(a->v_out)) & 15)
        return fail(TDIST_EINVAL, "quantised cache: outputs must lie on 16 bytes");
    p.starts = static_cast<const int*>(a->starts);
    p.lens = static_cast<const int*>(a->lens);
    p.table = static_cast<const int*>(a->table);
    // few rows: a CTA each, so that all lookups run side by side
    int per = qcache::MAX_ROWS;
    while (per > 1 && (a->rows + per - 1) / per < 8ll * tdist_host::sm_count()) per >>= 1;
    p.rows_per_cta = per;
    const long long grid = (a->rows + per - 1) / per;
    const dim3 blocks(static_cast<unsigned>(grid));
    const cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    cudaError_t e;
    if (a->bits == 8)
        e = (a->head_dim == 64 ? read_rows<8, 64>(blocks, stream, p) : (a->head_dim == 128 ? read_rows<8, 128>(blocks, stream, p) : read_rows<8, 256>(blocks, stream, p)));
    else
        e = (a->head_dim == 64 ? read_rows<4, 64>(blocks, stream, p) : (a->head_dim == 128 ? read_rows<4, 128>(blocks, stream, p) : read_rows<4, 256>(blocks, stream, p)));
    TDIST_CUDA_OK(e);
    return 0;
}
