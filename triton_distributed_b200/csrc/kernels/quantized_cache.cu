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
// Bound by bytes. A lane takes 8 values (16 bytes) of a k row and of the v row beside it when writing, 16 codes of each of two places when reading:
// two and four loads of each lane under way at once. Quotients of places by heads and page sizes go by a multiplication, rounding by
// the addition of 1.5 2^23, whose low byte is the code.
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

__device__ __forceinline__ void unpack8(const uint4& v, int is_f16, float (&f)[8]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (is_f16) {
            const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = t.x;
            f[2 * i + 1] = t.y;
        } else {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
// the largest bf16 that is not above x (x finite), as its 16 bits
__device__ __forceinline__ uint32_t bf16_down(float x) {
    const uint32_t u = __float_as_uint(x);
    return (u >> 16) + ((u >> 31) && (u & 0xffffu) ? 1u : 0u);
}

// LANES lanes hold a row, 8 values each
template <int BITS, int D>
__global__ void __launch_bounds__(THREADS) write_kernel(const Params p) {
    constexpr int LANES = D / 8, GROUP = BITS == 8 ? LANES : 8;   // lanes that share a scale
    const uint32_t item = static_cast<uint32_t>((static_cast<uint64_t>(blockIdx.x) * THREADS + threadIdx.x) / LANES);
    const int l = static_cast<int>(threadIdx.x) % LANES;
    pdl_wait_and_release();
    const long long t = quotient(item, p.head_mul, p.head_shift);
    const int h = static_cast<int>(item - static_cast<uint32_t>(t) * p.Hkv);
    const bool live = t < p.rows;
    const int slot = live ? p.slots[t] : -1;
    uint4 raw[2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
        raw[i] = live ? ld_v4(p.x[i] + t * p.x_token[i] + h * p.x_head[i] + l * 16) : make_uint4(0u, 0u, 0u, 0u);
    const int page = slot < 0 ? 0 : static_cast<int>(quotient(static_cast<uint32_t>(slot), p.page_mul, p.page_shift));
    const int row = slot - page * p.page_size;
    const bool kept = slot >= 0 && page < p.blocks;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        float f[8];
        unpack8(raw[i], p.is_f16, f);
        uint32_t top = 0;   // bits of the largest magnitude; a NaN's lie above an infinity's
        float lo = f[0], hi = f[0];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
            lo = fminf(lo, f[j]);
            hi = fmaxf(hi, f[j]);
        }
#pragma unroll
        for (int o = 1; o < GROUP; o <<= 1) {
            top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
            if (BITS == 4) {
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
                hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
        }
        const bool good = top < 0x7f800000u;
        uint8_t* dst = p.codes[i] + page * p.code_block + row * p.code_token + h * p.code_head;
        char* sdst = p.scales[i] + page * p.scale_block + h * p.scale_head + row * p.scale_token;
        if (BITS == 8) {
            const float a = fmaxf(good ? __uint_as_float(top) : 1.f, kLeast);
            const float inv = __fdiv_rn(127.f, a);
            uint32_t b[8];   // 1.5 2^23 + 128 + the code: the low byte is what is stored
#pragma unroll
            for (int j = 0; j < 8; ++j) b[j] = good ? __float_as_uint(__fadd_rn(__fmul_rn(f[j], inv), 12583040.f)) : 128u;
            const uint32_t w[2] = {__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                                   __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410)};
            if (kept) {
                *reinterpret_cast<uint2*>(dst + l * 8) = make_uint2(w[0], w[1]);
                if (l == 0) *reinterpret_cast<float*>(sdst) = good ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fffffffu);
            }
        } else {
            const uint32_t least = bf16_down(lo);
            const float base = __uint_as_float(least << 16);
            const float wide = fmaxf(__fdiv_rn(__fsub_rn(hi, base), 15.f), kLeast);
            const uint32_t step = bf16_down(-wide) & 0x7fffu;   // up: down of the negative (a range beyond fp32's: infinite)
            const float inv = __fdiv_rn(1.f, __uint_as_float(step << 16));
            uint32_t w = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                // (a NaN, from a range beyond fp32's, gives 0)
                const float c = fminf(15.f, fmaxf(0.f, __fmul_rn(__fsub_rn(f[j], base), inv)));
                w |= (good ? __float_as_uint(__fadd_rn(c, 12582912.f)) & 15u : 0u) << (4 * j);
            }
            if (kept) {
                *reinterpret_cast<uint32_t*>(dst + l * 4) = w;
                if ((l & 7) == 0) *reinterpret_cast<uint32_t*>(sdst + (l >> 3) * 4) = good ? step | (least << 16) : 0x7fff7fffu;
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

// A CTA takes `rows_per_cta` rows of the output: first a thread per row looks its place up, then LANES lanes read a (row, head)'s k and v.
template <int BITS, int D>
__global__ void __launch_bounds__(THREADS) read_kernel(const Params p) {
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
        if (a > 0 && r < p.starts[a]) {
            const int j = r - p.starts[a - 1];
            const int in_table = static_cast<int>(quotient(static_cast<uint32_t>(j), p.page_mul, p.page_shift));
            if (j < p.lens[a - 1] && in_table < p.max_blocks) {
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

#define TDIST_BY_CACHE(kernel, bits, dim, ...)                                                                      \
    do {                                                                                                            \
        cudaError_t e;                                                                                              \
        if (bits == 8)                                                                                              \
            e = dim == 64 ? tdist_host::launch_pdl(kernel<8, 64>, __VA_ARGS__)                                      \
                          : (dim == 128 ? tdist_host::launch_pdl(kernel<8, 128>, __VA_ARGS__) : tdist_host::launch_pdl(kernel<8, 256>, __VA_ARGS__)); \
        else                                                                                                        \
            e = dim == 64 ? tdist_host::launch_pdl(kernel<4, 64>, __VA_ARGS__)                                      \
                          : (dim == 128 ? tdist_host::launch_pdl(kernel<4, 128>, __VA_ARGS__) : tdist_host::launch_pdl(kernel<4, 256>, __VA_ARGS__)); \
        TDIST_CUDA_OK(e);                                                                                           \
    } while (0)

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
    const long long lanes = a->head_dim / 8, threads = a->rows * a->Hkv * lanes;
    const long long grid = (threads + qcache::THREADS - 1) / qcache::THREADS;
    if (a->rows * a->Hkv > 0x7ffffff0ll) return fail(TDIST_EINVAL, "quantised cache: too many rows in one call");
    TDIST_BY_CACHE(qcache::write_kernel, a->bits, a->head_dim, dim3(static_cast<unsigned>(grid)), qcache::THREADS, 0, static_cast<cudaStream_t>(a->stream), p);
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
    while (per > 1 && (a->rows + per - 1) / per < 4ll * tdist_host::sm_count()) per >>= 1;
    p.rows_per_cta = per;
    const long long grid = (a->rows + per - 1) / per;
    TDIST_BY_CACHE(qcache::read_kernel, a->bits, a->head_dim, dim3(static_cast<unsigned>(grid)), qcache::THREADS, 0, static_cast<cudaStream_t>(a->stream), p);
    return 0;
}
