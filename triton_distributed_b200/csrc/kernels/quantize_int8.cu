// Rows of bf16 / fp16 / fp32 to signed 8-bit integers with a scale each: a = max(max |x|, 2^-100), scale = a / 127, code = rint(x (127 / a)).
// A row with a NaN or an infinity gets a scale of NaN and codes of 0. Quotients and products are IEEE's (compiled without fast math), so the
// codes are those of the statement in torch.
//
// Bound by bytes: a CTA per row holds up to 64 values of it per thread in registers between the two passes; longer rows are read again (L2).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../device/ptx.cuh"
#include "../include/tdist.h"
#include "../runtime/host_common.h"

namespace tdist {
namespace quant8 {

constexpr int THREADS = 256, HELD = 8;       // HELD x 8 values of a thread stay in registers
constexpr float kLeast = 7.888609052210118e-31f;   // 2^-100

template <int DT>
__device__ __forceinline__ void load8(const char* row, long long i, float (&f)[8]) {
    if (DT == TDIST_F32) {
        const uint4 a = ld_v4(row + i * 32), b = ld_v4(row + i * 32 + 16);
        const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
    } else {
        const uint4 a = ld_v4(row + i * 16);
        const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (DT == TDIST_F16) {
                const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                f[2 * j] = t.x;
                f[2 * j + 1] = t.y;
            } else {
                f[2 * j] = __uint_as_float(w[j] << 16);
                f[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
            }
        }
    }
}

template <int DT>
__global__ void __launch_bounds__(THREADS) quantize_kernel(const char* x, long long row_bytes, int chunks, int8_t* out, float* scale) {
    __shared__ uint32_t top_s[THREADS / 32];
    pdl_wait_and_release();
    const char* row = x + static_cast<long long>(blockIdx.x) * row_bytes;
    const int t = static_cast<int>(threadIdx.x);
    float f[HELD][8];
    uint32_t top = 0;   // bits of the largest magnitude; a NaN's lie above an infinity's
#pragma unroll
    for (int i = 0; i < HELD; ++i) {
        if (t + i * THREADS < chunks) load8<DT>(row, t + i * THREADS, f[i]);
        else
#pragma unroll
            for (int j = 0; j < 8; ++j) f[i][j] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < HELD; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[i][j]) & 0x7fffffffu);
    for (int i = t + HELD * THREADS; i < chunks; i += THREADS) {
        float g[8];
        load8<DT>(row, i, g);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(g[j]) & 0x7fffffffu);
    }
    top = __reduce_max_sync(0xffffffffu, top);
    if ((t & 31) == 0) top_s[t >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) top = max(top, top_s[w]);
    const bool good = top < 0x7f800000u;
    const float a = fmaxf(good ? __uint_as_float(top) : 1.f, kLeast);
    const float inv = __fdiv_rn(127.f, a);
    if (t == 0) scale[blockIdx.x] = good ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7fffffffu);
    int8_t* dst = out + static_cast<long long>(blockIdx.x) * chunks * 8;
    auto put = [&](int i, const float (&v)[8]) {
        uint32_t w[2] = {0u, 0u};
#pragma unroll
        for (int j = 0; j < 8; ++j) w[j >> 2] |= (static_cast<uint32_t>(good ? __float2int_rn(__fmul_rn(v[j], inv)) : 0) & 255u) << (8 * (j & 3));
        *reinterpret_cast<uint2*>(dst + static_cast<long long>(i) * 8) = make_uint2(w[0], w[1]);
    };
#pragma unroll
    for (int i = 0; i < HELD; ++i)
        if (t + i * THREADS < chunks) put(t + i * THREADS, f[i]);
    for (int i = t + HELD * THREADS; i < chunks; i += THREADS) {
        float g[8];
        load8<DT>(row, i, g);
        put(i, g);
    }
}

}  // namespace quant8
}  // namespace tdist

using tdist_host::fail;

// x [rows, k] (row_stride elements from one to the next, k a multiple of 8) -> int8 [rows, k] and fp32 scales [rows]
extern "C" int tdist_quant_int8_rowwise(const void* x, long long row_stride, void* out, void* scale, long long rows, int k, int dtype, void* stream) {
    using namespace tdist::quant8;
    const int size = dtype == TDIST_F32 ? 4 : 2;
    if (rows < 0 || rows > 0x7fffffffll || k < 8 || k % 8) return fail(TDIST_EINVAL, "int8 quantiser: bad shape");
    if (dtype != TDIST_BF16 && dtype != TDIST_F16 && dtype != TDIST_F32) return fail(TDIST_EINVAL, "int8 quantiser: rows must be bf16, fp16 or fp32");
    if ((reinterpret_cast<uintptr_t>(x) & 15) || (row_stride * size) % 16 || (reinterpret_cast<uintptr_t>(out) & 7))
        return fail(TDIST_EINVAL, "int8 quantiser: rows must lie on 16 bytes");
    if (rows == 0) return 0;
    const dim3 grid(static_cast<unsigned>(rows));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const char* src = static_cast<const char*>(x);
    int8_t* dst = static_cast<int8_t*>(out);
    float* sc = static_cast<float*>(scale);
    cudaError_t e;
    if (dtype == TDIST_F32) e = tdist_host::launch_pdl(quantize_kernel<TDIST_F32>, grid, THREADS, 0, s, src, row_stride * size, k / 8, dst, sc);
    else if (dtype == TDIST_F16) e = tdist_host::launch_pdl(quantize_kernel<TDIST_F16>, grid, THREADS, 0, s, src, row_stride * size, k / 8, dst, sc);
    else e = tdist_host::launch_pdl(quantize_kernel<TDIST_BF16>, grid, THREADS, 0, s, src, row_stride * size, k / 8, dst, sc);
    TDIST_CUDA_OK(e);
    return 0;
}
