// Few-row GEMM of 8-bit integers for sm_100a: the product of gemm_int8_sm100.cu for a decode step's or a short prompt's tokens.
//
// Bound by reading B (the weights) once from HBM, and cut up as gemm_skinny_sm100.cu does it: 128 weight rows are the M operand of
// tcgen05.mma (kind::i8), up to 128 tokens its N operand, and the K ranges of a tile (`split` of them) form a cluster whose CTAs
// add their sums through shared memory, in 32-bit integers: exact in any order. CTA r of a cluster scales and writes the r-th share of the tokens.
//
// Measured: 16 x 6144 x 12288 17.0 us (75 MB, 11.6 at HBM's copy rate), 1 x 4096 x 4096 6.7 (2.6: start, one tile's latency, the exchange), 128 tokens 10.9.
//
// Warps (192 threads): 0 = TMA producer, 1 = MMA issuer and TMEM owner, 2..5 = epilogue. One tile per CTA, two CTAs per SM.
#include <cuda.h>
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <mutex>

#include "../device/ptx.cuh"
#include "../device/signal.cuh"
#include "../include/tdist.h"
#include "../runtime/host_common.h"
#include "gemm_int8.h"

namespace tdist {
namespace int8_skinny {

constexpr int ROWS = 128;      // weight rows per CTA (UMMA M)
constexpr int MAX_TOK = 128;   // tokens per CTA (UMMA N)
constexpr int BK = 128, UMMA_K = 32;   // values = bytes
constexpr int W_BYTES = ROWS * BK;
constexpr int MAX_STAGES = 6, MAX_SPLIT = 8;
constexpr int THREADS = 192;
constexpr int STAGE_AREA = 108 * 1024;   // with alignment and barriers below half of an SM's 227 KB: two CTAs per SM
constexpr int SMEM_BYTES = STAGE_AREA + 1024 + 256;
// the partials of one cluster share: split x ceil(tok / split) tokens x 128 rows of 32 bits
static_assert((MAX_TOK + MAX_SPLIT) * ROWS * 4 <= STAGE_AREA, "the partial sums reuse the stages");

constexpr int kKernelSkinny = 10;   // reported as the int8 GEMM

struct Params {
    CUtensorMap tm_w;   // {K, N}, box {128, 128}
    CUtensorMap tm_x;   // {K, M}, box {128, tok}
    const float *sa, *sb;
    void* out;          // [M, N] bf16 / fp16
    int m, n, k_blocks, tok, m_tiles, split, stages, is_f16, tmem_cols;
    WaitCtx wctx;
};

__global__ void __launch_bounds__(THREADS, 2) gemm_int8_skinny_kernel(const __grid_constant__ Params p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + STAGE_AREA);   // [0,S) full, [S,2S) empty, [2S] accumulator done
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * MAX_STAGES + 1);
    const int warp = static_cast<int>(threadIdx.x) >> 5;
    const int lane = static_cast<int>(threadIdx.x) & 31;
    const uint32_t bars_u32 = smem_u32(bars);
    auto bar_full = [&](uint32_t s) { return bars_u32 + 8u * s; };
    auto bar_empty = [&](uint32_t s) { return bars_u32 + 8u * (MAX_STAGES + s); };
    const uint32_t bar_done = bars_u32 + 8u * (2 * MAX_STAGES);

    const int tile = static_cast<int>(blockIdx.x) / p.split;
    const int part = static_cast<int>(blockIdx.x) - tile * p.split;   // = rank in the cluster
    const int m0 = (tile % p.m_tiles) * p.tok;    // the token tiles of one weight tile run side by side: it is read from HBM once
    const int n0 = (tile / p.m_tiles) * ROWS;
    const int kb0 = static_cast<int>(static_cast<long long>(p.k_blocks) * part / p.split);
    const int kb1 = static_cast<int>(static_cast<long long>(p.k_blocks) * (part + 1) / p.split);
    const uint32_t stage_bytes = W_BYTES + static_cast<uint32_t>(p.tok) * BK;
    const uint32_t stages = static_cast<uint32_t>(p.stages);

    if (threadIdx.x == 0) {
        prefetch_tensormap(&p.tm_w);
        prefetch_tensormap(&p.tm_x);
        for (uint32_t s = 0; s < stages; ++s) {
            mbar_init(bar_full(s), 1);
            mbar_init(bar_empty(s), 1);
        }
        mbar_init(bar_done, 1);
        fence_mbar_init();
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(tmem_slot), static_cast<uint32_t>(p.tmem_cols));
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(tmem_slot);
    pdl_wait_and_release();

    if (warp == 0) {
        if (lane == 0) {
            uint32_t s = 0, phase = 1;
            for (int kb = kb0; kb < kb1; ++kb) {
                mbar_wait(bar_empty(s), phase, p.wctx, 2);
                const uint32_t dst = smem_u32(smem) + s * stage_bytes;
                mbar_expect_tx(bar_full(s), stage_bytes);
                tma_load_2d(dst, &p.tm_w, bar_full(s), kb * BK, n0);
                tma_load_2d(dst + W_BYTES, &p.tm_x, bar_full(s), kb * BK, m0);
                if (++s == stages) {
                    s = 0;
                    phase ^= 1u;
                }
            }
        }
        __syncwarp();
    } else if (warp == 1) {
        if (lane == 0) {
            const uint32_t idesc = umma_idesc_s8(ROWS, static_cast<uint32_t>(p.tok));
            uint32_t s = 0, phase = 0;
            for (int kb = kb0; kb < kb1; ++kb) {
                mbar_wait(bar_full(s), phase, p.wctx, 4);
                tc_fence_after();
                const uint32_t src = smem_u32(smem) + s * stage_bytes;
                const uint64_t wdesc = umma_desc_k_sw128(src);
                const uint64_t xdesc = umma_desc_k_sw128(src + W_BYTES);
#pragma unroll
                for (int k = 0; k < BK / UMMA_K; ++k) umma_s8<1>(tmem_base, wdesc + 2 * k, xdesc + 2 * k, idesc, (kb != kb0 || k != 0) ? 1u : 0u);
                umma_commit(bar_empty(s));
                if (++s == stages) {
                    s = 0;
                    phase ^= 1u;
                }
            }
            umma_commit(bar_done);
        }
        __syncwarp();
    } else {
        mbar_wait(bar_done, 0, p.wctx, 5);
        tc_fence_after();
    }

    // ---- exchange: [source part][token of the share][weight row] 32-bit integers in every CTA's shared memory
    cluster_arrive();   // this CTA's MMAs (and with them its loads) are complete: its stages may be overwritten
    cluster_wait();
    const int live = min(p.tok, p.m - m0);
    const int per = (p.tok + p.split - 1) / p.split;
    int* sums = reinterpret_cast<int*>(smem);
    if (warp >= 2) {
        const int q = warp & 3;   // TMEM lane quadrant this warp may read
        const uint32_t mine = smem_u32(sums) + static_cast<uint32_t>((part * per * ROWS + q * 32 + lane) * 4);
        int owner = 0, j = 0;
        uint32_t dst = mapa_u32(mine, 0);
        for (int c = 0; c < live; c += 16) {
            uint32_t r[16];
            tmem_ld_32x16(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + static_cast<uint32_t>(c), r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                st_shared_cluster_f32(dst + static_cast<uint32_t>(j) * (ROWS * 4), __uint_as_float(r[i]));
                if (++j == per) {
                    j = 0;
                    owner = min(owner + 1, p.split - 1);
                    dst = mapa_u32(mine, static_cast<uint32_t>(owner));
                }
            }
        }
    }
    tc_fence_before();
    cluster_arrive();
    cluster_wait();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, static_cast<uint32_t>(p.tmem_cols));
    }
    const int t0 = part * per;
    const int items = min(per, live - t0) * (ROWS / 4);   // 4 columns of a token each; this CTA's share may be empty
    constexpr int UNROLL = 4;   // items per thread and step: their loads of one source part are in flight together
    for (int i0 = static_cast<int>(threadIdx.x); i0 < items; i0 += UNROLL * THREADS) {
        int4 acc[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) acc[u] = make_int4(0, 0, 0, 0);
        for (int s = 0; s < p.split; ++s) {
            const int4* src = reinterpret_cast<const int4*>(sums + s * per * ROWS);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                if (i0 + u * THREADS >= items) continue;
                const int4 v = src[i0 + u * THREADS];
                acc[u].x += v.x;
                acc[u].y += v.y;
                acc[u].z += v.z;
                acc[u].w += v.w;
            }
        }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) {
            const int i = i0 + u * THREADS;
            const int t = i / (ROWS / 4), c = (i % (ROWS / 4)) * 4;
            if (i >= items || n0 + c >= p.n) continue;   // N is a multiple of 8: all four columns or none
            const float sa = p.sa[m0 + t0 + t];
            const float4 sb = *reinterpret_cast<const float4*>(p.sb + n0 + c);
            const float x = static_cast<float>(acc[u].x) * sa * sb.x, y = static_cast<float>(acc[u].y) * sa * sb.y;
            const float z = static_cast<float>(acc[u].z) * sa * sb.z, v = static_cast<float>(acc[u].w) * sa * sb.w;
            const uint2 w = p.is_f16 ? make_uint2(pack_f16x2(x, y), pack_f16x2(z, v)) : make_uint2(pack_bf16x2(x, y), pack_bf16x2(z, v));
            *reinterpret_cast<uint2*>(static_cast<char*>(p.out) + (static_cast<size_t>(m0 + t0 + t) * p.n + n0 + c) * 2) = w;
        }
    }
}

}  // namespace int8_skinny
}  // namespace tdist

using namespace tdist;
using tdist_host::fail;

namespace {

// CTAs of the kernel that are resident at once when they come in clusters of `split` (a cluster needs its SMs in one GPC,
// so sizes that do not divide a GPC leave some unused). The occupancy query counts one CTA per SM here whatever the
// carveout; two do run (clusters of four, n6144 k12288: 192 CTAs finish sooner than 144 in clusters of three). Cached per device.
int int8_slots(int split) {
    using namespace tdist::int8_skinny;
    static int cache[64][MAX_SPLIT + 1] = {};
    static std::mutex lock;
    std::lock_guard<std::mutex> guard(lock);
    int dev = 0;
    const int nominal = 2 * tdist_host::sm_count() / split * split;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
        cudaGetLastError();
        return nominal;   // planning on a host without a GPU
    }
    int& slot = cache[dev][split];
    if (slot > 0) return slot;
    int clusters = 0;
    const void* fn = reinterpret_cast<const void*>(&gemm_int8_skinny_kernel);
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(nominal));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_BYTES) == cudaSuccess &&
        cudaOccupancyMaxActiveClusters(&clusters, fn, &cfg) == cudaSuccess && clusters > 0)
        slot = clusters * split <= tdist_host::sm_count() ? 2 * clusters * split : clusters * split;
    else
        slot = nominal;
    cudaGetLastError();
    return slot;
}

}  // namespace

namespace tdist_host {

bool int8_skinny_plan(int m, int n, int k, double other_s, SkinnyPlan* plan) {
    using namespace tdist::int8_skinny;
    if (m > 4 * MAX_TOK) return false;   // every further 128 tokens read the weights once more out of L2
    const int m_tiles = (m + MAX_TOK - 1) / MAX_TOK;
    const int tok = ((m + m_tiles - 1) / m_tiles + 15) / 16 * 16;
    const int n_tiles = (n + ROWS - 1) / ROWS;
    const int k_blocks = (k + BK - 1) / BK;
    const int tiles = n_tiles * m_tiles;
    // The model of gemm_skinny_sm100.cu, whose runs have the same bytes per K block: a CTA moves 70 GB/s
    // whatever its tile (twice the stages on a CTA that has its SM to itself changed nothing), HBM delivers 6.4 TB/s and
    // the two bend into one another; launch, first loads and the exchange of the partial sums cost 5.3 us and 15-50 ns per
    // token of the tile, the most where two CTAs share an SM; half of that again for every further round.
    const double stage = W_BYTES + tok * BK;
    const double hbm_s = (static_cast<double>(n) * k + static_cast<double>(m) * k + 2.0 * m * n) / 6.4e12;
    const int sms = tdist_host::sm_count();
    double best = 1e30;
    int best_split = 1;
    for (int split = 1; split <= MAX_SPLIT; ++split) {
        if (split > 1 && k_blocks < 3 * split) break;   // a part shorter than the pipeline only adds partial sums
        const int slots = int8_slots(split);
        const int ctas = tiles * split;
        const int blocks = (k_blocks + split - 1) / split;
        const int rounds = (ctas + slots - 1) / slots;
        const double sm_s = rounds * blocks * stage / 70e9;
        const double loads = std::pow(std::pow(sm_s * 1e6, 6) + std::pow(hbm_s * 1e6, 6), 1.0 / 6) * 1e-6;
        const double fixed = 5.3e-6 + tok * (15e-9 + 16e-9 / split + (ctas > sms ? 20e-9 : 0.0)) + 0.05e-6 * split;
        const double t = loads + fixed * (1 + 0.5 * (rounds - 1));
        if (t < best) {
            best = t;
            best_split = split;
        }
    }
    if (best >= (m > 2 * MAX_TOK ? 0.9 : 1.0) * other_s) return false;
    plan->tok = tok;
    plan->m_tiles = m_tiles;
    plan->n_tiles = n_tiles;
    plan->split = best_split;
    plan->stages = STAGE_AREA / (W_BYTES + tok * BK);
    if (plan->stages > MAX_STAGES) plan->stages = MAX_STAGES;
    plan->grid = tiles * best_split;
    return true;
}

int int8_skinny_run(const TdistGemmInt8Args* a, const SkinnyPlan& plan) {
    using namespace tdist::int8_skinny;
    Params p;
    memset(&p, 0, sizeof(p));
    const CUtensorMapDataType dt = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    const uint64_t K = a->k, N = a->n, M = a->m;
    const uint64_t strides[1] = {K};
    int rc;
    {
        const uint64_t dims[2] = {K, N};
        const uint32_t box[2] = {BK, ROWS};
        if ((rc = encode_tmap(&p.tm_w, dt, 1, 2, a->b, dims, strides, box, Swizzle::B128))) return rc;
    }
    {
        const uint64_t dims[2] = {K, M};
        const uint32_t box[2] = {BK, static_cast<uint32_t>(plan.tok)};
        if ((rc = encode_tmap(&p.tm_x, dt, 1, 2, a->a, dims, strides, box, Swizzle::B128))) return rc;
    }
    p.sa = static_cast<const float*>(a->sa);
    p.sb = static_cast<const float*>(a->sb);
    p.out = a->c;
    p.m = a->m;
    p.n = a->n;
    p.k_blocks = (a->k + BK - 1) / BK;
    p.tok = plan.tok;
    p.m_tiles = plan.m_tiles;
    p.split = plan.split;
    p.stages = plan.stages;
    p.is_f16 = a->dtype == TDIST_F16;
    p.tmem_cols = plan.tok <= 32 ? 32 : (plan.tok <= 64 ? 64 : 128);
    p.wctx.status = static_cast<Status*>(a->status);
    p.wctx.timeout_ns = a->timeout_ns;
    p.wctx.kernel_id = kKernelSkinny;
    int8_slots(plan.split);   // opts in to the shared memory on this device
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(plan.grid));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = static_cast<cudaStream_t>(a->stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(plan.split);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1] = pdl_attribute();
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    TDIST_CUDA_OK(cudaLaunchKernelEx(&cfg, gemm_int8_skinny_kernel, p));
    return 0;
}

}  // namespace tdist_host
