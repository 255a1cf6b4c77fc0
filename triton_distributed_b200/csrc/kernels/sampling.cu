// A token per row of logits: temperature, top-k, top-p, min-p, and the inverse of the cumulative weights at a given number.
//
//   w[i] = round(2^31 exp((x[i] - max) / temperature))          whole numbers: their sums do not depend on the order
//   order: by x, descending, ties by index; every filter keeps the first ones of it:
//     top-k   the first k
//     top-p   those with (sum of w before) < p (sum of the first k)
//     min-p   those with w >= min_p 2^31
//   token = the first index (by index) at which the sum of the kept w passes floor(u W), W = sum of the kept w
//   logprob = (x[token] - max) / temperature - log(W / 2^31),  log_norm = max / temperature + log(W / 2^31)
//
// Temperature 0, below or NaN: the largest logit (lowest index). A NaN logit counts as -inf; a row without anything above -inf gives token -1.
// Weights below 2^-32 of the largest are zero, at most V 2^-32 of the largest in all (200000 tokens: 4.7e-5).
//
// A row belongs to a cluster of 1 to 8 CTAs. Each reads its part from HBM once, into shared memory, and goes over it there: the maximum;
// for top-k a histogram of counts over bins that are linear in x (they spread logits evenly where bins of the bits would heap them on a few
// exponents), of long runs only of the elements in the bins that hold the k largest of the threads' own maxima; for top-p the sum W of the
// weights, then a list of the elements that can matter, x >= max + temperature y0, as all others together weigh less than
// (1 - p) W, and a histogram of their weights; the elements of the bin in which a filter
// cuts, at most kCand, whose places every CTA works out by comparing each with each; the kept sum of every warp's run of the
// row; then the run, its part and the element in which the number falls. A bin of more than kCand elements (flat rows, masked rows,
// ties) is cut again by the bits of x, 11 at a time; ties of one value beyond kCand are counted in the order of the index.
// What bounds it: the instructions per element and pass (a weight takes some 20, most of them expf's), with 16 to 32 warps an SM; 64 rows of
// 128256 bf16 with mixed settings 64 us, of which the slowest row's passes take 48 (sum 6, histogram 14, its bin's elements 5 and their
// order 5, kept sum 7, cluster barriers 6); 256 rows of 100003 fp32 162 us; 1 row of 32000 fp32 12.4 us, eight cluster barriers of
// 0.6 us among them. (512 threads: two CTAs per SM. Clusters of at most four / two: 64 / 78 us, 178 us / no room, 13.4 / 15.6 us. Sorting the bin's
// elements instead of comparing each with each: no faster at the 100 to 400 that a bin holds. One histogram without the bound
// from the threads' maxima: 41000 clocks instead of 22000 for the cut of a top-k row.)
// Compiled without fast math: the weights are those of a correctly rounded subtraction and product and CUDA's expf.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>

#include <cstring>
#include <mutex>
#include <string>

#include "../device/ptx.cuh"
#include "../include/tdist.h"
#include "../runtime/host_common.h"

namespace tdist {
namespace sampling {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kGroups = kBins / 16;
constexpr int kCand = 1024;
// Elements of a warp's run that can matter; more: the whole run is gone over, and the pass that looked for them is lost. Two CTAs' shared memory
// leaves room for less than twice as many. It holds what top-k leaves, and top-p's where the runs are short or steep; 128256 logits of deviation 2.5 in 64 runs leave 732
// at temperature 1, p 0.9. Without lists / with them: 1 x 32000 15.1 / 15.2 us, 64 x 128256 63.1 / 61.8, 256 x 100003 176 / 163.
constexpr int kList = 256;
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 65536;          // elements of a CTA: a bin's sums of 16-bit halves of the weights stay below 2^32
constexpr int kMaxSliceBytes = 180 * 1024;
constexpr float kOne = 2147483648.f;      // weight of the largest logit
constexpr float kSpan = 22.25f;           // weights of exp(-22.2) and less are zero
constexpr int kBoundFrom = 16;            // elements per thread from which on the threads' maxima are looked at first
constexpr int kAhead = 4;                 // 16-byte loads of a lane in flight

struct Params {
    const void* logits;
    long long stride;      // elements between rows
    int V, cl;
    const float *u, *temperature, *top_p, *min_p;   // per row, or nullptr: the values below
    const int* top_k;
    float one_temperature, one_top_p, one_min_p;
    int one_top_k;
    int* tokens;
    float* logprobs;
    float* log_norm;
};

struct Shared {
    // sums of the weights' 16-bit halves, or counts in lo; between two histograms the candidates in one row, and their weights
    union {
        uint32_t lo[kBins];
        unsigned long long row[kCand];
    };
    union {
        uint32_t hi[kBins];
        uint32_t row_w[kCand];
    };
    unsigned long long bins[kMaxCluster][16];         // the bins of one group
    unsigned long long group[kMaxCluster][kGroups];   // every CTA's histogram summed up by 16 bins, written by it into all CTAs
    unsigned long long cand[kCand];     // elements of the bin in which a filter cuts: every CTA's share, written by it into all CTAs
    uint16_t list[kWarps][kList];       // the warps' elements that can matter, by their number in the CTA's part
    float top[kMaxCluster];             // written by every CTA of the cluster
    unsigned long long mass[kMaxCluster];
    unsigned long long run[kWarps];     // sums of the warps' runs
    unsigned long long scan[kWarps];
    uint32_t n_mine, count[kMaxCluster];
    int bin;                            // the pick of a bin: its number (-1: none) and what lies before it
    unsigned long long before;
    unsigned long long cut;             // written by the thread that finds it
    int found;
};

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync_all() {
    cluster_arrive();
    cluster_wait();
}

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<float>(float v) { return v; }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v) { return T(v); }

// Order of the floats as whole numbers; x has no NaN and no -0.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
// (x, index) in the filters' order: larger is earlier
__device__ __forceinline__ unsigned long long place(float x, int i) {
    return (static_cast<unsigned long long>(order_key(x + 0.f)) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Params p) {
    constexpr int VEC = 16 / sizeof(T);
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Shared& s = *reinterpret_cast<Shared*>(smem_raw);
    uint4* part = reinterpret_cast<uint4*>(smem_raw + sizeof(Shared));   // this CTA's part of the row
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
    const int rank = static_cast<int>(blockIdx.x) % p.cl, row_no = static_cast<int>(blockIdx.x) / p.cl;
    cluster_arrive();   // its counterpart stands before the first store into another CTA
    if (tid == 0) s.found = -1;
    auto clear = [&]() {
        for (int i = tid; i < 2 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(s.lo)[i] = make_uint4(0u, 0u, 0u, 0u);
    };
    clear();
    pdl_wait_and_release();
    const float temperature = p.temperature ? p.temperature[row_no] : p.one_temperature;
    const float top_p = p.top_p ? p.top_p[row_no] : p.one_top_p;
    const float min_p = p.min_p ? p.min_p[row_no] : p.one_min_p;
    const int top_k = p.top_k ? p.top_k[row_no] : p.one_top_k;
    const bool greedy = !(temperature > 0.f);   // NaN too
    const bool by_k = top_k > 0 && top_k < p.V && !greedy, by_p = top_p < 1.f && !greedy;
    const uint32_t least = min_p > 0.f && !greedy ? static_cast<uint32_t>(ceil(static_cast<double>(fminf(min_p, 1.f)) * kOne)) : 0u;

    // The row as 16-byte vectors: vector v holds elements v * VEC - shift and on. This CTA's, and within them this warp's run, are contiguous.
    const T* row = static_cast<const T*>(p.logits) + row_no * p.stride;
    const int shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
    const int vecs = (shift + p.V + VEC - 1) / VEC;
    const int per_cta = (vecs + p.cl - 1) / p.cl;
    const int c0 = min(vecs, rank * per_cta), n_vec = min(vecs, c0 + per_cta) - c0;
    const int e0 = c0 * VEC - shift;   // index of the part's first element
    const int per_run = (n_vec + kWarps - 1) / kWarps;
    const int r0 = min(n_vec, warp * per_run), r1 = min(n_vec, r0 + per_run);

    // ---- the part into shared memory (elements beyond the row: -inf), the largest logit
    float top, best = -CUDART_INF_F;   // of the row, of this thread's elements
    {
        for (int v = r0 + lane; v < r1; v += 32 * kAhead) {
            uint4 raw[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                const int i = e0 + (v + 32 * a) * VEC;
                if (v + 32 * a >= r1) continue;
                if (i >= 0 && i + VEC <= p.V) {
                    raw[a] = ld_v4(row + i);
                } else {
                    T* t = reinterpret_cast<T*>(&part[v + 32 * a]);
                    for (int e = 0; e < VEC; ++e) t[e] = i + e >= 0 && i + e < p.V ? row[i + e] : from_float<T>(-CUDART_INF_F);
                    raw[a] = part[v + 32 * a];
                }
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (v + 32 * a >= r1) continue;
                const T* t = reinterpret_cast<const T*>(&raw[a]);
#pragma unroll
                for (int e = 0; e < VEC; ++e) best = fmaxf(best, to_float<T>(t[e]));   // NaN: the other one
                part[v + 32 * a] = raw[a];
            }
        }
        float m = best;
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        float* tops = reinterpret_cast<float*>(s.scan);
        if (lane == 0) tops[warp] = m;
        __syncthreads();
        cluster_wait();   // every CTA of the cluster runs
        if (warp == 0) {
            m = lane < kWarps ? tops[lane] : -CUDART_INF_F;
#pragma unroll
            for (int o = 8; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
            m = __shfl_sync(0xffffffffu, m, 0);
            if (lane < p.cl) st_shared_cluster_f32(mapa_u32(smem_u32(&s.top[rank]), lane), m);
        }
        cluster_sync_all();
        top = s.top[0];
        for (int r = 1; r < p.cl; ++r) top = fmaxf(top, s.top[r]);
        top += 0.f;   // no -0
    }
    if (top == -CUDART_INF_F) {   // alike in the whole cluster
        if (rank == 0 && tid == 0) {
            p.tokens[row_no] = -1;
            p.logprobs[row_no] = p.log_norm[row_no] = -CUDART_INF_F;
        }
        return;
    }
    const float row_top = top;
    if (top == CUDART_INF_F) {
        // infinite logits weigh alike and the others nothing: as 0 and -inf from here on
        for (int v = r0 + lane; v < r1; v += 32) {
            T* t = reinterpret_cast<T*>(&part[v]);
#pragma unroll
            for (int e = 0; e < VEC; ++e) t[e] = from_float<T>(to_float<T>(t[e]) == CUDART_INF_F ? 0.f : -CUDART_INF_F);
        }
        top = 0.f;
        __syncthreads();
    }

    const float inv = greedy ? 1.f : 1.f / temperature;
    auto scaled = [&](float x) { return __fmul_rn(__fsub_rn(x, top), inv); };
    auto weight = [&](float x) { return x == top ? 0x80000000u : __float2uint_rn(expf(scaled(x)) * kOne); };   // NaN, -inf: 0
    // Bins of equal width in x, the first at the top; from kBins - 1 on: all the rest. (Finite also for a temperature next to zero.)
    const float to_bin = fminf(inv * (kBins / kSpan), 1e30f);
    auto depth = [&](float x) { return (top - x) * to_bin; };
    const T* el = reinterpret_cast<const T*>(part);
    unsigned long long cut = 0ull;                          // the last place that is kept, and its logit
    float x_cut = -CUDART_INF_F;
    float low = greedy ? top : -CUDART_INF_F;               // less matters no more
    int listed = -1;
    const int run0 = r0 * VEC, run_n = (r1 - r0) * VEC;
    // fn(x, their numbers in the part) for the elements of this warp's run that are kept so far, four of a lane at a time, from the list
    // where there is one; the others appear as -inf. Without branches, so that four of them are under way at once, and not unrolled further:
    // the kernel goes through most of its code a few times per row.
    struct alignas(4 * sizeof(T)) Quad {
        T t[4];
    };
    const Quad* quads = reinterpret_cast<const Quad*>(part);
    auto sift = [&](float (&x)[4], const int (&at)[4]) {
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = x[u] >= low ? x[u] : -CUDART_INF_F;   // NaN: -inf
        if (cut != 0ull) {
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (x[u] == x_cut && place(x[u], e0 + at[u]) < cut) x[u] = -CUDART_INF_F;
        }
    };
    auto each = [&](auto&& fn) {
        if (listed >= 0) {
#pragma unroll 1
            for (int j = lane; j < listed; j += 128) {
                float x[4];
                int at[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    at[u] = j + 32 * u < listed ? s.list[warp][j + 32 * u] : -1;
                    x[u] = at[u] >= 0 ? to_float<T>(el[at[u]]) : -CUDART_INF_F;
                }
                sift(x, at);
                fn(x, at);
            }
        } else {
#pragma unroll 1
            for (int q = run0 / 4 + lane; q < (run0 + run_n) / 4; q += 32) {
                const Quad v = quads[q];
                float x[4] = {to_float<T>(v.t[0]), to_float<T>(v.t[1]), to_float<T>(v.t[2]), to_float<T>(v.t[3])};
                const int at[4] = {4 * q, 4 * q + 1, 4 * q + 2, 4 * q + 3};
                sift(x, at);
                fn(x, at);
            }
        }
    };
    // The list of the elements x >= low, if they are few.
    auto make_list = [&]() {
        int n = 0;
        listed = -1;
#pragma unroll 1
        for (int q0 = run0 / 4; q0 < (run0 + run_n) / 4; q0 += 32) {
            unsigned m = 0u;
            if (q0 + lane < (run0 + run_n) / 4) {
                const Quad v = quads[q0 + lane];
#pragma unroll
                for (int u = 0; u < 4; ++u) m |= (to_float<T>(v.t[u]) >= low ? 1u : 0u) << u;
            }
            if (!__any_sync(0xffffffffu, m != 0u)) continue;
            int upto = __popc(m);
            const int own = upto;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int k = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += k;
            }
            const int all = __shfl_sync(0xffffffffu, upto, 31);
            if (n + all > kList) return;   // too many: the run itself
            int to = n + upto - own;
            for (; m != 0u; m &= m - 1u) s.list[warp][to++] = static_cast<uint16_t>(4 * (q0 + lane) + __ffs(m) - 1);
            n += all;
        }
        __syncwarp();
        listed = n;
    };
    // Sums of the warps' runs and of the CTAs; all CTAs know them behind it.
    auto put_sum = [&](unsigned long long sum) {
        sum = warp_sum(sum);
        if (lane == 0) s.run[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            sum = warp_sum(lane < kWarps ? s.run[lane] : 0ull);
            if (lane < p.cl) st_cluster_u64(mapa_u32(smem_u32(&s.mass[rank]), lane), sum);
        }
        cluster_sync_all();
    };
    auto total_sum = [&]() {
        unsigned long long m = 0ull;
        for (int r = 0; r < p.cl; ++r) m += s.mass[r];
        return m;
    };
    // Index at which the sum of the values (those of put_sum) passes `target`, in s.found of the CTA that has it; -1 elsewhere.
    auto locate = [&](unsigned long long target, auto&& value) {
        for (int r = 0; r < rank; ++r) {
            const unsigned long long m = s.mass[r];
            if (target < m) return;
            target -= m;
        }
        if (target >= s.mass[rank]) return;
        int run = 0;
        while (run < kWarps - 1 && target >= s.run[run]) target -= s.run[run++];
        // that run, a part of it per warp
        const int q0 = min(n_vec, run * per_run) * VEC, q1 = min(n_vec, (run + 1) * per_run) * VEC;
        const int each_warp = (q1 - q0 + kWarps - 1) / kWarps;
        const int j0 = min(q1, q0 + warp * each_warp), j1 = min(q1, j0 + each_warp);
        unsigned long long own = 0ull;
        for (int j = j0 + lane; j < j1; j += 32) {
            const float x = to_float<T>(el[j]);
            if (x >= low) own += value(x, e0 + j);
        }
        own = warp_sum(own);
        if (lane == 0) s.scan[warp] = own;
        __syncthreads();
        unsigned long long before = 0ull;
        for (int w = 0; w < warp; ++w) before += s.scan[w];
        if (target < before || target >= before + s.scan[warp]) return;   // one warp stays
        target -= before;
        for (int j = j0; j < j1; j += 32) {
            own = 0ull;
            if (j + lane < j1) {
                const float x = to_float<T>(el[j + lane]);
                if (x >= low) own = value(x, e0 + j + lane);
            }
            unsigned long long upto = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long n = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += n;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, target < upto);
            if (hit != 0) {
                if (lane == __ffs(hit) - 1) s.found = e0 + j + lane;
                return;
            }
            target -= __shfl_sync(0xffffffffu, upto, 31);
        }
    };

    auto kept = [&](float x, int i) { return x > x_cut || (x == x_cut && place(x, i) >= cut); };
    constexpr int kOwn = kBins / kThreads, kShare = 16 / kOwn;   // bins of a thread, threads of a group
    // The bin in which the histogram's sum, from `before` on, reaches `goal`, and in `before` what lies before it; -1 and all there is if it
    // never does. By groups of 16 bins first.
    auto pick = [&](unsigned long long goal, unsigned long long& before) -> int {
        __syncthreads();
        unsigned long long m = 0ull;
#pragma unroll
        for (int e = 0; e < kOwn; ++e) m += s.lo[kOwn * tid + e] + (static_cast<unsigned long long>(s.hi[kOwn * tid + e]) << 16);
#pragma unroll
        for (int o = 1; o < kShare; o <<= 1) m += __shfl_xor_sync(0xffffffffu, m, o);
        for (int r = tid % kShare; r < p.cl; r += kShare) st_cluster_u64(mapa_u32(smem_u32(&s.group[rank][tid / kShare]), r), m);
        if (tid == 0) s.bin = -1;
        cluster_sync_all();
        unsigned long long own = 0ull, upto;
        if (tid < kGroups)
            for (int r = 0; r < p.cl; ++r) own += s.group[r][tid];
        upto = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long n = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += n;
        }
        if (lane == 31) s.scan[warp] = upto;
        __syncthreads();
        if (tid < kGroups) {
            unsigned long long at = before + upto - own;
            for (int w = 0; w < warp; ++w) at += s.scan[w];
            if (at < goal && goal <= at + own) {
                s.bin = tid;
                s.before = at;
            } else if (tid == kGroups - 1 && at + own < goal) {
                s.before = at + own;
            }
        }
        __syncthreads();
        const int group = s.bin;
        before = s.before;
        if (group < 0) return -1;
        // its bins, a thread per CTA and bin
        if (tid < 16 * p.cl) {
            const uint32_t b = 16u * group + (tid & 15);
            s.bins[tid >> 4][tid & 15] = ld_cluster_u32(mapa_u32(smem_u32(&s.lo[b]), tid >> 4)) +
                                         (static_cast<unsigned long long>(ld_cluster_u32(mapa_u32(smem_u32(&s.hi[b]), tid >> 4))) << 16);
        }
        __syncthreads();
        unsigned long long v = 0ull;
        for (int r = 0; r < p.cl; ++r) v += s.bins[r][lane & 15];
        upto = v;
#pragma unroll
        for (int o = 1; o < 16; o <<= 1) {
            const unsigned long long n = __shfl_up_sync(0xffffffffu, upto, o, 16);
            if ((lane & 15) >= o) upto += n;
        }
        const int e = __ffs(__ballot_sync(0xffffffffu, goal <= before + upto) & 0xffffu) - 1;   // every warp finds it
        before += __shfl_sync(0xffffffffu, upto - v, e);
        return 16 * group + e;
    };
    // Top-k of long runs: k threads have an element in the bins up to the one that holds the k-th of the threads' maxima, so the k-th
    // element is in these bins too.
    if (by_k && p.V / (kThreads * p.cl) >= kBoundFrom) {
        const float f = depth(row_top == CUDART_INF_F ? (best == row_top ? 0.f : -CUDART_INF_F) : best);
        if (f < kBins - 1) atomicAdd(&s.lo[static_cast<int>(f)], 1u);
        unsigned long long before = 0ull;
        const int bin = pick(static_cast<unsigned long long>(top_k), before);
        if (bin >= 0) {
            low = top - (bin + 1.01f) / to_bin - fabsf(top) * 1e-6f;
            make_list();
        }
        cluster_sync_all();   // nobody reads the histogram any more
        clear();
        __syncthreads();
    }
    // The first search cuts by count (top-k), the second by weight (top-p).
#pragma unroll 1
    for (int search = by_k ? 0 : 1; search < (by_p ? 2 : 1); ++search) {
        const bool count = search == 0;
        unsigned long long goal = static_cast<unsigned long long>(top_k);
        if (!count) {
            if (by_k && cut != 0ull) make_list();
            unsigned long long sum = 0ull;
            each([&](const float (&x)[4], const int (&)[4]) {
#pragma unroll
                for (int u = 0; u < 4; ++u) sum += weight(x[u]);
            });
            put_sum(sum);
            const unsigned long long all = total_sum();
            const double limit = ceil(static_cast<double>(top_p) * static_cast<double>(all));
            goal = limit > 1.0 ? static_cast<unsigned long long>(limit) : 1ull;
            if (goal > all) goal = all;
            if (cut == 0ull) {
                // Elements below y0 are beyond the cut, however many: V (2^31 exp(y0) + 1/2) < W - goal. A hundredth of slack for the
                // roundings of y0 and of the product.
                const double room = static_cast<double>(all - goal) / (static_cast<double>(p.V) * kOne) - 0.5 / kOne;
                if (room > 0.0) low = top + ((logf(static_cast<float>(room)) - 0.01f) * temperature - fabsf(top) * 1e-6f);
                make_list();
            }
            clear();
            __syncthreads();
        }
        // Looks for the place of the last element up to which the sum reaches `goal`: by bins of x, and, within a bin of more than kCand
        // elements, by bins of the bits.
        unsigned long long before = 0ull;   // of the elements in earlier bins
        float f0 = 0.f;                     // the bin
        uint32_t klo = 0u, khi = 0xffffffffu;
        int down = -1;                      // bits per bin; -1: bins of x
        unsigned long long got = 0ull;
        auto inside = [&](float x) {   // x of `each`
            const float f = fminf(depth(x), kBins - 0.5f);
            const uint32_t k = order_key(x + 0.f);
            return f >= f0 && f < f0 + 1.f && k >= klo && k <= khi;
        };
#pragma unroll 1
        while (true) {
            each([&](const float (&x)[4], const int (&)[4]) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    // by x: the rest is only looked into if these bins do not suffice
                    const float f = depth(x[u]);
                    const bool in = down < 0 ? f < kBins - 1 : inside(x[u]);
                    const int b = down < 0 ? static_cast<int>(f) : static_cast<int>((khi - order_key(x[u] + 0.f)) >> down);
                    if (in) {
                        const uint32_t w = count ? 1u : weight(x[u]);
                        if (w & 0xffffu) atomicAdd(&s.lo[b], w & 0xffffu);
                        if (w >> 16) atomicAdd(&s.hi[b], w >> 16);
                    }
                }
            });
            const int bin = pick(goal, before);
            if (bin < 0 && down >= 0) break;   // all are kept
            if (down < 0) {
                f0 = bin >= 0 ? bin : kBins - 1;             // all the rest
                klo = order_key(-3.402823466e38f);           // not -inf, whose weight is 0
            } else {
                khi -= static_cast<uint32_t>(bin) << down;
                const uint32_t width = down ? (1u << down) - 1u : 0u;
                klo = khi - klo > width ? khi - width : klo;
            }
            // ---- the bin's elements, if they are few: into every CTA
            const uint32_t share = kCand / p.cl;
            if (tid == 0) s.n_mine = 0u;
            cluster_sync_all();   // (and nobody reads the histogram or the candidates any more)
            each([&](const float (&x)[4], const int (&at)[4]) {
                bool any = false;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const float f = fminf(depth(x[u]), kBins - 0.5f);
                    any |= f >= f0 && f < f0 + 1.f;
                }
                if (!any) return;
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    if (!inside(x[u])) continue;
                    const uint32_t to = atomicAdd(&s.n_mine, 1u);
                    if (to >= share) continue;
                    const unsigned long long c = place(x[u], e0 + at[u]);
                    for (int r = 0; r < p.cl; ++r) st_cluster_u64(mapa_u32(smem_u32(&s.cand[rank * share + to]), r), c);
                }
            });
            __syncthreads();
            if (tid < p.cl) st_cluster_u32(mapa_u32(smem_u32(&s.count[rank]), tid), s.n_mine);
            cluster_sync_all();
            uint32_t most = 0u, n = 0u;
            for (int r = 0; r < p.cl; ++r) {
                most = max(most, s.count[r]);
                n += s.count[r];
            }
            if (most <= share) {
                // in one row, with their weights; then each is compared with all
                uint32_t base = 0u;
                for (int r = 0; r < p.cl; ++r) {
                    const uint32_t k = s.count[r];
                    for (uint32_t i = tid; i < k; i += kThreads) {
                        const unsigned long long c = s.cand[r * share + i];
                        s.row[base + i] = c;
                        s.row_w[base + i] = count ? 1u : weight(key_value(static_cast<uint32_t>(c >> 32)));
                    }
                    base += k;
                }
                if (tid == 0) s.cut = 0ull;
                __syncthreads();
                for (uint32_t i = tid; i < n; i += kThreads) {
                    const unsigned long long c = s.row[i];
                    unsigned long long m = before;
#pragma unroll 4
                    for (uint32_t j = 0; j < n; ++j) m += s.row[j] > c ? s.row_w[j] : 0u;
                    if (m < goal && goal <= m + s.row_w[i]) s.cut = c;
                }
                __syncthreads();
                got = s.cut;
                break;
            }
            if (klo == khi) {
                // more ties of one value than candidates: the first of them by index
                const float x0 = key_value(khi);
                const uint32_t w0 = count ? 1u : weight(x0);
                const unsigned long long ties = (goal - before + w0 - 1) / w0;
                auto one = [&](float x, int i) -> unsigned long long { return kept(x, i) && inside(x) ? 1ull : 0ull; };
                unsigned long long sum = 0ull;
                each([&](const float (&x)[4], const int (&)[4]) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) sum += inside(x[u]) ? 1u : 0u;
                });
                put_sum(sum);
                locate(ties - 1, one);
                __syncthreads();
                if (s.found >= 0 && tid < p.cl) st_cluster_u64(mapa_u32(smem_u32(&s.cut), tid), place(x0, s.found));
                cluster_sync_all();
                if (tid == 0) s.found = -1;
                got = s.cut;
                cluster_sync_all();
                break;
            }
            const int bits = 32 - __clz(khi - klo);
            down = bits > 11 ? bits - 11 : 0;
            clear();
            __syncthreads();
        }
        if (got != 0ull) {
            cut = got;
            x_cut = key_value(static_cast<uint32_t>(cut >> 32));
            low = fmaxf(low, x_cut);
        }
    }
    if (least > 0u) low = fmaxf(low, top + ((logf(static_cast<float>(least) / kOne) - 0.01f) * temperature - fabsf(top) * 1e-6f));

    auto value = [&](float x, int i) -> unsigned long long {
        if (!kept(x, i)) return 0ull;
        const uint32_t w = weight(x);
        return w >= least ? w : 0u;
    };
    unsigned long long sum = 0ull;
    each([&](const float (&x)[4], const int (&)[4]) {
        if (fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) == -CUDART_INF_F) return;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t w = weight(x[u]);
            sum += w >= least ? w : 0u;
        }
    });
    put_sum(sum);
    const unsigned long long total = total_sum();
    const double at = greedy ? 0.0 : floor(static_cast<double>(p.u[row_no]) * static_cast<double>(total));
    unsigned long long target = at > 0.0 ? static_cast<unsigned long long>(at) : 0ull;
    if (target >= total) target = total - 1;
    locate(target, value);
    __syncthreads();
    if (s.found >= 0 && tid == 0) {
        const float x = to_float<T>(el[s.found - e0]);
        const float norm = logf(static_cast<float>(total) / kOne);
        p.tokens[row_no] = s.found;
        p.logprobs[row_no] = greedy ? 0.f : __fsub_rn(x == top ? 0.f : scaled(x), norm);
        p.log_norm[row_no] = greedy ? row_top : __fadd_rn(__fmul_rn(row_top, inv), norm);
    }
}

}  // namespace sampling
}  // namespace tdist

using namespace tdist;
using tdist_host::fail;

namespace {

template <typename T>
int launch_sample(sampling::Params& p, int B, cudaStream_t stream) {
    using namespace sampling;
    static bool done[64] = {};
    static std::mutex setup_lock;
    int dev = 0;
    TDIST_CUDA_OK(cudaGetDevice(&dev));
    if (dev < 0 || dev >= 64) return fail(TDIST_EINVAL, "sample: device ordinal out of range");
    {
        std::lock_guard<std::mutex> guard(setup_lock);
        if (!done[dev]) {
            TDIST_CUDA_OK(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Shared)) + kMaxSliceBytes));
            done[dev] = true;
        }
    }
    // As many CTAs per row as fill the machine once (two fit an SM), of 2048 elements at least; and so many that a part leaves room for a
    // second CTA on its SM.
    constexpr int vec = 16 / static_cast<int>(sizeof(T));
    auto slice = [&](int cl) { return ((p.V + vec - 1 + vec - 1) / vec + cl - 1) / cl * 16; };   // bytes, wherever the row starts
    int cl = 1;
    while (cl < kMaxCluster && ((static_cast<long long>(B) * cl * 2 <= 2 * tdist_host::sm_count() && p.V / (cl * 2) >= 2048) || slice(cl) > 64 * 1024)) cl *= 2;
    if (slice(cl) > kMaxSliceBytes || slice(cl) / static_cast<int>(sizeof(T)) > kMaxSlice)
        return fail(TDIST_ELIMIT, "sample: at most 524032 logits per row, 368000 in fp32");
    p.cl = cl;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(B * cl));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared) + static_cast<size_t>(slice(cl));
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    cfg.attrs = attr;
    attr[cfg.numAttrs++] = tdist_host::pdl_attribute();
    cudaLaunchAttribute& dim = attr[cfg.numAttrs++];
    dim.id = cudaLaunchAttributeClusterDimension;
    dim.val.clusterDim.x = static_cast<unsigned>(cl);
    dim.val.clusterDim.y = 1;
    dim.val.clusterDim.z = 1;
    TDIST_CUDA_OK(cudaLaunchKernelEx(&cfg, sample_kernel<T>, p));
    return 0;
}

}  // namespace

extern "C" int tdist_sample(const TdistSampleArgs* a) {
    if (a == nullptr) return fail(TDIST_EINVAL, "sample: null args");
    if (a->B < 1 || a->V < 1) return fail(TDIST_EINVAL, "sample: B and V must be at least 1");
    if (a->V > sampling::kMaxCluster * sampling::kMaxSlice) return fail(TDIST_ELIMIT, "sample: at most 524032 logits per row, 368000 in fp32");
    if (a->B > 1 << 24) return fail(TDIST_ELIMIT, "sample: at most 2^24 rows");
    if (!a->logits || !a->u || !a->tokens || !a->logprobs || !a->log_norm) return fail(TDIST_EINVAL, "sample: null pointer");
    sampling::Params p;
    memset(&p, 0, sizeof(p));
    p.logits = a->logits;
    p.stride = a->stride;
    p.V = a->V;
    p.u = static_cast<const float*>(a->u);
    p.temperature = static_cast<const float*>(a->temperature);
    p.top_k = static_cast<const int*>(a->top_k);
    p.top_p = static_cast<const float*>(a->top_p);
    p.min_p = static_cast<const float*>(a->min_p);
    p.one_temperature = a->one_temperature;
    p.one_top_k = a->one_top_k;
    p.one_top_p = a->one_top_p;
    p.one_min_p = a->one_min_p;
    p.tokens = static_cast<int*>(a->tokens);
    p.logprobs = static_cast<float*>(a->logprobs);
    p.log_norm = static_cast<float*>(a->log_norm);
    cudaStream_t stream = static_cast<cudaStream_t>(a->stream);
    if (a->dtype == TDIST_BF16) return launch_sample<__nv_bfloat16>(p, a->B, stream);
    if (a->dtype == TDIST_F16) return launch_sample<__half>(p, a->B, stream);
    if (a->dtype == TDIST_F32) return launch_sample<float>(p, a->B, stream);
    return fail(TDIST_EINVAL, "sample: dtype must be bf16, fp16 or fp32");
}
