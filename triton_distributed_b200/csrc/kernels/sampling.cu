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
// Temperature 0: the largest logit (lowest index). NaN counts as -inf; a row without anything above -inf gives token -1.
// Weights below 2^-32 of the largest are zero: tokens that no 24-bit random number could have drawn.
//
// A row belongs to a cluster of 1 to 8 CTAs, each of which goes over its part of the row a few times (the first time from HBM,
// then from L2): maximum; sum of the weights, and where there are filters a histogram (count and weight) over bins that are linear in x,
// which spread logits evenly where bins of the bits would heap them on a few exponents; the elements of the bin in which a filter
// cuts, at most kCand of them, sorted in the first CTA; the kept sum of every warp's run of the row; then the run, its part and the
// element in which the number falls. A bin of more than kCand elements (flat rows, masked rows, ties) is cut again by
// the bits of x, 11 at a time; ties of one value beyond kCand are counted in the order of the index.
// Compiled without fast math: the weights are those of any correctly rounded subtraction and product and CUDA's expf.
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
constexpr int kCand = 2048;
constexpr int kMaxCluster = 8;
constexpr int kMaxSlice = 65536;          // elements of a CTA: a bin's sums of 16-bit halves of the weights stay below 2^32
constexpr float kOne = 2147483648.f;      // weight of the largest logit
constexpr float kSpan = 22.25f;           // weights of exp(-22.2) and less are zero
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
    uint32_t cnt[kBins], lo[kBins], hi[kBins];
    unsigned long long cand[kCand];     // first CTA: the candidates of all
    unsigned long long mine[kCand];     // this CTA's
    unsigned long long top[kMaxCluster];    // written by every CTA of the cluster
    unsigned long long mass[kMaxCluster];
    unsigned long long run[kWarps];     // sums of the warps' runs
    unsigned long long scan_m[kWarps];
    uint32_t scan_c[kWarps];
    uint32_t n_cand, n_mine, base;
    int bin;                            // the pick of a bin: its number, what lies before it, what is in it
    uint32_t bin_before, bin_count;
    unsigned long long bin_mass_before;
    unsigned long long cut, cut_mass;   // written by the first CTA or the one that finds it
    int found;
};

__device__ __forceinline__ void st_cluster_u64(uint32_t addr, unsigned long long v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t atom_add_cluster(uint32_t addr, uint32_t v) {
    uint32_t old;
    asm volatile("atom.shared::cluster.add.u32 %0, [%1], %2;" : "=r"(old) : "r"(addr), "r"(v) : "memory");
    return old;
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

// Order of the floats as whole numbers; x has no NaN and no -0.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x);
    return (b & 0x80000000u) ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k); }
// (x, index) in the filters' order: larger is earlier
__device__ __forceinline__ unsigned long long place(float x, int i) {
    return (static_cast<unsigned long long>(order_key(x)) << 32) | (0xffffffffu - static_cast<uint32_t>(i));
}

// The row as 16-byte vectors: vector v holds elements v * VEC - shift ...
template <typename T>
struct Row {
    static constexpr int VEC = 16 / sizeof(T);
    const T* p;
    int V, shift, vecs;

    __device__ __forceinline__ Row(const T* row, int n) : p(row), V(n) {
        shift = static_cast<int>((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        vecs = (shift + n + VEC - 1) / VEC;
    }
    __device__ __forceinline__ uint4 load(int v) const {
        const int i = v * VEC - shift;
        if (i >= 0 && i + VEC <= V) return ld_v4(p + i);
        union {
            uint4 q;
            T t[VEC];
        } u;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            T x;
            if constexpr (sizeof(T) == 4)
                x = -CUDART_INF_F;
            else
                x = T(-CUDART_INF_F);
            if (i + e >= 0 && i + e < V) x = *const_cast<const volatile T*>(p + i + e);
            u.t[e] = x;
        }
        return u.q;
    }
    // fn(x, index) for the elements of a loaded vector
    template <typename F>
    __device__ __forceinline__ void each(const uint4& raw, int v, F&& fn) const {
        const T* t = reinterpret_cast<const T*>(&raw);
        const int i0 = v * VEC - shift;
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const int i = i0 + e;
            if (i < 0 || i >= V) continue;
            float x = to_float<T>(t[e]) + 0.f;   // no -0
            x = x == x ? x : -CUDART_INF_F;
            fn(x, i);
        }
    }
    // the same for those of vectors [v0, v1), by one warp; indices rise within a lane
    template <typename F>
    __device__ __forceinline__ void walk(int v0, int v1, F&& fn) const {
        const int lane = static_cast<int>(threadIdx.x) & 31;
        for (int v = v0 + lane; v < v1; v += 32 * kAhead) {
            uint4 raw[kAhead];
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (v + 32 * a < v1) raw[a] = load(v + 32 * a);
#pragma unroll
            for (int a = 0; a < kAhead; ++a) {
                if (v + 32 * a >= v1) break;
                each(raw[a], v + 32 * a, fn);
            }
        }
    }
};

__device__ __forceinline__ unsigned long long warp_sum(unsigned long long v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Adds to bin b of the histogram; where all lanes that do so meet in one bin (ties), one of them adds for all.
__device__ __forceinline__ void add_bin(Shared& s, int b, uint32_t w, bool count, bool mass) {
    const unsigned act = __activemask();
    int same;
    __match_all_sync(act, b, &same);
    if (same) {
        const int n = __popc(act);
        const uint32_t l = __reduce_add_sync(act, w & 0xffffu), h = __reduce_add_sync(act, w >> 16);
        if ((threadIdx.x & 31) == static_cast<unsigned>(__ffs(act) - 1)) {
            if (count) atomicAdd(&s.cnt[b], n);
            if (mass) {
                atomicAdd(&s.lo[b], l);
                atomicAdd(&s.hi[b], h);
            }
        }
        return;
    }
    if (count) atomicAdd(&s.cnt[b], 1u);
    if (mass && w != 0) {
        atomicAdd(&s.lo[b], w & 0xffffu);
        if (w >> 16) atomicAdd(&s.hi[b], w >> 16);
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const Params p) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    Shared& s = *reinterpret_cast<Shared*>(smem_raw);
    const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
    const int rank = static_cast<int>(blockIdx.x) % p.cl, row_no = static_cast<int>(blockIdx.x) / p.cl;
    if (tid == 0) {
        s.found = -1;
        s.bin = 0;
        s.bin_before = s.bin_count = 0u;
        s.bin_mass_before = 0ull;
    }
    pdl_wait_and_release();
    const float temperature = p.temperature ? p.temperature[row_no] : p.one_temperature;
    const float top_p = p.top_p ? p.top_p[row_no] : p.one_top_p;
    const float min_p = p.min_p ? p.min_p[row_no] : p.one_min_p;
    int top_k = p.top_k ? p.top_k[row_no] : p.one_top_k;
    const bool greedy = temperature <= 0.f;
    if (top_k <= 0 || top_k >= p.V) top_k = 0;
    const bool by_k = top_k > 0, by_p = top_p < 1.f;
    const uint32_t least = min_p > 0.f ? static_cast<uint32_t>(ceil(static_cast<double>(fminf(min_p, 1.f)) * kOne)) : 0u;

    const Row<T> row(static_cast<const T*>(p.logits) + row_no * p.stride, p.V);
    // this CTA's vectors, and within them this warp's run: both contiguous
    const int per_cta = (row.vecs + p.cl - 1) / p.cl;
    const int c0 = min(row.vecs, rank * per_cta), c1 = min(row.vecs, c0 + per_cta);
    const int per_run = (c1 - c0 + kWarps - 1) / kWarps;
    const int r0 = min(c1, c0 + warp * per_run), r1 = min(c1, r0 + per_run);

    // ---- the largest logit, and the first index that has it
    {
        float best = -CUDART_INF_F;
        int at = -1;
        row.walk(r0, r1, [&](float x, int i) {
            if (x > best) {
                best = x;
                at = i;
            }
        });
        unsigned long long k = at >= 0 ? place(best, at) : 0ull;
#pragma unroll
        for (int o = 16; o; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
        if (lane == 0) s.run[warp] = k;
        __syncthreads();
        if (warp == 0) {
            k = lane < kWarps ? s.run[lane] : 0ull;
#pragma unroll
            for (int o = 8; o; o >>= 1) k = max(k, __shfl_xor_sync(0xffffffffu, k, o));
            k = __shfl_sync(0xffffffffu, k, 0);
            if (lane < p.cl) st_cluster_u64(mapa_u32(smem_u32(&s.top[rank]), lane), k);
        }
    }
    // histogram, empty
    for (int i = tid; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(s.cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
    cluster_sync_all();
    unsigned long long best = 0ull;
    for (int r = 0; r < p.cl; ++r) best = max(best, s.top[r]);
    const float top = best == 0ull ? -CUDART_INF_F : key_value(static_cast<uint32_t>(best >> 32));
    if (best == 0ull || greedy) {   // alike in the whole cluster; nobody's shared memory is read any more
        if (rank == 0 && tid == 0) {
            p.tokens[row_no] = best == 0ull ? -1 : static_cast<int>(0xffffffffu - static_cast<uint32_t>(best));
            p.logprobs[row_no] = best == 0ull ? -CUDART_INF_F : 0.f;
            p.log_norm[row_no] = top;
        }
        return;
    }

    const float inv = 1.f / temperature;
    auto scaled = [&](float x) { return x == top ? 0.f : __fmul_rn(__fsub_rn(x, top), inv); };
    auto weight = [&](float x) { return __float2uint_rn(expf(scaled(x)) * kOne); };
    const float to_bin = inv * (kBins / kSpan);
    auto bin_of = [&](float x) {   // falls with x
        const float f = x == top ? 0.f : (top - x) * to_bin;
        return f < kBins - 1 ? static_cast<int>(f) : kBins - 1;
    };
    // Sums of the warps' runs and of the CTAs, for a value per element; all CTAs know them behind it.
    auto sum_runs = [&](auto&& value) {
        unsigned long long sum = 0ull;
        row.walk(r0, r1, [&](float x, int i) { sum += value(x, i); });
        sum = warp_sum(sum);
        if (lane == 0) s.run[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            sum = warp_sum(lane < kWarps ? s.run[lane] : 0ull);
            if (lane < p.cl) st_cluster_u64(mapa_u32(smem_u32(&s.mass[rank]), lane), sum);
        }
        cluster_sync_all();
    };
    // Index at which the sum of the values (those of sum_runs) passes `target`, in s.found of the CTA that has it; -1 elsewhere.
    auto locate = [&](unsigned long long target, auto&& value) {
        for (int r = 0; r < rank; ++r) {
            const unsigned long long m = s.mass[r];
            if (target < m) return;
            target -= m;
        }
        if (target >= s.mass[rank]) return;
        int run = 0;
        while (run < kWarps - 1 && target >= s.run[run]) target -= s.run[run++];
        const int q0 = min(c1, c0 + run * per_run), q1 = min(c1, q0 + per_run);
        const int part = (q1 - q0 + kWarps - 1) / kWarps;
        const int v0 = min(q1, q0 + warp * part), v1 = min(q1, v0 + part);
        unsigned long long sum = 0ull;
        row.walk(v0, v1, [&](float x, int i) { sum += value(x, i); });
        sum = warp_sum(sum);
        if (lane == 0) s.scan_m[warp] = sum;
        __syncthreads();
        unsigned long long before = 0ull;
        for (int w = 0; w < warp; ++w) before += s.scan_m[w];
        if (target < before || target >= before + s.scan_m[warp]) return;   // one warp stays
        target -= before;
        for (int v = v0; v < v1; v += 32) {
            sum = 0ull;
            const bool has = v + lane < v1;
            uint4 raw = make_uint4(0u, 0u, 0u, 0u);
            if (has) {
                raw = row.load(v + lane);
                row.each(raw, v + lane, [&](float x, int i) { sum += value(x, i); });
            }
            unsigned long long upto = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const unsigned long long n = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += n;
            }
            const unsigned hit = __ballot_sync(0xffffffffu, target < upto);
            if (hit != 0) {
                if (lane == __ffs(hit) - 1) {
                    unsigned long long left = target - (upto - sum);
                    int at = -1;
                    row.each(raw, v + lane, [&](float x, int i) {
                        const unsigned long long m = value(x, i);
                        if (at < 0) {
                            if (left < m) at = i;
                            else left -= m;
                        }
                    });
                    s.found = at;
                }
                return;
            }
            target -= __shfl_sync(0xffffffffu, upto, 31);
        }
    };

    unsigned long long cut = 0ull;   // the last place that is kept
    if (by_k || by_p) {
        unsigned long long sum = 0ull;
        row.walk(r0, r1, [&](float x, int) {
            const uint32_t w = weight(x);
            sum += w;
            add_bin(s, bin_of(x), w, true, by_p);
        });
        sum = warp_sum(sum);
        if (lane == 0) s.run[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            sum = warp_sum(lane < kWarps ? s.run[lane] : 0ull);
            if (lane < p.cl) st_cluster_u64(mapa_u32(smem_u32(&s.mass[rank]), lane), sum);
        }
        cluster_sync_all();
        unsigned long long total = 0ull;
        for (int r = 0; r < p.cl; ++r) total += s.mass[r];

        // The cluster's histogram: four bins per thread, and what lies before them.
        uint32_t cnt[4], c_before;
        unsigned long long mass[4], m_before;
        auto merge = [&]() {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                cnt[e] = 0u;
                mass[e] = 0ull;
            }
            for (int r = 0; r < p.cl; ++r) {
                const uint4 c = ld_cluster_v4(mapa_u32(smem_u32(&s.cnt[4 * tid]), r));
                const uint4 l = ld_cluster_v4(mapa_u32(smem_u32(&s.lo[4 * tid]), r));
                const uint4 h = ld_cluster_v4(mapa_u32(smem_u32(&s.hi[4 * tid]), r));
                const uint32_t ca[4] = {c.x, c.y, c.z, c.w}, la[4] = {l.x, l.y, l.z, l.w}, ha[4] = {h.x, h.y, h.z, h.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    cnt[e] += ca[e];
                    mass[e] += la[e] + (static_cast<unsigned long long>(ha[e]) << 16);
                }
            }
            const uint32_t c = cnt[0] + cnt[1] + cnt[2] + cnt[3];
            const unsigned long long m = mass[0] + mass[1] + mass[2] + mass[3];
            uint32_t cu = c;
            unsigned long long mu = m;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const uint32_t cn = __shfl_up_sync(0xffffffffu, cu, o);
                const unsigned long long mn = __shfl_up_sync(0xffffffffu, mu, o);
                if (lane >= o) {
                    cu += cn;
                    mu += mn;
                }
            }
            if (lane == 31) {
                s.scan_c[warp] = cu;
                s.scan_m[warp] = mu;
            }
            __syncthreads();
            c_before = cu - c;
            m_before = mu - m;
            for (int w = 0; w < warp; ++w) {
                c_before += s.scan_c[w];
                m_before += s.scan_m[w];
            }
        };
        // The bin in which the count (or the weight) reaches `goal` (at least 1, at most all).
        auto pick = [&](bool count, unsigned long long goal) {
            __syncthreads();
            uint32_t c = c_before;
            unsigned long long m = m_before;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const unsigned long long a = count ? c : m, b = a + (count ? cnt[e] : mass[e]);
                if (a < goal && goal <= b) {
                    s.bin = 4 * tid + e;
                    s.bin_before = c;
                    s.bin_mass_before = m;
                    s.bin_count = cnt[e];
                }
                c += cnt[e];
                m += mass[e];
            }
            __syncthreads();
        };
        // The place of the last element up to which the count (or the weight) reaches `goal`; `upto`: the weight up to it.
        // `again`: another search follows, which starts from the first histogram.
        auto find_cut = [&](bool count, unsigned long long goal, bool again, unsigned long long& upto) {
            merge();
            pick(count, goal);
            const int bin0 = s.bin;
            uint32_t before = s.bin_before, n = s.bin_count, klo = 0u, khi = 0xffffffffu;
            unsigned long long m_above = s.bin_mass_before;
            auto inside = [&](float x) {
                const uint32_t k = order_key(x);
                return bin_of(x) == bin0 && k >= klo && k <= khi;
            };
            bool refined = false;
            while (n > kCand && klo < khi) {
                const int bits = 32 - __clz(khi - klo), shift = bits > 11 ? bits - 11 : 0;
                cluster_sync_all();   // everyone has read the histogram
                for (int i = tid; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(s.cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
                __syncthreads();
                row.walk(r0, r1, [&](float x, int) {
                    if (inside(x)) add_bin(s, static_cast<int>((khi - order_key(x)) >> shift), by_p ? weight(x) : 0u, true, by_p);
                });
                cluster_sync_all();
                merge();
                pick(count, goal - (count ? before : m_above));
                before += s.bin_before;
                m_above += s.bin_mass_before;
                n = s.bin_count;
                const uint32_t down = static_cast<uint32_t>(s.bin) << shift;
                khi -= down;
                const uint32_t width = shift ? (1u << shift) - 1u : 0u;
                klo = khi - klo > width ? khi - width : klo;
                refined = true;
            }
            if (n > kCand) {
                // more ties of one value than candidates: the first of them by index
                const float x0 = key_value(khi);
                const uint32_t w0 = weight(x0);
                const unsigned long long ties = count ? goal - before : (goal - m_above + w0 - 1) / w0;
                auto one = [&](float x, int) -> unsigned long long { return x == x0 ? 1ull : 0ull; };
                sum_runs(one);
                locate(ties - 1, one);
                __syncthreads();
                if (s.found >= 0 && tid < p.cl) st_cluster_u64(mapa_u32(smem_u32(&s.cut), tid), place(x0, s.found));
                cluster_sync_all();
                if (tid == 0) s.found = -1;
                upto = m_above + ties * w0;
            } else {
                if (tid == 0) s.n_mine = s.n_cand = 0u;
                cluster_sync_all();
                row.walk(r0, r1, [&](float x, int i) {
                    if (inside(x)) s.mine[atomicAdd(&s.n_mine, 1u)] = place(x, i);
                });
                __syncthreads();
                if (tid == 0) s.base = atom_add_cluster(mapa_u32(smem_u32(&s.n_cand), 0), s.n_mine);
                __syncthreads();
                for (uint32_t i = tid; i < s.n_mine; i += kThreads) st_cluster_u64(mapa_u32(smem_u32(&s.cand[s.base + i]), 0), s.mine[i]);
                cluster_sync_all();
                if (rank == 0) {
                    // sorted, earliest first
                    int size = 32;
                    while (size < static_cast<int>(n)) size <<= 1;
                    for (int i = tid; i < size; i += kThreads)
                        if (i >= static_cast<int>(n)) s.cand[i] = 0ull;
                    for (int k = 2; k <= size; k <<= 1)
                        for (int j = k >> 1; j > 0; j >>= 1) {
                            __syncthreads();
                            for (int i = tid; i < size / 2; i += kThreads) {
                                const int a = ((i & ~(j - 1)) << 1) | (i & (j - 1)), b = a | j;
                                const unsigned long long va = s.cand[a], vb = s.cand[b];
                                if (((a & k) == 0) == (va < vb)) {
                                    s.cand[a] = vb;
                                    s.cand[b] = va;
                                }
                            }
                        }
                    __syncthreads();
                    // weights before every candidate: kCand / kThreads of them per thread
                    constexpr int EACH = kCand / kThreads;
                    uint32_t w[EACH];
                    unsigned long long m = 0ull;
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const int i = tid * EACH + e;
                        w[e] = i < static_cast<int>(n) ? weight(key_value(static_cast<uint32_t>(s.cand[i] >> 32))) : 0u;
                        m += w[e];
                    }
                    unsigned long long acc = m;
#pragma unroll
                    for (int o = 1; o < 32; o <<= 1) {
                        const unsigned long long v = __shfl_up_sync(0xffffffffu, acc, o);
                        if (lane >= o) acc += v;
                    }
                    if (lane == 31) s.scan_m[warp] = acc;
                    __syncthreads();
                    acc -= m;
                    for (int i = 0; i < warp; ++i) acc += s.scan_m[i];
#pragma unroll
                    for (int e = 0; e < EACH; ++e) {
                        const int i = tid * EACH + e;
                        // the last one that is kept: the count ends here, or the weight reaches the goal with it
                        const bool last = count ? before + i + 1 == goal : (m_above + acc < goal && goal <= m_above + acc + w[e]);
                        if (i < static_cast<int>(n) && last) {
                            s.cut = s.cand[i];
                            s.cut_mass = m_above + acc + w[e];
                        }
                        acc += w[e];
                    }
                    __syncthreads();
                    if (tid > 0 && tid < p.cl) {
                        st_cluster_u64(mapa_u32(smem_u32(&s.cut), tid), s.cut);
                        st_cluster_u64(mapa_u32(smem_u32(&s.cut_mass), tid), s.cut_mass);
                    }
                }
                cluster_sync_all();
                upto = s.cut_mass;
            }
            const unsigned long long got = s.cut;
            cluster_sync_all();
            if (refined && again) {
                for (int i = tid; i < 3 * kBins / 4; i += kThreads) reinterpret_cast<uint4*>(s.cnt)[i] = make_uint4(0u, 0u, 0u, 0u);
                __syncthreads();
                row.walk(r0, r1, [&](float x, int) { add_bin(s, bin_of(x), by_p ? weight(x) : 0u, true, by_p); });
                cluster_sync_all();
            }
            return got;
        };
        unsigned long long kept = total;
        if (by_k) cut = find_cut(true, static_cast<unsigned long long>(top_k), by_p, kept);
        if (by_p) {
            const double limit = ceil(static_cast<double>(top_p) * static_cast<double>(kept));
            unsigned long long goal = limit > 1.0 ? static_cast<unsigned long long>(limit) : 1ull;
            if (goal > kept) goal = kept;
            unsigned long long unused;
            cut = find_cut(false, goal, false, unused);
        }
    }

    auto value = [&](float x, int i) -> unsigned long long {
        if (place(x, i) < cut) return 0ull;
        const uint32_t w = weight(x);
        return w >= least ? w : 0u;
    };
    sum_runs(value);
    unsigned long long total = 0ull;
    for (int r = 0; r < p.cl; ++r) total += s.mass[r];
    const double at = floor(static_cast<double>(p.u[row_no]) * static_cast<double>(total));
    unsigned long long target = at > 0.0 ? static_cast<unsigned long long>(at) : 0ull;
    if (target >= total) target = total - 1;
    locate(target, value);
    __syncthreads();
    if (s.found >= 0 && tid == 0) {
        const float x = to_float<T>(row.p[s.found]) + 0.f;
        const float norm = logf(static_cast<float>(total) / kOne);
        p.tokens[row_no] = s.found;
        p.logprobs[row_no] = __fsub_rn(scaled(x), norm);
        p.log_norm[row_no] = __fadd_rn(__fmul_rn(top, inv), norm);
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
            TDIST_CUDA_OK(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(sizeof(Shared))));
            done[dev] = true;
        }
    }
    // As many CTAs per row as fill the machine once (two fit an SM), of 2048 elements at least; a CTA takes kMaxSlice at most.
    int cl = 1;
    while (cl < kMaxCluster && ((static_cast<long long>(B) * cl * 2 <= 2 * tdist_host::sm_count() && p.V / (cl * 2) >= 2048) || p.V / cl + 32 > kMaxSlice))
        cl *= 2;
    p.cl = cl;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(static_cast<unsigned>(B * cl));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = sizeof(Shared);
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
    if (a->V > sampling::kMaxCluster * (sampling::kMaxSlice - 32)) return fail(TDIST_ELIMIT, "sample: at most 524032 logits per row");
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
