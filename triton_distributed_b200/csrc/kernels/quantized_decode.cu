// Decode attention over a quantised cache: the call's checks, its kernel's arguments, and the kernel that adds up what the CTAs of quantized_decode.cuh
// leave in a workspace.
#include "quantized_decode.cuh"

namespace tdist {
namespace qdecode {

// Shares: the sums of a segment that several CTAs have pieces of. Block (c, h): head h of the segment whose second piece is CTA c's first; its
// first piece is in CTA info.z / 2 (its last piece where info.z is odd), the others are the first ones of every per_b-th CTA from c to info.w.
// Four threads per two dimensions.
template <int D>
__global__ void __launch_bounds__(2 * D) merge_kernel(const float* part, const int4* info, int per_b, int heads, bool is_f16, void* out) {
    constexpr int GROUPS = 4;
    __shared__ float a_s[GROUPS][D], l_s[GROUPS], m_s[GROUPS];
    pdl_wait_and_release();
    const int4 x = info[blockIdx.x];
    const int h = static_cast<int>(blockIdx.y);
    if (x.x < 0 || h >= x.y) return;
    const int group = static_cast<int>(threadIdx.x) / (D / 2), d = static_cast<int>(threadIdx.x) % (D / 2) * 2;
    const int c = static_cast<int>(blockIdx.x), count = (x.w - c) / per_b + 2;
    auto at = [&](int i) { return part + (static_cast<size_t>(i == 0 ? x.z : 2 * (c + (i - 1) * per_b)) * heads + h) * (D + 2); };
    float m = kNoScore, l = 0.f, a0 = 0.f, a1 = 0.f;
#pragma unroll 4
    for (int i = group; i < count; i += GROUPS) {
        const float* src = at(i);
        const float mi = src[D], li = src[D + 1];
        const float2 v = *reinterpret_cast<const float2*>(src + d);
        const float m_new = fmaxf(m, mi);
        const float fa = exp2f(m - m_new), fb = exp2f(mi - m_new);
        l = l * fa + li * fb;
        a0 = a0 * fa + v.x * fb;
        a1 = a1 * fa + v.y * fb;
        m = m_new;
    }
    a_s[group][d] = a0;
    a_s[group][d + 1] = a1;
    if (d == 0) {
        l_s[group] = l;
        m_s[group] = m;
    }
    __syncthreads();
    if (group != 0) return;
    m = kNoScore;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) m = fmaxf(m, m_s[i]);
    l = a0 = a1 = 0.f;
#pragma unroll
    for (int i = 0; i < GROUPS; ++i) {
        const float f = exp2f(m_s[i] - m);
        l += l_s[i] * f;
        a0 += a_s[i][d] * f;
        a1 += a_s[i][d + 1] * f;
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    const uint32_t w = is_f16 ? pack_f16x2(a0 * inv, a1 * inv) : pack_bf16x2(a0 * inv, a1 * inv);
    *reinterpret_cast<uint32_t*>(static_cast<char*>(out) + ((static_cast<size_t>(x.x) + h) * D + d) * 2) = w;
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
    if (a->splits < 0 || a->splits > MAX_CLUSTER || a->shares < 0 || (a->splits == 0 && a->shares > 0 && (a->part == nullptr || c.B > MAX_SHARED)))
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
    int l = 0;
    while ((1ll << l) < c.page_size) ++l;
    const bool paged = c.page_size == 1 << l && l >= 4 && ((c.code_block | c.code_token | c.scale_block | c.scale_token << l) >> 32) == 0;
    // PAGED: t >> l. Otherwise, with 2^l >= page_size, the multiplier ceil(2^(31 + l) / page_size) is off by less than one, so its product with
    // t < 2^31 by less than 2^31, and the quotient's fraction is at most 1 - 1 / page_size
    p.page_shift = paged ? l : 31 + l;
    p.page_mul = static_cast<uint32_t>(((1ull << (31 + l)) + static_cast<uint64_t>(c.page_size) - 1) / static_cast<uint64_t>(c.page_size));
    p.max_blocks = c.max_blocks;
    p.blocks = c.blocks;
    p.splits = a->splits > 0 ? a->splits : 1;
    p.shares = a->splits > 0 ? 0 : a->shares;
    const bool small = a->splits == 0 && a->shares == 0;
    p.B = c.B;
    p.window = a->window;
    p.sinks = a->sinks;
    const long long keys = static_cast<long long>(c.max_blocks) * c.page_size;
    p.table_keys = static_cast<int>(keys < 0x7fffffc0ll ? keys : 0x7fffffc0ll);
    const bool f16 = c.dtype == TDIST_F16;
    p.scale = a->scale;
    // a cap below 2^-60 makes all weights alike as 2^-60 does, whose inverse fp32 has
    p.soft_cap = a->soft_cap > 0.f && a->soft_cap < 8.673617379884035e-19f ? 8.673617379884035e-19f : a->soft_cap;
    const long long segments = static_cast<long long>(c.B) * c.Hkv * p.head_tiles, grid = p.shares > 0 ? static_cast<long long>(p.shares) * c.Hkv * p.head_tiles : segments * p.splits;
    if (grid > 0x7fffffffll) return fail(TDIST_EINVAL, "quantised decode: too many sequences");
    if (p.shares > 0) {
        // (tiles are counted in 32 bits)
        if (c.B * static_cast<long long>((p.table_keys + TOK - 1) / TOK + 2) > 0x7fffffffll) return fail(TDIST_EINVAL, "quantised decode: too many keys to deal out in shares");
        if (a->scratch < grid * (4 + 2ll * 8 * nh * (c.head_dim + 2))) return fail(TDIST_EINVAL, "quantised decode: too little scratch");
        p.info = reinterpret_cast<int4*>(p.part);
        p.part += 4 * grid;
    }
    const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
    const int rc = c.bits == 8 ? launch_bits<8>(p, c.head_dim, nh, paged, f16, small, static_cast<int>(grid), stream)
                               : launch_bits<4>(p, c.head_dim, nh, paged, f16, small, static_cast<int>(grid), stream);
    if (rc) return rc;
    if (p.shares > 0) {
        const dim3 blocks(static_cast<unsigned>(grid), static_cast<unsigned>(8 * nh));
        const int per_b = c.Hkv * p.head_tiles;
        const float* part = p.part;
        const int4* info = p.info;
        cudaError_t e;
        if (c.head_dim == 64) e = tdist_host::launch_pdl(merge_kernel<64>, blocks, 128, 0, stream, part, info, per_b, 8 * nh, f16, a->out);
        else if (c.head_dim == 128) e = tdist_host::launch_pdl(merge_kernel<128>, blocks, 256, 0, stream, part, info, per_b, 8 * nh, f16, a->out);
        else e = tdist_host::launch_pdl(merge_kernel<256>, blocks, 512, 0, stream, part, info, per_b, 8 * nh, f16, a->out);
        TDIST_CUDA_OK(e);
    }
    return 0;
}
