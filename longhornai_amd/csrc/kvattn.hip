// kvattn.hip -- attention of new (drafted) tokens over the paged 8-bit cache
// (layout in kvcommon.hpp) and over one another, for gfx950.
//
//   s_j = scale * q . k_j          over the sequence's cached tokens and those
//   o   = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)     new ones its mask names
// Keys and values of cached tokens are code * scale; a token whose page is
// missing is not seen; a query that sees nothing gives zeros.
#include <cmath>

#include "kvcommon.hpp"

namespace lhq {
namespace {

struct AttnArgs {
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* k_new;
    int64_t k_stride;
    const uint16_t* v_new;
    int64_t v_stride;
    const uint64_t* tree;
    const int32_t* offsets;
    const int32_t* lengths;
    KvCache c;
    uint16_t* out;
    int n_seqs, capacity, max_new, heads;
    float scale;
};

template <bool FP8>
__device__ __forceinline__ float code_value(uint8_t b) {
    if constexpr (FP8) return e4m3_to_f32(b);
    else return static_cast<float>(static_cast<int8_t>(b));
}

// One wave per (new token, query head); 64 keys at a time, one a lane, then
// every lane its channels d = lane + 64 i.
template <bool FP8>
__global__ __launch_bounds__(64) void kv_attn_plain_kernel(AttnArgs a) {
    __shared__ float qs[kKvMaxDim], ps[64];
    const int row = blockIdx.x, hq = blockIdx.y, lane = threadIdx.x;
    const int D = a.c.D, Dp = a.c.Dp(), h = hq / (a.heads / a.c.heads);
    const KvUnit u = kv_find_unit(row, a.n_seqs, [&](int s) {
        const KvRows r = kv_rows(a.offsets, s, a.capacity);
        return static_cast<int64_t>(r.hi - r.lo);
    });
    if (u.seq >= a.n_seqs || u.nth >= a.max_new) return;
    const KvRows r = kv_rows(a.offsets, u.seq, a.capacity);
    const int tok = r.lo + static_cast<int>(u.nth), T = min(r.hi - r.lo, a.max_new);
    const int64_t L = min<int64_t>(max(a.lengths[u.seq], 0), static_cast<int64_t>(a.c.max_pages) * kKvPage);
    for (int d = lane; d < D; d += 64) qs[d] = bf16_to_f32(a.q[tok * a.q_stride + hq * D + d]) * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[kKvMaxDim / 64] = {};
    auto step = [&](bool seen, float s, auto value) {
        if (!__ballot(seen)) return;
        float top = seen ? s : -INFINITY;
        for (int x = 32; x; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
        const float mn = fmaxf(m, top);
        const float f = m == -INFINITY ? 0.0f : expf(m - mn), p = seen ? expf(s - mn) : 0.0f;
        m = mn;
        float sum = p;
        for (int x = 32; x; x >>= 1) sum += __shfl_xor(sum, x, 64);
        l = l * f + sum;
        ps[lane] = p;
        __syncthreads();
        for (int i = 0; i < kKvMaxDim / 64; ++i) {
            const int d = lane + 64 * i;
            if (d >= D) break;
            float acc = o[i] * f;
            for (int t = 0; t < 64; ++t)
                if (ps[t] != 0.0f) acc += ps[t] * value(t, d);
            o[i] = acc;
        }
        __syncthreads();
    };
    for (int64_t p = 0; p * kKvPage < L; ++p) {
        const int page = a.c.page(u.seq, p);
        if (page < 0) continue;
        const uint8_t* kc = a.c.k + a.c.code_base(page, h);
        const uint8_t* vc = a.c.v + a.c.code_base(page, h);
        const float *ks = a.c.ks + a.c.scale_base(page, h), *vs = a.c.vs + a.c.scale_base(page, h);
        const bool in = p * kKvPage + lane < L;
        float s = 0.0f;
        if (in)
            for (int d = 0; d < D; ++d) s += qs[d] * code_value<FP8>(kc[lane * Dp + d]);
        step(in, in ? s * ks[lane] : 0.0f, [&](int t, int d) { return vs[t] * code_value<FP8>(vc[d * kKvPage + kv_slot(t)]); });
    }
    if (a.k_new) {
        float s = 0.0f;
        const uint64_t seen = a.tree ? a.tree[tok] : ~uint64_t{0} >> (63 - u.nth);
        const bool in = lane < T && ((seen >> lane) & 1);
        if (in)
            for (int d = 0; d < D; ++d) s += qs[d] * bf16_to_f32(a.k_new[(r.lo + lane) * a.k_stride + h * D + d]);
        step(in, s, [&](int t, int d) { return bf16_to_f32(a.v_new[(r.lo + t) * a.v_stride + h * D + d]); });
    }
    for (int i = 0; i < kKvMaxDim / 64; ++i) {
        const int d = lane + 64 * i;
        if (d < D) a.out[(static_cast<int64_t>(tok) * a.heads + hq) * D + d] = f32_to_bf16(l == 0.0f ? 0.0f : o[i] / l);
    }
}

}  // namespace
}  // namespace lhq

using namespace lhq;

extern "C" {

int64_t lhq_kv_attn_workspace_bytes(int n_seqs, int row_capacity, int max_new, int max_pages, int n_heads,
                                    int n_kv_heads, int head_dim) {
    (void)n_seqs, (void)row_capacity, (void)max_new, (void)max_pages, (void)n_heads, (void)n_kv_heads, (void)head_dim;
    return 0;
}

int lhq_kv_attn_bf16(const uint16_t* q, int64_t q_stride, const uint16_t* k_new, int64_t k_stride,
                     const uint16_t* v_new, int64_t v_stride, const uint64_t* tree, const int32_t* offsets,
                     const int32_t* lengths, const int32_t* block_table, const uint8_t* k_codes,
                     const float* k_scales, const uint8_t* v_codes, const float* v_scales, uint16_t* out, int format,
                     int n_seqs, int row_capacity, int max_new, int max_pages, int num_pages, int n_heads,
                     int n_kv_heads, int head_dim, float scale, void* workspace, int64_t workspace_bytes,
                     void* stream) {
    const char* fn = "kv_attn_bf16";
    const KvCache c{const_cast<uint8_t*>(k_codes), const_cast<float*>(k_scales), const_cast<uint8_t*>(v_codes),
                    const_cast<float*>(v_scales), block_table, max_pages, num_pages, n_kv_heads, head_dim};
    if (int st = kv_check(fn, c, format, n_seqs, row_capacity)) return st;
    LHQ_REQUIRE(n_heads > 0 && n_heads % n_kv_heads == 0, "%s: %d query heads are no multiple of %d kv heads", fn,
                n_heads, n_kv_heads);
    LHQ_SUPPORTED(n_heads <= 65535, "%s: %d query heads are over 65535", fn, n_heads);
    LHQ_REQUIRE(max_new >= 0, "%s: bad max_new %d", fn, max_new);
    LHQ_SUPPORTED(max_new <= kKvMaxNew, "%s: max_new %d is over %d", fn, max_new, kKvMaxNew);
    LHQ_REQUIRE(std::isfinite(scale) && scale > 0.0f, "%s: scale %g is not finite and positive", fn, scale);
    LHQ_REQUIRE((k_new == nullptr) == (v_new == nullptr), "%s: new keys without values, or values without keys", fn);
    LHQ_REQUIRE(q_stride >= static_cast<int64_t>(n_heads) * head_dim, "%s: q rows of stride %lld are under %d heads of %d",
                fn, static_cast<long long>(q_stride), n_heads, head_dim);
    LHQ_REQUIRE(!k_new || (k_stride >= static_cast<int64_t>(n_kv_heads) * head_dim &&
                           v_stride >= static_cast<int64_t>(n_kv_heads) * head_dim),
                "%s: new rows of strides %lld, %lld are under %d heads of %d", fn, static_cast<long long>(k_stride),
                static_cast<long long>(v_stride), n_kv_heads, head_dim);
    LHQ_REQUIRE(workspace_bytes >= 0, "%s: negative workspace size", fn);
    LHQ_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "%s: workspace must be 16-byte aligned", fn);
    if (n_seqs == 0 || row_capacity == 0 || max_new == 0) return LHQ_OK;
    if (int st = kv_check_pointers(fn, c)) return st;
    LHQ_REQUIRE(q && offsets && lengths && out, "%s: null pointer", fn);
    const AttnArgs a{q,     q_stride, k_new, k_stride, v_new,        v_stride, tree,    offsets,
                     lengths, c,      out,   n_seqs,   row_capacity, max_new,  n_heads, scale};
    const dim3 grid(row_capacity, n_heads);
    if (format == LHQ_KV_FP8) kv_attn_plain_kernel<true><<<grid, 64, 0, as_stream(stream)>>>(a);
    else kv_attn_plain_kernel<false><<<grid, 64, 0, as_stream(stream)>>>(a);
    return check_launch(fn);
}

}  // extern "C"
