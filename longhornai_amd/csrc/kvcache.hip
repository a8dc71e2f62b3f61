// kvcache.hip -- writing the paged 8-bit key/value cache and reading it back
// (layout in kvcommon.hpp), for gfx950.
//
// The quantizer is the per-row rule of quant.hip with a row = one token of one
// kv head: scale = max|x| / 127 (448 for e4m3), 1 for a row of zeros, code =
// x * (1 / scale) rounded to nearest even; NaN never wins the maximum.  The
// same IEEE operations in the same order, no multiply-add fused.
#include <algorithm>
#include <type_traits>

#include "kvcommon.hpp"

#pragma clang fp contract(off)

namespace lhq {
namespace {

constexpr int kThreads = 256;

// Eight elements of a row as fp32, elements from `left` on as zero.  VEC: rows
// are 16-byte aligned and head_dim is a multiple of 8.
template <bool VEC>
__device__ __forceinline__ void load8(const float* p, int left, float (&x)[8]) {
    if constexpr (VEC) {
        f32x4_t a = {0.f, 0.f, 0.f, 0.f}, b = a;
        if (left > 0) {
            a = *reinterpret_cast<const f32x4_t*>(p);
            b = *reinterpret_cast<const f32x4_t*>(p + 4);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = j < left ? p[j] : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t* p, int left, float (&x)[8]) {
    if constexpr (VEC) {
        u32x4_t w = {0, 0, 0, 0};
        if (left > 0) w = *reinterpret_cast<const u32x4_t*>(p);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = j < left ? bf16_to_f32(p[j]) : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(float* p, int left, const float (&x)[8]) {
    if constexpr (VEC) {
        if (left > 0) {
            *reinterpret_cast<f32x4_t*>(p) = f32x4_t{x[0], x[1], x[2], x[3]};
            *reinterpret_cast<f32x4_t*>(p + 4) = f32x4_t{x[4], x[5], x[6], x[7]};
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = x[j];
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(uint16_t* p, int left, const float (&x)[8]) {
    if constexpr (VEC) {
        if (left > 0)
            *reinterpret_cast<u32x4_t*>(p) = u32x4_t{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                                     pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = f32_to_bf16(x[j]);
    }
}

// Codes of eight values with scale and reciprocal of a row whose maximum is m.
template <bool FP8>
__device__ __forceinline__ u32x2_t quant8(const float (&x)[8], float m, float& scale) {
    scale = m > 0.0f ? m / (FP8 ? 448.0f : 127.0f) : 1.0f;
    const float inv = 1.0f / scale;
    u32x2_t w;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const float* y = x + 4 * j;
        if constexpr (FP8) {
            w[j] = pack_e4m3x2(y[0] * inv, y[1] * inv) | (pack_e4m3x2(y[2] * inv, y[3] * inv) << 16);
        } else {
            auto q = [inv](float v) { return static_cast<uint32_t>(sat_rint(v * inv, 127)) & 0xffu; };
            w[j] = q(y[0]) | (q(y[1]) << 8) | (q(y[2]) << 16) | (q(y[3]) << 24);
        }
    }
    return w;
}
template <bool FP8>
__device__ __forceinline__ float code_value(uint32_t w, int j) {
    const uint8_t b = static_cast<uint8_t>(w >> (8 * j));
    if constexpr (FP8) return e4m3_to_f32(b);
    else return static_cast<float>(static_cast<int8_t>(b));
}

// Pages that n tokens from position `start` on touch.
__device__ __forceinline__ uint32_t tile_count(int64_t start, int64_t n) {
    return n > 0 ? static_cast<uint32_t>(((start + n - 1) >> 6) - (start >> 6) + 1) : 0u;
}

// The tile of a workgroup: tokens [t0, t1) of page `p` of sequence seq; token
// t is row row0 + t of the list of new rows.
struct Tile { int seq, t0, t1; int64_t p, row0; };
__device__ __forceinline__ Tile find_tile(const int32_t* offsets, const int32_t* start, int n_seqs, int capacity) {
    KvRows mine{0, 0};
    int mine_start = 0;
    const KvUnit u = kv_find_unit(blockIdx.x, n_seqs, [&](int s) {
        mine = kv_rows(offsets, s, capacity);
        mine_start = start[s];
        return tile_count(mine_start, mine.hi - mine.lo);
    });
    if (u.seq >= n_seqs) return {n_seqs, 0, 0, 0, 0};
    const int lo = __builtin_amdgcn_readlane(mine.lo, u.lane), hi = __builtin_amdgcn_readlane(mine.hi, u.lane);
    const int64_t s0 = __builtin_amdgcn_readlane(mine_start, u.lane), p = (s0 >> 6) + u.nth;
    const int64_t a = s0 - (p << 6), b = a + (hi - lo);
    return {u.seq, static_cast<int>(max<int64_t>(a, 0)), static_cast<int>(min<int64_t>(b, kKvPage)), p, lo - a};
}

// Write: one workgroup per (tile, head).  1 << LB lanes (eight channels each)
// take a token: row maximum by shuffles, key codes straight to the token's
// row, value codes to LDS as [token][Dp]; then the value tile leaves
// transposed, 16 bytes a lane where a lane's 16 tokens are all new, else four
// tokens or one at a time (bytes of other tokens are never touched).
template <typename T, bool FP8, int LB, bool VEC>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                            int64_t k_stride, int64_t v_stride,
                                                            const int32_t* __restrict__ rows,
                                                            const int32_t* __restrict__ offsets,
                                                            const int32_t* __restrict__ start, KvCache c, int n_seqs,
                                                            int n_rows, int capacity) {
    constexpr int kPitch = (8 << LB) + 4;
    __shared__ uint32_t vt[kKvPage * kPitch / 4];
    __shared__ int ok[kKvPage];
    const Tile tile = find_tile(offsets, start, n_seqs, capacity);
    if (tile.seq >= n_seqs) return;
    const int page = c.page(tile.seq, tile.p);
    if (page < 0) return;  // nowhere to write: dropped
    const int h = blockIdx.y, Dp = c.Dp();
    const int64_t cb = c.code_base(page, h), sb = c.scale_base(page, h);
    if (threadIdx.x < kKvPage) ok[threadIdx.x] = 0;
    __syncthreads();
    const int d = (threadIdx.x & ((1 << LB) - 1)) * 8;
    for (int t = tile.t0 + (threadIdx.x >> LB); t < tile.t1; t += kThreads >> LB) {
        int64_t row = tile.row0 + t;
        if (rows) row = rows[row];
        const bool in = row >= 0 && row < n_rows;  // (the same for all of a token's lanes)
        if (!in) continue;
        float x[8], y[8];
        load8<VEC>(k + row * k_stride + h * c.D + d, c.D - d, x);
        load8<VEC>(v + row * v_stride + h * c.D + d, c.D - d, y);
        float mk = 0.0f, mv = 0.0f;
        auto amax = [](float m, float a) { return a > m ? a : m; };
#pragma unroll
        for (int j = 0; j < 8; ++j) mk = amax(mk, fabsf(x[j])), mv = amax(mv, fabsf(y[j]));
#pragma unroll
        for (int o = 1; o < (1 << LB); o <<= 1) {
            mk = amax(mk, __shfl_xor(mk, o, 64));
            mv = amax(mv, __shfl_xor(mv, o, 64));
        }
        float sk, sv;
        const u32x2_t wk = quant8<FP8>(x, mk, sk), wv = quant8<FP8>(y, mv, sv);
        if (d < Dp) *reinterpret_cast<u32x2_t*>(c.k + cb + t * Dp + d) = wk;
        vt[(t * kPitch + d) / 4] = wv[0];
        vt[(t * kPitch + d) / 4 + 1] = wv[1];
        if (d == 0) {
            c.ks[sb + t] = sk;
            c.vs[sb + t] = sv;
            ok[t] = 1;
        }
    }
    __syncthreads();
    const uint64_t written = __ballot(ok[threadIdx.x & 63] != 0);
    const uint8_t* vb = reinterpret_cast<const uint8_t*>(vt);
    for (int i = threadIdx.x; i < Dp * 4; i += kThreads) {
        const int g = i & 3, dd = i >> 2;
        uint8_t* out = c.v + cb + static_cast<int64_t>(dd) * kKvPage + 16 * g;
        u32x4_t w;
        uint32_t full = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // q = 2s + h: tokens 16q + 4g + r
            const int t = 16 * q + 4 * g;
            w[q] = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r) w[q] |= static_cast<uint32_t>(vb[(t + r) * kPitch + dd]) << (8 * r);
            full |= (((written >> t) & 15) == 15 ? 1u : 0u) << q;
        }
        if (full == 15) {
            *reinterpret_cast<u32x4_t*>(out) = w;
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int t = 16 * q + 4 * g;
                if ((full >> q) & 1) {
                    *reinterpret_cast<uint32_t*>(out + 4 * q) = w[q];
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if ((written >> (t + r)) & 1) out[4 * q + r] = static_cast<uint8_t>(w[q] >> (8 * r));
                }
            }
        }
    }
}

// Read: one workgroup per (tile, head): x = code * scale, rounded once to the
// output type; the value tile is turned in LDS.  A position without a page
// reads as zero.
template <typename T, bool FP8, int LB, bool VEC>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvCache c, const int32_t* __restrict__ offsets,
                                                           const int32_t* __restrict__ start, T* __restrict__ k_out,
                                                           T* __restrict__ v_out, int n_seqs, int capacity) {
    constexpr int kPitch = (8 << LB) + 4;
    __shared__ uint32_t vt[kKvPage * kPitch / 4];
    const Tile tile = find_tile(offsets, start, n_seqs, capacity);
    if (tile.seq >= n_seqs) return;
    const int page = c.page(tile.seq, tile.p);
    const int h = blockIdx.y, Dp = c.Dp();
    const int64_t cb = c.code_base(max(page, 0), h), sb = c.scale_base(max(page, 0), h);
    uint8_t* vb = reinterpret_cast<uint8_t*>(vt);
    if (page >= 0) {
        for (int i = threadIdx.x; i < Dp * 4; i += kThreads) {
            const int g = i & 3, dd = i >> 2;
            const u32x4_t w = *reinterpret_cast<const u32x4_t*>(c.v + cb + static_cast<int64_t>(dd) * kKvPage + 16 * g);
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    vb[(16 * q + 4 * g + r) * kPitch + dd] = static_cast<uint8_t>(w[q] >> (8 * r));
        }
    }
    __syncthreads();
    const int d = (threadIdx.x & ((1 << LB) - 1)) * 8;
    if (d >= c.D) return;
    for (int t = tile.t0 + (threadIdx.x >> LB); t < tile.t1; t += kThreads >> LB) {
        const int64_t at = ((tile.row0 + t) * c.heads + h) * c.D + d;
        float x[8] = {}, y[8] = {};
        if (page >= 0) {
            const u32x2_t wk = *reinterpret_cast<const u32x2_t*>(c.k + cb + t * Dp + d);
            const float sk = c.ks[sb + t], sv = c.vs[sb + t];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[j] = code_value<FP8>(wk[j / 4], j & 3) * sk;
                y[j] = code_value<FP8>(vt[(t * kPitch + d) / 4 + j / 4], j & 3) * sv;
            }
        }
        store8<VEC>(k_out + at, c.D - d, x);
        store8<VEC>(v_out + at, c.D - d, y);
    }
}

// Workgroups that cover every list of n_seqs sequences with `capacity` rows in
// all: n rows touch at most (n + 62) / 64 + 1 pages, and at most n.
unsigned tile_bound(int n_seqs, int capacity) {
    const int64_t seqs = std::min(n_seqs, capacity);
    const int64_t most = (static_cast<int64_t>(capacity) + 62 * seqs) / kKvPage + seqs;
    return static_cast<unsigned>(std::min<int64_t>(most, capacity));
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// f(lane bits, vectors) with the lanes that a row of D channels needs.
template <typename F>
void by_row(int D, bool vec, F f) {
    using std::integral_constant;
    auto go = [&](auto lb) {
        if (vec) f(lb, std::true_type{});
        else f(lb, std::false_type{});
    };
    if (D <= 64) go(integral_constant<int, 3>{});
    else if (D <= 128) go(integral_constant<int, 4>{});
    else go(integral_constant<int, 5>{});
}

template <typename T>
int kv_write(const char* fn, const T* k, const T* v, int64_t k_stride, int64_t v_stride, const int32_t* rows,
             const int32_t* offsets, const int32_t* start, const KvCache& c, int format, int n_seqs, int n_rows,
             int capacity, void* stream) {
    if (int st = kv_check(fn, c, format, n_seqs, capacity)) return st;
    LHQ_REQUIRE(n_rows >= 0, "%s: bad row count %d", fn, n_rows);
    LHQ_REQUIRE(k_stride >= static_cast<int64_t>(c.heads) * c.D && v_stride >= static_cast<int64_t>(c.heads) * c.D,
                "%s: row strides %lld, %lld are under %d heads of %d", fn, static_cast<long long>(k_stride),
                static_cast<long long>(v_stride), c.heads, c.D);
    if (n_seqs == 0 || capacity == 0 || n_rows == 0) return LHQ_OK;
    if (int st = kv_check_pointers(fn, c)) return st;
    LHQ_REQUIRE(k && v && offsets && start, "%s: null pointer", fn);
    constexpr int kPer16 = 16 / sizeof(T);
    const bool vec = c.D % 8 == 0 && aligned16(k) && aligned16(v) && k_stride % kPer16 == 0 && v_stride % kPer16 == 0;
    const dim3 grid(tile_bound(n_seqs, capacity), c.heads);
    by_row(c.D, vec, [&](auto lb, auto ve) {
        auto launch = [&](auto fp8) {
            kv_write_kernel<T, fp8(), lb(), ve()><<<grid, kThreads, 0, as_stream(stream)>>>(
                k, v, k_stride, v_stride, rows, offsets, start, c, n_seqs, n_rows, capacity);
        };
        if (format == LHQ_KV_FP8) launch(std::true_type{});
        else launch(std::false_type{});
    });
    return check_launch(fn);
}

template <typename T>
int kv_read(const char* fn, const KvCache& c, const int32_t* offsets, const int32_t* start, T* k_out, T* v_out,
            int format, int n_seqs, int capacity, void* stream) {
    if (int st = kv_check(fn, c, format, n_seqs, capacity)) return st;
    if (n_seqs == 0 || capacity == 0) return LHQ_OK;
    if (int st = kv_check_pointers(fn, c)) return st;
    LHQ_REQUIRE(offsets && start && k_out && v_out, "%s: null pointer", fn);
    const bool vec = c.D % 8 == 0 && aligned16(k_out) && aligned16(v_out);
    const dim3 grid(tile_bound(n_seqs, capacity), c.heads);
    by_row(c.D, vec, [&](auto lb, auto ve) {
        auto launch = [&](auto fp8) {
            kv_read_kernel<T, fp8(), lb(), ve()><<<grid, kThreads, 0, as_stream(stream)>>>(c, offsets, start, k_out,
                                                                                          v_out, n_seqs, capacity);
        };
        if (format == LHQ_KV_FP8) launch(std::true_type{});
        else launch(std::false_type{});
    });
    return check_launch(fn);
}

}  // namespace
}  // namespace lhq

using lhq::KvCache;

extern "C" {

int64_t lhq_kv_codes_bytes(int num_pages, int n_kv_heads, int head_dim) {
    if (num_pages < 0 || n_kv_heads <= 0 || head_dim <= 0 || head_dim > lhq::kKvMaxDim) return 0;
    return static_cast<int64_t>(num_pages) * n_kv_heads * lhq::kKvPage * lhq::kv_padded(head_dim);
}
int64_t lhq_kv_scales_bytes(int num_pages, int n_kv_heads) {
    if (num_pages < 0 || n_kv_heads <= 0) return 0;
    return static_cast<int64_t>(num_pages) * n_kv_heads * lhq::kKvPage * 4;
}

int lhq_kv_write_f32(const float* k, const float* v, int64_t k_stride, int64_t v_stride, const int32_t* rows,
                     const int32_t* offsets, const int32_t* start, const int32_t* block_table, uint8_t* k_codes,
                     float* k_scales, uint8_t* v_codes, float* v_scales, int format, int n_seqs, int n_rows,
                     int row_capacity, int max_pages, int num_pages, int n_kv_heads, int head_dim, void* stream) {
    return lhq::kv_write("kv_write_f32", k, v, k_stride, v_stride, rows, offsets, start,
                         KvCache{k_codes, k_scales, v_codes, v_scales, block_table, max_pages, num_pages, n_kv_heads,
                                 head_dim},
                         format, n_seqs, n_rows, row_capacity, stream);
}
int lhq_kv_write_bf16(const uint16_t* k, const uint16_t* v, int64_t k_stride, int64_t v_stride, const int32_t* rows,
                      const int32_t* offsets, const int32_t* start, const int32_t* block_table, uint8_t* k_codes,
                      float* k_scales, uint8_t* v_codes, float* v_scales, int format, int n_seqs, int n_rows,
                      int row_capacity, int max_pages, int num_pages, int n_kv_heads, int head_dim, void* stream) {
    return lhq::kv_write("kv_write_bf16", k, v, k_stride, v_stride, rows, offsets, start,
                         KvCache{k_codes, k_scales, v_codes, v_scales, block_table, max_pages, num_pages, n_kv_heads,
                                 head_dim},
                         format, n_seqs, n_rows, row_capacity, stream);
}

int lhq_kv_read_f32(const uint8_t* k_codes, const float* k_scales, const uint8_t* v_codes, const float* v_scales,
                    const int32_t* offsets, const int32_t* start, const int32_t* block_table, float* k_out,
                    float* v_out, int format, int n_seqs, int row_capacity, int max_pages, int num_pages,
                    int n_kv_heads, int head_dim, void* stream) {
    return lhq::kv_read("kv_read_f32",
                        KvCache{const_cast<uint8_t*>(k_codes), const_cast<float*>(k_scales),
                                const_cast<uint8_t*>(v_codes), const_cast<float*>(v_scales), block_table, max_pages,
                                num_pages, n_kv_heads, head_dim},
                        offsets, start, k_out, v_out, format, n_seqs, row_capacity, stream);
}
int lhq_kv_read_bf16(const uint8_t* k_codes, const float* k_scales, const uint8_t* v_codes, const float* v_scales,
                     const int32_t* offsets, const int32_t* start, const int32_t* block_table, uint16_t* k_out,
                     uint16_t* v_out, int format, int n_seqs, int row_capacity, int max_pages, int num_pages,
                     int n_kv_heads, int head_dim, void* stream) {
    return lhq::kv_read("kv_read_bf16",
                        KvCache{const_cast<uint8_t*>(k_codes), const_cast<float*>(k_scales),
                                const_cast<uint8_t*>(v_codes), const_cast<float*>(v_scales), block_table, max_pages,
                                num_pages, n_kv_heads, head_dim},
                        offsets, start, k_out, v_out, format, n_seqs, row_capacity, stream);
}

}  // extern "C"
