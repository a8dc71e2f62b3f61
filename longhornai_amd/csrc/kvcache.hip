// kvcache.hip -- writing the paged 8-bit key/value cache and reading it back
// (layout in kvcommon.hpp), for gfx950.
//
// The quantizer is the per-row rule of quant.hip with a row = one token of one
// kv head: scale = max|x| / 127 (448 for e4m3), 1 for a row of zeros, code =
// x * (1 / scale) rounded to nearest even; NaN never wins the maximum.  The
// same IEEE operations in the same order, no multiply-add fused.
//
// Both ways are bound by memory from a few thousand tokens on, below that by
// the launch and one workgroup's chain of loads.  8 x 4096 tokens of 8 heads of
// 128, bf16 and e4m3, 203 MB each way: write 57 us with inputs that change (3.6
// TB/s; 42 to 49 where they lie partly in the last-level cache), read 31 us (6.5,
// the results partly in that cache); one token of 16 sequences: 5.7 and 3.8 us.
// Turning the value tile in bytes rather than dwords, one row after the other,
// took 55 and 42 us where this takes 42 and 31.
#include <algorithm>
#include <type_traits>

#include "kvcommon.hpp"

#pragma clang fp contract(off)

namespace lhq {
namespace {

constexpr int kThreads = 256;

// Eight elements of a row from channel d on as fp32, those past D as zero.
// VEC: rows are 16-byte aligned and D is a multiple of 8.  No branch: loads of
// several rows stay in flight together.
template <bool VEC>
__device__ __forceinline__ void load8(const float* row, int d, int D, float (&x)[8]) {
    if constexpr (VEC) {
        const float* p = row + (d < D ? d : 0);
        const f32x4_t a = *reinterpret_cast<const f32x4_t*>(p), b = *reinterpret_cast<const f32x4_t*>(p + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = a[j], x[4 + j] = b[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = row[min(d + j, D - 1)];
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = d + (VEC ? 0 : j) < D ? x[j] : 0.0f;
}
template <bool VEC>
__device__ __forceinline__ void load8(const uint16_t* row, int d, int D, float (&x)[8]) {
    if constexpr (VEC) {
        u32x4_t w = *reinterpret_cast<const u32x4_t*>(row + (d < D ? d : 0));
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (d >= D) w[j] = 0;
            x[2 * j] = __uint_as_float(w[j] << 16);
            x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
        }
    } else {
        uint16_t y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = row[min(d + j, D - 1)];
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = d + j < D ? bf16_to_f32(y[j]) : 0.0f;
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

// Codes of eight values with scale and reciprocal of a row whose maximum is m,
// whatever the row holds.
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
// The values of eight codes, times their scale.
template <bool FP8>
__device__ __forceinline__ void values8(u32x2_t w, float scale, float (&x)[8]) {
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        if constexpr (FP8) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[j], true);
            x[4 * j] = lo[0] * scale;
            x[4 * j + 1] = lo[1] * scale;
            x[4 * j + 2] = hi[0] * scale;
            x[4 * j + 3] = hi[1] * scale;
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[4 * j + i] = static_cast<float>(static_cast<int8_t>(w[j] >> (8 * i))) * scale;
        }
    }
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
    const KvUnit u = kv_find_unit(blockIdx.y + blockIdx.z * gridDim.y, n_seqs, [&](int s) {
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

__device__ __forceinline__ uint32_t magnitude(const float (&x)[8]) {  // bits of max |x|; NaN is over infinity
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(x[j]) & 0x7fffffffu);
    return m;
}
// The same codes as quant8 for a row of finite values whose reciprocal scale is
// finite: nothing saturates (the largest value is within a rounding of 127 or
// 448), so int8 takes the low byte of the sum with 1.5 * 2^23, whose last bit
// is 1, and e4m3 the conversion of values that are quartered below 2^-9.
template <bool FP8>
__device__ __forceinline__ u32x2_t quant8_plain(const float (&x)[8], float inv) {
    u32x2_t w;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        float y[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            y[i] = x[4 * j + i] * inv;
            if constexpr (FP8) y[i] *= fabsf(y[i]) < 0x1p-9f ? 0.25f : 1.0f;
            else y[i] += 12582912.0f;
        }
        if constexpr (FP8) {
            const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
            w[j] = static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true));
        } else {
            const uint32_t lo = __builtin_amdgcn_perm(__float_as_uint(y[1]), __float_as_uint(y[0]), 0x0c0c0400u);
            const uint32_t hi = __builtin_amdgcn_perm(__float_as_uint(y[3]), __float_as_uint(y[2]), 0x04000c0cu);
            w[j] = lo | hi;
        }
    }
    return w;
}
template <int CTRL>
__device__ __forceinline__ float quad(float x) {
    return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, false));
}

// Four dwords of four bytes, turned: byte j of out[i] is byte i of in[j].
__device__ __forceinline__ void turn4(const uint32_t (&in)[4], uint32_t (&out)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(in[1], in[0], 0x05010400u), b = __builtin_amdgcn_perm(in[3], in[2], 0x05010400u);
    const uint32_t c = __builtin_amdgcn_perm(in[1], in[0], 0x07030602u), d = __builtin_amdgcn_perm(in[3], in[2], 0x07030602u);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100u);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    out[2] = __builtin_amdgcn_perm(d, c, 0x05040100u);
    out[3] = __builtin_amdgcn_perm(d, c, 0x07060302u);
}
// A page's value codes in LDS: [token][kPitch bytes].  The turn between tokens
// and channels reads and writes it in dwords, a lane group g at tokens 4 g on:
// 16 dwords over a multiple of 64 keeps the four groups on banks of their own.
template <int LB>
constexpr int kValuePitch = (8 << LB) + 16;

// Write: one workgroup per (tile, head).  1 << LB lanes (eight channels each)
// take a token, up to four tokens of theirs in flight: row maximum across
// lanes, key codes straight to the token's row, value codes to LDS; then the
// value tile leaves turned, four channels of 16 tokens a lane, 16 bytes at a
// time where those tokens are all new, else four tokens or one at a time
// (bytes of other tokens are never touched).
template <typename T, bool FP8, int LB, bool VEC>
__global__ __launch_bounds__(kThreads) void kv_write_kernel(const T* __restrict__ k, const T* __restrict__ v,
                                                            int64_t k_stride, int64_t v_stride,
                                                            const int32_t* __restrict__ rows,
                                                            const int32_t* __restrict__ offsets,
                                                            const int32_t* __restrict__ start, KvCache c, int n_seqs,
                                                            int n_rows, int capacity) {
    constexpr int kPitch = kValuePitch<LB>, kPer = kThreads >> LB, kPasses = kKvPage / kPer < 4 ? kKvPage / kPer : 4;
    __shared__ __attribute__((aligned(16))) uint32_t vt[kKvPage * kPitch / 4];
    __shared__ int ok[kKvPage];
    const Tile tile = find_tile(offsets, start, n_seqs, capacity);
    if (tile.seq >= n_seqs) return;
    const int page = c.page(tile.seq, tile.p);
    if (page < 0) return;  // nowhere to write: dropped
    const int h = blockIdx.x, Dp = c.Dp();
    const int64_t cb = c.code_base(page, h), sb = c.scale_base(page, h);
    if (threadIdx.x < kKvPage) ok[threadIdx.x] = 0;
    __syncthreads();
    const int d = (threadIdx.x & ((1 << LB) - 1)) * 8;
    for (int t0 = tile.t0; t0 < tile.t1; t0 += kPasses * kPer) {
        float x[kPasses][8], y[kPasses][8];
        bool in[kPasses];  // (the same for all of a token's lanes)
        int64_t row[kPasses];
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int t = t0 + i * kPer + (threadIdx.x >> LB);
            row[i] = tile.row0 + min(t, tile.t1 - 1);
            if (rows) row[i] = rows[row[i]];
            in[i] = t < tile.t1 && row[i] >= 0 && row[i] < n_rows;
            if (!in[i]) row[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            load8<VEC>(k + row[i] * k_stride + h * c.D, d, c.D, x[i]);
            load8<VEC>(v + row[i] * v_stride + h * c.D, d, c.D, y[i]);
        }
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            if (t0 + i * kPer >= tile.t1) break;
            const int t = t0 + i * kPer + (threadIdx.x >> LB);
            u32x2_t wk, wv;
            float sk, sv;
            auto umax = [](uint32_t m, uint32_t n) { return max(m, n); };
            const uint32_t bk = row_max<LB>(magnitude(x[i]), umax), bv = row_max<LB>(magnitude(y[i]), umax);
            // (from 2^-100 on, and of zeros, the scale's reciprocal is finite)
            auto plain = [](uint32_t m) { return m - 0x0d800000u < 0x7f800000u - 0x0d800000u || m == 0; };
            if (__ballot(!plain(bk) || !plain(bv)) == 0) {
                // Even lanes divide for the keys, odd ones for the values.
                const float m = __uint_as_float(threadIdx.x & 1 ? bv : bk);
                const float scale = m > 0.0f ? m / (FP8 ? 448.0f : 127.0f) : 1.0f, inv = 1.0f / scale;
                sk = quad<0xA0>(scale);  // quad_perm 0, 0, 2, 2
                sv = quad<0xF5>(scale);  // quad_perm 1, 1, 3, 3
                wk = quant8_plain<FP8>(x[i], quad<0xA0>(inv));
                wv = quant8_plain<FP8>(y[i], quad<0xF5>(inv));
            } else {
                float mk = 0.0f, mv = 0.0f;
                auto amax = [](float m, float a) { return a > m ? a : m; };  // NaN never wins
#pragma unroll
                for (int j = 0; j < 8; ++j) mk = amax(mk, fabsf(x[i][j])), mv = amax(mv, fabsf(y[i][j]));
                wk = quant8<FP8>(x[i], row_max<LB>(mk, amax), sk);
                wv = quant8<FP8>(y[i], row_max<LB>(mv, amax), sv);
                // An infinite reciprocal makes NaN of the zeros past D: their codes are zero all the same.
                const int own = 8 * min(max(c.D - d, 0), 8);
                const uint64_t keep = own == 64 ? ~uint64_t{0} : (uint64_t{1} << own) - 1;
                wk &= __builtin_bit_cast(u32x2_t, keep);
                wv &= __builtin_bit_cast(u32x2_t, keep);
            }
            if (!in[i]) continue;
            if (d < Dp) *reinterpret_cast<u32x2_t*>(c.k + cb + t * Dp + d) = wk;
            *reinterpret_cast<u32x2_t*>(vt + (t * kPitch + d) / 4) = wv;
            if (d == 0) {
                c.ks[sb + t] = sk;
                c.vs[sb + t] = sv;
                ok[t] = 1;
            }
        }
    }
    __syncthreads();
    const uint64_t written = __ballot(ok[threadIdx.x & 63] != 0);
    for (int i = threadIdx.x; i < Dp; i += kThreads) {
        const int g = i & 3, dd = 4 * (i >> 2);
        uint8_t* out = c.v + cb + static_cast<int64_t>(dd) * kKvPage + 16 * g;
        u32x4_t w[4];
        uint32_t full = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {  // q = 2s + h: tokens 16q + 4g + r
            const int t = 16 * q + 4 * g;
            uint32_t by_token[4], by_channel[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) by_token[r] = vt[((t + r) * kPitch + dd) / 4];
            turn4(by_token, by_channel);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j][q] = by_channel[j];
            full |= (((written >> t) & 15) == 15 ? 1u : 0u) << q;
        }
        if (full == 15) {
#pragma unroll
            for (int j = 0; j < 4; ++j) *reinterpret_cast<u32x4_t*>(out + j * kKvPage) = w[j];
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t some = (written >> (16 * q + 4 * g)) & 15;
                if (some == 15) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) *reinterpret_cast<uint32_t*>(out + j * kKvPage + 4 * q) = w[j][q];
                } else if (some != 0) {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if ((some >> r) & 1)
#pragma unroll
                            for (int j = 0; j < 4; ++j)
                                out[j * kKvPage + 4 * q + r] = static_cast<uint8_t>(w[j][q] >> (8 * r));
                }
            }
        }
    }
}

// Read: one workgroup per (tile, head): x = code * scale, rounded once to the
// output type; the value tile is turned in LDS while the keys are on their
// way.  A position without a page reads as zero.
template <typename T, bool FP8, int LB, bool VEC>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(KvCache c, const int32_t* __restrict__ offsets,
                                                           const int32_t* __restrict__ start, T* __restrict__ k_out,
                                                           T* __restrict__ v_out, int n_seqs, int capacity) {
    constexpr int kPitch = kValuePitch<LB>, kPer = kThreads >> LB, kPasses = kKvPage / kPer < 4 ? kKvPage / kPer : 4;
    __shared__ __attribute__((aligned(16))) uint32_t vt[kKvPage * kPitch / 4];
    const Tile tile = find_tile(offsets, start, n_seqs, capacity);
    if (tile.seq >= n_seqs) return;
    const int page = c.page(tile.seq, tile.p);
    const int h = blockIdx.x, Dp = c.Dp();
    const int64_t cb = c.code_base(max(page, 0), h), sb = c.scale_base(max(page, 0), h);
    const int d = (threadIdx.x & ((1 << LB) - 1)) * 8;
    u32x2_t wk[kPasses];
    float sk[kPasses], sv[kPasses];
    auto load_keys = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int t = min(t0 + i * kPer + static_cast<int>(threadIdx.x >> LB), kKvPage - 1);
            wk[i] = *reinterpret_cast<const u32x2_t*>(c.k + cb + t * Dp + (d < Dp ? d : 0));
            sk[i] = c.ks[sb + t];
            sv[i] = c.vs[sb + t];
        }
    };
    if (page >= 0) {
        load_keys(tile.t0);
        for (int i = threadIdx.x; i < Dp; i += kThreads) {
            const int g = i & 3, dd = 4 * (i >> 2);
            const uint8_t* from = c.v + cb + static_cast<int64_t>(dd) * kKvPage + 16 * g;
            u32x4_t w[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const u32x4_t*>(from + j * kKvPage);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const uint32_t by_channel[4] = {w[0][q], w[1][q], w[2][q], w[3][q]};
                uint32_t by_token[4];
                turn4(by_channel, by_token);
#pragma unroll
                for (int r = 0; r < 4; ++r) vt[((16 * q + 4 * g + r) * kPitch + dd) / 4] = by_token[r];
            }
        }
    }
    __syncthreads();
    if (d >= c.D) return;
    for (int t0 = tile.t0; t0 < tile.t1; t0 += kPasses * kPer) {
        if (page >= 0 && t0 > tile.t0) load_keys(t0);
#pragma unroll
        for (int i = 0; i < kPasses; ++i) {
            const int t = t0 + i * kPer + (threadIdx.x >> LB);
            if (t >= tile.t1) break;
            const int64_t at = ((tile.row0 + t) * c.heads + h) * c.D + d;
            float x[8] = {}, y[8] = {};
            if (page >= 0) {
                values8<FP8>(wk[i], sk[i], x);
                values8<FP8>(*reinterpret_cast<const u32x2_t*>(vt + (t * kPitch + d) / 4), sv[i], y);
            }
            store8<VEC>(k_out + at, c.D - d, x);
            store8<VEC>(v_out + at, c.D - d, y);
        }
    }
}

// Workgroups that cover every list of n_seqs sequences with `capacity` rows in
// all: n rows touch at most (n + 62) / 64 + 1 pages, and at most n.
unsigned tile_bound(int n_seqs, int capacity) {
    const int64_t seqs = std::min(n_seqs, capacity);
    const int64_t most = (static_cast<int64_t>(capacity) + 62 * seqs) / kKvPage + seqs;
    return static_cast<unsigned>(std::min<int64_t>(most, capacity));
}

// Heads, tiles: blockIdx.y + blockIdx.z * gridDim.y.  Workgroups that start
// together have the heads of a token, whose rows lie side by side.
dim3 tile_grid(int n_seqs, int capacity, int heads) {
    const unsigned tiles = tile_bound(n_seqs, capacity), y = std::min(tiles, 32768u);
    return dim3(heads, y, (tiles + y - 1) / y);
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
    const dim3 grid = tile_grid(n_seqs, capacity, c.heads);
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
    const dim3 grid = tile_grid(n_seqs, capacity, c.heads);
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
