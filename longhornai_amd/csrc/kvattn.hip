// kvattn.hip -- attention of new (drafted) tokens over the paged 8-bit cache
// (layout in kvcommon.hpp) and over one another, for gfx950.
//
//   s_j = scale * q . k_j          over the sequence's cached tokens and those
//   o   = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)     new ones its mask names
// Keys and values of cached tokens are code * scale; a token whose page is
// missing is not seen; a query that sees nothing gives zeros.
//
// One pass over the cache with a running maximum and sum.  A wave owns 16 * NQ
// queries of one kv head (the new tokens' query heads that share it) and every
// NW-th page of a range; its pages come to its own part of LDS, so no wave
// waits for another until the end, where the waves of the workgroup join their
// sums.  Both products are 16x16x32 MFMAs on transposed tiles: S^T = K Q^T
// leaves a lane with 4 adjacent tokens of one query for each 16-token tile,
// which is what it needs as the B operand of O^T = V^T P^T when the value codes
// lie in kv_slot order -- no exchange between lanes, and a query's maximum and
// rescaling factor are one register.
// Precision: key codes are exact in bf16 and meet the queries' own bf16; value
// codes are exact in fp16, and a weight times its value scale is rounded once
// to fp16.  That product is held relative to 2^e, e the running exponent of the
// largest value scale that the wave has met: the rounding is 2^-11 of itself
// down to 2^-24 of that scale, under that 2^-35 of the scale.  New tokens have
// their own exponents and each query one for those it sees, so a query's result
// depends on nothing that it does not see, to the bit; 0.15 us of a decode call,
// 0.5 of a tree's (one exponent for all of a wave's new tokens erased what stood
// beside an unseen 2^40).
//
// Measured with inputs that change (32 or 64 query heads over 8 kv heads of
// 128): decode of 4 x 131072 tokens 193 us, 5.7 TB/s, where a 4 GiB read streams
// at 6.35 -- bound by memory.  Trees of 64 over 4 x 8192 tokens 88 to 97 us at
// settled clocks, 710 to 780 TFLOP/s of the 1246 of a large library product (103
// to 117 us in the first 200 calls after a pause).  There the matrix cores are
// busy 35% of a SIMD's cycles and vector instructions issue in 67%, together all
// of them: the two hardly overlap.  A page of 32 queries takes a wave 64 MFMAs
// of 16 clocks and about 400 vector instructions, converting codes and weighing
// scores; two waves of a SIMD share its vector unit, which takes 4.2 to 4.4
// clocks for a conversion, a permute or a multiply-add, 8.2 for an exponential,
// 2.2 for a sum.  Small calls are bound by their ends: 4 us to find a workgroup's
// share and fetch its queries and first page, 2 to 3 to join.
// Tried and slower: 64 queries a wave with a SIMD to itself (trees of 64 152
// us); pages shared by the query waves of a workgroup with a barrier a page,
// its halves in turn at the products and the softmax (110).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kvcommon.hpp"

namespace lhq {
namespace {

#define LHQ_LDS_AS __attribute__((address_space(3)))
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8_t;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2_t;
typedef __attribute__((ext_vector_type(2))) uint16_t u16x2_t;

// The running maximum follows the scores only when one is over it by more
// than 2^kLag (rarely, after the first pages): weights go up to 2^kLag and,
// times value scales held at 2^kTop, stay within fp16's 65504.
constexpr float kLag = 4.0f;
constexpr int kTop = 11;
// New tokens: the exponent that a query has while it sees none; the room that
// fp32 sums have over an exponent e, so that 32 products of 2^29, at to <= e +
// kRoom, stay under 2^(34 - 29 + kTop + kRoom) = 2^100; the highest e that new
// tokens set.  A query's excess is at most 129 - kHighest - kRoom = 105: the sum
// of its weights, 2^-105 or more, is a normal number.
constexpr int kNothing = -400, kRoom = 84, kHighest = -60;

constexpr int kJoinRows = 4;     // rows of a workgroup that joins splits, a wave each
constexpr int kMostSplits = 64;  // of a sequence: a lane each when they are joined

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
    int n_seqs, capacity, max_new, heads, group;  // group: query heads of a kv head
    float scale2;          // scale * log2 e: weights are powers of two
    bool vec_out;          // rows of out: 8-byte stores
    int pages_per_split;   // a sequence of p pages has ceil(p / this) splits
    int splits;            // the most of one sequence
    float* ws_ml;          // [row][query head][split] {maximum, sum}
    float* ws_o;           // [row][query head][split][Dp]
};

__device__ __forceinline__ int cached(const AttnArgs& a, int s) {
    return static_cast<int>(min<int64_t>(max(a.lengths[s], 0), static_cast<int64_t>(a.c.max_pages) * kKvPage));
}
__device__ __forceinline__ int split_count(const AttnArgs& a, int length) {
    if (a.splits == 1) return 1;
    const int pages = (length + kKvPage - 1) / kKvPage;
    return max(1, (pages + a.pages_per_split - 1) / a.pages_per_split);
}
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Four codes as two pairs of bf16 or of fp16 (exact either way).
template <bool FP8>
__device__ __forceinline__ u32x2_t codes_bf16(uint32_t w) {
    if constexpr (FP8) {
        return {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false)),
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true))};
    } else {
        auto f = [w](int j) { return static_cast<float>(static_cast<int8_t>(w >> (8 * j))); };
        return {pack_bf16x2(f(0), f(1)), pack_bf16x2(f(2), f(3))};
    }
}
template <bool FP8>
__device__ __forceinline__ u32x2_t codes_f16(uint32_t w) {
    if constexpr (FP8) {
        return {__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false)),
                __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true))};
    } else {
        // code + 128 in the mantissa of 1024, less 1152
        const uint32_t b = w ^ 0x80808080u;
        constexpr uint32_t kExp = 0x64646464u;
        const f16x2_t off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
        auto pair = [off](uint32_t u) {
            return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, u) + off);
        };
        return {pair(__builtin_amdgcn_perm(kExp, b, 0x04010400u)), pair(__builtin_amdgcn_perm(kExp, b, 0x04030402u))};
    }
}
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {  // rounds to nearest even
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(lhq_f32x2{a, b}, f16x2_t));
}
__device__ __forceinline__ f32x4_t mfma_f16_16x16x32(u32x4_t a, u32x4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                  0, 0, 0);
}

// Eight bf16 of a row from channel ch on, those past D as zero: one 16-byte
// load at any alignment, of the row's last 8 channels where fewer are left
// (and shifted down).  SMALL: D may be under 8.
template <bool SMALL>
__device__ __forceinline__ u32x4_t load_channels(const uint16_t* row, int ch, int D) {
    uint64_t w[2] = {0, 0};
    if (SMALL && D < 8) {
        if (ch == 0)
#pragma unroll 1
            for (int j = D - 1; j >= 0; --j) {
                w[1] = (w[1] << 16) | (w[0] >> 48);
                w[0] = (w[0] << 16) | row[j];
            }
    } else {
        const int at = min(ch, D - 8), down = 16 * (ch - at), by = down & 63;
        __builtin_memcpy(w, row + at, 16);
        if (D % 8) {
            const uint64_t lo = down >= 64 ? w[1] : w[0], hi = down >= 64 ? 0 : w[1];
            w[0] = (lo >> by) | ((hi << 1) << (63 - by));
            w[1] = hi >> by;
        }
        if (ch >= D) w[0] = w[1] = 0;
    }
    return {static_cast<uint32_t>(w[0]), static_cast<uint32_t>(w[0] >> 32), static_cast<uint32_t>(w[1]),
            static_cast<uint32_t>(w[1] >> 32)};
}

// The arguments once more, from where the launch left them: a kernel that
// takes the ones of a later stage from here does not hold them through its
// main loop (they would be spilled there).
typedef const __attribute__((address_space(4))) AttnArgs* LateArgs;
__device__ __forceinline__ LateArgs late_args() {
    auto p = (LateArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return p;
}

// The first channel of lane group g in k step i: 64 channels are two steps, of
// which a group takes 16 adjacent ones (one 16-byte load of key codes); the
// 32 left over when the steps are odd in number give 8 to a group.
template <int KS>
__device__ __forceinline__ int step_channel(int i, int g) {
    return i < KS / 2 * 2 ? 64 * (i / 2) + 16 * g + 8 * (i & 1) : 32 * i + 8 * g;
}

// A page's keys in LDS: rows of Dp bytes, the 16-byte chunk j of row r in place
// j ^ key_swizzle(r).  The lanes of an operand read have 16 rows and one chunk
// for each lane group; with this the 16 lanes that LDS serves at a time (lane
// bit 5 and the parity of bits 2..4 are the same in them) meet 16 different
// 16-byte bank groups.  Rows of an odd number of 32 bytes do so as they are.
// Keys come in by LDS DMA because a wave reads 64 adjacent chunks that way: in
// operand order, 16 rows apart, the same loads reach 9.7 TB/s of the L2's 33.
template <int KS>
__device__ __forceinline__ int key_swizzle(int r) {
    if constexpr (KS == 2) return (r >> 1) & 2;
    else if constexpr (KS == 4) return (r >> 1) & 7;
    else if constexpr (KS == 6) return (r >> 2) & 2;
    else if constexpr (KS == 8) return ((r & 1) << 2) | ((r & 2) << 2) | ((r >> 2) & 2);
    else return 0;
}
// The same for values, which lie as operands already (channel row c of 64 bytes,
// lane group g's 16 at 16 g): group g's chunk of row c is in place g ^ this.
__device__ __forceinline__ int value_swizzle(int c) { return (c >> 1) & 2; }

// LDS DMA: 16 bytes a lane, from this lane's address + OFFSET to `to` + OFFSET +
// 16 * lane.
template <int OFFSET>
__device__ __forceinline__ void dma16(const void* from, void* to);
#define LHQ_DMA16(offset)                                                           \
    template <>                                                                     \
    __device__ __forceinline__ void dma16<offset>(const void* from, void* to) {     \
        __builtin_amdgcn_global_load_lds(from, (LHQ_LDS_AS void*)to, 16, offset, 0); \
    }
LHQ_DMA16(0)
LHQ_DMA16(1024)
LHQ_DMA16(2048)
LHQ_DMA16(3072)
#undef LHQ_DMA16
// KiB 4 part .. 4 part + 3 of a page's 2 KS: KiB n from `from` + 1024 n + place(n) to `to` + 1024 n + 16 * lane.
template <int KS, typename Place>
__device__ __forceinline__ void fetch(int part, const uint8_t* from, uint8_t* to, Place place) {
    const int n = 4 * part;  // (with one address on either side)
    dma16<0>(from + 1024 * n + place(n), to + 1024 * n);
    dma16<1024>(from + 1024 * n + place(n + 1), to + 1024 * n);
    if (n + 2 < 2 * KS) dma16<2048>(from + 1024 * n + place(n + 2), to + 1024 * n);
    if (n + 2 < 2 * KS) dma16<3072>(from + 1024 * n + place(n + 3), to + 1024 * n);
}
// A page's keys from LDS as operands: k steps 2 i and 2 i + 1 of tile t.
template <int KS>
__device__ __forceinline__ void read_keys(const uint8_t* keys, u32x4_t (&k)[(KS + 1) / 2][4]) {
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
    for (int i = 0; i < (KS + 1) / 2; ++i)
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint8_t* row = keys + (16 * t + c) * 32 * KS;
            if (2 * i + 1 < KS) {
                k[i][t] = *reinterpret_cast<const u32x4_t*>(row + 16 * ((4 * i + g) ^ key_swizzle<KS>(c)));
            } else {
                const u32x2_t y = *reinterpret_cast<const u32x2_t*>(row + 64 * i + 8 * g);
                k[i][t] = u32x4_t{y[0], y[1], 0, 0};
            }
        }
}
// Step i of a page's S^T.
template <int KS, int NQ, bool FP8>
__device__ __forceinline__ void score(int i, const u32x4_t (&k)[(KS + 1) / 2][4], const u32x4_t (&q)[NQ][KS],
                                      f32x4_t (&x)[NQ][4]) {
    // (a step of channels over all tiles: no product waits for the one before it)
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const u32x2_t lo = codes_bf16<FP8>(k[i / 2][t][2 * (i & 1)]), hi = codes_bf16<FP8>(k[i / 2][t][2 * (i & 1) + 1]);
        const u32x4_t key = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int n = 0; n < NQ; ++n)
            x[n][t] = mfma_bf16_16x16x32(key, q[n][i], i == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : x[n][t]);
    }
}

// The waves of a workgroup at most; two a SIMD where 256 registers hold a
// wave's page, queries and sums, else one.
template <int KS>
constexpr int most_waves() { return KS <= 4 ? 8 : 4; }

// LDS of a wave: its page and the factors of its tokens, then its sums [QB][Dp + 4] and its maxima and sums of
// weights [2][QB].
template <int KS, int NQ>
constexpr int sums_floats() { return 16 * NQ * (32 * KS + 4 + 2); }
template <int KS>
constexpr int page_bytes() { return 4 * KS * 1024 + 512; }

// Four channels of a result row from channel ch on.
__device__ __forceinline__ void store_row(uint16_t* row, int ch, int D, const f32x4_t& sum, float weight, bool vec) {
    f32x4_t y;
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = weight == 0.0f ? 0.0f : sum[j] / weight;  // nothing seen: zeros
    if (vec) {
        if (ch < D) *reinterpret_cast<u32x2_t*>(row + ch) = u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (ch + j < D) row[ch + j] = f32_to_bf16(y[j]);
    }
}

// A workgroup's share: rows [r0, ...) of the (new token, query head of the kv
// head) list of a sequence, and its pages [p0, p1).
struct Unit {
    int seq, h, G, lo, T, R, r0, L, pages, split, splits, p0, p1;
    float per_token;  // 1 / G
    // The token of row r of the list: r / G, under 64.
    __device__ int token(int r) const {
        const int t = static_cast<int>(static_cast<float>(r) * per_token);  // at most one off
        return t + (r >= (t + 1) * G) - (r < t * G);
    }
    __device__ int64_t out_row(int r, int heads) const {
        const int t = token(r);
        return static_cast<int64_t>(lo + t) * heads + h * G + r - t * G;
    }
};
// BLOCK rows a workgroup; false past the end of the list.
__device__ __forceinline__ bool find_share(const AttnArgs& a, int block, Unit& u) {
    u.h = blockIdx.x;
    u.G = a.group;
    u.per_token = 1.0f / static_cast<float>(a.group);
    int lane_lo = 0, lane_T = 0, lane_L = 0;
    const KvUnit f = kv_find_unit(blockIdx.y + blockIdx.z * gridDim.y, a.n_seqs, [&](int s) {
        const KvRows r = kv_rows(a.offsets, s, a.capacity);
        lane_lo = r.lo;
        lane_T = min(r.hi - r.lo, a.max_new);
        lane_L = cached(a, s);
        return static_cast<uint32_t>((lane_T * u.G + block - 1) / block) * split_count(a, lane_L);
    });
    if (f.seq >= a.n_seqs) return false;
    u.seq = f.seq;
    u.lo = __builtin_amdgcn_readlane(lane_lo, f.lane);
    u.T = __builtin_amdgcn_readlane(lane_T, f.lane);
    u.R = u.T * u.G;
    u.L = __builtin_amdgcn_readlane(lane_L, f.lane);
    u.pages = (u.L + kKvPage - 1) / kKvPage;
    u.splits = split_count(a, u.L);
    const int blocks = (u.R + block - 1) / block;
    if (u.splits == 1) {
        u.split = 0;
        u.r0 = f.nth * block;
        u.p0 = 0;
        u.p1 = u.pages;
    } else {  // (under 2^25 pages and 64 splits)
        u.split = f.nth / blocks;
        u.r0 = (f.nth - u.split * blocks) * block;
        u.p0 = static_cast<uint32_t>(u.pages * u.split) / static_cast<uint32_t>(u.splits);
        u.p1 = (static_cast<uint32_t>(u.pages) * (u.split + 1)) / static_cast<uint32_t>(u.splits);
    }
    return true;
}
// The operands of the 16 queries from row r on, column lane & 15 (past the
// last row: that one again, whose results no one reads).
template <int KS>
__device__ __forceinline__ void load_queries(const AttnArgs& a, const Unit& u, int r, u32x4_t (&q)[KS]) {
    const int lane = threadIdx.x & 63, row = min(r + (lane & 15), u.R - 1), t = u.token(row);
    const uint16_t* from = a.q + (u.lo + t) * a.q_stride + (u.h * u.G + row - t * u.G) * a.c.D;
#pragma unroll
    for (int i = 0; i < KS; ++i) q[i] = load_channels<KS == 1>(from, step_channel<KS>(i, lane >> 4), a.c.D);
}

// What a wave holds: sums o (channels 16 i + 4 g + j of query 16 n + c at
// o[n][i][j], c = lane & 15, g = lane >> 4), scores or weights x of 64 tokens
// (token 16 t + 4 g + j at x[n][t][j]), the running maximum m and this lane's
// part l of the sum of weights.
template <int KS, int NQ>
struct Sums {
    static constexpr int CT = 2 * KS, QB = 16 * NQ, kPitch = 32 * KS + 4;
    f32x4_t o[NQ][CT], x[NQ][4];
    float m[NQ], l[NQ];
    int e;       // o is relative to 2^(e - kTop)
    bool fresh;  // a query of the wave has no scores so far

    __device__ __forceinline__ void clear() {
        fresh = true;
        e = -200;  // (under every exponent: the first value scale that is not zero sets it)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = l[n] = 0.0f;
#pragma unroll
            for (int i = 0; i < CT; ++i) o[n][i] = f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
    }
    __device__ __forceinline__ void raise(int to) {  // to > e
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][i][j] = ldexpf(o[n][i][j], max(e - to, -400));
        e = to;
    }
    // The exponent that a maximum asks for; infinite and NaN ones ask for the largest.
    static __device__ __forceinline__ int exponent(float v) {
        return v < INFINITY ? __builtin_amdgcn_frexp_expf(v) : 128;
    }
    static __device__ __forceinline__ float across(float v) {  // maximum over the four lane groups
        v = fmaxf(v, __shfl_xor(v, 16, 64));
        return fmaxf(v, __shfl_xor(v, 32, 64));
    }
    // The value scale of token `lane` -> the factor of its weights.
    __device__ __forceinline__ float factor(float vs) {
        float top = fabsf(vs);
        if (__ballot(top > ldexpf(1.0f, e))) {
            for (int d = 32; d; d >>= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
            raise(max(e, __builtin_amdgcn_readfirstlane(exponent(top))));
        }
        return ldexpf(vs, kTop - e);
    }
    // Of x (products q . k), times ks the scores: a query's first ones set its maximum.
    __device__ __forceinline__ void start(const f32x4_t (&ks)[4]) {
        bool all = true;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) top = fmaxf(top, x[n][t][j] * ks[t][j]);
            top = across(top);
            // (a maximum's own weight is at least 2^-kLag, 2^-105 where new tokens took an excess)
            const bool first = across(l[n]) == 0.0f;
            if (first && top != -INFINITY) m[n] = top;  // (a missing page, or a mask that leaves nothing, sets nothing)
            all &= !first || top != -INFINITY;
        }
        fresh = __ballot(!all) != 0;
    }
    // Products of query tile n -> scores less the maximum, which follows when one is over it by more than kLag.
    __device__ __forceinline__ void follow(int n, const f32x4_t (&ks)[4]) {
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                x[n][t][j] = __builtin_fmaf(x[n][t][j], ks[t][j], -m[n]);
                top = fmaxf(top, x[n][t][j]);
            }
        if (__ballot(top > kLag)) {
            top = across(top);  // (of the other queries nothing moves: what they see decides nothing here)
            const float to = m[n] + (top > kLag ? top : 0.0f), by = to - m[n], f = exp2_(-by);
            m[n] = to;
            l[n] *= f;
#pragma unroll
            for (int i = 0; i < CT; ++i) o[n][i] *= f;
#pragma unroll
            for (int t = 0; t < 4; ++t) x[n][t] -= by;
        }
    }
    // Products -> weights; times w they are the operands p of the second product.
    __device__ __forceinline__ void weigh(const f32x4_t (&ks)[4], const f32x4_t (&w)[4], u32x4_t (&p)[NQ][2]) {
        if (fresh) start(ks);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            follow(n, ks);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                f32x4_t y;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = exp2_(x[n][t][j]);
                    l[n] += y[j];
                }
                p[n][t / 2][2 * (t & 1)] = pack_f16x2(y[0] * w[t][0], y[1] * w[t][1]);
                p[n][t / 2][2 * (t & 1) + 1] = pack_f16x2(y[2] * w[t][2], y[3] * w[t][3]);
            }
        }
    }
    // The last page's tokens past the length are not seen.
    __device__ __forceinline__ void cut(int left) {
        left = __builtin_amdgcn_readfirstlane(left);
        asm volatile("" : "+s"(left));  // (else made selects on every page)
        const int g = (threadIdx.x & 63) >> 4;
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int n = 0; n < NQ; ++n) x[n][t][j] = 16 * t + 4 * g + j < left ? x[n][t][j] : -INFINITY;
    }
    // The bytes of tokens 16 t + 4 g + (0..3) that are under `left`.
    static __device__ __forceinline__ uint32_t bytes_in(int t, int left) {
        const int in = min(max(left - 16 * t - 4 * ((static_cast<int>(threadIdx.x) & 63) >> 4), 0), 4);
        return in == 4 ? 0xffffffffu : (1u << (8 * in)) - 1;
    }

    // The new tokens' own keys and values: tokens t0 .. t0 + 31 that there are (at least one), before any page.
    // Each has an exponent of its own, that of its largest value, and each query one of the largest weighted value
    // that it sees: what a query does not see, however large, takes no bits from what it does.
    __device__ __forceinline__ void new_tokens(LateArgs late, const Unit& u, int t0, int D, const u32x4_t (&q)[NQ][KS]) {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
        uint32_t seen[NQ];  // of those 32
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int t = u.token(min(u.r0 + 16 * n + c, u.R - 1));
            uint64_t word = late->tree ? late->tree[u.lo + t] : ~uint64_t{0} >> (63 - t);
            word &= ~uint64_t{0} >> (64 - u.T);
            seen[n] = static_cast<uint32_t>(word >> t0);
        }
        // Value rows as they come, all loads in flight together: channel 16 i + c of tokens t and t + 1,
        // t = t0 + 16 (j / 2) + 4 g + 2 (j % 2), clamped to a row and a channel that are there.
        const uint16_t* new_values = late->v_new + u.lo * late->v_stride + u.h * D;
        uint32_t raw[CT][4];
        auto load_raw = [&] {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int t = t0 + 16 * (j / 2) + 4 * g + 2 * (j % 2);
                const uint16_t* row = new_values + min(t, u.T - 1) * late->v_stride;
                const uint16_t* odd = new_values + min(t + 1, u.T - 1) * late->v_stride;
#pragma unroll
                for (int i = 0; i < CT; ++i) {
                    const int ch = min(16 * i + c, D - 1);
                    raw[i][j] = row[ch] | static_cast<uint32_t>(odd[ch]) << 16;
                }
            }
        };
        if constexpr (NQ == 1) load_raw();  // (early where registers are free)
        const uint16_t* new_keys = late->k_new + u.lo * late->k_stride + u.h * D;
        f32x4_t ks[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) ks[t][j] = late->scale2;
#pragma unroll
            for (int n = 0; n < NQ; ++n) x[n][t] = f32x4_t{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
            if (t >= 2) continue;
            const uint16_t* row = new_keys + min(t0 + 16 * t + c, u.T - 1) * late->k_stride;
            u32x4_t key[KS];
#pragma unroll
            for (int i = 0; i < KS; ++i) key[i] = load_channels<KS == 1>(row, step_channel<KS>(i, g), D);
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int i = 0; i < KS; ++i) y = mfma_bf16_16x16x32(key[i], q[n][i], y);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if ((seen[n] >> (16 * t + 4 * g + j)) & 1) x[n][t][j] = y[j];
            }
        }
        start(ks);
#pragma unroll
        for (int n = 0; n < NQ; ++n) follow(n, ks);
        if constexpr (NQ > 1) load_raw();
        u16x2_t size[4];  // the largest of this lane's channels of two tokens, as in raw
        auto grow = [&] {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                size[j] = u16x2_t{0, 0};
#pragma unroll
                for (int i = 0; i < CT; ++i)
                    size[j] = __builtin_elementwise_max(size[j], __builtin_bit_cast(u16x2_t, raw[i][j] & 0x7fff7fffu));
            }
        };
        grow();
        const u16x2_t all = __builtin_elementwise_max(__builtin_elementwise_max(size[0], size[1]),
                                                      __builtin_elementwise_max(size[2], size[3]));
        const uint64_t not_finite = __ballot(max(all[0], all[1]) >= 0x7f80);
        if (not_finite) {  // kept out of the product, in which they would reach queries that do not see them
            uint32_t inf = 0x7f80u;
            asm volatile("" : "+s"(inf));  // (else made 64 selects on every call)
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    if ((raw[i][j] & inf) == inf) raw[i][j] &= 0xffff0000u;
                    if (((raw[i][j] >> 16) & inf) == inf) raw[i][j] &= 0xffffu;
                }
            grow();
        }
        // Each of this lane group's eight tokens, whose weights this lane has too: the exponent of its largest value,
        // biased by 126 and at least 14 (2^-112, by which smaller values are exact in fp16 too); x[n][t][j]'s is te[t][j].
        u16x2_t exps[4];
        float te[2][4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const u16x2_t top = row_max<4>(size[j], [](u16x2_t a, u16x2_t b) { return __builtin_elementwise_max(a, b); });
            exps[j] = __builtin_elementwise_max(top >> 7, u16x2_t{14, 14});
#pragma unroll
            for (int half = 0; half < 2; ++half) te[j / 2][2 * (j % 2) + half] = static_cast<float>(exps[j][half]) - 126.0f;
        }
        // Values as fp16 under 2^15 and weights up to 2^14 of the query's largest (either keeps a normal number down
        // to 2^-28 of that): the products are relative to 2^(to - 29).
        int to[NQ], most = kNothing;
        u32x4_t p[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float top = static_cast<float>(kNothing);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    l[n] += exp2_(x[n][t][j]);
                    x[n][t][j] += te[t][j];
                    top = fmaxf(top, x[n][t][j]);
                }
            top = ceilf(across(top));
            to[n] = static_cast<int>(top);
            most = max(most, to[n]);
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                f32x4_t y;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = exp2_(x[n][t][j] - (top - 14.0f));
                p[n][2 * t] = pack_f16x2(y[0], y[1]);
                p[n][2 * t + 1] = pack_f16x2(y[2], y[3]);
            }
        }
#pragma unroll
        for (int i = 0; i < CT; ++i) {
            u32x4_t val;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                val[j] = pack_f16x2(ldexpf(__uint_as_float(raw[i][j] << 16), 141 - exps[j][0]),
                                    ldexpf(__uint_as_float(raw[i][j] & 0xffff0000u), 141 - exps[j][1]));
#pragma unroll
            for (int n = 0; n < NQ; ++n) o[n][i] = mfma_f16_16x16x32(val, p[n], o[n][i]);
        }
        // To one exponent, so low that a page's value scales keep their bits beside it (the sums are fp32 and lose
        // none).  A query whose values are too large for that takes the excess into its maximum.
        most = row_max<4>(most, [](int a, int b) { return max(a, b); });
        e = min(max(__builtin_amdgcn_readfirstlane(most) - kRoom, -200), kHighest);
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const int excess = max(to[n] - e - kRoom, 0);
            m[n] += static_cast<float>(excess);
            l[n] = ldexpf(l[n], -excess);
#pragma unroll
            for (int i = 0; i < CT; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][i][j] = ldexpf(o[n][i][j], to[n] - 29 + kTop - e - excess);
        }
        if (not_finite)  // a query that sees such a value takes it as it is, the others do not
#pragma unroll 1
            for (int t = t0; t < min(u.T, t0 + 32); ++t) {
                const uint16_t* row = new_values + t * late->v_stride;
#pragma unroll
                for (int i = 0; i < CT; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float y = bf16_to_f32(row[min(16 * i + 4 * g + j, D - 1)]);
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
                            o[n][i][j] += !(fabsf(y) < INFINITY) && ((seen[n] >> (t - t0)) & 1) ? y : 0.0f;
                    }
            }
    }
    // This wave's sums to LDS, as they are (2^e applied).
    __device__ __forceinline__ void put(float* to) {
        const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float sum = l[n];
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (g == 0) {
                to[QB * kPitch + 16 * n + c] = sum == 0.0f ? -INFINITY : m[n];
                to[QB * kPitch + QB + 16 * n + c] = sum;
            }
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                f32x4_t y;
#pragma unroll
                for (int j = 0; j < 4; ++j) y[j] = ldexpf(o[n][i][j], e - kTop);
                *reinterpret_cast<f32x4_t*>(to + (16 * n + c) * kPitch + 16 * i + 4 * g) = y;
            }
        }
    }
};

// The waves' sums in LDS -> results, or a split's part of them.
template <int KS, int NQ, int WAVES>
__device__ __forceinline__ void join_waves(const float* lds, LateArgs late, const Unit& u, int D) {
    constexpr int Dp = 32 * KS, QB = 16 * NQ, kPitch = Dp + 4, step = sums_floats<KS, NQ>();
    for (int n = threadIdx.x; n < QB * (Dp / 4); n += 64 * WAVES) {
        const int qr = n / (Dp / 4), ch = 4 * (n % (Dp / 4)), r = u.r0 + qr;
        if (r >= u.R) break;
        const float* at = lds + qr * kPitch + ch;
        const float* ml = lds + QB * kPitch + qr;
        float m[WAVES], l[WAVES], top = -INFINITY;
        f32x4_t o[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            m[w] = ml[w * step];
            l[w] = ml[w * step + QB];
            o[w] = *reinterpret_cast<const f32x4_t*>(at + w * step);
        }
#pragma unroll
        for (int w = 0; w < WAVES; ++w) top = fmaxf(top, m[w]);
        const float ref = top == -INFINITY ? 0.0f : top;
        f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
        float weight = 0.0f;
#pragma unroll
        for (int w = 0; w < WAVES; ++w) {
            const float f = exp2_(m[w] - ref);
            weight += l[w] * f;
            sum += o[w] * f;
        }
        const int64_t row = u.out_row(r, late->heads);
        if (u.splits == 1) {
            store_row(late->out + row * D, ch, D, sum, weight, late->vec_out);
        } else {
            const int64_t part = row * late->splits + u.split;
            *reinterpret_cast<f32x4_t*>(late->ws_o + part * Dp + ch) = sum;
            if (ch == 0) {
                late->ws_ml[2 * part] = top;
                late->ws_ml[2 * part + 1] = weight;
            }
        }
    }
}

// Every wave has the workgroup's 16 * NQ queries and pages of its own, which
// come to its own place in LDS by DMA.  A page's operands are read to registers
// at once, and its place takes the next page while this one is worked on.  No
// wave waits for another before the end.
template <int KS, int NQ, bool FP8>
__global__ __launch_bounds__(64 * most_waves<KS>(), KS <= 4 ? 2 : 1) void kv_attn_kernel(AttnArgs a) {
    constexpr int CT = 2 * KS;
    extern __shared__ __attribute__((aligned(16))) uint8_t attn_lds[];
    Unit u;
    if (!find_share(a, 16 * NQ, u)) return;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4, h = u.h, D = a.c.D;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), NW = blockDim.x >> 6;
    uint8_t* keys = attn_lds + wave * page_bytes<KS>();
    uint8_t* values = keys + 2 * KS * 1024;

    float* factors = reinterpret_cast<float*>(values + 2 * KS * 1024);  // of scores, of weights; by token

    float ks = 0.0f, vs = 0.0f;  // of token `lane`
    // A page's fetch in parts: its scales and keys, then its values (the values last: the wait for the keys counts
    // on it).
    constexpr int kParts = (KS + 1) / 2;
    const uint8_t *from_k = nullptr, *from_v = nullptr;
    auto aim = [&](int page) {
        ks = a.c.ks[a.c.scale_base(page, h) + lane];
        vs = a.c.vs[a.c.scale_base(page, h) + lane];
        from_k = a.c.k + a.c.code_base(page, h);
        from_v = a.c.v + a.c.code_base(page, h);
    };
    auto load_part = [&](int part) {
        if (part < kParts)
            fetch<KS>(part, from_k, keys, [lane](int n) -> uint32_t {
                return 16 * (lane ^ key_swizzle<KS>((64 * n + lane) / (2 * KS)));
            });
        else
            fetch<KS>(part - kParts, from_v, values,
                      [lane](int) -> uint32_t { return 16 * (lane ^ value_swizzle(lane >> 2)); });
        asm volatile("" ::: "memory");  // (in order)
    };
    auto load_page = [&](int page) {
        aim(page);
#pragma unroll
        for (int part = 0; part < 2 * kParts; ++part) load_part(part);
    };
    // pages p0 + wave, + NW, ...
    const int mine = u.p0 + wave < u.p1 ? (u.p1 - u.p0 - wave + NW - 1) / NW : 0;
    int ids = 0;
    auto page_id = [&](int it) {  // 64 entries of the block table at a time, one a lane
        if ((it & 63) == 0) {
            const int p = u.p0 + wave + (it + lane) * NW;
            ids = p < u.p1 ? a.c.page(u.seq, p) : -1;
        }
        return __builtin_amdgcn_readlane(ids, it & 63);
    };
    int page = -1;
    if (mine > 0) {
        page = page_id(0);
        load_page(max(page, 0));  // (a missing page's place is taken by page 0, of which no token is seen)
    }
    u32x4_t q[NQ][KS];
#pragma unroll
    for (int n = 0; n < NQ; ++n) load_queries<KS>(a, u, u.r0 + 16 * n, q[n]);
    Sums<KS, NQ> z;
    z.clear();
    // The new tokens first, 32 at a time, by the waves whose turn it is after the last page (at least four waves
    // for at most 64 tokens): their rows are fetched while the first page is on its way.  After the pages they
    // took up to 4% of a call more (decode of 64 ragged sequences, replays over one set of inputs, 44.3 us for 42.9),
    // and more registers.
    const int turn = __builtin_amdgcn_readfirstlane((wave + NW - (u.p1 - u.p0) % NW) % NW);
    if (late_args()->k_new && u.split == u.splits - 1 && 32 * turn < u.T) z.new_tokens(late_args(), u, 32 * turn, D, q);
    for (int it = 0; it < mine; ++it) {
        const int left = page < 0 ? 0 : min(u.L - (u.p0 + wave + it * NW) * kKvPage, kKvPage);
        // The keys have landed: at least the CT loads of values were issued after them.
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(CT) : "memory");
        u32x4_t k[(KS + 1) / 2][4], v[CT], w[NQ][2];
        read_keys<KS>(keys, k);
        const bool in = lane < left;  // what the last page holds past the length counts for nothing
        factors[lane] = in ? ks * a.scale2 : 1.0f;
        factors[64 + lane] = z.factor(in ? vs : 0.0f);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < CT; ++i)
            v[i] = *reinterpret_cast<const u32x4_t*>(values + 1024 * i + 64 * c + 16 * (g ^ value_swizzle(c)));
        const int next = it + 1 < mine ? page_id(it + 1) : -1;
        const bool more = it + 1 < mine;
        __builtin_amdgcn_sched_barrier(0);
        // The SIMD's other wave is kept off the matrix cores until this one's product is through: left
        // alone the two run every product and every softmax at the same time, one unit idle in turn.
        __builtin_amdgcn_s_setprio(2);
#pragma unroll
        for (int i = 0; i < KS; ++i) {
            score<KS, NQ, FP8>(i, k, q, z.x);
            if (more) {  // parts of the next page's fetch between the steps (all before them: 42.9 us for 42.2)
                if (i == 0) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // (this page has been read)
                    aim(max(next, 0));
                }
#pragma unroll
                for (int part = i * 2 * kParts / KS; part < (i + 1) * 2 * kParts / KS; ++part) load_part(part);
            }
        }
        __builtin_amdgcn_s_setprio(0);
        if (left < kKvPage) {
            z.cut(left);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint32_t bytes = z.bytes_in(t, left);
#pragma unroll
                for (int i = 0; i < CT; ++i) v[i][t] &= bytes;
            }
        }
        f32x4_t k2[4], f[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            k2[t] = *reinterpret_cast<const f32x4_t*>(factors + 16 * t + 4 * g);
            f[t] = *reinterpret_cast<const f32x4_t*>(factors + 64 + 16 * t + 4 * g);
        }
        z.weigh(k2, f, w);
        __builtin_amdgcn_s_setprio(2);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < CT; ++i) {
                const u32x2_t lo = codes_f16<FP8>(v[i][2 * s]), hi = codes_f16<FP8>(v[i][2 * s + 1]);
                const u32x4_t val = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
                for (int n = 0; n < NQ; ++n) z.o[n][i] = mfma_f16_16x16x32(val, w[n][s], z.o[n][i]);
            }
        __builtin_amdgcn_s_setprio(0);
        page = next;
    }

    const LateArgs late = late_args();
    __syncthreads();  // (the pages' place is taken)
    float* sums = reinterpret_cast<float*>(attn_lds);
    z.put(sums + wave * sums_floats<KS, NQ>());
    __syncthreads();
    if constexpr (KS <= 4)
        if (NW == 8) return join_waves<KS, NQ, 8>(sums, late, u, D);
    join_waves<KS, NQ, 4>(sums, late, u, D);
}

// Joins the splits of a sequence's rows, in order of position: a wave takes one
// (new token, query head) row of a kv head.  4 to 5 us, a launch's cost, from 24
// splits of 16 rows to 3 of 400.
__global__ __launch_bounds__(256) void kv_attn_join_kernel(AttnArgs a) {
    const int G = a.group, D = a.c.D, Dp = a.c.Dp(), h = blockIdx.x;
    int lane_lo = 0, lane_T = 0, lane_L = 0;
    const KvUnit u = kv_find_unit(blockIdx.y + blockIdx.z * gridDim.y, a.n_seqs, [&](int s) {
        const KvRows r = kv_rows(a.offsets, s, a.capacity);
        lane_lo = r.lo;
        lane_T = min(r.hi - r.lo, a.max_new);
        lane_L = cached(a, s);
        return static_cast<uint32_t>((lane_T * G + kJoinRows - 1) / kJoinRows);
    });
    if (u.seq >= a.n_seqs) return;
    const int splits = split_count(a, __builtin_amdgcn_readlane(lane_L, u.lane));
    if (splits == 1) return;  // (its rows are there already)
    const int lo = __builtin_amdgcn_readlane(lane_lo, u.lane), R = __builtin_amdgcn_readlane(lane_T, u.lane) * G;
    const int lane = threadIdx.x & 63;
    // lanes that share the splits of 4 channels
    const int share = Dp <= 64 ? 4 : Dp <= 128 ? 2 : 1, ch = 4 * (lane & (64 / share - 1)), first = lane / (64 / share);
    const int r = u.nth * kJoinRows + (threadIdx.x >> 6);
    if (r >= R) return;
    const int64_t row = static_cast<int64_t>(lo + r / G) * a.heads + h * G + r % G, part = row * a.splits;
    const float* from = a.ws_o + part * Dp + min(ch, Dp - 4);
    const float m = lane < splits ? a.ws_ml[2 * (part + lane)] : -INFINITY;
    const float l = lane < splits ? a.ws_ml[2 * (part + lane) + 1] : 0.0f;
    float f = 0.0f, weight = 0.0f;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < splits; s0 += 8 * share) {
        f32x4_t y[8];  // eight splits a lane in flight; past the last one, that again, unused
#pragma unroll
        for (int k = 0; k < 8; ++k)
            y[k] = *reinterpret_cast<const f32x4_t*>(from + min(s0 + k * share + first, splits - 1) * Dp);
        if (s0 == 0) {
            float top = m;
            for (int s = 32; s; s >>= 1) top = fmaxf(top, __shfl_xor(top, s, 64));
            f = exp2_(m - (top == -INFINITY ? 0.0f : top));
            weight = l * f;
            for (int s = 32; s; s >>= 1) weight += __shfl_xor(weight, s, 64);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int s = s0 + k * share + first;
            const float fs = __shfl(f, s & 63, 64);
            if (s < splits) sum += y[k] * fs;
        }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        if (share >= 2) sum[j] += __shfl_xor(sum[j], 32, 64);
        if (share == 4) sum[j] += __shfl_xor(sum[j], 16, 64);
    }
    if (first == 0) store_row(a.out + row * D, ch, D, sum, weight, a.vec_out);
}

// How a call is laid out: query tiles of a wave, waves of a workgroup, splits
// of a sequence, workgroups.
struct Plan {
    int tiles, waves, pages_per_split, splits;
    int64_t units, join_units;  // per kv head
    int64_t ml_bytes, bytes;
};
int64_t unit_bound(int n_seqs, int capacity, int max_new, int G, int block) {
    const int64_t seqs = std::min(n_seqs, capacity);
    return std::min(static_cast<int64_t>(capacity) * G / block + seqs,
                    seqs * ((static_cast<int64_t>(max_new) * G + block - 1) / block));
}
// Splits and waves by an estimate of the time, in us, from what small calls
// measured.  For each 32 channels a workgroup costs 1.5 (one tile of queries)
// or 2 to set up and to finish, a page of a wave 0.45 or 1; 0.6 of that where
// it has a SIMD for itself, 1.1 of two tiles in workgroups of eight waves, which
// are in step with one another.  Splitting adds the launch that joins, 4.5 and
// 0.075 a split, and the parts' way through memory.  2048 waves are resident (1024 with over 128 channels).
// The host knows the longest length there may be, not the lengths: the estimate
// is that of all sequences having that and that of three tenths of the work
// being there (ragged lengths), added.  Measured: decode of 4 x 4096 tokens in 8
// splits 14.6 us, in one 19.4; of 16 x 2048 in one 19.2, in two 21.7; trees of
// 12 over 2500 ragged tokens in 3 or 5 splits 24, in one 31; trees of 64 over 4 x
// 8192 in one 97, in two 116.
// A split is a share of the table's width, of which a sequence far shorter than
// that has few: one token over 8192 takes 12.4 us with a table of 128 or 256
// pages, 14.6 with 512, 18.7 with 1024, 26.7 with 2048 (16 such sequences 48 us
// with any).  And with kMostSplits one sequence and one kv head have 64
// workgroups at most: 131072 tokens of 4 query heads 24 us, 1.4 TB/s.
Plan make_plan(int n_seqs, int capacity, int max_new, int max_pages, int heads, int kv_heads, int D, int64_t ws_bytes) {
    const int G = heads / kv_heads, KS = kv_padded(D) / 32;
    Plan p{};
    p.tiles = max_new * G <= 16 ? 1 : 2;
    p.units = unit_bound(n_seqs, capacity, max_new, G, 16 * p.tiles);
    p.join_units = unit_bound(n_seqs, capacity, max_new, G, kJoinRows);
    const int64_t units = std::max<int64_t>(1, p.units * kv_heads), rows = static_cast<int64_t>(capacity) * heads;
    const int64_t resident = KS <= 4 ? 2048 : 1024;
    const double ends = (p.tiles == 1 ? 1.5 : 2.0) * KS, page = (p.tiles == 1 ? 0.45 : 1.0) * KS;
    double best = HUGE_VAL;
    auto consider = [&](int64_t want) {
        const int per = std::max<int>(1, (max_pages + want - 1) / want), splits = std::max(1, (max_pages + per - 1) / per);
        const int64_t ml_bytes = splits == 1 ? 0 : (rows * splits * 8 + 15) / 16 * 16;
        const int64_t bytes = splits == 1 ? 0 : ml_bytes + rows * splits * 32 * KS * 4;
        if (bytes > ws_bytes) return;
        const int64_t groups = units * splits, some = n_seqs > 1 ? std::max<int64_t>(1, groups * 3 / 10) : groups;
        for (int waves = 4; waves <= (KS <= 4 ? 8 : 4); waves += 4) {
            const int64_t slots = resident / waves;
            auto time = [&](int64_t n) {
                const double share = waves == 8 ? (p.tiles == 1 ? 1.0 : 1.1) : KS <= 4 && n <= slots / 2 ? 0.6 : 1.0;
                return static_cast<double>((n + slots - 1) / slots) * (ends + (per + waves - 1) / waves * page * share);
            };
            const double cost = time(groups) + time(some) + (splits > 1 ? 9.0 + 0.15 * splits + static_cast<double>(bytes) * 0.5e-6 : 0.0);
            if (cost >= best) continue;
            best = cost;
            p.waves = waves;
            p.splits = splits;
            p.pages_per_split = per;
            p.ml_bytes = ml_bytes;
            p.bytes = bytes;
        }
    };
    for (int n : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, kMostSplits})
        if (n == 1 || n <= max_pages) consider(n);
    for (int64_t slots : {resident / 4, resident / 8})  // as many as are resident
        if (slots / units > 1) consider(std::min<int64_t>(slots / units, kMostSplits));
    return p;
}

// kv heads, units: blockIdx.y + blockIdx.z * gridDim.y
dim3 unit_grid(int heads, int64_t units) {
    const unsigned y = static_cast<unsigned>(std::min<int64_t>(units, 32768));
    return dim3(heads, y, static_cast<unsigned>((units + y - 1) / y));
}

template <auto Kern>
int launch(const char* fn, const AttnArgs& a, const Plan& p, size_t lds, hipStream_t s) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(Kern),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (attr != hipSuccess) return set_error(LHQ_ERR_HIP, "%s: dynamic LDS attribute: %s", fn, hipGetErrorString(attr));
    Kern<<<unit_grid(a.c.heads, p.units * p.splits), 64 * p.waves, lds, s>>>(a);
    return check_launch(fn);
}
template <int KS, bool FP8>
int launch(const char* fn, const AttnArgs& a, const Plan& p, hipStream_t s) {
    const int wave = std::max(4 * (p.tiles == 1 ? sums_floats<KS, 1>() : sums_floats<KS, 2>()), page_bytes<KS>());
    const size_t lds = p.waves * wave;
    if (p.tiles == 1) return launch<&kv_attn_kernel<KS, 1, FP8>>(fn, a, p, lds, s);
    return launch<&kv_attn_kernel<KS, 2, FP8>>(fn, a, p, lds, s);
}

}  // namespace
}  // namespace lhq

using namespace lhq;

extern "C" {

int64_t lhq_kv_attn_workspace_bytes(int n_seqs, int row_capacity, int max_new, int max_pages, int n_heads,
                                    int n_kv_heads, int head_dim) {
    if (n_seqs < 0 || row_capacity < 0 || max_new < 0 || max_new > kKvMaxNew || max_pages < 0 || n_kv_heads <= 0 ||
        n_heads <= 0 || n_heads % n_kv_heads != 0 || head_dim <= 0 || head_dim > kKvMaxDim)
        return 0;
    return make_plan(n_seqs, row_capacity, max_new, max_pages, n_heads, n_kv_heads, head_dim, INT64_MAX).bytes;
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
    const float scale2 = scale * 1.4426950408889634f;  // weights are powers of two
    LHQ_REQUIRE(std::isfinite(scale2) && scale > 0.0f, "%s: scale %g is not positive and finite, also times log2 e", fn,
                scale);
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
    auto odd = [](const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; };
    AttnArgs a{q,        q_stride, k_new,  k_stride,     v_new,   v_stride, tree, offsets, lengths, c, out,
               n_seqs, row_capacity, max_new, n_heads, n_heads / n_kv_heads, scale2};
    if (num_pages == 0) a.c.max_pages = 0;  // (no page to stand in for a missing one)
    a.vec_out = head_dim % 4 == 0 && !odd(out, 8);
    const Plan p = make_plan(n_seqs, row_capacity, max_new, max_pages, n_heads, n_kv_heads, head_dim,
                             workspace ? workspace_bytes : 0);
    LHQ_SUPPORTED(p.units * p.splits * n_kv_heads * p.waves < INT32_MAX / 64 &&
                      (p.splits == 1 || p.join_units * n_kv_heads < INT32_MAX / 256),
                  "%s: %lld query blocks of %d heads are over the grid", fn, static_cast<long long>(p.units), n_kv_heads);
    a.pages_per_split = p.pages_per_split;
    a.splits = p.splits;
    a.ws_ml = static_cast<float*>(workspace);
    a.ws_o = a.ws_ml + p.ml_bytes / 4;
    const hipStream_t s = as_stream(stream);
    int st = LHQ_OK;
    auto go = [&](auto ks) {
        st = format == LHQ_KV_FP8 ? launch<ks(), true>(fn, a, p, s) : launch<ks(), false>(fn, a, p, s);
    };
    switch (kv_padded(head_dim) / 32) {
        case 1: go(std::integral_constant<int, 1>{}); break;
        case 2: go(std::integral_constant<int, 2>{}); break;
        case 3: go(std::integral_constant<int, 3>{}); break;
        case 4: go(std::integral_constant<int, 4>{}); break;
        case 5: go(std::integral_constant<int, 5>{}); break;
        case 6: go(std::integral_constant<int, 6>{}); break;
        case 7: go(std::integral_constant<int, 7>{}); break;
        default: go(std::integral_constant<int, 8>{}); break;
    }
    if (st != LHQ_OK || p.splits == 1) return st;
    kv_attn_join_kernel<<<unit_grid(n_kv_heads, p.join_units), 256, 0, s>>>(a);
    return check_launch(fn);
}

}  // extern "C"
