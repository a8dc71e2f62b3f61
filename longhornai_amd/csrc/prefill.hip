// prefill.hip -- causal attention of prompts and of prompts' chunks, with the
// paged 8-bit cache (layout in kvcommon.hpp) or without, for gfx950.
//
//   s_j = scale * q . k_j           over the sequence's cached tokens and its new
//   o   = sum_j e^(s_j - m) v_j / sum_j e^(s_j - m)     ones up to the token itself
//
// One pass with a running maximum and sum.  A workgroup has 128 or 256 (new token,
// query head) rows of one kv head (block_rows says which), four or eight waves of 32
// rows each, and walks the keys 64 at a time: pages of the cache, then tiles of the
// new tokens.  A tile comes to LDS once for all waves, in bf16 (codes are exact
// there), while they work on the one before it.  Both products are 32x32x16 MFMAs on
// transposed tiles: S^T = K Q^T leaves a lane with 4 adjacent keys of one row, four
// times over, which is what it needs as the B operand of O^T = V^T P^T when V^T's
// keys come in that order; a row's maximum and sum are one register each.
// Precision: scores, weights' sums and results are fp32; a weight (of a cached
// token, times its value scale) is rounded once to bf16, at 2^-8 of itself, which has
// the range of both and needs no exponent of its own (down to scales of 2^-115 or so:
// below them weights leave its normal numbers); the result is rounded to bf16.
//
// Bound: a tile for 256 rows of 128 channels is 2048 clocks of a SIMD's matrix work,
// about 1900 of its vector work (exponentials half of it) and 256 KB of LDS reads,
// 2048 clocks at the 128 bytes a clock that LDS gives at most; two waves a SIMD
// overlap them to 3600.  Measured on several cards, 32 heads over 8 of 128: 16384
// tokens 1.98 to 2.1 ms (1050 to 1110 TFLOPS, where a bf16 product of 8192^3 reaches
// 1190 to 1250), 16 prompts of up to 2048 205 to 217 us (730 to 770), 4 of up to 200
// 12.3 to 12.5 us.
// Pages cost the conversion of their codes beside it: 512 tokens of 64 heads over
// 32768 of e4m3 601 to 640 us (870 to 920 TFLOPS).  Of 64 rows a wave, which halves
// the LDS reads but leaves one wave a SIMD: 2290 us where this takes 1985, also with
// the products of the next tile interleaved with the weights of this one.
#include <algorithm>
#include <cmath>
#include <type_traits>
#include <utility>

#include "kvcommon.hpp"

namespace lhq {
namespace {

#define LHQ_LDS_AS __attribute__((address_space(3)))
typedef __attribute__((ext_vector_type(4))) short s16x4_t;

// The running maximum follows the scores only when one is over it by more than
// 2^kLag: weights go up to 2^kLag, which costs none of their bits.
constexpr float kLag = 6.0f;
constexpr int kMostSplits = 64;  // of a block's keys
constexpr int kLeastTiles = 8;   // of a split: the launch that joins takes as long as some tiles
constexpr int kJoinRows = 8;     // of a workgroup that joins splits: half a wave a row

struct PrefillArgs {
    const uint16_t* q;
    int64_t q_stride;
    const uint16_t* k_new;
    int64_t k_stride;
    const uint16_t* v_new;
    int64_t v_stride;
    const int32_t* offsets;
    const int32_t* lengths;
    KvCache c;
    uint16_t* out;
    int n_seqs, capacity, heads, group;  // group: query heads of a kv head
    float scale2;          // scale * log2 e: weights are powers of two
    bool vec_new;          // rows of k_new, v_new: 16-byte loads at 32-bit offsets from a tile's first
    bool vec_out;          // rows of out: 16-byte stores
    bool clear_rest;       // rows of no sequence become zeros
    int slots;             // workgroups of a kv head that are on the chip at once, 0: no splitting
    int block_rows;        // rows of a workgroup
    int part_rows;         // rows of a part in the workspace
    float* ws_o;           // [kv head][part][part_rows][Dp]
    float* ws_ml;          // [kv head][part][part_rows] {maximum, sum}
};

// Bytes of LDS: two tiles of keys and values, two pages' factors, a flag.
template <int KS>
constexpr int lds_bytes() { return 4 * KS * 4096 + 1024 + 16; }

// A sequence: its first row, new tokens, cached tokens; the list of blocks.
struct Seq {
    int lo, T, L, blocks, tiles;
};
__device__ __forceinline__ Seq seq_of(const PrefillArgs& a, int s) {
    if (s >= a.n_seqs) return {0, 0, 0, 0, 0};
    const KvRows r = kv_rows(a.offsets, s, a.capacity);
    Seq q;
    q.lo = r.lo;
    q.T = r.hi - r.lo;
    q.L = a.c.max_pages == 0 ? 0 : static_cast<int>(min<int64_t>(max(a.lengths[s], 0), static_cast<int64_t>(a.c.max_pages) * kKvPage));
    q.blocks = (q.T * a.group + a.block_rows - 1) / a.block_rows;
    q.tiles = (q.L + kKvPage - 1) / kKvPage + (a.k_new ? (q.T + kKvPage - 1) / kKvPage : 0);
    return q;
}
__device__ __forceinline__ int split_count(const Seq& q, int target) {
    return q.tiles <= target ? 1 : min((q.tiles + target - 1) / target, kMostSplits);
}
// Tiles that a split has at most: all blocks' tiles over the workgroups wanted, or
// half of that where the parts would not all be on the chip at once (a finer grain
// leaves less over at the end).  Blocks that have more are split, into less than 4 *
// slots parts in all: a block of t > target tiles has ceil(t / target) < 2 t / target.
__device__ __forceinline__ int split_target(const PrefillArgs& a, const Seq& first) {
    if (a.slots == 0) return INT32_MAX;
    auto over_all = [&](auto of) {  // (held at 2^32 - 1)
        uint32_t sum = 0;
        for (int base = 0; base < a.n_seqs; base += 64) {
            const uint32_t x = of(base == 0 ? first : seq_of(a, base + (threadIdx.x & 63)));
            sum = __builtin_elementwise_add_sat(sum, static_cast<uint32_t>(__builtin_amdgcn_readlane(kv_scan(x), 63)));
        }
        return sum;
    };
    const uint32_t work = over_all([](const Seq& q) {
        return static_cast<uint32_t>(min(static_cast<uint64_t>(q.blocks) * q.tiles, uint64_t{0xffffffff}));
    });
    if (work == 0xffffffff) return INT32_MAX;  // (more than the chip has workgroups, by far)
    auto target = [work](uint32_t slots) { return max(kLeastTiles, static_cast<int>(min(work / slots, 0x7ffffffeu)) + 1); };
    const int once = target(a.slots);
    const uint32_t units = over_all([once](const Seq& q) { return static_cast<uint32_t>(q.blocks) * split_count(q, once); });
    return units <= static_cast<uint32_t>(a.slots) ? once : target(2 * a.slots);
}
// (`first` is the lane's of the first 64 sequences, `target` split_target's.)
// The unit with number `unit` in the list that has count(sequence, splits) units
// of each sequence in turn: the sequence, the unit's number within it, and the
// parts (split blocks times their splits) of the sequences before it.  Past the
// end of the list seq is n_seqs and nth counts from there.
struct Found { int seq, nth, splits, parts; Seq q; };
template <typename Count>
__device__ __forceinline__ Found find_unit(const PrefillArgs& a, const Seq& first, int target, uint32_t unit, Count count) {
    const int lane = threadIdx.x & 63;
    uint32_t parts = 0;
    for (int base = 0; base < a.n_seqs; base += 64) {
        const Seq q = base == 0 ? first : seq_of(a, base + lane);
        const int splits = split_count(q, target);
        const uint32_t sum = kv_scan(count(q, splits)), own = splits > 1 ? q.blocks * splits : 0, upto = kv_scan(own);
        const uint64_t over = __ballot(sum > unit);
        if (over) {
            const int l = __builtin_ctzll(over);
            auto of = [l](int x) { return __builtin_amdgcn_readlane(x, l); };
            const uint32_t before = l > 0 ? __builtin_amdgcn_readlane(sum, l - 1) : 0u;
            return {base + l, static_cast<int>(unit - before), of(splits), static_cast<int>(parts) + of(upto - own),
                    {of(q.lo), of(q.T), of(q.L), of(q.blocks), of(q.tiles)}};
        }
        unit -= __builtin_amdgcn_readlane(sum, 63);
        parts += __builtin_amdgcn_readlane(upto, 63);
    }
    return {a.n_seqs, static_cast<int>(unit), 1, 0, {0, 0, 0, 0, 0}};
}

// ---- tiles in LDS -----------------------------------------------------------
// Keys, and values of new tokens: [32 channels][64 tokens][64 bytes], the 16-byte
// chunk j of token t at place j ^ ((t >> 2) & 3): the 16 lanes of an operand read
// that LDS serves at a time have one chunk of 16 tokens, which lie in 16 different
// places of 256 bytes.
// Values of cached tokens: [channel][128 bytes], the chunk of keys 16 s + {4 h ..
// 4 h + 3, 8 + 4 h .. + 3} at place (2 s + h) ^ ((channel >> 1) & 7), as above.
__device__ __forceinline__ int token_place(int t, int chunk) { return t * 64 + 16 * (chunk ^ ((t >> 2) & 3)); }
__device__ __forceinline__ int value_place(int ch, int chunk) { return ch * 128 + 16 * (chunk ^ ((ch >> 1) & 7)); }

__device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0, 0, 0, 0};

// 16 bytes a lane from `from` + lane_at + OFFSET to LDS address `to` + OFFSET + 16 *
// lane, without a register on the way.  In assembly: the compiler makes every later
// LDS read wait for the builtin's.  arrived() waits for them all.  m0 is named as written:
// the compiler keeps no variable there (and warns of that), but sets it ahead of
// instructions of its own, and may take an earlier setting for still there.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int OFFSET>
__device__ __forceinline__ void dma16(const void* from, uint32_t lane_at, uint32_t to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 offset:%3"
                 :: "s"(to), "v"(lane_at), "s"(from), "n"(OFFSET) : "m0", "memory");
}
__device__ __forceinline__ void dma16_any(const void* from, uint32_t to) {  // an address a lane
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" :: "s"(to), "v"(from) : "m0", "memory");
}
#pragma clang diagnostic pop
__device__ __forceinline__ void arrived() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ uint32_t lds_address(const void* p) {
    return static_cast<uint32_t>(reinterpret_cast<uintptr_t>((LHQ_LDS_AS const void*)p));
}

// Keys or values of a sequence's new tokens on their way to LDS, a tile of 64 after
// the other.  Tokens past the last one are that one again (no row sees them); channels
// past D are zero.
template <int KS, int W>
struct NewTiles {
    const uint16_t* from;  // the next tile's first row, this kv head
    int64_t stride;        // of rows
    uint32_t lane_at;      // this lane's bytes in a whole tile, from there
    uint32_t wave_at;      // this wave's part of a tile in LDS
    int j0, past;          // the next tile's first token, that past the last tile

    // A wave brings 16 tokens (wave & 3) of every (W / 4)th 32 channels; four lanes a token.
    static __device__ __forceinline__ int token() { return 16 * ((threadIdx.x >> 6) & 3) + ((threadIdx.x & 63) >> 2); }
    static __device__ __forceinline__ int channel() {  // of the first 32
        const int lane = threadIdx.x & 63;
        return 32 * (threadIdx.x >> 8) + 8 * ((lane & 3) ^ ((lane >> 4) & 3));
    }
    __device__ __forceinline__ void aim(const uint16_t* rows, int64_t stride_, int lo, int h, int D, int j0_, int past_) {
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        j0 = j0_;
        past = past_;
        stride = stride_;
        from = rows + (lo + static_cast<int64_t>(j0)) * stride + h * D;
        lane_at = token() * static_cast<uint32_t>(2 * stride) + 2 * channel();
        wave_at = 4096 * (wave >> 2) + 1024 * (wave & 3);
    }
    template <int... M>
    __device__ __forceinline__ void whole(uint32_t at, uint32_t to, std::integer_sequence<int, M...>) const {
        constexpr int kStep = W / 4;
        // (an odd number of 32 channels: the upper waves of eight have one fewer)
        ((kStep * M + kStep <= KS || __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) + kStep * M < KS
              ? dma16<64 * kStep * M>(from, at, to + (4096 - 64) * kStep * M) : void()), ...);
    }
    // The next tile to `to`, if there is one.
    __device__ __forceinline__ void fetch(const PrefillArgs& a, int T, uint8_t* to) {
        if (j0 >= past) return;
        const int D = a.c.D;
        constexpr int kMost = (KS + W / 4 - 1) / (W / 4);
        if (a.vec_new) {
            uint32_t at = lane_at;
            if (j0 + kKvPage > T) at = min(token(), T - 1 - j0) * static_cast<uint32_t>(2 * stride) + 2 * channel();
            const uint32_t lds = lds_address(to) + wave_at;
            if (D == 32 * KS) {
                whole(at, lds, std::make_integer_sequence<int, kMost>{});
            } else {
#pragma unroll
                for (int m = 0; m < kMost; ++m) {
                    const int more = 32 * (W / 4) * m;
                    if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 8) + W / 4 * m >= KS) break;
                    const uint8_t* lane = reinterpret_cast<const uint8_t*>(from) + at + 2 * more;
                    dma16_any(channel() + more < D ? lane : reinterpret_cast<const uint8_t*>(kZeros), lds + 128 * more);
                }
            }
        } else {
            for (int n = threadIdx.x; n < 64 * 4 * KS; n += 64 * W) {
                const int t = n & 63, ch = 8 * (n >> 6);
                const uint16_t* row = from + static_cast<int64_t>(min(t, T - 1 - j0)) * stride;
                *reinterpret_cast<u32x4_t*>(to + (ch >> 5) * 4096 + token_place(t, (ch >> 3) & 3)) = load_channels<KS == 1>(row, ch, D);
            }
        }
        from += kKvPage * stride;
        j0 += kKvPage;
    }
};

// Four codes as two pairs of bf16 (exact).
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

// A page on its way: 32 codes of keys (a token's 32 channels) or of values (a
// channel's 32 keys of one half) a thread and task, and a scale.
template <int KS, int W>
struct PageLoad {
    static constexpr int kTasks = (2 * KS + W - 1) / W;
    u32x4_t w[kTasks][2];
    float factor;

    __device__ __forceinline__ void load(const KvCache& c, int page, int h) {
        const uint8_t *k = c.k + c.code_base(page, h), *v = c.v + c.code_base(page, h);
        const int tid = threadIdx.x;
#pragma unroll
        for (int i = 0; i < kTasks; ++i) {
            const int n = tid + 64 * W * i;  // (the same side for all of a wave)
            if (n < 64 * KS) {
                w[i][0] = *reinterpret_cast<const u32x4_t*>(k + 32 * n);
                w[i][1] = *reinterpret_cast<const u32x4_t*>(k + 32 * n + 16);
            } else if (n < 128 * KS) {
                const int m = n - 64 * KS;  // channel m >> 1, keys' half m & 1
                w[i][0] = *reinterpret_cast<const u32x4_t*>(v + 64 * (m >> 1) + 16 * (m & 1));
                w[i][1] = *reinterpret_cast<const u32x4_t*>(v + 64 * (m >> 1) + 16 * (m & 1) + 32);
            }
        }
        if (tid < 64) factor = c.ks[c.scale_base(page, h) + tid];
        else if (tid < 128) factor = c.vs[c.scale_base(page, h) + tid - 64];
    }
    // `left` tokens of the page count; codes and value scales of the others become zero.
    template <bool FP8>
    __device__ __forceinline__ void store(int left, float scale2, uint8_t* keys, uint8_t* values, float* factors) {
        const int tid = threadIdx.x;
#pragma unroll
        for (int i = 0; i < kTasks; ++i) {
            const int n = tid + 64 * W * i;
            if (n < 64 * KS) {
                const int t = n / KS, kb = n % KS;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const u32x2_t lo = codes_bf16<FP8>(w[i][j >> 1][2 * (j & 1)]), hi = codes_bf16<FP8>(w[i][j >> 1][2 * (j & 1) + 1]);
                    *reinterpret_cast<u32x4_t*>(keys + 4096 * kb + token_place(t, j)) = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
                }
            } else if (n < 128 * KS) {
                const int m = n - 64 * KS, ch = m >> 1, half = m & 1;
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    uint32_t x = w[i][0][s], y = w[i][1][s];  // keys 16 s + 4 half on, and 8 further
                    if (left < kKvPage) {
                        auto keep = [left](uint32_t codes, int t) {
                            const int in = left - t;
                            return in >= 4 ? codes : in <= 0 ? 0u : codes & ((1u << (8 * in)) - 1);
                        };
                        x = keep(x, 16 * s + 4 * half);
                        y = keep(y, 16 * s + 4 * half + 8);
                    }
                    const u32x2_t lo = codes_bf16<FP8>(x), hi = codes_bf16<FP8>(y);
                    *reinterpret_cast<u32x4_t*>(values + value_place(ch, 2 * s + half)) = u32x4_t{lo[0], lo[1], hi[0], hi[1]};
                }
            }
        }
        if (tid < 64) factors[tid] = factor * scale2;
        else if (tid < 128) factors[tid] = tid - 64 < left ? factor : 0.0f;
    }
};

// The halves of a dword that are bf16 infinities or NaN, as a mask.
__device__ __forceinline__ uint32_t odd_halves(uint32_t w) {
    return ((w & 0x7f80u) == 0x7f80u ? 0xffffu : 0u) | ((w & 0x7f800000u) == 0x7f800000u ? 0xffff0000u : 0u);
}
// (Once they have arrived.)  A product with a zero weight would make NaN of such a value: in tiles that some
// row does not see whole, they become zeros here (each wave those that it brought)
// and are added at the end to the rows that see them.  Returns whether there were any.
template <int KS, int W>
__device__ __forceinline__ bool clear_odd(const PrefillArgs& a, uint8_t* values) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    bool any = false;
    auto clear = [&](uint8_t* at) {
        u32x4_t w = *reinterpret_cast<const u32x4_t*>(at), bad;
#pragma unroll
        for (int j = 0; j < 4; ++j) bad[j] = odd_halves(w[j]);
        if ((bad[0] | bad[1] | bad[2] | bad[3]) == 0) return;
        any = true;
        *reinterpret_cast<u32x4_t*>(at) = w & ~bad;
    };
    if (a.vec_new) {
        for (int kb = wave >> 2; kb < KS; kb += W / 4) clear(values + 4096 * kb + 1024 * (wave & 3) + 16 * lane);
    } else {
        for (int n = threadIdx.x; n < 64 * 4 * KS; n += 64 * W) clear(values + (n >> 8) * 4096 + token_place(n & 63, (n >> 6) & 3));
    }
    return __ballot(any) != 0;
}

__device__ __forceinline__ float odd_or_zero(float x) { return fabsf(x) < INFINITY ? 0.0f : x; }

// ---- a wave's rows ----------------------------------------------------------
__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32, 64); }

// A wave's 32 rows: row lane & 31 is this lane's, with keys and channels 8 a + 4
// (lane >> 5) + (0..3) of every 32.
template <int KS>
struct Rows {
    static constexpr int NT = KS <= 4 ? 2 : 1;  // 32-key tiles whose scores are held at a time
    u32x4_t q[2 * KS];
    f32x16_t o[KS];
    float m, l;     // maximum, this lane's part of the weights' sum
    float above;    // a score so far over the maximum moves it

    __device__ __forceinline__ void clear() {
        m = l = 0.0f;
        above = -INFINITY;
#pragma unroll
        for (int i = 0; i < KS; ++i) o[i] = 0.0f;
    }
    // A score, `top` in this lane's keys, is over the maximum by more than 2^kLag in
    // some row of the wave: those rows' maximum moves (what other rows see
    // decides nothing).
    __device__ __forceinline__ void raise(float top) {
        top = fmaxf(top, other_half(top));
        if (!(top > above)) return;
        const float f = above == -INFINITY ? 0.0f : exp2_(m - top);
        m = top;
        above = top + kLag;
        l *= f;
#pragma unroll
        for (int i = 0; i < KS; ++i) o[i] *= f;
    }
    // Products of the rows with keys 32 t0 on of a tile, operands read kAhead ahead.
    template <int N>
    __device__ __forceinline__ void products(const uint8_t* keys, int t0, f32x16_t (&x)[N]) const {
        constexpr int kAll = 2 * KS * N, kMost = KS <= 4 ? 8 : KS <= 6 ? 4 : 2, kAhead = kAll < kMost ? kAll : kMost;
        const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
        const uint8_t* k0 = keys + token_place(c, g);
        const uint8_t* k1 = keys + token_place(c, 2 + g);
        auto key = [&](int n) {  // 32 keys n % N, channels 16 (n / N) on
            return *reinterpret_cast<const u32x4_t*>((n / N & 1 ? k1 : k0) + 4096 * (n / N >> 1) + 2048 * (t0 + n % N));
        };
        u32x4_t k[kAhead];
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kAhead; ++n) k[n] = key(n);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int n = 0; n < kAll; ++n) {
            if (n < N) x[n] = 0.0f;
            x[n % N] = mfma_bf16_32x32x16(k[n % kAhead], q[n / N], x[n % N]);
            if (n + kAhead < kAll) k[n % kAhead] = key(n + kAhead);
            __builtin_amdgcn_sched_barrier(0);
        }
    }
    // Only the first `limit` keys of the tile are seen; returns this lane's largest product with them.
    template <int N>
    __device__ __forceinline__ float mask(int t0, int limit, f32x16_t (&x)[N]) const {
        int left = limit - 32 * t0 - 4 * static_cast<int>((threadIdx.x & 63) >> 5);
        asm volatile("" : "+v"(left));  // (else made selects on every tile)
        float top = -INFINITY;
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                x[t][j] = 32 * t + 8 * (j >> 2) + (j & 3) < left ? x[t][j] : -INFINITY;
                top = fmaxf(top, x[t][j]);
            }
        return top;
    }
    // Products after the mask and with the maximum moved where they are far over it.
    template <int N>
    __device__ __forceinline__ void settle(const PrefillArgs& a, int t0, bool masked, int limit, f32x16_t (&x)[N]) {
        float top = -INFINITY;
        if (masked) {
            top = mask(t0, limit, x);
        } else {
#pragma unroll
            for (int t = 0; t < N; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) top = fmaxf(top, x[t][j]);
        }
        top *= a.scale2;
        if (__ballot(top > above)) raise(top);
    }
    // Products -> weights as operands.
    template <int N>
    __device__ __forceinline__ void weigh(const PrefillArgs& a, const f32x16_t (&x)[N], u32x4_t (&p)[2 * N]) {
#pragma unroll
        for (int t = 0; t < N; ++t)
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                f32x4_t y;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    y[j] = exp2_(__builtin_fmaf(x[t][4 * b + j], a.scale2, -m));
                    l += y[j];
                }
                p[2 * t + (b >> 1)][2 * (b & 1)] = pack_bf16x2(y[0], y[1]);
                p[2 * t + (b >> 1)][2 * (b & 1) + 1] = pack_bf16x2(y[2], y[3]);
            }
    }
    // O^T += V^T P^T of new tokens 32 t0 on of a tile.
    template <int N>
    __device__ __forceinline__ void add(const uint8_t* values, int t0, const u32x4_t (&p)[2 * N]) {
        const int lane = threadIdx.x & 63, g = lane >> 5;
        // a lane's address in a transposing read: token 4 g + (lane & 15) / 4, channels 16 (lane >> 4 & 1) + 4 (lane & 3) on
        const int tok = 4 * g + ((lane & 15) >> 2), chunk = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        const uint8_t* at[2] = {values + token_place(tok, chunk) + 8 * (lane & 1), values + token_place(tok + 8, chunk) + 8 * (lane & 1)};
#pragma unroll
        for (int s = 0; s < 2 * N; ++s)
#pragma unroll
            for (int i = 0; i < KS; ++i) {
                u32x2_t w[2];
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    w[e] = __builtin_bit_cast(u32x2_t, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                               (LHQ_LDS_AS s16x4_t*)(at[e] + 4096 * i + 1024 * (2 * t0 + s))));
                o[i] = mfma_bf16_32x32x16(u32x4_t{w[0][0], w[0][1], w[1][0], w[1][1]}, p[s], o[i]);
            }
    }
    // One page.  masked (the same for the wave): a row sees the first `limit` tokens of it.
    __device__ __forceinline__ void page(const uint8_t* keys, const uint8_t* values, const float* factors, bool masked,
                                         int limit) {
        const int lane = threadIdx.x & 63, c = lane & 31, g = lane >> 5;
#pragma unroll
        for (int t0 = 0; t0 < 2; t0 += NT) {
            f32x16_t x[NT];
            products(keys, t0, x);
            // scores less the maximum
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4_t f = *reinterpret_cast<const f32x4_t*>(factors + 32 * (t0 + t) + 8 * b + 4 * g);
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[t][4 * b + j] = __builtin_fmaf(x[t][4 * b + j], f[j], -m);
                }
            if (masked) {
                int left = limit - 32 * t0 - 4 * g;
                asm volatile("" : "+v"(left));  // (else made selects on every page)
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int j = 0; j < 16; ++j) x[t][j] = 32 * t + 8 * (j >> 2) + (j & 3) < left ? x[t][j] : -INFINITY;
            }
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) top = fmaxf(top, x[t][j]);
            if (__ballot(top > above - m)) {
                const float was = m;
                raise(top + m);
#pragma unroll
                for (int t = 0; t < NT; ++t) x[t] += was - m;
            }
            u32x4_t p[2 * NT];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int b = 0; b < 4; ++b) {
                    const f32x4_t f = *reinterpret_cast<const f32x4_t*>(factors + 64 + 32 * (t0 + t) + 8 * b + 4 * g);
                    f32x4_t y;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        y[j] = exp2_(x[t][4 * b + j]);
                        l += y[j];
                        y[j] *= f[j];
                    }
                    p[2 * t + (b >> 1)][2 * (b & 1)] = pack_bf16x2(y[0], y[1]);
                    p[2 * t + (b >> 1)][2 * (b & 1) + 1] = pack_bf16x2(y[2], y[3]);
                }
#pragma unroll
            for (int s = 0; s < 2 * NT; ++s)
#pragma unroll
                for (int i = 0; i < KS; ++i) {
                    const u32x4_t v = *reinterpret_cast<const u32x4_t*>(values + 4096 * i + value_place(c, 2 * (2 * t0 + s) + g));
                    o[i] = mfma_bf16_32x32x16(v, p[s], o[i]);
                }
        }
    }
    // One tile of new tokens, its products and then its weights.
    __device__ __forceinline__ void tile(const PrefillArgs& a, const uint8_t* keys, const uint8_t* values, bool masked, int limit) {
#pragma unroll
        for (int t0 = 0; t0 < 2; t0 += NT) {
            f32x16_t x[NT];
            u32x4_t p[2 * NT];
            products(keys, t0, x);
            settle(a, t0, masked, limit, x);
            weigh(a, x, p);
            add<NT>(values, t0, p);
        }
    }
};

// Rows of no sequence: zeros, by the workgroups that have no block (one at least).
__device__ void clear_rest(const PrefillArgs& a, int nth, int count) {
    const int lo = a.n_seqs ? kv_rows(a.offsets, 0, a.capacity).lo : 0;
    const int hi = a.n_seqs ? kv_rows(a.offsets, a.n_seqs - 1, a.capacity).hi : 0;
    const int64_t width = static_cast<int64_t>(a.group) * a.c.D, at = blockIdx.x * width;  // a kv head's part of a row
    for (int64_t row = nth; row < a.capacity; row += count) {
        if (row >= lo && row < hi) {
            row += (hi - 1 - row) / count * count;  // the last of this workgroup's that is inside
            continue;
        }
        uint16_t* to = a.out + row * a.heads * a.c.D + at;
        if (a.vec_out)
            for (int64_t n = 8 * threadIdx.x; n < width; n += 8 * blockDim.x) *reinterpret_cast<u32x4_t*>(to + n) = u32x4_t{0, 0, 0, 0};
        else
            for (int64_t n = threadIdx.x; n < width; n += blockDim.x) to[n] = 0;
    }
}

// MODE 0: no cache, 1: int8, 2: e4m3.  W waves, each with 32 rows.
template <int KS, int MODE, int W>
__global__ __launch_bounds__(64 * W, 2) void prefill_kernel(PrefillArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint8_t prefill_lds[];
    constexpr int kTile = KS * 4096, kRows = 32 * W;
    const uint32_t unit = blockIdx.y + blockIdx.z * gridDim.y;
    const Seq first_seq = seq_of(a, threadIdx.x & 63);
    const Found u = find_unit(a, first_seq, split_target(a, first_seq), unit, [](const Seq& q, int splits) { return static_cast<uint32_t>(q.blocks) * splits; });
    if (u.seq >= a.n_seqs) {
        if (a.clear_rest) clear_rest(a, u.nth, static_cast<int>(gridDim.y * gridDim.z - unit) + u.nth);
        return;
    }
    const int h = blockIdx.x, G = a.group, D = a.c.D, R = u.q.T * G, lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = u.nth % u.splits;
    const int block = u.q.blocks - 1 - u.nth / u.splits;  // those with the most keys first
    const int r0 = block * kRows, pages = (u.q.L + kKvPage - 1) / kKvPage;
    const int tiles = pages + (a.k_new ? ((min(r0 + kRows, R) - 1) / G) / kKvPage + 1 : 0);
    const int first = static_cast<int>(static_cast<int64_t>(tiles) * split / u.splits);
    const int end = static_cast<int>(static_cast<int64_t>(tiles) * (split + 1) / u.splits);
    auto place = [&](int t) { return prefill_lds + ((t - first) & 1) * 2 * kTile; };  // of tile t
    auto factors = [&](int t) { return reinterpret_cast<float*>(prefill_lds + 4 * kTile) + 128 * ((t - first) & 1); };
    int* odd = reinterpret_cast<int*>(prefill_lds + 4 * kTile + 1024);  // infinite or NaN values were cleared

    // this wave's rows: (token, query head) pairs of the kv head; past the last one, that again, which is not kept
    const bool some = r0 + 32 * wave < R;
    const int r = min(r0 + 32 * wave + (lane & 31), R - 1), token = r / G;
    const int low = __builtin_amdgcn_readlane(token, 0), high = __builtin_amdgcn_readlane(token, 31);
    PageLoad<KS, W> page_load;
    int ids = 0;
    auto page_id = [&](int t) {  // 64 entries of the block table at a time, one a lane
        if (((t - first) & 63) == 0) ids = t + lane < pages ? a.c.page(u.seq, t + lane) : -1;
        return __builtin_amdgcn_readlane(ids, (t - first) & 63);
    };
    bool there = false, next_there = false;  // whether a page is
    // the first tile of new tokens that some row of the block does not see whole
    const int partly = pages + (r0 / G + 1) / kKvPage;
    auto fetch_page = [&](int t) {
        const int id = page_id(t);
        next_there = id >= 0;
        if (next_there) page_load.load(a.c, id, h);
    };
    auto page_arrives = [&](int t) {
        there = next_there;
        if (there) page_load.template store<MODE == 2>(min(u.q.L - t * kKvPage, kKvPage), a.scale2, place(t), place(t) + kTile, factors(t));
    };
    NewTiles<KS, W> keys, values;
    const int page_end = MODE == 0 ? first : min(end, max(first, pages));
    {
        const int j0 = (page_end - pages) * kKvPage, past = (end - pages) * kKvPage;
        keys.aim(a.k_new, a.k_stride, u.q.lo, h, D, j0, past);
        values.aim(a.v_new, a.v_stride, u.q.lo, h, D, j0, past);
    }
    auto values_arrive = [&](int t, uint8_t* at) {
        if (t < end && t >= partly && clear_odd<KS, W>(a, at) && lane == 0) *odd = 1;
    };
    if (first < page_end) {
        fetch_page(first);
    } else {
        keys.fetch(a, u.q.T, place(first));
        values.fetch(a, u.q.T, place(first) + kTile);
    }
    Rows<KS> z;
    {
        const uint16_t* from = a.q + (u.q.lo + token) * a.q_stride + static_cast<int64_t>(h * G + r - token * G) * D;
#pragma unroll
        for (int i = 0; i < 2 * KS; ++i) z.q[i] = load_channels<KS == 1>(from, 16 * i + 8 * (lane >> 5), D);
    }
    z.clear();

    if (threadIdx.x == 0) *odd = 0;
    arrived();
    __syncthreads();
    if (first < page_end) page_arrives(first);
    else values_arrive(first, place(first) + kTile);
    __syncthreads();
    int t = first;
    if constexpr (MODE != 0) {
        for (; t < page_end; ++t) {
            uint8_t *now = place(t), *next = place(t + 1);
            if (t + 1 < page_end) {
                fetch_page(t + 1);
            } else {
                keys.fetch(a, u.q.T, next);
                values.fetch(a, u.q.T, next + kTile);
            }
            if (some && there) {
                const int left = min(u.q.L - t * kKvPage, kKvPage);
                z.page(now, now + kTile, factors(t), left < kKvPage, left);
            }
            if (t + 1 < page_end) {
                page_arrives(t + 1);
            } else {
                arrived();
                values_arrive(t + 1, next + kTile);
            }
            __syncthreads();
        }
    }
    // New tokens.
    auto masked = [&](int t) { return (t - pages) * kKvPage + kKvPage - 1 > low; };
    auto limit = [&](int t) { return token - (t - pages) * kKvPage + 1; };
    const int last = some ? min(end - 1, pages + high / kKvPage) : first - 1;  // the last tile that this wave sees
    uint8_t *now = place(t), *next = place(t + 1);
    for (; t < end; ++t) {
        keys.fetch(a, u.q.T, next);
        values.fetch(a, u.q.T, next + kTile);
        if (t <= last) z.tile(a, now, now + kTile, masked(t), limit(t));
        arrived();
        values_arrive(t + 1, next + kTile);
        __syncthreads();
        uint8_t* was = now;
        now = next;
        next = was;
    }

    if (!some) return;
    z.l += other_half(z.l);
    const int g = lane >> 5, mine = 32 * wave + (lane & 31);
    // Infinite or NaN values that a row sees: its sum is what they add to, whatever they
    // weigh.  A tile that some row does not see whole holds none of them any more; in the
    // others they left the products infinite or NaN (0 times infinity, where the weight or
    // a move of the maximum is 0).  get(channel) and set(channel, value) are this lane's
    // row's; all lanes of the wave call this.  Read in rows: a prompt of 16384 that holds
    // such values takes up to 9.6 ms, 5.9 with one token of them, 2.3 without.
    const bool some_odd = *odd != 0;
    float all = 0.0f;
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) all = __builtin_fmaf(z.o[i][j], 0.0f, all);
    auto settle_odd = [&](auto get, auto set) {
        const bool sums = fabsf(z.l) < INFINITY && r0 + mine < R, blank = z.l == 0.0f && all != 0.0f;
        if (!some_odd && __ballot(sums && all != 0.0f) == 0) return;
        const int from = (max(first, pages) - pages) * kKvPage, whole = (min(end, max(first, partly)) - pages) * kKvPage;
        const int past = min((end - pages) * kKvPage, token + 1);
        const uint16_t* rows = a.v_new + u.q.lo * a.v_stride + static_cast<int64_t>(h) * D;
        auto value = [&](int n, int ch) { return odd_or_zero(bf16_to_f32(rows[n * a.v_stride + ch])); };
        // those that all of the wave's rows see: a lane has channels lane, lane + 64, ..
        float seen[(KS + 1) / 2] = {};
        if (__ballot(sums && all != 0.0f) != 0) {
#pragma unroll 8
            for (int n = from; n < whole; ++n)
#pragma unroll
                for (int m = 0; m < (KS + 1) / 2; ++m) seen[m] += value(n, min(64 * m + lane, D - 1));
        }
#pragma unroll
        for (int m = 0; m < (KS + 1) / 2; ++m)
            for (int c = 0; c < min(64, D - 64 * m); ++c) {
                const int ch = 64 * m + c;
                const bool own = sums && (ch >> 2 & 1) == g;
                const float before = __shfl(seen[m], c, 64);
                float sum = own && (blank || !(fabsf(get(ch)) < INFINITY)) ? before : 0.0f;
                if (some_odd)
                    for (int n = max(from, whole); n < past; ++n) sum += value(n, ch);
                if (own && sum != 0.0f) set(ch, sum);
            }
    };
    if (u.splits > 1) {
        const bool kept = r0 + mine < R;
        const int64_t part = static_cast<int64_t>(h) * 4 * a.slots + u.parts + block * u.splits + split;
        const int64_t at = part * a.part_rows + mine;
        if (kept && g == 0) {
            a.ws_ml[2 * at] = z.l == 0.0f ? -INFINITY : z.m;
            a.ws_ml[2 * at + 1] = z.l;
        }
        float* to = a.ws_o + at * (32 * KS);
        if (kept) {
#pragma unroll
            for (int i = 0; i < KS; ++i)
#pragma unroll
                for (int b = 0; b < 4; ++b)
                    *reinterpret_cast<f32x4_t*>(to + 32 * i + 8 * b + 4 * g) =
                        f32x4_t{z.o[i][4 * b], z.o[i][4 * b + 1], z.o[i][4 * b + 2], z.o[i][4 * b + 3]};
        }
        settle_odd([&](int ch) { return to[ch]; }, [&](int ch, float y) { to[ch] = y; });
        return;
    }
    // Results to LDS (the tiles' place is free), from there in rows: the chunk j of row
    // c at place j ^ (c & kTurn).
    constexpr int kChunks = 4 * KS, kTurn = KS % 4 == 0 ? 15 : KS % 2 == 0 ? 7 : 3;
    uint8_t* rows = prefill_lds + wave * 32 * 16 * kChunks;
    auto chunk_at = [&](int row, int chunk) { return rows + 16 * (row * kChunks + (chunk ^ (row & kTurn))); };
    const float by = z.l == 0.0f ? 0.0f : 1.0f / z.l;  // nothing seen: zeros
#pragma unroll
    for (int i = 0; i < KS; ++i)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float y[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) y[j] = z.l == 0.0f ? 0.0f : z.o[i][4 * b + j] * by;
            *reinterpret_cast<u32x2_t*>(chunk_at(lane & 31, 4 * i + b) + 8 * g) = u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        }
    auto result = [&](int ch) { return reinterpret_cast<uint16_t*>(chunk_at(lane & 31, ch >> 3)) + (ch & 7); };
    settle_odd([&](int ch) { return bf16_to_f32(*result(ch)); }, [&](int ch, float y) { *result(ch) = f32_to_bf16(y); });
    const int out_row = token * a.heads + r - token * G;  // of (sequence, kv head)
    uint16_t* out = a.out + (static_cast<int64_t>(u.q.lo) * a.heads + h * G) * D;
    for (int n = lane; n < 32 * kChunks; n += 64) {
        const int row = n / kChunks, ch = 8 * (n % kChunks), left = D - ch;
        uint16_t* to = out + static_cast<int64_t>(__shfl(out_row, row, 64)) * D + ch;
        if (r0 + 32 * wave + row >= R) break;
        const u32x4_t w = *reinterpret_cast<const u32x4_t*>(chunk_at(row, n % kChunks));
        if (left <= 0) continue;
        if (a.vec_out) {
            *reinterpret_cast<u32x4_t*>(to) = w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (j < left) to[j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
        }
    }
}

// Joins the parts of split blocks in order of position: kJoinRows rows of a
// block a workgroup, four channels a thread at a time.  Bound by latency (finding
// the block, then the parts' loads), 5 us, and where there are many rows by memory: 14
// us for 32768 rows of 128 channels in two parts, 34 MB written and read again.
struct Joined {
    float top = -INFINITY, weight = 0.0f;
    f32x4_t sum = {0.f, 0.f, 0.f, 0.f};

    // The next N parts, on their way together: those of maxima and sums at ml, of products at o.
    template <int N>
    __device__ __forceinline__ void add(const float*& ml, int64_t ml_step, const float*& o, int64_t o_step) {
        float m[N], l[N];
        f32x4_t y[N];
#pragma unroll
        for (int k = 0; k < N; ++k) {
            m[k] = ml[0];
            l[k] = ml[1];
            y[k] = *reinterpret_cast<const f32x4_t*>(o);
            ml += ml_step;
            o += o_step;
        }
        float most = top;
#pragma unroll
        for (int k = 0; k < N; ++k) most = fmaxf(most, m[k]);
        if (most != -INFINITY) {
            const float f = exp2_(top - most);
            if (f != 0.0f) {
                weight *= f;
                sum *= f;
            } else {  // infinities and NaN have no weight that makes them nothing
                weight = odd_or_zero(weight);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] = odd_or_zero(sum[j]);
            }
            top = most;
        }
#pragma unroll
        for (int k = 0; k < N; ++k) {
            const float f = m[k] == -INFINITY ? 0.0f : exp2_(m[k] - most);
            if (f != 0.0f) {
                weight += l[k] * f;
                sum += y[k] * f;
            } else {
                weight += odd_or_zero(l[k]);
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[j] += odd_or_zero(y[k][j]);
            }
        }
    }
};
__device__ void join_rows(const PrefillArgs& a, const Found& u) {
    const int h = blockIdx.x, G = a.group, D = a.c.D, Dp = a.c.Dp(), R = u.q.T * G;
    const int chunks = a.block_rows / kJoinRows, block = u.nth / chunks, from = u.nth % chunks * kJoinRows;
    const int64_t part = static_cast<int64_t>(h) * 4 * a.slots + u.parts + block * u.splits;
    const int64_t ml_step = 2 * a.part_rows, o_step = static_cast<int64_t>(a.part_rows) * Dp;
    // thread n: the channels 4 n on of the rows, Dp a row
    const int row = from + static_cast<int>(threadIdx.x) / 32, r = block * a.block_rows + row;
    if (r >= R) return;
    const float* const ml0 = a.ws_ml + part * ml_step + 2 * row;
    const float* const o0 = a.ws_o + part * o_step + static_cast<int64_t>(row) * Dp;
    uint16_t* out = a.out + (static_cast<int64_t>(u.q.lo + r / G) * a.heads + h * G + r % G) * D;
    for (int ch = 4 * (threadIdx.x % 32); ch < D; ch += 128) {
        const float *ml = ml0, *o = o0 + ch;
        Joined z;
        int left = u.splits;
        for (; left >= 8; left -= 8) z.add<8>(ml, ml_step, o, o_step);
        if (left & 4) z.add<4>(ml, ml_step, o, o_step);
        if (left & 2) z.add<2>(ml, ml_step, o, o_step);
        if (left & 1) z.add<1>(ml, ml_step, o, o_step);
        const float by = 1.0f / z.weight;
        float y[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) y[j] = z.weight == 0.0f ? odd_or_zero(z.sum[j]) : z.sum[j] * by;
        if (a.vec_out) {
            *reinterpret_cast<u32x2_t*>(out + ch) = u32x2_t{pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3])};
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (ch + j < D) out[ch + j] = f32_to_bf16(y[j]);
        }
    }
}
__global__ __launch_bounds__(256) void prefill_join_kernel(PrefillArgs a) {
    auto chunks = [&](const Seq& q) { return static_cast<uint32_t>(q.T * a.group + kJoinRows - 1) / kJoinRows; };
    const Seq first = seq_of(a, threadIdx.x & 63);
    const int target = split_target(a, first);
    // (how many there are is known here alone; the grid is as many as run at once)
    for (uint32_t unit = blockIdx.y;;) {
        Found u = find_unit(a, first, target, unit, [&](const Seq& q, int splits) { return splits > 1 ? chunks(q) : 0u; });
        if (u.seq >= a.n_seqs) return;
        for (const int end = static_cast<int>(chunks(u.q)); u.nth < end; u.nth += gridDim.y, unit += gridDim.y) join_rows(a, u);
    }
}

// ---- host -------------------------------------------------------------------

int compute_units() {
    int dev = 0, n = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess || n <= 0) {
        (void)hipGetLastError();
        return 256;
    }
    return n;
}
// Rows of a workgroup.  256, eight waves, bring a tile to LDS half as often; 128 make
// two workgroups of a CU, which wait for different things, where LDS and registers
// hold two (without a cache, up to 128 channels), and leave less over at the end.
// Measured, 128 / 256 rows, 32 heads over 8: 2048 tokens 52 / 61 us, 16 prompts of up
// to 2048 212 / 219, 4096 tokens 154 / 142, 16384 2054 / 2019; 64 channels, 8192
// tokens 317 / 360; 96 channels 433 / 444; 16 heads over 4 of 192 483 / 384, of 256
// 931 / 602.  With a cache a page is made bf16 by all waves: 256.
int block_rows(int mode, int D, int n_seqs, int capacity, int heads) {
    const int64_t blocks = static_cast<int64_t>(capacity) * heads / 256, cus = compute_units();
    if (mode != 0) return 256;
    if (D > 128) return blocks >= cus ? 256 : 128;
    return D > 96 && blocks >= 2 * cus && capacity / std::max(n_seqs, 1) >= 4096 ? 256 : 128;
}
// Workgroups of a kv head that are on the chip at once: one a CU.  None (no splits)
// where the rows fill it four times over, or where splits would have too few tiles
// each.  Measured with splits / without: 128 tokens over 16384, 32 heads over 8, 67 /
// 579 us; 512 tokens of 64 heads over 32768 613 / 1141; 24 sequences, most of which
// decode, over up to 4096 172 / 203.
int want_slots(int block_rows, int capacity, int heads, int kv_heads, int64_t most_tiles) {
    const int cus = compute_units();
    const int64_t rows = static_cast<int64_t>(capacity) * (heads / kv_heads);
    if (rows / block_rows * kv_heads >= 4 * cus || most_tiles <= 2 * kLeastTiles) return 0;
    return std::max(1, cus / kv_heads);
}
int64_t part_bytes(int rows, int D) { return static_cast<int64_t>(rows) * (kv_padded(D) + 2) * 4; }
int part_rows(int block_rows, int capacity, int heads, int kv_heads) {
    return static_cast<int>(std::min<int64_t>(block_rows, static_cast<int64_t>(capacity) * (heads / kv_heads)));
}

dim3 unit_grid(int heads, int64_t units) {
    const unsigned y = static_cast<unsigned>(std::min<int64_t>(units, 32768));
    return dim3(heads, y, static_cast<unsigned>((units + y - 1) / y));
}

template <int KS, int MODE, int W>
int launch(const char* fn, const PrefillArgs& a, dim3 grid, hipStream_t s) {
    static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void*>(&prefill_kernel<KS, MODE, W>),
                                                       hipFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024);
    if (attr != hipSuccess) return set_error(LHQ_ERR_HIP, "%s: dynamic LDS attribute: %s", fn, hipGetErrorString(attr));
    prefill_kernel<KS, MODE, W><<<grid, 64 * W, lds_bytes<KS>(), s>>>(a);
    return check_launch(fn);
}

bool odd(const void* p, uintptr_t n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) != 0; }

int prefill(const char* fn, PrefillArgs a, int mode, int clear_rest, float scale, void* workspace, int64_t workspace_bytes, void* stream) {
    const int D = a.c.D, kv_heads = a.c.heads;
    LHQ_REQUIRE(a.heads > 0 && a.heads % kv_heads == 0, "%s: %d query heads are no multiple of %d kv heads", fn, a.heads, kv_heads);
    LHQ_SUPPORTED(a.heads <= 65535, "%s: %d query heads are over 65535", fn, a.heads);
    a.group = a.heads / kv_heads;
    a.block_rows = block_rows(mode, D, a.n_seqs, a.capacity, a.heads);
    LHQ_SUPPORTED(static_cast<int64_t>(a.capacity) * a.heads < INT32_MAX - a.block_rows, "%s: %d rows of %d heads are over 2^31", fn, a.capacity, a.heads);
    a.scale2 = scale * 1.4426950408889634f;  // weights are powers of two
    LHQ_REQUIRE(std::isfinite(a.scale2) && scale > 0.0f, "%s: scale %g is not positive and finite, also times log2 e", fn, scale);
    LHQ_REQUIRE((a.k_new == nullptr) == (a.v_new == nullptr), "%s: new keys without values, or values without keys", fn);
    LHQ_REQUIRE(a.q_stride >= static_cast<int64_t>(a.heads) * D, "%s: q rows of stride %lld are under %d heads of %d", fn,
                static_cast<long long>(a.q_stride), a.heads, D);
    LHQ_REQUIRE(!a.k_new || (a.k_stride >= static_cast<int64_t>(kv_heads) * D && a.v_stride >= static_cast<int64_t>(kv_heads) * D),
                "%s: new rows of strides %lld, %lld are under %d heads of %d", fn, static_cast<long long>(a.k_stride),
                static_cast<long long>(a.v_stride), kv_heads, D);
    LHQ_REQUIRE(workspace_bytes >= 0, "%s: negative workspace size", fn);
    LHQ_REQUIRE(!odd(workspace, 16), "%s: workspace must be 16-byte aligned", fn);
    if (a.capacity == 0 || (a.n_seqs == 0 && !clear_rest)) return LHQ_OK;
    if (a.n_seqs == 0) a.c.max_pages = 0;  // (no table and no lengths then)
    if (mode != 0)
        if (int st = kv_check_pointers(fn, a.c)) return st;
    LHQ_REQUIRE(a.q && a.offsets && a.out && (mode == 0 || a.n_seqs == 0 || a.lengths), "%s: null pointer", fn);
    if (mode == 0) LHQ_REQUIRE(a.k_new, "%s: null pointer", fn);
    // Workgroups read keys and values in no order with the writing of results; of the
    // queries each reads its own before it writes them.
    const int64_t q_width = static_cast<int64_t>(a.heads) * D, kv_width = static_cast<int64_t>(kv_heads) * D;
    auto meets = [&a, q_width](const uint16_t* rows, int64_t stride, int64_t width) {
        const int64_t out = reinterpret_cast<intptr_t>(a.out), x = reinterpret_cast<intptr_t>(rows);
        const int64_t ahead = out - x - 2 * width;  // the first row that ends behind out's start
        const int64_t row = ahead < 0 ? 0 : ahead / (2 * stride) + 1;
        return row < a.capacity && x + 2 * stride * row < out + 2 * q_width * a.capacity;
    };
    const bool in_place = a.q == a.out && (a.q_stride == q_width || a.capacity == 1);
    LHQ_REQUIRE((in_place || !meets(a.q, a.q_stride, q_width)) &&
                    (!a.k_new || (!meets(a.k_new, a.k_stride, kv_width) && !meets(a.v_new, a.v_stride, kv_width))),
                "%s: the result overlaps queries, new keys or new values", fn);
    if (a.c.num_pages == 0) a.c.max_pages = 0;
    a.vec_new = D % 8 == 0 && !odd(a.k_new, 16) && !odd(a.v_new, 16) && a.k_stride % 8 == 0 && a.v_stride % 8 == 0 &&
                a.k_stride < (1 << 24) && a.v_stride < (1 << 24);
    a.vec_out = D % 8 == 0 && !odd(a.out, 16);
    a.clear_rest = clear_rest != 0;
    const int64_t tiles = a.c.max_pages + (a.k_new ? (static_cast<int64_t>(a.capacity) + kKvPage - 1) / kKvPage : 0);
    a.part_rows = part_rows(a.block_rows, a.capacity, a.heads, kv_heads);
    // as many parts as there is room for, four a slot
    const int64_t room = workspace ? workspace_bytes / part_bytes(a.part_rows, D) / (4 * kv_heads) : 0;
    a.slots = static_cast<int>(std::min<int64_t>(want_slots(a.block_rows, a.capacity, a.heads, kv_heads, tiles), room));
    const int64_t parts = static_cast<int64_t>(kv_heads) * 4 * a.slots;
    a.ws_o = static_cast<float*>(workspace);
    a.ws_ml = a.ws_o + parts * a.part_rows * kv_padded(D);
    const int64_t rows = static_cast<int64_t>(a.capacity) * a.group;
    const int64_t units = rows / a.block_rows + std::min(a.n_seqs, a.capacity) + 4 * a.slots + (clear_rest ? 1 : 0);
    LHQ_SUPPORTED(units * kv_heads < INT32_MAX / (2 * a.block_rows), "%s: %lld query blocks of %d heads are over the grid", fn,
                  static_cast<long long>(units), kv_heads);
    const dim3 grid = unit_grid(kv_heads, units);
    const hipStream_t s = as_stream(stream);
    int st = LHQ_OK;
    auto go = [&](auto ks) {
        st = mode == 1 ? launch<ks(), 1, 8>(fn, a, grid, s) : mode == 2 ? launch<ks(), 2, 8>(fn, a, grid, s) :
             a.block_rows == 128 ? launch<ks(), 0, 4>(fn, a, grid, s) : launch<ks(), 0, 8>(fn, a, grid, s);
    };
    switch (kv_padded(D) / 32) {
        case 1: go(std::integral_constant<int, 1>{}); break;
        case 2: go(std::integral_constant<int, 2>{}); break;
        case 3: go(std::integral_constant<int, 3>{}); break;
        case 4: go(std::integral_constant<int, 4>{}); break;
        case 5: go(std::integral_constant<int, 5>{}); break;
        case 6: go(std::integral_constant<int, 6>{}); break;
        case 7: go(std::integral_constant<int, 7>{}); break;
        default: go(std::integral_constant<int, 8>{}); break;
    }
    if (st != LHQ_OK || a.slots == 0) return st;
    // (a split block has two parts or more: less than two a slot)
    const int join_units = static_cast<int>(std::min<int64_t>(static_cast<int64_t>(2 * a.slots) * (a.block_rows / kJoinRows), 2048 / kv_heads + 1));
    prefill_join_kernel<<<dim3(kv_heads, join_units), 256, 0, s>>>(a);
    return check_launch(fn);
}

}  // namespace
}  // namespace lhq

using namespace lhq;

extern "C" {

int64_t lhq_prefill_workspace_bytes(int n_seqs, int row_capacity, int n_heads, int n_kv_heads, int head_dim) {
    if (n_seqs <= 0 || row_capacity <= 0 || n_kv_heads <= 0 || n_kv_heads > 65535 || n_heads <= 0 || n_heads % n_kv_heads != 0 ||
        head_dim <= 0 || head_dim > kKvMaxDim)
        return 0;
    int64_t most = 0;
    for (int rows : {128, 256})
        most = std::max(most, static_cast<int64_t>(n_kv_heads) * 4 * want_slots(rows, row_capacity, n_heads, n_kv_heads, INT64_MAX) *
                                  part_bytes(part_rows(rows, row_capacity, n_heads, n_kv_heads), head_dim));
    return most;
}

int lhq_attn_prompt_bf16(const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride, const uint16_t* v,
                         int64_t v_stride, const int32_t* offsets, uint16_t* out, int n_seqs, int row_capacity,
                         int n_heads, int n_kv_heads, int head_dim, float scale, int clear_rest,
                         void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "attn_prompt_bf16";
    const KvCache c{nullptr, nullptr, nullptr, nullptr, nullptr, 0, 0, n_kv_heads, head_dim};
    if (int st = kv_check(fn, c, LHQ_KV_INT8, n_seqs, row_capacity)) return st;
    const PrefillArgs a{q, q_stride, k, k_stride, v, v_stride, offsets, nullptr, c, out, n_seqs, row_capacity, n_heads};
    return prefill(fn, a, 0, clear_rest, scale, workspace, workspace_bytes, stream);
}

int lhq_kv_prefill_bf16(const uint16_t* q, int64_t q_stride, const uint16_t* k_new, int64_t k_stride,
                        const uint16_t* v_new, int64_t v_stride, const int32_t* offsets, const int32_t* lengths,
                        const int32_t* block_table, const uint8_t* k_codes, const float* k_scales,
                        const uint8_t* v_codes, const float* v_scales, uint16_t* out, int format, int n_seqs,
                        int row_capacity, int max_pages, int num_pages, int n_heads, int n_kv_heads, int head_dim,
                        float scale, int clear_rest, void* workspace, int64_t workspace_bytes, void* stream) {
    const char* fn = "kv_prefill_bf16";
    const KvCache c{const_cast<uint8_t*>(k_codes), const_cast<float*>(k_scales), const_cast<uint8_t*>(v_codes),
                    const_cast<float*>(v_scales), block_table, max_pages, num_pages, n_kv_heads, head_dim};
    if (int st = kv_check(fn, c, format, n_seqs, row_capacity)) return st;
    const PrefillArgs a{q, q_stride, k_new, k_stride, v_new, v_stride, offsets, lengths, c, out, n_seqs, row_capacity, n_heads};
    return prefill(fn, a, format == LHQ_KV_FP8 ? 2 : 1, clear_rest, scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
