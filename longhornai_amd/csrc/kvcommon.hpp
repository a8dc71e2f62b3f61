// kvcommon.hpp -- the paged 8-bit key/value cache: layout, argument checks and
// the device-side list of (sequence, page) tiles that its kernels walk.
//
// A page holds kKvPage = 64 tokens of every kv head, one byte a value, with
// Dp = head_dim rounded up to 32 (the k extent of one 16x16x32 MFMA):
//   keys    [page][head][64 tokens][Dp]   a token's row is contiguous
//   values  [page][head][Dp][64 tokens]   a channel's row holds the page's
//     tokens in kv_slot order, so that 8 adjacent bytes are the k elements
//     that one lane of a 16x16x32 MFMA takes from two score tiles that the
//     lane itself holds (see kvattn.hip)
//   scales  [page][head][64] fp32, for keys and for values
// Values past head_dim in a row are zero codes.
#pragma once

#include "common.hpp"

namespace lhq {

constexpr int kKvPage = 64;
constexpr int kKvMaxDim = 256;
constexpr int kKvMaxNew = 64;  // new tokens of one sequence: a 64-bit mask each

__host__ __device__ constexpr int kv_padded(int D) { return (D + 31) / 32 * 32; }
// Place of page token t in a value row: lane group g = (t >> 2) & 3 owns bytes
// 16g .. 16g+15: token 32s + 16h + 4g + r at 16g + 8s + 4h + r.
__host__ __device__ constexpr int kv_slot(int t) {
    return 16 * ((t >> 2) & 3) + 8 * (t >> 5) + 4 * ((t >> 4) & 1) + (t & 3);
}

struct KvCache {
    uint8_t* k;
    float* ks;
    uint8_t* v;
    float* vs;
    const int32_t* table;  // [n_seqs][max_pages]
    int max_pages, num_pages, heads, D;
    __host__ __device__ int Dp() const { return kv_padded(D); }
    // The pool page that holds page p of sequence s, or -1.
    __device__ int page(int s, int64_t p) const {
        if (p < 0 || p >= max_pages) return -1;
        const int id = table[static_cast<int64_t>(s) * max_pages + p];
        return id >= 0 && id < num_pages ? id : -1;
    }
    __device__ int64_t code_base(int page, int h) const {
        return (static_cast<int64_t>(page) * heads + h) * kKvPage * Dp();
    }
    __device__ int64_t scale_base(int page, int h) const {
        return (static_cast<int64_t>(page) * heads + h) * kKvPage;
    }
};

// Rows [lo, hi) of sequence s by the offsets table, inside [0, capacity]
// whatever the table holds.
struct KvRows { int lo, hi; };
__device__ __forceinline__ KvRows kv_rows(const int32_t* offsets, int s, int capacity) {
    const int lo = min(max(offsets[s], 0), capacity);
    return {lo, min(max(offsets[s + 1], lo), capacity)};
}

// Sums over the lanes up to each one, of numbers under 2^32, held at 2^32 - 1.
__device__ __forceinline__ uint32_t kv_scan(uint32_t x) {
#define LHQ_SCAN_STEP(ctrl, rows)                                                                           \
    x = __builtin_elementwise_add_sat(                                                                      \
        x, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), ctrl, rows, 0xf, false)))
    LHQ_SCAN_STEP(0x111, 0xf);  // row_shr:1, 2, 4, 8: within 16 lanes
    LHQ_SCAN_STEP(0x112, 0xf);
    LHQ_SCAN_STEP(0x114, 0xf);
    LHQ_SCAN_STEP(0x118, 0xf);
    LHQ_SCAN_STEP(0x142, 0xa);  // row_bcast:15 to rows 1 and 3
    LHQ_SCAN_STEP(0x143, 0xc);  // row_bcast:31 to the upper half
#undef LHQ_SCAN_STEP
    return x;
}

// Maximum over 1 << LB adjacent lanes (8, 16 or 32), the same in all of them.
template <int LB, typename T, typename Max>
__device__ __forceinline__ T row_max(T m, Max max_of) {
#define LHQ_MAX_STEP(ctrl)                                                                               \
    m = max_of(m, __builtin_bit_cast(T, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, m), ctrl, \
                                                                    0xf, 0xf, false)))
    LHQ_MAX_STEP(0xB1);   // quad_perm 1, 0, 3, 2
    LHQ_MAX_STEP(0x4E);   // quad_perm 2, 3, 0, 1
    LHQ_MAX_STEP(0x141);  // row_half_mirror: the other quad of 8 lanes
    if constexpr (LB >= 4) LHQ_MAX_STEP(0x140);  // row_mirror: the other half of 16
#undef LHQ_MAX_STEP
    if constexpr (LB >= 5) m = max_of(m, __shfl_xor(m, 16, 64));
    return m;
}

// The unit with number `unit` in the list that has count(s) units of sequence
// 0, then those of sequence 1, ...: its sequence, its number within it and the
// lane that counted the sequence (what count left in that lane's variables is
// the sequence's), the same in every lane; seq = n_seqs past the end of the
// list.  Each wave scans the sequences by itself, 64 at a time (no barrier; a
// batch of 64 is one step).  A sum held at 2^32 - 1 is over every unit.
struct KvUnit { int seq, nth, lane; };
template <typename Count>
__device__ __forceinline__ KvUnit kv_find_unit(uint32_t unit, int n_seqs, Count count) {
    const int lane = threadIdx.x & 63;
    for (int base = 0; base < n_seqs; base += 64) {
        const int s = base + lane;
        const uint32_t sum = kv_scan(s < n_seqs ? count(s) : 0u);
        const uint64_t over = __ballot(sum > unit);
        if (over) {
            const int l = __builtin_ctzll(over);
            const uint32_t before = l > 0 ? __builtin_amdgcn_readlane(sum, l - 1) : 0u;
            return {base + l, static_cast<int>(unit - before), l};
        }
        unit -= __builtin_amdgcn_readlane(sum, 63);
    }
    return {n_seqs, 0, 0};
}

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

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

// Checks that all entry points of the cache share; `fn` names the caller.
inline int kv_check(const char* fn, const KvCache& c, int format, int n_seqs, int row_capacity) {
    LHQ_REQUIRE(format == LHQ_KV_INT8 || format == LHQ_KV_FP8, "%s: unknown cache format %d", fn, format);
    LHQ_REQUIRE(n_seqs >= 0 && row_capacity >= 0, "%s: bad counts (%d sequences, %d rows)", fn, n_seqs, row_capacity);
    LHQ_REQUIRE(c.max_pages >= 0 && c.num_pages >= 0 && c.heads > 0 && c.D > 0,
                "%s: bad cache dims (pages %d of %d, heads %d, head_dim %d)", fn, c.max_pages, c.num_pages, c.heads,
                c.D);
    LHQ_SUPPORTED(c.D <= kKvMaxDim, "%s: head_dim %d is over %d", fn, c.D, kKvMaxDim);
    LHQ_SUPPORTED(c.heads <= 65535, "%s: %d kv heads are over 65535", fn, c.heads);
    LHQ_SUPPORTED(static_cast<int64_t>(c.max_pages) * kKvPage < (int64_t{1} << 31),
                  "%s: sequences of 2^31 tokens", fn);
    return LHQ_OK;
}
// The pointers, wanted once there is something to do.
inline int kv_check_pointers(const char* fn, const KvCache& c) {
    LHQ_REQUIRE(c.num_pages == 0 || (c.k && c.ks && c.v && c.vs), "%s: null cache pointer", fn);
    LHQ_REQUIRE(c.max_pages == 0 || c.table, "%s: null block table", fn);
    auto odd = [](const void* p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) != 0; };
    LHQ_REQUIRE(!odd(c.k, 16) && !odd(c.v, 16), "%s: cache codes must be 16-byte aligned", fn);
    LHQ_REQUIRE(!odd(c.ks, 16) && !odd(c.vs, 16), "%s: cache scales must be 16-byte aligned", fn);
    return LHQ_OK;
}

}  // namespace lhq
