// kvplan.hip -- a serving step's tables from the requests' lengths, for gfx950:
// pages handed back and out, offsets, positions and cache slots of the new
// rows (lhq_kv_plan, lhq_kv_plan_owned).
//
// The free pages are a stack.  Pages of sequences that are over are pushed in
// order of sequence and page, then those of new tokens are popped in that order
// (all pushes come first, whatever the order of sequences), so every entry's
// place follows from prefix sums and no atomic decides anything.  Which entries of
// its row a sequence has pages in follows from its length, or is counted in `owned`:
// those of rejected tokens, and those granted before the stack ran out, are the
// sequence's then though its length does not reach them.  The sums run
// over all sequences, so one workgroup does them; the rows, which only read
// what it wrote, are done by it too where they are few and by a launch of their
// own where they are many.  Bound by latency, a chain of loads and scans: 256 decoding
// sequences 5.9 us (a pass 12.7, the host's); 48 prompts, 40243 rows, 12.1 to 12.6 and
// 4.0, most of it the pages of those sequences, which are all one wave's: a wave serves
// the 64 sequences beside one another of its lanes, one after the other.
#include <algorithm>

#include "kvcommon.hpp"

namespace lhq {
namespace {

constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;
// Rows that the planning workgroup does itself: four a thread.
constexpr int kPlanRows = 4 * kPlanThreads;
constexpr int kRowThreads = 256;

struct PlanArgs {
    const int32_t* lengths;
    const int32_t* new_tokens;
    const uint64_t* tree;
    const int32_t* left;
    int32_t* left_out;
    int32_t* free_pages;
    int32_t* table;
    int32_t* offsets;
    int32_t* positions;
    int64_t* slots;
    int32_t* owned;  // entries of its row that a sequence has, or null: those of its tokens
    int n_seqs, capacity, max_pages, num_pages;
};

// Tokens that a sequence holds, as its table row can name them.
__device__ __forceinline__ int held(const PlanArgs& a, int s) {
    return static_cast<int>(min<int64_t>(max(a.lengths[s], 0), static_cast<int64_t>(a.max_pages) * kKvPage));
}
__device__ __forceinline__ int owned(const PlanArgs& a, int s) { return min(max(a.owned[s], 0), a.max_pages); }
__device__ __forceinline__ int pages_of(int64_t tokens) { return static_cast<int>((tokens + kKvPage - 1) / kKvPage); }

// Sums over the threads before this one (below 2^32 in all, else held there);
// `total` is that of all threads.  lds: a place that no thread reads any more.
__device__ __forceinline__ uint32_t scan_before(uint32_t x, uint32_t* lds, uint32_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t upto = kv_scan(x);
    if (lane == 63) lds[wave] = upto;
    __syncthreads();
    const uint32_t waves = kv_scan(lane < kPlanWaves ? lds[lane] : 0u);
    total = __builtin_amdgcn_readlane(waves, kPlanWaves - 1);
    const uint32_t before = wave > 0 ? __builtin_amdgcn_readlane(waves, wave - 1) : 0u;
    return __builtin_elementwise_add_sat(before, upto - x);
}
// f(lane, its x) for each lane of the wave that has x > 0, in order.
template <typename F>
__device__ __forceinline__ void each_lane(int x, F f) {
    for (uint64_t some = __ballot(x > 0); some; some &= some - 1) {
        const int l = __builtin_ctzll(some);
        f(l, __builtin_amdgcn_readlane(x, l));
    }
}

// Row r: the last sequence whose offset is not over r owns it, if its rows
// reach that far.
template <typename Length>
__device__ __forceinline__ void plan_row(const PlanArgs& a, const int32_t* offsets, Length length_of, int r) {
    int lo = 0, hi = a.n_seqs;  // offsets[lo] <= r (offsets[0] = 0), offsets[hi] > r or hi = n_seqs
    while (hi - lo > 1) {
        const int mid = lo + (hi - lo) / 2;
        if (offsets[mid] <= r) lo = mid;
        else hi = mid;
    }
    int position = -1;
    int64_t slot = -1;
    if (a.n_seqs > 0 && r < offsets[lo + 1]) {
        const int first = offsets[lo], length = length_of(lo), i = r - first;
        const int64_t at = static_cast<int64_t>(length) + i, p = at / kKvPage;
        int64_t depth = i;
        if (a.tree) {  // ancestors of a drafted token, itself among them
            const int T = min(offsets[lo + 1] - first, 64);
            const uint64_t own = T == 64 ? ~uint64_t{0} : (uint64_t{1} << T) - 1;
            depth = max(static_cast<int>(__popcll(a.tree[r] & own)) - 1, 0);
        }
        position = static_cast<int>(min<int64_t>(length + depth, INT32_MAX));
        const int page = p < a.max_pages ? a.table[static_cast<int64_t>(lo) * a.max_pages + p] : -1;
        if (page >= 0 && page < a.num_pages) slot = static_cast<int64_t>(page) * kKvPage + at % kKvPage;
    }
    a.positions[r] = position;
    if (a.slots) a.slots[r] = slot;
}

// ROWS: the rows too (n_seqs <= kPlanThreads, capacity <= kPlanRows).
template <bool ROWS>
__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanArgs a) {
    __shared__ uint32_t sums[3][kPlanWaves];
    __shared__ int offs[kPlanThreads + 1], lengths[kPlanThreads];
    const int lane = threadIdx.x & 63, wave_first = static_cast<int>(threadIdx.x) - lane;
    uint32_t have = static_cast<uint32_t>(min(max(a.left[0], 0), a.num_pages));  // pages on the stack
    // the first 1024 sequences' lengths and new tokens stay in registers
    auto length_of = [&](int s) { return s < a.n_seqs ? held(a, s) : 0; };
    auto new_of = [&](int s) { return s < a.n_seqs ? a.new_tokens[s] : 0; };
    const int length0 = length_of(threadIdx.x), new0 = new_of(threadIdx.x);

    // Pages of sequences that are over, 1024 sequences at a time, a wave its own 64.
    for (int base = 0; base < a.n_seqs; base += kPlanThreads) {
        const int s = base + static_cast<int>(threadIdx.x);
        const int n = base ? new_of(s) : new0;
        const int had = n >= 0 ? 0 : a.owned ? owned(a, s) : pages_of(base ? length_of(s) : length0);
        if (!__syncthreads_or(had)) continue;
        auto entry = [&](int l, int p, int pages) {
            const int id = p < pages ? a.table[static_cast<int64_t>(base + wave_first + l) * a.max_pages + p] : -1;
            return id < a.num_pages ? id : -1;
        };
        int valid = 0;  // entries of this lane's sequence that are pages
        each_lane(had, [&](int l, int pages) {
            int sum = 0;
            for (int p = lane; p - lane < pages; p += 64) sum += __popcll(__ballot(entry(l, p, pages) >= 0));
            if (lane == l) valid = sum;
        });
        uint32_t total;
        const uint32_t before = scan_before(static_cast<uint32_t>(valid), sums[0], total);
        each_lane(had, [&](int l, int pages) {
            int64_t at = static_cast<int64_t>(have) + static_cast<uint32_t>(__builtin_amdgcn_readlane(before, l));
            for (int p = lane; p - lane < pages; p += 64) {
                const int id = entry(l, p, pages);
                const uint64_t all = __ballot(id >= 0);
                const int64_t to = at + __popcll(all & ((uint64_t{1} << lane) - 1));
                // (more pages than there are: some were handed back twice; the stack keeps to its size)
                if (id >= 0 && to < a.num_pages) a.free_pages[to] = id;
                at += __popcll(all);
            }
        });
        have = min(__builtin_elementwise_add_sat(have, total), static_cast<uint32_t>(a.num_pages));
    }
    __syncthreads();  // (what is on the stack now is seen by all)

    // Offsets, and the new tokens' pages.
    uint32_t rows = 0, asked = 0;
    for (int base = 0; base < a.n_seqs; base += kPlanThreads) {
        const int s = base + static_cast<int>(threadIdx.x);
        const int length = base ? length_of(s) : length0;
        const uint32_t want = static_cast<uint32_t>(max(base ? new_of(s) : new0, 0)), cap = static_cast<uint32_t>(a.capacity);
        uint32_t total;
        const uint32_t before = __builtin_elementwise_add_sat(rows, scan_before(want, sums[1], total));
        const int lo = static_cast<int>(min(before, cap)), hi = static_cast<int>(min(__builtin_elementwise_add_sat(before, want), cap));
        rows = __builtin_elementwise_add_sat(rows, total);
        int from = pages_of(length), takes = 0;
        if (s < a.n_seqs) {
            a.offsets[s + 1] = hi;
            if (s == 0) a.offsets[0] = 0;
            if constexpr (ROWS) {
                offs[s + 1] = hi;
                if (s == 0) offs[0] = 0;
                lengths[s] = length;
            }
            if (a.owned) from = max(from, owned(a, s));
            if (hi > lo) takes = max(min(pages_of(static_cast<int64_t>(length) + hi - lo), a.max_pages) - from, 0);
        }
        const uint32_t mine = __builtin_elementwise_add_sat(asked, scan_before(static_cast<uint32_t>(takes), sums[2], total));
        asked = __builtin_elementwise_add_sat(asked, total);
        if (a.owned && s < a.n_seqs) {
            if ((base ? new_of(s) : new0) < 0) a.owned[s] = 0;
            else if (takes > 0 && mine < have) a.owned[s] = from + static_cast<int>(min(static_cast<uint32_t>(takes), have - mine));
        }
        auto take = [&](int seq, int p, uint32_t nth) {
            a.table[static_cast<int64_t>(seq) * a.max_pages + p] = nth < have ? a.free_pages[have - 1 - nth] : -1;
        };
        // one page by the sequence's lane, more by its wave
        if (takes == 1) take(s, from, mine);
        each_lane(takes > 1 ? takes : 0, [&](int l, int pages) {
            const int p0 = __builtin_amdgcn_readlane(from, l);
            const uint32_t nth = __builtin_amdgcn_readlane(mine, l);
            for (int p = lane; p < pages; p += 64) take(base + wave_first + l, p0 + p, __builtin_elementwise_add_sat(nth, static_cast<uint32_t>(p)));
        });
    }
    __syncthreads();  // (left may be left_out: everyone has read it)
    if (threadIdx.x == 0) {
        a.left_out[0] = static_cast<int32_t>(have - min(have, asked));
        a.left_out[1] = static_cast<int32_t>(min(asked - min(have, asked), 0x7fffffffu));
        if (a.n_seqs == 0) a.offsets[0] = 0;
    }
    if constexpr (ROWS) {
        for (int r = threadIdx.x; r < a.capacity; r += kPlanThreads) plan_row(a, offs, [&](int s) { return lengths[s]; }, r);
    }
}

__global__ __launch_bounds__(kRowThreads) void kv_plan_rows_kernel(PlanArgs a) {
    const int r = static_cast<int>(blockIdx.x * kRowThreads + threadIdx.x);
    if (r < a.capacity) plan_row(a, a.offsets, [&](int s) { return held(a, s); }, r);
}

}  // namespace
}  // namespace lhq

using namespace lhq;

namespace {

int plan(const char* fn, const PlanArgs& a, void* stream) {
    LHQ_REQUIRE(a.n_seqs >= 0 && a.capacity >= 0, "%s: bad counts (%d sequences, %d rows)", fn, a.n_seqs, a.capacity);
    LHQ_REQUIRE(a.max_pages >= 0 && a.num_pages >= 0, "%s: bad page counts (%d of a sequence, %d in all)", fn, a.max_pages,
                a.num_pages);
    LHQ_SUPPORTED(static_cast<int64_t>(a.max_pages) * kKvPage < (int64_t{1} << 31), "%s: sequences of 2^31 tokens", fn);
    LHQ_SUPPORTED(a.capacity <= INT32_MAX - kPlanRows && a.n_seqs <= INT32_MAX - kPlanThreads,
                  "%s: %d rows of %d sequences are over 2^31 - 4097 or 2^31 - 1025", fn, a.capacity, a.n_seqs);
    LHQ_REQUIRE(a.left && a.left_out && a.offsets, "%s: null pointer", fn);
    LHQ_REQUIRE(a.n_seqs == 0 || (a.lengths && a.new_tokens), "%s: null lengths", fn);
    LHQ_REQUIRE(a.num_pages == 0 || a.free_pages, "%s: null list of free pages", fn);
    LHQ_REQUIRE(a.n_seqs == 0 || a.max_pages == 0 || a.table, "%s: null block table", fn);
    LHQ_REQUIRE(a.capacity == 0 || a.positions, "%s: null positions", fn);
    const hipStream_t s = as_stream(stream);
    if (a.n_seqs <= kPlanThreads && a.capacity <= kPlanRows) {
        kv_plan_kernel<true><<<1, kPlanThreads, 0, s>>>(a);
        return check_launch(fn);
    }
    kv_plan_kernel<false><<<1, kPlanThreads, 0, s>>>(a);
    if (int st = check_launch(fn)) return st;
    if (a.capacity == 0) return LHQ_OK;
    kv_plan_rows_kernel<<<(a.capacity + kRowThreads - 1) / kRowThreads, kRowThreads, 0, s>>>(a);
    return check_launch(fn);
}

}  // namespace

extern "C" {

int lhq_kv_plan(const int32_t* lengths, const int32_t* new_tokens, const uint64_t* tree, const int32_t* left,
                int32_t* left_out, int32_t* free_pages, int32_t* block_table, int32_t* offsets, int32_t* positions,
                int64_t* slots, int n_seqs, int row_capacity, int max_pages, int num_pages, void* stream) {
    return plan("kv_plan", {lengths, new_tokens, tree, left, left_out, free_pages, block_table, offsets, positions, slots,
                            nullptr, n_seqs, row_capacity, max_pages, num_pages}, stream);
}

int lhq_kv_plan_owned(const int32_t* lengths, const int32_t* new_tokens, const uint64_t* tree, const int32_t* left,
                      int32_t* left_out, int32_t* free_pages, int32_t* block_table, int32_t* owned, int32_t* offsets,
                      int32_t* positions, int64_t* slots, int n_seqs, int row_capacity, int max_pages, int num_pages,
                      void* stream) {
    const char* fn = "kv_plan_owned";
    LHQ_REQUIRE(n_seqs <= 0 || owned, "%s: null counts of owned pages", fn);
    return plan(fn, {lengths, new_tokens, tree, left, left_out, free_pages, block_table, offsets, positions, slots, owned,
                     n_seqs, row_capacity, max_pages, num_pages}, stream);
}

}  // extern "C"
