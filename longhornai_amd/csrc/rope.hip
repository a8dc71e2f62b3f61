// rope.hip -- queries and keys turned by their positions, with the RMS norm of
// each head in the same pass where a layer has one, for gfx950.
//
//   y = x / sqrt(mean(x^2) + eps) * w             of a head (no weight: y = x)
//   (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin) * gain
// for each pair (a, b) of the first rot_dim channels: (i, i + rot_dim / 2), or
// (2i, 2i + 1) when interleaved; the other channels are y.  fp32 from the input
// to one rounding at the end.
//
// The angle of a pair is position * turns[i], turns[i] being the fraction of a
// full turn per position in units of 2^-64: the product modulo 2^64 is the angle
// itself, whole turns gone, exact for every position (position * frequency in
// fp32 is off by 2^-24 of the angle, 0.008 rad at position 131072).  Its nearest
// quarter turn comes off as an integer too, and what is left, at most pi / 4,
// goes through the Taylor series of sine and cosine.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "kvcommon.hpp"

namespace lhq {
namespace {

constexpr int kRopeThreads = 256;

template <typename T>
struct RopeArgs {
    const T* x[2];         // queries, keys
    int64_t in_stride[2];
    T* y[2];
    int64_t out_stride[2];
    const T* weight[2];
    int heads[2];
    const int32_t* positions;
    const uint64_t* turns;
    int n_rows, D, rot;
    float eps, gain;
};

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(uint16_t x) { return bf16_to_f32(x); }
__device__ __forceinline__ void put(float* p, float x) { *p = x; }
__device__ __forceinline__ void put(uint16_t* p, float x) { *p = f32_to_bf16(x); }

// cos and sin of an angle in units of 2^-64 turns.
__device__ __forceinline__ void turn(uint64_t angle, float& c, float& s) {
    const uint32_t top = static_cast<uint32_t>(angle >> 32);  // 2^-32 turns: 1.5e-9 rad
    const uint32_t quarter = (top + 0x20000000u) >> 30;
    const float x = static_cast<float>(static_cast<int32_t>(top - (quarter << 30))) * 1.4629180792671596e-9f;  // 2 pi / 2^32
    const float x2 = x * x;
    // to x^9 and x^10: the next terms are under 2e-9 and 2e-10 of pi / 4's
    const float sx = x + x * x2 * (-1.6666667e-1f + x2 * (8.3333333e-3f + x2 * (-1.9841270e-4f + x2 * 2.7557319e-6f)));
    const float cx = 1.0f + x2 * (-0.5f + x2 * (4.1666667e-2f + x2 * (-1.3888889e-3f + x2 * (2.4801587e-5f + x2 * -2.7557319e-7f))));
    const float a = quarter & 1 ? sx : cx, b = quarter & 1 ? cx : sx;
    c = (quarter + 1) & 2 ? -a : a;
    s = quarter & 2 ? -b : b;
}

// A wave a (row, head): lane l has pairs l, l + 64 of the channels; those past
// rot_dim go in twos that are not turned.  For the heads that rope_vec_kernel does not
// take: of an odd size (75 channels: 402 us for 32768 rows of 32 and 8 heads in bf16,
// 1 TB/s), or of more than 128 channels whose pairs are cut into no vectors.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(kRopeThreads) void rope_kernel(RopeArgs<T> a) {
    const int lane = threadIdx.x & 63, pairs = a.rot / 2, units = (a.D + 1) / 2;
    const int64_t row = blockIdx.x;
    const int position = a.positions[row];
    for (int h = blockIdx.y * (kRopeThreads / 64) + (threadIdx.x >> 6); h < a.heads[0] + a.heads[1];
         h += gridDim.y * (kRopeThreads / 64)) {
        const int of = h < a.heads[0] ? 0 : 1, head = of ? h - a.heads[0] : h;
        const T* x = a.x[of] + row * a.in_stride[of] + static_cast<int64_t>(head) * a.D;
        T* y = a.y[of] + row * a.out_stride[of] + static_cast<int64_t>(head) * a.D;
        const T* w = a.weight[of];
        T in[2][2];
        int at[2][2];
        bool there[2][2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int u = lane + 64 * k;
            at[k][0] = u < pairs && !INTERLEAVED ? u : 2 * u;
            at[k][1] = u < pairs && !INTERLEAVED ? u + pairs : 2 * u + 1;
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                there[k][e] = u < units && at[k][e] < a.D;
                in[k][e] = there[k][e] ? x[at[k][e]] : T(0);
            }
        }
        if (position < 0) {  // no position: passed on as it is
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e)
                    if (there[k][e]) y[at[k][e]] = in[k][e];
            continue;
        }
        double by = 1.0;
        if (w) {
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 2; ++e) sum += static_cast<double>(to_f32(in[k][e])) * to_f32(in[k][e]);
            for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d, 64);
            by = 1.0 / sqrt(sum / a.D + a.eps);
        }
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int u = lane + 64 * k;
            float v[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                v[e] = to_f32(in[k][e]);
                if (w && there[k][e]) v[e] = static_cast<float>(v[e] * by) * to_f32(w[at[k][e]]);
            }
            if (u < pairs) {
                float c, s;
                turn(static_cast<uint64_t>(position) * a.turns[u], c, s);
                c *= a.gain;
                s *= a.gain;
                const float p = v[0] * c - v[1] * s, q = v[1] * c + v[0] * s;
                v[0] = p;
                v[1] = q;
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (there[k][e]) put(y + at[k][e], v[e]);
        }
    }
}

// Sum over 1 << LB adjacent lanes (4 to 64), the same in all of them.
template <int LB, typename S>
__device__ __forceinline__ S lanes_sum(S x) {
#pragma unroll
    for (int d = 1; d < 1 << LB; d <<= 1) x += __shfl_xor(x, d, 64);
    return x;
}
// V channels, up to 16 bytes, at any alignment.
template <typename T, int V>
struct Vector {
    static constexpr int kWords = (V * sizeof(T) + 3) / 4;
    uint32_t w[kWords];

    __device__ __forceinline__ void load(const T* from) {
        w[0] = 0;  // (of one bf16 the upper half)
        __builtin_memcpy(w, from, V * sizeof(T));
    }
    __device__ __forceinline__ void store(T* to) const { __builtin_memcpy(to, w, V * sizeof(T)); }
    __device__ __forceinline__ void unpack(float (&x)[V]) const {
#pragma unroll
        for (int j = 0; j < V; ++j) {
            if constexpr (sizeof(T) == 4) x[j] = __uint_as_float(w[j]);
            else x[j] = __uint_as_float(j % 2 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
        }
    }
    __device__ __forceinline__ void pack(const float (&x)[V]) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < V; ++j) w[j] = __float_as_uint(x[j]);
        } else if constexpr (V == 1) {
            w[0] = f32_to_bf16(x[0]);
        } else {
#pragma unroll
            for (int j = 0; j < V / 2; ++j) w[j] = pack_bf16x2(x[2 * j], x[2 * j + 1]);
        }
    }
};

// Rows whose heads are whole vectors of V channels: a lane has two vectors of a head,
// of which each pair has its channels in the lane, 1 << LB lanes a head, kHeads heads of
// a row beside one another.  The workgroup makes its rows' cosines and sines once, one
// or two a thread, through LDS, and a lane keeps its own for all the heads it goes
// through, of which kBatch are on their way at a time.
// Bound by memory: 32768 rows of 32 and 8 heads of 128 in bf16, 671 MB in and out, 121
// to 125 us, 5.4 to 5.5 TB/s (a copy of 1 GiB: 5.1; rope_kernel 435); 16384 in fp32, as
// many bytes, 127 (273).  A few rows: 4.2 us of launch
// and loads one after the other.
template <int LB>
constexpr int heads_of() { return std::min(8, kRopeThreads >> LB); }
template <typename T, int V>
constexpr int batch_of() { return V * sizeof(T) >= 8 ? 4 : 8; }
template <typename T, int V, bool INTERLEAVED, int LB>
__global__ __launch_bounds__(kRopeThreads) void rope_vec_kernel(RopeArgs<T> a) {
    constexpr int kHeads = heads_of<LB>(), kBatch = batch_of<T, V>(), kRows = (kRopeThreads >> LB) / kHeads, kPairs = V << LB;
    __shared__ __attribute__((aligned(16))) float cosines[kRows][kPairs], sines[kRows][kPairs];
    const int pairs = a.rot / 2, first_row = blockIdx.x * kRows;
    for (int n = threadIdx.x; n < kRows * kPairs; n += kRopeThreads) {
        const int row = first_row + n / kPairs, i = n % kPairs;
        if (row >= a.n_rows || i >= pairs) continue;
        float c, s;
        turn(static_cast<uint64_t>(max(a.positions[row], 0)) * a.turns[i], c, s);
        cosines[n / kPairs][i] = c * a.gain;
        sines[n / kPairs][i] = s * a.gain;
    }
    __syncthreads();
    const int group = threadIdx.x >> LB, unit = threadIdx.x & ((1 << LB) - 1), r = group / kHeads;
    const int64_t row = first_row + r;
    const int units = a.D / (2 * V), heads = a.heads[0] + a.heads[1];
    const bool turned = unit * V < pairs, in = unit < units;
    if (row >= a.n_rows) return;
    const bool somewhere = a.positions[row] >= 0;
    // this lane's vectors of a head
    const int at0 = turned && !INTERLEAVED ? unit * V : 2 * unit * V;
    const int at1 = turned && !INTERLEAVED ? unit * V + pairs : 2 * unit * V + V;
    float c[V], s[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        c[j] = cosines[r][unit * V + j];
        s[j] = sines[r][unit * V + j];
    }
    float w0[V], w1[V];
    int side = -1;
    bool norm = false;
    for (int h0 = blockIdx.y * kBatch * kHeads + group % kHeads; h0 < heads; h0 += gridDim.y * kBatch * kHeads) {
        Vector<T, V> x0[kBatch], x1[kBatch];
        T* to[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int h = min(h0 + k * kHeads, heads - 1);  // (past the last one that again, not kept)
            const int of = h >= a.heads[0], head = of ? h - a.heads[0] : h;
            const T* from = (of ? a.x[1] + row * a.in_stride[1] : a.x[0] + row * a.in_stride[0]) + static_cast<int64_t>(head) * a.D;
            to[k] = (of ? a.y[1] + row * a.out_stride[1] : a.y[0] + row * a.out_stride[0]) + static_cast<int64_t>(head) * a.D;
            if (in) {
                x0[k].load(from + at0);
                x1[k].load(from + at1);
            }
        }
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const int h = h0 + k * kHeads, of = h >= a.heads[0];
            if (h >= heads) break;
            if (of != side) {
                side = of;
                const T* w = a.weight[of];
                norm = w != nullptr;
                if (norm && in) {
                    Vector<T, V> v;
                    v.load(w + at0);
                    v.unpack(w0);
                    v.load(w + at1);
                    v.unpack(w1);
                }
            }
            if (somewhere) {
                float y0[V], y1[V];
                x0[k].unpack(y0);
                x1[k].unpack(y1);
                if (norm) {
                    float sum = 0.0f;
#pragma unroll
                    for (int j = 0; j < V; ++j) sum += y0[j] * y0[j] + y1[j] * y1[j];
                    sum = lanes_sum<LB>(in ? sum : 0.0f);
                    const float mean = sum / static_cast<float>(a.D) + a.eps;
                    float by = __builtin_amdgcn_rsqf(mean);
                    if (!(mean >= 0x1p-60f && sum < 0x1p126f)) {  // squares out of fp32's range
                        double all = 0.0;
#pragma unroll
                        for (int j = 0; j < V; ++j)
                            all += static_cast<double>(y0[j]) * y0[j] + static_cast<double>(y1[j]) * y1[j];
                        const double d = 1.0 / sqrt(lanes_sum<LB>(in ? all : 0.0) / a.D + a.eps);
#pragma unroll
                        for (int j = 0; j < V; ++j) {  // (the factor itself may be out of it)
                            y0[j] = static_cast<float>(y0[j] * d);
                            y1[j] = static_cast<float>(y1[j] * d);
                        }
                        by = 1.0f;
                    }
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        y0[j] = y0[j] * by * w0[j];
                        y1[j] = y1[j] * by * w1[j];
                    }
                }
                if (turned) {
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        // (adjacent pairs: of the first vector, then of the second; of one channel each, both)
                        constexpr bool kAdjacent = INTERLEAVED && V > 1;
                        float& p = kAdjacent ? (2 * j < V ? y0[2 * j % V] : y1[2 * j % V]) : y0[j];
                        float& q = kAdjacent ? (2 * j < V ? y0[(2 * j + 1) % V] : y1[(2 * j + 1) % V]) : y1[j];
                        const float t = p * c[j] - q * s[j];
                        q = q * c[j] + p * s[j];
                        p = t;
                    }
                }
                x0[k].pack(y0);
                x1[k].pack(y1);
            }
            if (in) {
                x0[k].store(to[k] + at0);
                x1[k].store(to[k] + at1);
            }
        }
    }
}

// Whether rope_vec_kernel takes a call with vectors of V channels: heads of whole ones on
// 64 lanes, pairs (or channels that are not turned) in the same lane.
template <typename T, int V>
bool whole_vectors(const RopeArgs<T>& a, bool interleaved) {
    return a.D % (2 * V) == 0 && a.D <= 128 * V && (interleaved ? a.rot % (2 * V) == 0 : a.rot / 2 % V == 0);
}
template <typename T, int V, bool INTERLEAVED>
void launch_vec(const RopeArgs<T>& a, hipStream_t s) {
    const int units = a.D / (2 * V), heads = a.heads[0] + a.heads[1];
    auto go = [&](auto lb) {
        constexpr int kHeads = heads_of<lb()>(), kBatch = batch_of<T, V>(), kRows = (kRopeThreads >> lb()) / kHeads;
        const unsigned x = static_cast<unsigned>((a.n_rows + kRows - 1) / kRows);
        // a workgroup for each batch of heads while there are too few for the chip
        const unsigned y = std::min((heads + kBatch * kHeads - 1) / (kBatch * kHeads), static_cast<int>(1 + 2048 / x));
        rope_vec_kernel<T, V, INTERLEAVED, lb()><<<dim3(x, y), kRopeThreads, 0, s>>>(a);
    };
    // (as many lanes a head as kKvMaxDim channels can need)
    if (units <= 4) return go(std::integral_constant<int, 2>{});
    if (units <= 8) return go(std::integral_constant<int, 3>{});
    if (units <= 16) return go(std::integral_constant<int, 4>{});
    if constexpr (kKvMaxDim / (2 * V) > 16)
        if (units <= 32) return go(std::integral_constant<int, 5>{});
    if constexpr (kKvMaxDim / (2 * V) > 32) go(std::integral_constant<int, 6>{});
}
// The widest vectors that the call's channels can be cut into; whether there are any.
// Measured, 32768 rows of 32 and 8 heads in bf16, in place, two sets of inputs in turn,
// widest vectors / rope_kernel: of 128 channels 121 / 435 us (vectors of 8), 124 of 128
// turned 153 / 440 (2), 126 of 128 225 / 441 (1), 40 40 / 316 (4), 100 133 / 421 (2); of
// 64 rows 10.6 / 10.6, the host's.
template <typename T, int V>
bool by_vectors(const RopeArgs<T>& a, bool interleaved, hipStream_t s) {
    if (whole_vectors<T, V>(a, interleaved)) {
        if (interleaved) launch_vec<T, V, true>(a, s);
        else launch_vec<T, V, false>(a, s);
        return true;
    }
    if constexpr (V > 1) return by_vectors<T, V / 2>(a, interleaved, s);
    return false;
}

template <typename T>
int rope(const char* fn, const T* q, int64_t q_stride, const T* k, int64_t k_stride, const int32_t* positions,
         const uint64_t* turns, const T* q_weight, const T* k_weight, float eps, float gain, T* q_out,
         int64_t q_out_stride, T* k_out, int64_t k_out_stride, int interleaved, int n_rows, int n_heads, int n_kv_heads,
         int D, int rot, void* stream) {
    LHQ_REQUIRE(n_rows >= 0, "%s: bad row count %d", fn, n_rows);
    LHQ_SUPPORTED(n_rows <= (1 << 23), "%s: %d rows are over 2^23", fn, n_rows);
    LHQ_REQUIRE(n_heads >= 0 && n_kv_heads >= 0 && D > 0, "%s: bad dims (heads %d and %d, head_dim %d)", fn, n_heads,
                n_kv_heads, D);
    LHQ_SUPPORTED(D <= kKvMaxDim, "%s: head_dim %d is over %d", fn, D, kKvMaxDim);
    LHQ_SUPPORTED(n_heads <= 65535 && n_kv_heads <= 65535, "%s: %d or %d heads are over 65535", fn, n_heads, n_kv_heads);
    LHQ_REQUIRE(rot >= 0 && rot <= D && rot % 2 == 0, "%s: rot_dim %d is no even part of head_dim %d", fn, rot, D);
    LHQ_REQUIRE(interleaved == 0 || interleaved == 1, "%s: interleaved is %d, not 0 or 1", fn, interleaved);
    LHQ_REQUIRE(std::isfinite(gain), "%s: gain %g is not finite", fn, gain);
    LHQ_REQUIRE(std::isfinite(eps) && eps >= 0.0f, "%s: eps %g is negative or not finite", fn, eps);
    const int64_t q_width = static_cast<int64_t>(n_heads) * D, k_width = static_cast<int64_t>(n_kv_heads) * D;
    LHQ_REQUIRE(q_stride >= q_width && q_out_stride >= q_width && k_stride >= k_width && k_out_stride >= k_width,
                "%s: strides %lld, %lld, %lld, %lld are under rows of %lld and %lld", fn,
                static_cast<long long>(q_stride), static_cast<long long>(q_out_stride),
                static_cast<long long>(k_stride), static_cast<long long>(k_out_stride),
                static_cast<long long>(q_width), static_cast<long long>(k_width));
    if (n_rows == 0 || n_heads + n_kv_heads == 0) return LHQ_OK;
    LHQ_REQUIRE((n_heads == 0 || (q && q_out)) && (n_kv_heads == 0 || (k && k_out)) && positions && (rot == 0 || turns),
                "%s: null pointer", fn);
    // Waves read and write in no order: a result may lie where its own input does, else where none of them does.
    auto apart = [n_rows](const T* x, int64_t xs, int64_t xw, const T* y, int64_t ys, int64_t yw) {
        if (xw == 0 || yw == 0 || x + (n_rows - 1) * xs + xw <= y || y + (n_rows - 1) * ys + yw <= x) return true;
        const int64_t by = ((y - x) % xs + xs) % xs;  // columns of one wider matrix
        return xs == ys && by >= xw && by + yw <= xs;
    };
    auto in_place = [n_rows](const T* x, int64_t xs, const T* y, int64_t ys) { return x == y && (xs == ys || n_rows == 1); };
    const bool q_in_place = in_place(q, q_stride, q_out, q_out_stride), k_in_place = in_place(k, k_stride, k_out, k_out_stride);
    LHQ_REQUIRE((q_in_place || apart(q, q_stride, q_width, q_out, q_out_stride, q_width)) &&
                    (k_in_place || apart(k, k_stride, k_width, k_out, k_out_stride, k_width)) &&
                    apart(q, q_stride, q_width, k_out, k_out_stride, k_width) &&
                    apart(k, k_stride, k_width, q_out, q_out_stride, q_width) &&
                    apart(q_out, q_out_stride, q_width, k_out, k_out_stride, k_width),
                "%s: a result overlaps an input or the other result", fn);
    RopeArgs<T> a{{q, k},         {q_stride, k_stride}, {q_out, k_out}, {q_out_stride, k_out_stride},
                  {q_weight, k_weight}, {n_heads, n_kv_heads}, positions, turns, n_rows, D, rot, eps, gain};
    const hipStream_t s = as_stream(stream);
    if (by_vectors<T, 16 / sizeof(T)>(a, interleaved != 0, s)) return check_launch(fn);
    const int heads = n_heads + n_kv_heads;
    const dim3 grid(n_rows, std::min((heads + 3) / 4, 65535));
    if (interleaved) rope_kernel<T, true><<<grid, kRopeThreads, 0, s>>>(a);
    else rope_kernel<T, false><<<grid, kRopeThreads, 0, s>>>(a);
    return check_launch(fn);
}

}  // namespace
}  // namespace lhq

using namespace lhq;

extern "C" {

int lhq_rope_f32(const float* q, int64_t q_stride, const float* k, int64_t k_stride, const int32_t* positions,
                 const uint64_t* turns, const float* q_weight, const float* k_weight, float eps, float gain,
                 float* q_out, int64_t q_out_stride, float* k_out, int64_t k_out_stride, int interleaved, int n_rows,
                 int n_heads, int n_kv_heads, int head_dim, int rot_dim, void* stream) {
    return rope("rope_f32", q, q_stride, k, k_stride, positions, turns, q_weight, k_weight, eps, gain, q_out,
                q_out_stride, k_out, k_out_stride, interleaved, n_rows, n_heads, n_kv_heads, head_dim, rot_dim, stream);
}

int lhq_rope_bf16(const uint16_t* q, int64_t q_stride, const uint16_t* k, int64_t k_stride, const int32_t* positions,
                  const uint64_t* turns, const uint16_t* q_weight, const uint16_t* k_weight, float eps, float gain,
                  uint16_t* q_out, int64_t q_out_stride, uint16_t* k_out, int64_t k_out_stride, int interleaved,
                  int n_rows, int n_heads, int n_kv_heads, int head_dim, int rot_dim, void* stream) {
    return rope("rope_bf16", q, q_stride, k, k_stride, positions, turns, q_weight, k_weight, eps, gain, q_out,
                q_out_stride, k_out, k_out_stride, interleaved, n_rows, n_heads, n_kv_heads, head_dim, rot_dim, stream);
}

}  // extern "C"
