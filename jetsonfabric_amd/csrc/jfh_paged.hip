// gfx950 kernels of the paged-cache operators (jfh_paged.hpp).
#include "jfh_paged.hpp"

#include <hip/hip_runtime.h>

#include <type_traits>

namespace jfh::paged {

namespace {

using half8 = _Float16 __attribute__((ext_vector_type(8)));
using bhalf8 = __bf16 __attribute__((ext_vector_type(8)));
using float4v = float __attribute__((ext_vector_type(4)));
using float16v = float __attribute__((ext_vector_type(16)));

constexpr float kLn2 = 0.693147180559945309F, kLog2e = 1.44269504088896341F;

enum : uint32_t { kF32 = 1, kF16 = 2, kBF16 = 3 };

template <typename... KArgs, typename... Args>
hipError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, hipStream_t stream, const Args&... args) {
    static_assert((std::is_same_v<KArgs, Args> && ...), "arguments are passed by address");
    // a launch holds fewer than 2^32 threads
    if (static_cast<uint64_t>(grid.x) * block.x > 0xFFFFFFFFULL) return hipErrorInvalidConfiguration;
    void* p[] = {const_cast<void*>(static_cast<const void*>(&args))...};
    return hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, block, p, 0, stream);
}

// ---------------------------------------------------------------- rotary positions

// N values of a row as floats; the type is uniform over the launch.
template <int N>
__device__ __forceinline__ void load(const void* data, int64_t at, uint32_t type, float (&x)[N]) {
    if constexpr (N == 8) {
        if (type == kF32) {
            const float4v* p = reinterpret_cast<const float4v*>(static_cast<const float*>(data) + at);
            const float4v a = p[0], b = p[1];
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
        } else if (type == kF16) {
            const half8 v = *reinterpret_cast<const half8*>(static_cast<const _Float16*>(data) + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
        } else {
            const bhalf8 v = *reinterpret_cast<const bhalf8*>(static_cast<const __bf16*>(data) + at);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
        }
    } else {
        static_assert(N == 1);
        x[0] = type == kF32   ? static_cast<const float*>(data)[at]
               : type == kF16 ? static_cast<float>(static_cast<const _Float16*>(data)[at])
                              : static_cast<float>(static_cast<const __bf16*>(data)[at]);
    }
}

template <bool PAST, typename V>
__device__ __forceinline__ void put(V* to, V v) {
    if constexpr (PAST) __builtin_nontemporal_store(v, to);
    else *to = v;
}

// The one rounding to the output's type, to nearest. PAST: past the caches, for rows that they could not hold.
template <int N, bool PAST = false>
__device__ __forceinline__ void store(void* data, int64_t at, uint32_t type, const float (&x)[N]) {
    if constexpr (N == 8) {
        if (type == kF32) {
            float4v* p = reinterpret_cast<float4v*>(static_cast<float*>(data) + at);
            put<PAST>(p, float4v{x[0], x[1], x[2], x[3]});
            put<PAST>(p + 1, float4v{x[4], x[5], x[6], x[7]});
        } else if (type == kF16) {
            half8 v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = static_cast<_Float16>(x[i]);
            put<PAST>(reinterpret_cast<half8*>(static_cast<_Float16*>(data) + at), v);
        } else {
            bhalf8 v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = static_cast<__bf16>(x[i]);
            put<PAST>(reinterpret_cast<bhalf8*>(static_cast<__bf16*>(data) + at), v);
        }
    } else {
        static_assert(N == 1);
        if (type == kF32) static_cast<float*>(data)[at] = x[0];
        else if (type == kF16) static_cast<_Float16*>(data)[at] = static_cast<_Float16>(x[0]);
        else static_cast<__bf16*>(data)[at] = static_cast<__bf16>(x[0]);
    }
}

constexpr int kRotateThreads = 256;
constexpr int kRotateRows = 4;  // most rows of a work-group

// cos and sin of every pair of `rows` rows from row0, times the rotation's size. The angle is a product of doubles in
// turns, reduced by whole turns before it becomes a float: far positions keep an error of 2^-24 of half a turn.
__device__ __forceinline__ void row_angles(const Rotation& r, const int32_t* __restrict__ positions, int row0, int rows,
                                           float2 (*cs)[kMaxRotPairs]) {
    const int pairs = static_cast<int>(r.n_rot / 2);
    for (int t = threadIdx.x; t < rows * pairs; t += kRotateThreads) {
        const int row = t / pairs, i = t - row * pairs;
        double turns = static_cast<double>(positions[row0 + row]) * r.turns[i];
        turns -= rint(turns);
        float s, c;
        sincospif(static_cast<float>(2.0 * turns), &s, &c);
        cs[row][i] = float2{c * r.size, s * r.size};
    }
}

// Unit u of a head: N pairs for u < pairs / N, then N values that stay.
template <int N, bool PAST>
__device__ __forceinline__ void rotate_unit(const Rotation& r, const float2* cs, int u, const void* x, int64_t x_at,
                                            uint32_t x_type, void* y, int64_t y_at, uint32_t y_type) {
    const int half = static_cast<int>(r.n_rot / 2);
    if (u * N < half) {
        const int lo = r.interleaved ? 2 * u * N : u * N;
        const int hi = r.interleaved ? lo + N : half + u * N;
        float a[N], b[N];
        load(x, x_at + lo, x_type, a);
        load(x, x_at + hi, x_type, b);
        const float2* t = cs + u * N;
        if (r.interleaved) {
            float v[2 * N];
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = a[i], v[N + i] = b[i];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = v[2 * i], q = v[2 * i + 1];
                v[2 * i] = p * t[i].x - q * t[i].y;
                v[2 * i + 1] = p * t[i].y + q * t[i].x;
            }
#pragma unroll
            for (int i = 0; i < N; ++i) a[i] = v[i], b[i] = v[N + i];
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float p = a[i], q = b[i];
                a[i] = p * t[i].x - q * t[i].y;
                b[i] = p * t[i].y + q * t[i].x;
            }
        }
        store<N, PAST>(y, y_at + lo, y_type, a);
        store<N, PAST>(y, y_at + hi, y_type, b);
    } else {
        const int d = static_cast<int>(r.n_rot) + (u * N - half);
        float a[N];
        load(x, x_at + d, x_type, a);
        store<N, PAST>(y, y_at + d, y_type, a);
    }
}

// Bound by the rows' bytes, one read and one write. A work-group computes the angles of its rows once for all heads;
// a thread owns a unit, so rows may be rotated in place. 4096 rows of 48 heads of 128 bf16 values: 17 us, 5.9 TB/s; two
// rows: 3 us.
template <int N, bool PAST>
__global__ __launch_bounds__(kRotateThreads) void k_rotate(Rotation r, Rows x, const int32_t* __restrict__ positions,
                                                           Rows y, int rows_per_group) {
    __shared__ float2 cs[kRotateRows][kMaxRotPairs];
    const int row0 = static_cast<int>(blockIdx.x) * rows_per_group;
    const int rows = min(rows_per_group, static_cast<int>(x.rows) - row0);
    row_angles(r, positions, row0, rows, cs);
    __syncthreads();
    const int units = static_cast<int>(r.n_rot / 2 + (x.head_dim - r.n_rot)) / N;
    const int tasks = static_cast<int>(x.heads) * units;
    for (int t = static_cast<int>(blockIdx.y) * kRotateThreads + threadIdx.x; t < rows * tasks;
         t += static_cast<int>(gridDim.y) * kRotateThreads) {
        const int row = t / tasks, left = t - row * tasks;
        const int head = left / units, u = left - head * units;
        rotate_unit<N, PAST>(r, cs[row], u, x.data, (row0 + row) * x.row_stride + head * x.head_stride, x.type, y.data,
                             (row0 + row) * y.row_stride + head * y.head_stride, y.type);
    }
}

// New rows into their pages: keys rotated where the step gives a rotation, values as they are, weight 0 and the row's
// position for every K/V head. Rows of no sequence, before slot 0 or on absent pages are not written. The dependent loads
// of a row's place (row starts, length, table) come before the bytes: 4095 rows of three sequences, 4 K/V heads of 128
// bf16 values, 9.0 us; 18 rows 4 us.
template <int N>
__global__ __launch_bounds__(kRotateThreads) void k_append(Rotation r, Cache c, Batch b, Rows k, Rows v,
                                                           const int32_t* __restrict__ positions, int rows_per_group) {
    __shared__ float2 cs[kRotateRows][kMaxRotPairs];
    __shared__ int32_t pages[kRotateRows], slots[kRotateRows];
    const int row0 = static_cast<int>(blockIdx.x) * rows_per_group;
    const int rows = min(rows_per_group, static_cast<int>(k.rows) - row0);
    if (static_cast<int>(threadIdx.x) < rows) {
        const int row = row0 + threadIdx.x;
        Span span;
        const int s = sequence_of(b, k.rows, row, &span);
        const int slot = s >= 0 ? span.first + (row - span.row0) : -1;
        pages[threadIdx.x] = slot >= 0 && slot < span.len ? page_of(c, b, s, slot) : -1;
        slots[threadIdx.x] = slot;
    }
    if (r.n_rot) row_angles(r, positions, row0, rows, cs);
    __syncthreads();
    const int ku = static_cast<int>(r.n_rot / 2 + (k.head_dim - r.n_rot)) / N, vu = static_cast<int>(v.head_dim) / N;
    const int heads = static_cast<int>(c.n_head_kv);
    const int tasks = heads * (ku + vu + 1);
    for (int t = static_cast<int>(blockIdx.y) * kRotateThreads + threadIdx.x; t < rows * tasks;
         t += static_cast<int>(gridDim.y) * kRotateThreads) {
        const int row = t / tasks;
        int left = t - row * tasks;
        const int page = pages[row], slot = slots[row];
        if (page < 0) continue;
        const int64_t at = slot_offset(c, page, slot);
        if (left < heads * ku) {
            const int head = left / ku;
            rotate_unit<N, false>(r, cs[row], left - head * ku, k.data, (row0 + row) * k.row_stride + head * k.head_stride,
                                  k.type, c.k, at + head * c.head_stride, c.type);
        } else if ((left -= heads * ku) < heads * vu) {
            const int head = left / vu, d = (left - head * vu) * N;
            float x[N];
            load(v.data, (row0 + row) * v.row_stride + head * v.head_stride + d, v.type, x);
            store(c.v, at + head * c.head_stride + d, c.type, x);
        } else {
            const int64_t i = slot_index(c, page, left - heads * vu, slot);
            if (c.weights) c.weights[i] = 0.0F;
            if (c.positions) c.positions[i] = positions[row0 + row];
        }
    }
}

// ---------------------------------------------------------------- attention

template <typename T> struct Values;
template <> struct Values<_Float16> {
    using v8 = half8;
    static constexpr uint32_t kExponent = 0x7C00;
    static constexpr float kRaised = 15.0F;  // base-2 logarithm of a row's largest weight
    static __device__ __forceinline__ float4v mfma(v8 a, v8 b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float16v mfma(v8 a, v8 b, float16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
    }
};
template <> struct Values<__bf16> {
    using v8 = bhalf8;
    static constexpr uint32_t kExponent = 0x7F80;
    static constexpr float kRaised = 0.0F;
    static __device__ __forceinline__ float4v mfma(v8 a, v8 b, float4v c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
    static __device__ __forceinline__ float16v mfma(v8 a, v8 b, float16v c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
    }
};

// Over the four lanes l, l ^ 16, l ^ 32, l ^ 48.
__device__ __forceinline__ float groups_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float groups_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// Over the two lanes l, l ^ 32.
__device__ __forceinline__ float halves_max(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float halves_sum(float v) {
    const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Whether one of two 16-bit values is infinite or NaN.
template <typename T>
__device__ __forceinline__ bool nonfinite(uint32_t two) {
    constexpr uint32_t e = Values<T>::kExponent;
    return (two & e) == e || (two & (e << 16)) == (e << 16);
}

// Takes an infinity or NaN out of a half of two 16-bit values: 0 in its place, bit j in mark (+inf, -inf, NaN).
template <typename T>
__device__ __forceinline__ void take_nonfinite(uint32_t& two, int half, int j, uint32_t (&mark)[3]) {
    constexpr uint32_t exponent = Values<T>::kExponent, mantissa = 0x7FFFU & ~exponent;
    const uint32_t x = two >> (16 * half) & 0xFFFFU;
    const bool odd = (x & exponent) == exponent, nan = odd && (x & mantissa) != 0;
    mark[0] |= static_cast<uint32_t>(odd && !nan && !(x >> 15)) << j;
    mark[1] |= static_cast<uint32_t>(odd && !nan && (x >> 15)) << j;
    mark[2] |= static_cast<uint32_t>(nan) << j;
    if (odd) two &= half ? 0x0000FFFFU : 0xFFFF0000U;
}

// A sum to which visible infinities and NaN belong (any positive weight of theirs gives the same).
__device__ __forceinline__ float with_nonfinite(float sum, bool pos, bool neg, bool nan) {
    if (pos) sum += INFINITY;
    if (neg) sum -= INFINITY;
    return nan ? NAN : sum;
}

// Column c of eight rows of 16-bit values, two to a word.
template <int VW>
__device__ __forceinline__ uint4 column(const uint32_t (&v)[8][VW], int c) {
    const uint32_t pick = c % 2 ? 0x07060302U : 0x05040100U;
    return uint4{__builtin_amdgcn_perm(v[1][c / 2], v[0][c / 2], pick), __builtin_amdgcn_perm(v[3][c / 2], v[2][c / 2], pick),
                 __builtin_amdgcn_perm(v[5][c / 2], v[4][c / 2], pick), __builtin_amdgcn_perm(v[7][c / 2], v[6][c / 2], pick)};
}

// 2^x for the sums of slots whose maximum lies x below the row's: never 0, or an infinite sum would become NaN. (2^-149 of
// a sum of finite values is nothing beside any that count.)
__device__ __forceinline__ float share_of(float x) { return fmaxf(exp2f(x), 1.4e-45F); }

// Weight of sums with maximum m among others with maximum `now`. A part that has seen nothing (l = 0) weighs nothing; one
// whose scores are NaN (m = -inf, l NaN) goes on as such.
__device__ __forceinline__ float split_share(float m, float l, float now) {
    return l == 0.0F ? 0.0F : m == -INFINITY ? 1.0F : share_of(m - now);
}

// Weights are 2^(score - top), where `top` is a row's running maximum (base 2) less kRaised: the largest one is the power
// of two 2^kRaised, which no type rounds, and f16 keeps full precision 29 octaves below it and numbers 40 below (from 1
// on it would be 14 and 25, while long rows of small weights still count). Sums leave a kernel with the factor taken out.
struct Sums {
    float top, l, unit;  // maximum, sum of weights, what the sums of V are multiplied by
};
template <typename T>
__device__ __forceinline__ Sums lowered(float top, float l) {
    constexpr float unit = 1.0F / static_cast<float>(1U << static_cast<int>(Values<T>::kRaised));
    return Sums{top + Values<T>::kRaised, l * unit, unit};
}

// Eight values of a row from column d, 0 from column dim on.
template <typename T>
__device__ __forceinline__ typename Values<T>::v8 row_piece(const T* row, int d, int dim) {
    uint4 x = *reinterpret_cast<const uint4*>(row + (d < dim ? d : 0));
    if (d >= dim) x = uint4{0, 0, 0, 0};
    return __builtin_bit_cast(typename Values<T>::v8, x);
}

// Query m of a K/V head's rows * group queries is head m % group of the sequence's row m / group.
struct Query {
    int row, head;
};
__device__ __forceinline__ Query query_of(int m, int group, uint32_t kv_head) {
    const int row = m / group;
    return Query{row, static_cast<int>(kv_head) * group + (m - row * group)};
}

// Few query rows: o = softmax(scale q K^T) V for up to 16 MT queries of a K/V head, 8 waves (4 of wide heads) that divide its
// keys.
//
// The bytes of K and V bound it where there are enough of them, and their latency elsewhere. A wave takes tiles of 32 keys
// from global memory to registers, in the layout of the rows: S^T = K Q^T on 16x16x32 products has a K row's 16 bytes per
// lane as its A operand. O^T += V^T P^T wants 8 keys of one column per lane; lane (i, g) loads rows 16 u + 4 g + r (u = 0,
// 1, r = 0..3), columns VEC i .. VEC i + VEC - 1, and 16-bit permutes of those rows give the operands of VEC products, the
// c-th of columns VEC i + c. The keys of lane group g are those whose scores the group holds after S^T, so P needs no
// exchange between lanes. No LDS on the way: the next tile's K is requested as soon as the scores are there, its V after
// the product with P, and the pages of the one after it are looked up meanwhile.
// Running maximum and sum are f32, base 2. P goes to its product as two values of the cache's type, the second what the
// rounding of the first left, so that the one rounding that counts is the output's: the bytes bound the call, and the
// second product costs it 0 to 2 % (eight rows over up to 32701 positions, bf16: 104 us, error against 64 bits 1.66e-3,
// with P rounded once 104 us and 1.77e-3; head dim 64, f16, 30000: 37.3 us and 2.03e-4, 36.6 and 2.18e-4).
// Eight rows of 40 heads over 4087 to 32701 positions, bf16: 102 us and 5 for the join, 5.8 TB/s of K and V; one row over
// 257: 10.9 us, latency. Head dims above 128 take 285 registers, one wave per SIMD: eight sequences of 30000 positions, 4
// heads of one K/V head of 256, 58 us, 4.2 TB/s.
constexpr int kFewKeys = 32;  // keys of a wave's tile
template <int HDP> constexpr int kFewWaves = HDP <= 128 ? 8 : 4;

template <typename T, int HDP, int MT>
__global__ __launch_bounds__(64 * kFewWaves<HDP>) void k_attend_few(Attend a, int group) {
    using V = Values<T>;
    using v8 = typename V::v8;
    constexpr int VEC = HDP / 16;   // columns per lane of V
    constexpr int KC = HDP / 32;    // products per 16 keys of S^T
    constexpr int VW = VEC / 2;     // words per lane and V row
    constexpr int kChunk = VW < 4 ? VW : 4;  // words of one load
    constexpr int OS = HDP + 4;     // floats per query of the waves' sums in LDS
    constexpr int kWaves = kFewWaves<HDP>, kThreads = 64 * kWaves;
    __shared__ float part_o[kWaves][16][OS];
    __shared__ float part_m[kWaves][16], part_l[kWaves][16];
    __shared__ uint4 q_lds[MT][KC][64];

    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16;
    const uint32_t pairs = a.cache.n_head_kv * a.batch.n_seq;  // K/V heads of sequences
    const uint32_t split = blockIdx.x % a.splits, pair = blockIdx.x / a.splits % pairs;
    const uint32_t h = pair % a.cache.n_head_kv, s = pair / a.cache.n_head_kv;
    const int m0 = static_cast<int>(blockIdx.x / a.splits / pairs) * 16 * MT;
    const Span span = sequence_span(a.batch, a.q.rows, s);
    const int queries = span.rows * group;
    if (m0 >= queries) return;
    const int dim = static_cast<int>(a.cache.head_dim);
    const auto sees = [&](int m) { return a.causal ? slots_seen(span, m / group) : span.len; };  // slots of query m
    const int least = sees(m0), end = sees(min(queries, m0 + 16 * MT) - 1);  // seen by all queries here, by any

    // the split's tiles: equal parts of the sequence's, whole rounds of the waves
    const int tiles = (span.len + kFewKeys - 1) / kFewKeys;
    const int per = (tiles + static_cast<int>(a.splits) * kWaves - 1) / (static_cast<int>(a.splits) * kWaves) * kWaves;
    const int t0 = min(static_cast<int>(split) * per, tiles), t1 = min(min(tiles, t0 + per), (end + kFewKeys - 1) / kFewKeys);

    const T* k_head = static_cast<const T*>(a.cache.k) + h * a.cache.head_stride;
    const T* v_head = static_cast<const T*>(a.cache.v) + h * a.cache.head_stride;

    // Offsets of the lane's K rows of a tile and a bit per key that is there: in use, and on a page.
    struct Keys {
        int64_t at[2];
        uint32_t present;  // bit 16 u + e: key 16 u + e
    };
    const auto look_up = [&](int t) {
        Keys x;
        x.present = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int slot = t * kFewKeys + 16 * u + i;
            const int page = slot < end ? page_of(a.cache, a.batch, s, slot) : -1;
            x.at[u] = page >= 0 ? slot_offset(a.cache, page, slot) : 0;  // of a row that is not there: any that is
            x.present |= (static_cast<uint32_t>(__ballot(page >= 0)) & 0xFFFFU) << (16 * u);
        }
        return x;
    };
    v8 k[2][KC];
    uint32_t v[8][VW];
    const auto fetch_k = [&](const Keys& x) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int c = 0; c < KC; ++c) {
                const int d = 32 * c + 8 * g;
                k[u][c] = *reinterpret_cast<const v8*>(k_head + x.at[u] + (d < dim ? d : 0));
            }
        }
    };
    // V is read once where sequences share no pages, so a load of a lane's 16 bytes of whole rows (head dims 65 to 128)
    // leaves nothing in the caches. Eight sequences of 30000 positions, 40 heads: head dim 128 161 us, 176 through them;
    // 96 137 and 140; 72 125 and 119; 128 with all pages shared 107 and 101. Of 8000, which stay in the caches from call to
    // call, 23.6 and 23.1. Loads of parts of rows (K's, and V's of other head dims) lose what the neighbouring loads find
    // there (27.0 and 29.6 us).
    typedef uint32_t Words __attribute__((ext_vector_type(kChunk)));
    const auto fetch_v = [&](const Keys& keys) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const T* row = v_head + __shfl(keys.at[j / 4], 4 * g + j % 4);
#pragma unroll
            for (int w = 0; w < VW; w += kChunk) {
                const int d = VEC * i + 2 * w;
                const Words* p = reinterpret_cast<const Words*>(row + (d < dim ? d : 0));
                const Words x = VW == 4 ? __builtin_nontemporal_load(p) : *p;
                __builtin_memcpy(&v[j][w], &x, sizeof x);
            }
        }
    };

    Keys now{}, next{};
    if (t0 + wave < t1) {
        now = look_up(t0 + wave);
        fetch_k(now);
        fetch_v(now);
        if (t0 + wave + kWaves < t1) next = look_up(t0 + wave + kWaves);
    }

    // queries to LDS in operand order, zeros behind the last one and beyond head_dim
    for (int e = threadIdx.x; e < MT * KC * 64; e += kThreads) {
        const int l = e % 64, c = e / 64 % KC, mt = e / 64 / KC;
        const int m = m0 + 16 * mt + l % 16, d = 32 * c + 8 * (l / 16);
        uint4 x{0, 0, 0, 0};
        if (m < queries && d < dim) {
            const Query q = query_of(m, group, h);
            x = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.q.data) + (span.row0 + q.row) * a.q.row_stride +
                                                q.head * a.q.head_stride + d);
        }
        q_lds[mt][c][l] = x;
    }
    __syncthreads();

    int limit[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) limit[mt] = sees(min(m0 + 16 * mt + i, queries - 1));
    float4v o[MT][VEC];
    float top[MT], sum[MT];
    const auto walk = [&](auto again) __attribute__((always_inline)) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
            top[mt] = -INFINITY;
            sum[mt] = 0.0F;
#pragma unroll
            for (int c = 0; c < VEC; ++c) o[mt][c] = float4v{0.0F, 0.0F, 0.0F, 0.0F};
        }

        for (int t = t0 + wave; t < t1; t += kWaves) {
            if constexpr (again) {
                now = look_up(t);
                fetch_k(now);
                fetch_v(now);
            }
            const int base = t * kFewKeys;
            const bool whole = now.present == 0xFFFFFFFFU;
            const bool hidden = base + kFewKeys > least;  // some query here does not see some of the tile
            if (dim < HDP) {  // beyond head_dim Q is 0, and what it meets must be a number
#pragma unroll
                for (int c = 0; c < KC; ++c) {
                    if (32 * c + 8 * g >= dim) k[0][c] = k[1][c] = __builtin_bit_cast(v8, uint4{0, 0, 0, 0});
                }
            }
            float4v sc[MT][2];
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) sc[mt][0] = sc[mt][1] = float4v{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
            for (int c = 0; c < KC; ++c) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const v8 q = __builtin_bit_cast(v8, q_lds[mt][c][lane]);
                    sc[mt][0] = V::mfma(k[0][c], q, sc[mt][0]);
                    sc[mt][1] = V::mfma(k[1][c], q, sc[mt][1]);
                }
            }
            if (!again && t + kWaves < t1) fetch_k(next);

            // scores of keys base + 16 u + 4 g + r, query i
            uint32_t seen[MT];
            if (again || !whole || hidden) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    seen[mt] = 0;
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int e = 16 * (j / 4) + 4 * g + j % 4;
                        const bool see = (now.present >> e & 1U) && base + e < limit[mt];
                        seen[mt] |= static_cast<uint32_t>(see) << j;
                        if (!see) sc[mt][j / 4][j % 4] = -INFINITY;
                    }
                }
            }
            float most[MT];
            bool rise = false;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                most[mt] = sc[mt][0][0];
#pragma unroll
                for (int j = 1; j < 8; ++j) most[mt] = fmaxf(most[mt], sc[mt][j / 4][j % 4]);
                most[mt] = groups_max(most[mt]) * a.scale_log2 - V::kRaised;
                rise |= most[mt] > top[mt];
            }
            if (__ballot(rise)) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const float to = fmaxf(top[mt], most[mt]);
                    const float shrink = to == -INFINITY ? 1.0F : share_of(top[mt] - to);
                    top[mt] = to;
                    sum[mt] *= shrink;
#pragma unroll
                    for (int c = 0; c < VEC; ++c) o[mt][c] *= shrink;
                }
            }
            v8 p[MT], rest[MT];  // weights, what their rounding left
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) {
                const float ref = top[mt] == -INFINITY ? 0.0F : top[mt];
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(sc[mt][j / 4][j % 4], a.scale_log2, -ref));
                    sum[mt] += w;
                    p[mt][j] = static_cast<T>(w);
                    rest[mt][j] = static_cast<T>(w - static_cast<float>(p[mt][j]));
                }
            }
            if (!whole) {  // what is not there must be a number: its weight is 0 (columns beyond head_dim go nowhere)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    if (now.present >> (16 * (j / 4) + 4 * g + j % 4) & 1U) continue;
#pragma unroll
                    for (int w = 0; w < VW; ++w) v[j][w] = 0;
                }
            }
            bool odd = false;
            if constexpr (again) {
#pragma unroll
                for (int j = 0; j < 8; ++j) {
#pragma unroll
                    for (int w = 0; w < VW; ++w) odd |= nonfinite<T>(v[j][w]);
                }
            }
            // marks of the infinities and NaN of V, taken out for the product, go to LDS by column, a byte per lane group
            uint32_t* marks = reinterpret_cast<uint32_t*>(part_o[wave]);  // [3][HDP], the wave's own until the loop ends
            const bool any_odd = __ballot(odd) != 0;
            if (any_odd) {
#pragma unroll
                for (int c = 0; c < VEC; ++c) {
                    uint32_t mark[3] = {0, 0, 0};
#pragma unroll
                    for (int j = 0; j < 8; ++j) take_nonfinite<T>(v[j][c / 2], c % 2, j, mark);
#pragma unroll
                    for (int n = 0; n < 3; ++n) reinterpret_cast<uint8_t*>(marks + n * HDP + VEC * i + c)[g] = static_cast<uint8_t>(mark[n]);
                }
            }
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
                const v8 x = __builtin_bit_cast(v8, column<VW>(v, c));
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) o[mt][c] = V::mfma(x, rest[mt], V::mfma(x, p[mt], o[mt][c]));
            }
            if (any_odd) {
                asm volatile("" ::: "memory");
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    // the query's keys: bit 8 g + j
                    uint32_t see = seen[mt] << (8 * g);
                    see |= __shfl_xor(see, 16);
                    see |= __shfl_xor(see, 32);
#pragma unroll
                    for (int c = 0; c < VEC; ++c) {
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int d = VEC * (4 * g + r) + c;
                            o[mt][c][r] = with_nonfinite(o[mt][c][r], marks[d] & see, marks[HDP + d] & see, marks[2 * HDP + d] & see);
                            asm volatile("" ::: "memory");  // one column's marks at a time: the sums leave few registers
                        }
                    }
                }
            }
            if (!again && t + kWaves < t1) {
                fetch_v(next);
                now = next;
                if (t + 2 * kWaves < t1) next = look_up(t + 2 * kWaves);
            }
        }
        float odd = 0.0F;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
            for (int c = 0; c < VEC; ++c) {
#pragma unroll
                for (int r = 0; r < 4; ++r) odd = fmaf(o[mt][c][r], 0.0F, odd);
            }
        }
        return __ballot(odd != odd) != 0;
    };
    // A sum that is not finite at the end has met infinities or NaN of V, whose weight may be 0 (hidden, or rounded to 0): the
    // wave walks its tiles again and takes them out of V.
    if (walk(std::false_type{})) walk(std::true_type{});

    // the waves' sums, 16 queries at a time
    const int64_t all = static_cast<int64_t>(a.q.rows) * a.q.heads;
    const bool complete = a.splits == 1;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
        if (m0 + 16 * mt >= queries) break;
        __syncthreads();
        const float wave_l = groups_sum(sum[mt]);
        const Sums all_seen = lowered<T>(top[mt], wave_l);
        if (g == 0) part_m[wave][i] = all_seen.top, part_l[wave][i] = all_seen.l;
        // lane (i, g) holds columns VEC (4 g + r) + c of query i
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
            for (int c = 0; c < VEC; c += 4) {
                *reinterpret_cast<float4v*>(&part_o[wave][i][VEC * (4 * g + r) + c]) =
                    float4v{o[mt][c][r], o[mt][c + 1][r], o[mt][c + 2][r], o[mt][c + 3][r]};
            }
        }
        __syncthreads();
        constexpr int kPer = kThreads / 16;  // threads of a query
        const int n = threadIdx.x / kPer, m = m0 + 16 * mt + n;
        if (m >= queries) continue;
        float high = part_m[0][n];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) high = fmaxf(high, part_m[w][n]);
        float share[kWaves], l = 0.0F;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            share[w] = split_share(part_m[w][n], part_l[w][n], high);
            l += part_l[w][n] * share[w];
        }
        const Query q = query_of(m, group, h);
        const int64_t row = span.row0 + q.row, at = row * a.q.heads + q.head;
        const float scale = all_seen.unit * (!complete ? 1.0F : l == 0.0F ? 0.0F : 1.0F / l);
        for (int d = threadIdx.x % kPer * 8; d < dim; d += 8 * kPer) {
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[e] = 0.0F;
#pragma unroll
                for (int w = 0; w < kWaves; ++w) {
                    if (share[w] != 0.0F) x[e] += part_o[w][n][d + e] * share[w];
                }
                x[e] *= scale;
            }
            if (complete) store(a.out.data, row * a.out.row_stride + q.head * a.out.head_stride + d, a.out.type, x);
            else if (l != 0.0F) store(a.partial, (split * all + at) * dim + d, kF32, x);
        }
        if (threadIdx.x % kPer == 0) {
            if (!complete) *reinterpret_cast<float2*>(a.marks + 2 * (split * all + at)) = float2{high, l};
            else if (a.lse) a.lse[at] = high * kLn2 + logf(l);
        }
    }
}

// Many query rows: 128 queries of a K/V head per work-group, 32 per wave, over tiles of KT keys that the work-group stages
// in LDS, double-buffered: while a tile is multiplied, the next one's rows are on their way to registers, and the offsets
// of the one after it are looked up (pages of any size: one lookup per key).
//
// 32x32x16 products: S^T = K Q^T has a query per lane and leaves a lane the scores of keys 8 b + 4 g + r (b = 0..3) of a
// 32-key block; eight consecutive ones are the B operand of O^T += V^T P^T over 16 keys in that order, so P stays in
// its lane. V goes to LDS transposed, in pieces of 8 keys in the same order (16-bit permutes on the way), so both
// operands are 16-byte LDS reads. A row of LDS is one piece longer than its values, so that lanes on consecutive rows spread
// over the banks, and every read of a tile has one address register and an immediate. Block e of O^T has columns HB n + e
// (HB blocks), whose rows in LDS follow one another. 32 queries per wave need a byte of LDS for 16 operations, which the
// LDS gives at the matrix cores' rate; 64 would need half, and twice the registers.
// Statistics as in k_attend_few. P is rounded to the cache's type once, half a step per weight: the products bound this
// form, and a second one for what the rounding leaves takes 2048 rows over 8192 positions of 7B heads from 280 to 368 us
// (f16: error against 64 bits 2.5e-4, with the second product 2.1e-4, of which the output's own rounding is nearly all).
// 2048 rows of 28 heads over 8192 positions of 4 K/V heads of 128 values, f16:
// 272 us, 780 TFLOP/s; products and the softmax's instructions share the time, 36 % and about half of a SIMD's cycles.
// Head dims above 128: 325 registers, one wave per SIMD.
constexpr int kTileThreads = 256;
constexpr int kTileWaves = kTileThreads / 64;
constexpr int kTileQueries = 32 * kTileWaves;

template <int HDP> constexpr int kTileKeys = HDP <= 128 ? 64 : 32;

template <typename T, int HDP>
__global__ __launch_bounds__(kTileThreads, HDP <= 128 ? 2 : 1) void k_attend_tile(Attend a, int group) {
    using V = Values<T>;
    using v8 = typename V::v8;
    constexpr int KT = kTileKeys<HDP>;
    constexpr int KB = KT / 32;     // key blocks of S^T
    constexpr int KC = HDP / 16;    // products per block of S^T
    constexpr int HB = HDP / 32;    // column blocks of O^T
    constexpr int CH = HDP / 8;     // pieces of a K row
    constexpr int KP = KT * CH / kTileThreads;  // pieces of K per thread
    constexpr int VG = KT / 8;      // pieces of a V column
    constexpr int V4 = HDP / 4;     // threads per piece row: four columns each
    constexpr int VT = VG * V4;     // threads that stage V
    static_assert(VT <= kTileThreads && KT <= 64 && kTileThreads % CH == 0);
    constexpr unsigned long long kAllKeys = ~0ULL >> (64 - KT);
    constexpr int KS = CH + 1, VS = VG + 1;  // pieces of a row in LDS
    __shared__ uint4 k_lds[2][KT * KS];
    __shared__ uint4 v_lds[2][HDP * VS];
    __shared__ int64_t offsets[3][KT];
    __shared__ unsigned long long there[3];
    // the keys (bits) whose V is +inf, -inf, NaN, by column and piece
    __shared__ alignas(8) uint8_t marks[2][3][HDP][8];
    __shared__ bool odd[2][kTileWaves];

    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int n = lane % 32, g = lane / 32;
    const uint32_t pairs = a.cache.n_head_kv * a.batch.n_seq;
    const uint32_t pair = blockIdx.x % pairs, split = blockIdx.x / pairs % a.splits;
    const uint32_t h = pair % a.cache.n_head_kv, s = pair / a.cache.n_head_kv;
    const Span span = sequence_span(a.batch, a.q.rows, s);
    const int queries = span.rows * group;
    // the last tile of queries, which sees most, first
    const int m0 = ((queries + kTileQueries - 1) / kTileQueries - 1 - static_cast<int>(blockIdx.x / pairs / a.splits)) * kTileQueries;
    if (m0 < 0) return;
    const int dim = static_cast<int>(a.cache.head_dim);

    const int wm = m0 + 32 * wave, m = wm + n;
    const Query query = query_of(min(m, queries - 1), group, h);
    const int64_t row = span.row0 + query.row;
    v8 q[KC];
    {
        const T* x = static_cast<const T*>(a.q.data) + row * a.q.row_stride + query.head * a.q.head_stride;
#pragma unroll
        for (int c = 0; c < KC; ++c) {
            const int d = 16 * c + 8 * g;
            uint4 y = *reinterpret_cast<const uint4*>(x + (d < dim ? d : 0));
            if (d >= dim) y = uint4{0, 0, 0, 0};
            q[c] = __builtin_bit_cast(v8, y);
        }
    }
    const auto sees = [&](int query_index) {  // slots that a query sees
        return a.causal ? slots_seen(span, min(query_index, queries - 1) / group) : span.len;
    };
    const int limit = sees(m), least = sees(wm), end = sees(m0 + kTileQueries - 1);

    const int tiles = (span.len + KT - 1) / KT;
    const int per = (tiles + static_cast<int>(a.splits) - 1) / static_cast<int>(a.splits);
    const int t0 = static_cast<int>(split) * per, t1 = min(min(tiles, t0 + per), (end + KT - 1) / KT);

    const T* k_head = static_cast<const T*>(a.cache.k) + h * a.cache.head_stride;
    const T* v_head = static_cast<const T*>(a.cache.v) + h * a.cache.head_stride;

    const auto look_up = [&](int t) {
        if (wave != 0) return;
        const int slot = t * KT + lane;
        const int page = lane < KT && slot < end ? page_of(a.cache, a.batch, s, slot) : -1;
        // of a row that is not there: any that is
        if (lane < KT) offsets[t % 3][lane] = page >= 0 ? slot_offset(a.cache, page, slot) : 0;
        const unsigned long long mask = __ballot(page >= 0);
        if (lane == 0) there[t % 3] = mask;
    };
    uint4 kr[KP];
    uint2 vr[8];
    const int v_at = 4 * (tid % V4), v_piece = tid / V4;
    const int k_at = 8 * (tid % CH);
    const T* k_from = k_head + (k_at < dim ? k_at : 0);
    const T* v_from = v_head + (v_at < dim ? v_at : 0);
    const auto fetch = [&](int t) {
        const int64_t* at = offsets[t % 3];
#pragma unroll
        for (int p = 0; p < KP; ++p) {
            kr[p] = *reinterpret_cast<const uint4*>(k_from + at[(tid + kTileThreads * p) / CH]);
        }
        if (VT == kTileThreads || tid < VT) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                vr[j] = *reinterpret_cast<const uint2*>(v_from + at[16 * (v_piece / 2) + 8 * (j / 4) + 4 * (v_piece % 2) + j % 4]);
            }
        }
    };
    const auto stage = [&](int t, auto again) __attribute__((always_inline)) {
        const int b = t % 2;
#pragma unroll
        for (int p = 0; p < KP; ++p) {
            if (k_at >= dim) kr[p] = uint4{0, 0, 0, 0};
            k_lds[b][(tid + kTileThreads * p) / CH * KS + tid % CH] = kr[p];
        }
        bool any = false;
        if (VT == kTileThreads || tid < VT) {
            const unsigned long long present = there[t % 3];
            if (present != kAllKeys || v_at >= dim) {  // what is not there must be a number: its weight is 0
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const int key = 16 * (v_piece / 2) + 8 * (j / 4) + 4 * (v_piece % 2) + j % 4;
                    if (!(present >> key & 1ULL) || v_at >= dim) vr[j] = uint2{0, 0};
                }
            }
            if constexpr (again) {
#pragma unroll
                for (int j = 0; j < 8; ++j) any |= nonfinite<T>(vr[j].x) || nonfinite<T>(vr[j].y);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t mark[3] = {0, 0, 0};
                    if (any) {
#pragma unroll
                        for (int j = 0; j < 8; ++j) take_nonfinite<T>(e < 2 ? vr[j].x : vr[j].y, e % 2, j, mark);
                    }
#pragma unroll
                    for (int k = 0; k < 3; ++k) marks[b][k][v_at + e][v_piece] = static_cast<uint8_t>(mark[k]);
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t pick = e % 2 ? 0x07060302U : 0x05040100U;
                const auto two = [&](int j) {
                    return e < 2 ? __builtin_amdgcn_perm(vr[j + 1].x, vr[j].x, pick) : __builtin_amdgcn_perm(vr[j + 1].y, vr[j].y, pick);
                };
                v_lds[b][((v_at + e) % HB * 32 + (v_at + e) / HB) * VS + v_piece] = uint4{two(0), two(2), two(4), two(6)};
            }
        }
        if constexpr (again) {
            any = __ballot(any) != 0;
            if (lane == 0) odd[b][wave] = any;
        }
    };

    float16v o[HB];
    float top, sum;
    const auto walk = [&](auto again) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < HB; ++e) {
#pragma unroll
            for (int r = 0; r < 16; ++r) o[e][r] = 0.0F;
        }
        top = -INFINITY;
        sum = 0.0F;

        if (t0 < t1) {
            look_up(t0);
            look_up(t0 + 1);
            __syncthreads();
            fetch(t0);
            stage(t0, again);
            __syncthreads();
        }
        for (int t = t0; t < t1; ++t) {
            const int b = t % 2, base = t * KT;
            if (t + 1 < t1) fetch(t + 1);
            if (t + 2 < t1) look_up(t + 2);

            float16v sc[KB];
#pragma unroll
            for (int e = 0; e < KB; ++e) {
#pragma unroll
                for (int r = 0; r < 16; ++r) sc[e][r] = 0.0F;
            }
#pragma unroll
            for (int c = 0; c < KC; ++c) {
#pragma unroll
                for (int e = 0; e < KB; ++e) {
                    const uint4 k = k_lds[b][(32 * e + n) * KS + 2 * c + g];
                    sc[e] = V::mfma(__builtin_bit_cast(v8, k), q[c], sc[e]);
                }
            }
            const unsigned long long present = there[t % 3];
            const bool hidden = base + KT > least;
            if (hidden || present != kAllKeys) {
#pragma unroll
                for (int e = 0; e < KB; ++e) {
                    // keys 32 e + 4 g + 8 (r / 4) + r % 4
                    const uint32_t here = static_cast<uint32_t>(present >> (32 * e + 4 * g));
                    const int left = limit - base - 32 * e - 4 * g;
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int key = 8 * (r / 4) + r % 4;
                        if (key >= left || !(here >> key & 1U)) sc[e][r] = -INFINITY;
                    }
                }
            }
            float most = sc[0][0];
#pragma unroll
            for (int e = 0; e < KB; ++e) {
#pragma unroll
                for (int r = 0; r < 16; ++r) most = fmaxf(most, sc[e][r]);
            }
            most = halves_max(most) * a.scale_log2 - V::kRaised;
            if (__ballot(most > top)) {
                const float now = fmaxf(top, most);
                const float shrink = now == -INFINITY ? 1.0F : share_of(top - now);
                top = now;
                sum *= shrink;
#pragma unroll
                for (int e = 0; e < HB; ++e) o[e] *= shrink;
            }
            const float ref = top == -INFINITY ? 0.0F : top;
            v8 p[KB][2];
#pragma unroll
            for (int e = 0; e < KB; ++e) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(sc[e][r], a.scale_log2, -ref));
                    sum += w;
                    p[e][r / 8][r % 8] = static_cast<T>(w);
                }
            }
#pragma unroll
            for (int c = 0; c < 2 * KB; ++c) {
#pragma unroll
                for (int e = 0; e < HB; ++e) {
                    const uint4 v = v_lds[b][(32 * e + n) * VS + 2 * c + g];
                    o[e] = V::mfma(__builtin_bit_cast(v8, v), p[c / 2][c % 2], o[e]);
                }
            }
            if (again && (odd[b][0] || odd[b][1] || odd[b][2] || odd[b][3])) {
                // what the tile's V has of infinities and NaN, staged as 0 for all waves, for the queries that see them
                unsigned long long seen = 0;
                for (int k = 0; k < KT; ++k) {
                    const int key = 16 * (k / 16) + 8 * (k % 8 / 4) + 4 * (k / 8 % 2) + k % 4;
                    seen |= static_cast<unsigned long long>(base + key < limit && (present >> key & 1ULL)) << k;
                }
#pragma unroll
                for (int e = 0; e < HB; ++e) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int d = HB * (8 * (r / 4) + 4 * g + r % 4) + e;
                        const auto any = [&](int k) {
                            return (*reinterpret_cast<const unsigned long long*>(marks[b][k][d]) & seen) != 0;
                        };
                        o[e][r] = with_nonfinite(o[e][r], any(0), any(1), any(2));
                        asm volatile("" ::: "memory");  // one column's marks at a time: the sums leave few registers
                    }
                }
            }
            if (t + 1 < t1) stage(t + 1, again);
            __syncthreads();
        }
        if (again || t0 >= t1) return false;
        float not_finite = 0.0F;
#pragma unroll
        for (int e = 0; e < HB; ++e) {
#pragma unroll
            for (int r = 0; r < 16; ++r) not_finite = fmaf(o[e][r], 0.0F, not_finite);
        }
        const bool any = __ballot(not_finite != not_finite) != 0;
        if (lane == 0) odd[0][wave] = any;
        __syncthreads();
        return odd[0][0] || odd[0][1] || odd[0][2] || odd[0][3];
    };
    // as in k_attend_few: where some sum is not finite at the end, the work-group walks its tiles again
    if (walk(std::false_type{})) {
        __syncthreads();
        walk(std::true_type{});
    }

    if (m >= queries) return;
    const Sums seen = lowered<T>(top, halves_sum(sum));
    const float l = seen.l;
    const int64_t at = row * a.q.heads + query.head, all = static_cast<int64_t>(a.q.rows) * a.q.heads;
    const bool whole = a.splits == 1;
    if (g == 0) {
        if (!whole) *reinterpret_cast<float2*>(a.marks + 2 * (split * all + at)) = float2{seen.top, l};
        else if (a.lse) a.lse[at] = seen.top * kLn2 + logf(l);
    }
    if (!whole && l == 0.0F) return;  // nothing seen: the join does not read it
    const float scale = seen.unit * (whole ? (l == 0.0F ? 0.0F : 1.0F / l) : 1.0F);
    // rows 8 b + 4 g + r of the blocks: 4 HB consecutive columns, four at a time
#pragma unroll
    for (int b = 0; b < 4; ++b) {
#pragma unroll
        for (int f = 0; f < HB; ++f) {
            const int d = HB * (8 * b + 4 * g) + 4 * f;
            if (d >= dim) continue;
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = o[(4 * f + e) % HB][4 * b + (4 * f + e) / HB] * scale;
            if (whole) {
                T* to = static_cast<T*>(a.out.data) + row * a.out.row_stride + query.head * a.out.head_stride + d;
                const T y[4] = {static_cast<T>(x[0]), static_cast<T>(x[1]), static_cast<T>(x[2]), static_cast<T>(x[3])};
                __builtin_memcpy(__builtin_assume_aligned(to, 8), y, 8);
            } else {
                *reinterpret_cast<float4v*>(a.partial + (split * all + at) * dim + d) = float4v{x[0], x[1], x[2], x[3]};
            }
        }
    }
}

// Joins the splits of a row and head: 32 (head dims up to 128: 16) threads hold a partial's columns 8 each, `takers` such
// groups take every takers-th split of a row and head, and a work-group has as many rows and heads as that leaves room for.
// Rows of no sequence are left as they are. Latency bounds short joins, so a thread's first partial and marks are requested
// before anything else is known; what no split wrote is not used. 720 rows and heads of 22 splits: 7.4 us.
constexpr int kJoinThreads = 256;

__global__ __launch_bounds__(kJoinThreads) void k_attend_join(Attend a, int takers) {
    __shared__ float part[16][kMaxHeadDim];
    __shared__ float2 part_mark[16];
    const int64_t all = static_cast<int64_t>(a.q.rows) * a.q.heads;
    const int dim = static_cast<int>(a.cache.head_dim), splits = static_cast<int>(a.splits);
    const int wide = dim <= 128 ? 16 : 32, unit = threadIdx.x / wide, d = threadIdx.x % wide * 8;
    const int taker = unit % takers, joins = kJoinThreads / wide / takers;
    const int64_t at = min(blockIdx.x * static_cast<int64_t>(joins) + unit / takers, all - 1);
    const float2* marks = reinterpret_cast<const float2*>(a.marks) + at;
    float2 mark{-INFINITY, 0.0F};
    float y[8] = {};
    if (taker < splits) {
        mark = marks[taker * all];
        if (d < dim) load(a.partial, (taker * all + at) * dim + d, kF32, y);
    }
    const int row = static_cast<int>(at / a.q.heads), head = static_cast<int>(at - row * static_cast<int64_t>(a.q.heads));
    Span span;
    const bool owned = sequence_of(a.batch, a.q.rows, row, &span) >= 0 && blockIdx.x * static_cast<int64_t>(joins) + unit / takers < all;

    float x[8] = {}, top = -INFINITY, l = 0.0F;
    if (owned) {
        for (int s = taker; s < splits; s += takers) {
            if (s != taker) {
                mark = marks[s * all];
                if (d < dim) load(a.partial, (s * all + at) * dim + d, kF32, y);
            }
            if (mark.y == 0.0F) continue;  // nothing seen: the split wrote no sums
            const float high = fmaxf(top, mark.x), before = split_share(top, l, high), share = split_share(mark.x, mark.y, high);
            top = high;
            l = l * before + mark.y * share;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = x[e] * before + y[e] * share;
        }
    }
    if (takers > 1) {
        if (d < dim) store(part[unit], d, kF32, x);
        if (d == 0) part_mark[unit] = float2{top, l};
        __syncthreads();
        if (taker != 0 || !owned) return;
        for (int t = 0; t < takers; ++t) top = fmaxf(top, part_mark[unit + t].x);
        l = 0.0F;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.0F;
        for (int t = 0; t < takers; ++t) {
            const float2 other = part_mark[unit + t];
            const float share = split_share(other.x, other.y, top);
            if (other.y == 0.0F) continue;
            l += other.y * share;
            if (d < dim) {
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] += part[unit + t][d + e] * share;
            }
        }
    }
    if (!owned) return;
    if (d == 0 && a.lse) a.lse[at] = top * kLn2 + logf(l);
    if (d >= dim) return;
    const float scale = l == 0.0F ? 0.0F : 1.0F / l;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] *= scale;
    store(a.out.data, row * a.out.row_stride + head * a.out.head_stride + d, a.out.type, x);
}

// ---------------------------------------------------------------- attention weights

// weights[slot] += sum over the step's queries of a K/V head of exp(scale q k - lse): the columns of the probabilities,
// summed. A wave owns 16 U slots, whose K rows stay in registers as A operands of 16x16x32 products, and goes over the
// queries. Each sum has one owner and one order, so results do not depend on the launch.

constexpr int kWeighThreads = 256;
constexpr int kWeighWaves = kWeighThreads / 64;
constexpr int kFewWeighSlots = 32;  // of a wave

// The K rows of a wave's slots, zeros beyond head_dim; where their weights lie, -1 for slots that are not there.
template <typename T, int U, int KC>
__device__ __forceinline__ void weighed_rows(const Weigh& a, uint32_t s, uint32_t h, int len, int base,
                                             typename Values<T>::v8 (&k)[U][KC], int64_t (&index)[U]) {
    const int i = threadIdx.x % 16, g = threadIdx.x % 64 / 16;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int slot = base + 16 * u + i;
        const int page = slot < len ? page_of(a.cache, a.batch, s, slot) : -1;
        index[u] = page >= 0 ? slot_index(a.cache, page, h, slot) : -1;
        const T* row = static_cast<const T*>(a.cache.k) + h * a.cache.head_stride + (page >= 0 ? slot_offset(a.cache, page, slot) : 0);
#pragma unroll
        for (int c = 0; c < KC; ++c) k[u][c] = row_piece<T>(row, 32 * c + 8 * g, static_cast<int>(a.cache.head_dim));
    }
}

// A query's lse in base 2 and 2^-(what its rounding left), which goes into the sums: without it every weight of the query
// has the rounding's error, 2^-24 of an lse that may be large.
__device__ __forceinline__ float2 lse_base2(float lse) {
    constexpr float kLog2eRest = 1.92596303e-8F;  // log2(e) - kLog2e
    const float ref = lse * kLog2e, rest = fmaf(lse, kLog2eRest, fmaf(lse, kLog2e, -ref));
    return float2{ref, fabsf(lse) < INFINITY ? exp2f(-rest) : 1.0F};
}

// sum += the weights of 16 queries (lane i's: its lse in base 2, the slots it sees) for the wave's slots from `base`. All
// seen: every query sees every one of the slots.
template <typename T, bool ALL_SEEN, int U, int KC>
__device__ __forceinline__ void weigh_queries(const Weigh& a, int base, const typename Values<T>::v8 (&k)[U][KC],
                                              const typename Values<T>::v8 (&q)[KC], float2 ref, int limit, float4v (&sum)[U]) {
    const int g = threadIdx.x % 64 / 16;
    float4v sc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sc[u] = float4v{0.0F, 0.0F, 0.0F, 0.0F};
#pragma unroll
    for (int c = 0; c < KC; ++c) {
#pragma unroll
        for (int u = 0; u < U; ++u) sc[u] = Values<T>::mfma(k[u][c], q[c], sc[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float p = __builtin_amdgcn_exp2f(fmaf(sc[u][r], a.scale_log2, -ref.x));
            sum[u][r] = fmaf(ALL_SEEN || base + 16 * u + 4 * g + r < limit ? p : 0.0F, ref.y, sum[u][r]);
        }
    }
}

// Few queries: the K rows' bytes bound the call. 32 slots per wave, the queries' operands straight from memory. Eight rows
// of 40 heads over 2177 positions: 13 us, 2.8 TB/s of K and weights.
template <typename T, int HDP>
__global__ __launch_bounds__(kWeighThreads) void k_weigh_few(Weigh a, int group, int blocks) {
    using v8 = typename Values<T>::v8;
    constexpr int KC = HDP / 32, U = kFewWeighSlots / 16;
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int i = lane % 16, g = lane / 16;
    const uint32_t pair = blockIdx.x / blocks;
    const uint32_t h = pair % a.cache.n_head_kv, s = pair / a.cache.n_head_kv;
    const Span span = sequence_span(a.batch, a.q.rows, s);
    const int base = (static_cast<int>(blockIdx.x % blocks) * kWeighWaves + wave) * kFewWeighSlots;
    const int queries = span.rows * group;
    if (base >= span.len || queries == 0) return;

    int64_t index[U];
    v8 k[U][KC];
    weighed_rows<T>(a, s, h, span.len, base, k, index);
    float4v sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] = float4v{0.0F, 0.0F, 0.0F, 0.0F};
    // from the first row that sees slot `base`
    for (int m0 = a.causal ? rows_before(span, base) * group / 16 * 16 : 0; m0 < queries; m0 += 16) {
        const Query query = query_of(min(m0 + i, queries - 1), group, h);
        const int64_t row = span.row0 + query.row;
        const T* x = static_cast<const T*>(a.q.data) + row * a.q.row_stride + query.head * a.q.head_stride;
        v8 q[KC];
#pragma unroll
        for (int c = 0; c < KC; ++c) q[c] = row_piece<T>(x, 32 * c + 8 * g, static_cast<int>(a.cache.head_dim));
        const float lse = a.lse[row * a.q.heads + query.head];
        // a row that saw nothing adds nothing
        const int limit = m0 + i >= queries || lse == -INFINITY ? 0 : a.causal ? slots_seen(span, query.row) : span.len;
        weigh_queries<T, false>(a, base, k, q, lse_base2(lse), limit, sum);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float x = sum[u][r];
#pragma unroll
            for (int o = 1; o < 16; o *= 2) x += __shfl_xor(x, o);
            const int64_t to = __shfl(index[u], 4 * g + r);
            if (i == 0 && to >= 0) a.cache.weights[to] += x;
        }
    }
}

// Many queries: products and exponentials bound the call, after the traffic of Q, which every work-group reads for its
// slots. So a work-group has 256 slots (128 of wide heads) and stages 64 queries at a time in LDS for its four waves,
// double-buffered; where that leaves the chip idle, the queries are divided into `splits` parts, whose sums go to the
// workspace and are added in order. 1777 rows of 28 heads over 3999 positions: 77 us and 4 for the sum, 500 TFLOP/s.
template <int HDP> constexpr int kWeighTiles = HDP <= 128 ? 4 : 2;  // 16-slot tiles of a wave

template <typename T, int HDP>
__global__ __launch_bounds__(kWeighThreads, 2) void k_weigh_many(Weigh a, int group, int blocks) {
    using v8 = typename Values<T>::v8;
    constexpr int KC = HDP / 32, U = kWeighTiles<HDP>, CH = HDP / 8, QS = CH + 1, QT = 64, KP = QT * CH / kWeighThreads;
    __shared__ uint4 q_lds[2][QT * QS];
    __shared__ float2 refs[2][QT];
    __shared__ int limits[2][QT];
    const int tid = threadIdx.x, lane = tid % 64, wave = tid / 64;
    const int i = lane % 16, g = lane / 16;
    const uint32_t split = blockIdx.x / blocks % a.splits, pair = blockIdx.x / blocks / a.splits;
    const uint32_t h = pair % a.cache.n_head_kv, s = pair / a.cache.n_head_kv;
    const Span span = sequence_span(a.batch, a.q.rows, s);
    const int group_base = static_cast<int>(blockIdx.x % blocks) * kWeighWaves * 16 * U, base = group_base + wave * 16 * U;
    const int queries = span.rows * group;
    if (group_base >= span.len) return;
    const int dim = static_cast<int>(a.cache.head_dim);

    int64_t index[U];
    v8 k[U][KC];
    weighed_rows<T>(a, s, h, span.len, base, k, index);

    // the split's queries, in whole tiles, from the first row that sees the work-group's first slot
    const int from = a.causal ? rows_before(span, group_base) * group / QT : 0;
    const int tiles = (queries + QT - 1) / QT - from, per = (tiles + static_cast<int>(a.splits) - 1) / static_cast<int>(a.splits);
    const int t0 = from + min(static_cast<int>(split) * per, tiles), t1 = from + min(static_cast<int>(split + 1) * per, tiles);

    // the thread's pieces of a tile: rows tid / CH + p (256 / CH), advanced by a tile at a time
    uint4 staged[KP];
    int at_row[KP], at_head[KP];
    const int row_step = QT / group, head_step = QT - row_step * group;
#pragma unroll
    for (int p = 0; p < KP; ++p) {
        const Query query = query_of(QT * t0 + (tid + kWeighThreads * p) / CH, group, 0);
        at_row[p] = query.row;
        at_head[p] = query.head;
    }
    const auto fetch = [&] {
#pragma unroll
        for (int p = 0; p < KP; ++p) {
            const int64_t row = span.row0 + min(at_row[p], span.rows - 1), head = static_cast<int>(h) * group + at_head[p];
            const int d = 8 * (tid % CH);
            staged[p] = __builtin_bit_cast(uint4, row_piece<T>(static_cast<const T*>(a.q.data) + row * a.q.row_stride +
                                                                   head * a.q.head_stride, d, dim));
            at_row[p] += row_step;
            at_head[p] += head_step;
            if (at_head[p] >= group) at_head[p] -= group, ++at_row[p];
        }
    };
    const auto stage = [&](int t) {
        const int b = t % 2;
#pragma unroll
        for (int p = 0; p < KP; ++p) q_lds[b][(tid + kWeighThreads * p) / CH * QS + tid % CH] = staged[p];
        if (tid < QT) {
            const int m = QT * t + tid;
            const Query query = query_of(min(m, queries - 1), group, h);
            const float lse = a.lse[(span.row0 + query.row) * static_cast<int64_t>(a.q.heads) + query.head];
            // a row that saw nothing adds nothing
            limits[b][tid] = m >= queries || lse == -INFINITY ? 0 : a.causal ? slots_seen(span, query.row) : span.len;
            refs[b][tid] = lse_base2(lse);
        }
    };

    float4v sum[U];
#pragma unroll
    for (int u = 0; u < U; ++u) sum[u] = float4v{0.0F, 0.0F, 0.0F, 0.0F};
    if (t0 < t1) {
        fetch();
        stage(t0);
    }
    __syncthreads();
    for (int t = t0; t < t1; ++t) {
        const int b = t % 2;
        if (t + 1 < t1) fetch();
        const auto weigh = [&](auto all_seen) {
#pragma unroll
            for (int w = 0; w < QT / 16; ++w) {
                v8 q[KC];
#pragma unroll
                for (int c = 0; c < KC; ++c) q[c] = __builtin_bit_cast(v8, q_lds[b][(16 * w + i) * QS + 4 * c + g]);
                weigh_queries<T, all_seen>(a, base, k, q, refs[b][16 * w + i], limits[b][16 * w + i], sum);
            }
        };
        if (__ballot(limits[b][lane % QT] < base + 16 * U) == 0) weigh(std::true_type{});
        else weigh(std::false_type{});
        if (t + 1 < t1) stage(t + 1);
        __syncthreads();
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float x = sum[u][r];
#pragma unroll
            for (int o = 1; o < 16; o *= 2) x += __shfl_xor(x, o);
            const int64_t to = __shfl(index[u], 4 * g + r);
            const int slot = base + 16 * u + 4 * g + r;
            if (i != 0 || slot >= span.len) continue;
            if (a.splits > 1) a.partial[(static_cast<int64_t>(split) * a.cache.n_head_kv * a.batch.n_seq + pair) * a.batch.max_length + slot] = x;
            else if (to >= 0) a.cache.weights[to] += x;
        }
    }
}

__global__ __launch_bounds__(kWeighThreads) void k_weigh_join(Weigh a, int blocks) {
    const uint32_t pair = blockIdx.x / blocks;
    const uint32_t h = pair % a.cache.n_head_kv, s = pair / a.cache.n_head_kv;
    const int slot = static_cast<int>(blockIdx.x % blocks) * kWeighThreads + threadIdx.x;
    if (slot >= span_length(a.batch, s)) return;
    const int page = page_of(a.cache, a.batch, s, slot);
    if (page < 0) return;
    const int64_t all = static_cast<int64_t>(a.cache.n_head_kv) * a.batch.n_seq;
    float x = 0.0F;
    for (uint32_t n = 0; n < a.splits; ++n) x += a.partial[(n * all + pair) * a.batch.max_length + slot];
    a.cache.weights[slot_index(a.cache, page, h, slot)] += x;
}

// ---------------------------------------------------------------- cutting a cache

// What stays of a K/V head's slots: the `budget` first in the order (protected, heavier, lower slot). One work-group per
// sequence and K/V head turns the order into 32-bit keys in LDS, finds the budget-th largest by its digits (counts of 2048
// bins: 11, 11 and 10 bits), and lists the slots below the budget that go and those above that stay, both ascending: the
// latter move into the former, the others stay where they are. Integer counts and scans only, so the lists do not depend
// on the launch. Latency bounds it: the passes over weights and positions have BATCH slots per thread in flight, and
// read caches of up to 8192 slots once. 16 K/V heads of 16384 slots 23 us, 32 of 4097 12.3 us, of which the counts are half.
constexpr int kSelectThreads = 1024;
constexpr int kSelectBins = 2048;
constexpr int kSelectRun = 63;  // most slots of a thread's run, bits of a word
static_assert(kSelectRun * kSelectThreads <= static_cast<int>(kSlotStep));
constexpr int kSelectFew = 8192, kSelectMany = 36864;  // keys in LDS; later slots' are computed again where they are used

// Order of weights as unsigned integers, 1 for NaN (nothing is lighter), 0 free.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 1U;
    const uint32_t b = __float_as_uint(w + 0.0F);  // -0 is 0
    return b >> 31 ? ~b : b | 0x80000000U;
}

// Inclusive sum over the lanes of a wave: within rows of 16, then from row to row.
__device__ __forceinline__ int wave_sum_upto(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // row_shr 1, 2, 4, 8
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // the last of rows 0 and 2 to rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);  // that of row 1 to rows 2 and 3
    return v;
}

// Exclusive sum over the work-group of two counts; `all` gets their totals.
__device__ __forceinline__ int2 exclusive_sum(int2 v, int2* waves, int2* all) {
    const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const int2 x{wave_sum_upto(v.x), wave_sum_upto(v.y)};
    __syncthreads();
    if (lane == 63) waves[wave] = x;
    __syncthreads();
    int2 before{0, 0}, sum{0, 0};
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) {
        const int2 y = waves[w];
        if (w == wave) before = sum;
        sum.x += y.x;
        sum.y += y.y;
    }
    *all = sum;
    return int2{before.x + x.x - v.x, before.y + x.y - v.y};
}

template <int CAP, int BATCH>
__global__ __launch_bounds__(kSelectThreads) void k_evict_select(Evict a) {
    static_assert(2 * BATCH * kSelectThreads <= static_cast<int>(kSlotStep));
    constexpr bool kStay = CAP <= BATCH * kSelectThreads;  // the first batch, in registers from pass to pass
    __shared__ uint32_t keys[CAP];
    __shared__ uint32_t bins[kSelectBins];
    __shared__ int2 waves[kSelectThreads / 64];
    __shared__ uint32_t found[2];
    const int tid = threadIdx.x;
    const uint32_t h = blockIdx.x % a.cache.n_head_kv, s = blockIdx.x / a.cache.n_head_kv;
    int32_t* list = a.lists + static_cast<int64_t>(blockIdx.x) * (1 + 2 * static_cast<int64_t>(a.width));
    const int len = span_length(a.batch, s), budget = a.budget;
    if (len <= budget) {
        if (tid == 0) list[0] = -1;
        return;
    }
    // where the weights and positions of the thread's next slots lie, -1 on absent pages
    const auto look_up = [&](int t0, int64_t (&at)[BATCH]) {
        int page[BATCH];
#pragma unroll
        for (int e = 0; e < BATCH; ++e) page[e] = page_of(a.cache, a.batch, s, min(t0 + e * kSelectThreads, len - 1));
#pragma unroll
        for (int e = 0; e < BATCH; ++e) {
            const int t = min(t0 + e * kSelectThreads, len - 1);
            at[e] = page[e] >= 0 ? slot_index(a.cache, page[e], h, t) : -1;
        }
    };

    // the newest position
    int newest = INT32_MIN;
    int64_t first_at[kStay ? BATCH : 1];
    int first_p[kStay ? BATCH : 1];
    float first_w[kStay ? BATCH : 1];
    for (int t0 = tid; t0 < len; t0 += BATCH * kSelectThreads) {
        int64_t at[BATCH];
        look_up(t0, at);
        int p[BATCH];
#pragma unroll
        for (int e = 0; e < BATCH; ++e) p[e] = a.cache.positions[max(at[e], static_cast<int64_t>(0))];
        if constexpr (kStay) {
            if (t0 == tid) {
#pragma unroll
                for (int e = 0; e < BATCH; ++e) {
                    first_at[e] = at[e];
                    first_p[e] = p[e];
                    first_w[e] = a.cache.weights[max(at[e], static_cast<int64_t>(0))];
                }
            }
        }
#pragma unroll
        for (int e = 0; e < BATCH; ++e) newest = max(newest, at[e] >= 0 ? p[e] : INT32_MIN);
    }
#pragma unroll
    for (int o = 32; o; o /= 2) newest = max(newest, __shfl_xor(newest, o));
    if (tid % 64 == 0) waves[tid / 64].x = newest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) newest = max(newest, waves[w].x);
    const int64_t recent = static_cast<int64_t>(newest) - a.recent;

    // Protected slots have the largest key, and so have an absent page's slots below the budget, whose place nothing can
    // take; its others have 0. Where that is more than the budget (`crowded`), protected slots are in the order of their
    // weights and the others at 0.
    const auto key_of = [&](int t, int64_t at, int p, float w, bool crowded, bool& keep) {
        keep = at < 0 ? t < budget : p < a.first || p > recent;
        if (at < 0 || (keep && !crowded)) return keep ? 0xFFFFFFFFU : 0U;
        return crowded && !keep ? 0U : weight_key(w);
    };
    const auto fill = [&](bool crowded) {
        int held = 0;
        for (int t0 = tid; t0 < len; t0 += BATCH * kSelectThreads) {
            int64_t at[BATCH];
            int p[BATCH];
            float w[BATCH];
            if (kStay && t0 == tid) {
#pragma unroll
                for (int e = 0; e < BATCH; ++e) {
                    const int f = kStay ? e : 0;
                    at[e] = first_at[f], p[e] = first_p[f], w[e] = first_w[f];
                }
            } else {
                look_up(t0, at);
#pragma unroll
                for (int e = 0; e < BATCH; ++e) {
                    p[e] = a.cache.positions[max(at[e], static_cast<int64_t>(0))];
                    w[e] = a.cache.weights[max(at[e], static_cast<int64_t>(0))];
                }
            }
#pragma unroll
            for (int e = 0; e < BATCH; ++e) {
                const int t = t0 + e * kSelectThreads;
                if (t >= len) continue;
                bool keep;
                const uint32_t k = key_of(t, at[e], p[e], w[e], crowded, keep);
                held += keep;
                if (t < CAP) keys[t] = k;
            }
        }
        return held;
    };
    int2 all;
    exclusive_sum(int2{fill(false), 0}, waves, &all);
    const bool crowded = all.x >= budget;
    if (crowded) fill(true);
    const auto key_at = [&](int t) {
        if (t < CAP) return keys[t];
        const int page = page_of(a.cache, a.batch, s, t);
        const int64_t at = page >= 0 ? slot_index(a.cache, page, h, t) : -1;
        bool keep;
        return key_of(t, at, at < 0 ? 0 : a.cache.positions[at], at < 0 ? 0.0F : a.cache.weights[at], crowded, keep);
    };

    uint32_t prefix = 0, mask = 0;
    int need = budget;
    for (int shift = 21; shift >= 0; shift -= shift == 21 ? 11 : 10) {  // 21, 10, 0
        const uint32_t digit = shift ? 2047U : 1023U;
        for (int e = tid; e < kSelectBins; e += kSelectThreads) bins[e] = 0;
        __syncthreads();
        const auto count = [&](uint32_t k) {
            if ((k & mask) == prefix) atomicAdd(&bins[k >> shift & digit], 1U);
        };
        if (len <= CAP) {
#pragma unroll 8
            for (int t = tid; t < len; t += kSelectThreads) count(keys[t]);
        } else {
            for (int t = tid; t < len; t += kSelectThreads) count(key_at(t));
        }
        __syncthreads();
        // thread l has bins 2047 - 2 l and 2046 - 2 l: those of larger keys come first
        const int hi = static_cast<int>(bins[kSelectBins - 1 - 2 * tid]), lo = static_cast<int>(bins[kSelectBins - 2 - 2 * tid]);
        const int above = exclusive_sum(int2{hi + lo, 0}, waves, &all).x;
        if (above < need && above + hi + lo >= need) {
            const bool upper = above + hi >= need;
            found[0] = kSelectBins - (upper ? 1 : 2) - 2 * tid;
            found[1] = upper ? above : above + hi;
        }
        __syncthreads();
        prefix |= found[0] << shift;
        mask |= digit << shift;
        need -= static_cast<int>(found[1]);
    }

    // `need` of the slots with key `prefix` stay, the lowest. A thread owns a run of slots (an odd number, for the LDS
    // banks) as bits of two words; sequences beyond 63 slots per thread take several rounds.
    int equals = 0;      // of earlier rounds
    int2 moves{0, 0};
    for (int round = 0; round < len; round += kSelectRun * kSelectThreads) {
        const int upto = min(len - round, kSelectRun * kSelectThreads);
        const int run = ((upto + kSelectThreads - 1) / kSelectThreads) | 1;
        const int t0 = round + min(tid * run, upto), count = min(run, round + upto - t0);
        unsigned long long larger = 0, equal = 0;
        const auto compare = [&](int e, uint32_t k) {
            larger |= static_cast<unsigned long long>(k > prefix) << e;
            equal |= static_cast<unsigned long long>(k == prefix) << e;
        };
        if (len <= CAP) {
#pragma unroll 8
            for (int e = 0; e < count; ++e) compare(e, keys[t0 + e]);
        } else {
            for (int e = 0; e < count; ++e) compare(e, key_at(t0 + e));
        }
        int room = need - equals - exclusive_sum(int2{__popcll(equal), 0}, waves, &all).x;
        equals += all.x;
        unsigned long long stays = larger;
        for (unsigned long long left = equal; left && room > 0; left &= left - 1, --room) stays |= left & -left;
        const int below = clamped(budget - t0, 0, count);  // of the run
        const unsigned long long inside = (1ULL << below) - 1, owned = (1ULL << count) - 1;
        unsigned long long goes = ~stays & inside, comes = stays & owned & ~inside;
        const int2 before = exclusive_sum(int2{__popcll(goes), __popcll(comes)}, waves, &all);
        // the lists hold what a cache that nobody else writes can need
        for (int n = moves.x + before.x; goes && n < a.width; goes &= goes - 1) list[1 + n++] = t0 + __ffsll(goes) - 1;
        for (int n = moves.y + before.y; comes && n < a.width; comes &= comes - 1) list[1 + a.width + n++] = t0 + __ffsll(comes) - 1;
        moves.x += all.x;
        moves.y += all.y;
    }
    if (tid == 0) list[0] = min(min(moves.x, moves.y), a.width);
}

// 16 threads per moving position: its K and V rows, its weight and its position. 16 K/V heads, 16384 slots cut to 2048:
// 7.8 us, 3.8 TB/s.
constexpr int kMoveThreads = 256;
constexpr int kMoveSlots = 32;  // of a work-group

__global__ __launch_bounds__(kMoveThreads) void k_evict_move(Evict a, int chunks) {
    const uint32_t pair = blockIdx.x / chunks;
    const uint32_t h = pair % a.cache.n_head_kv, s = pair / a.cache.n_head_kv;
    const int chunk = static_cast<int>(blockIdx.x % chunks);
    const int32_t* list = a.lists + static_cast<int64_t>(pair) * (1 + 2 * static_cast<int64_t>(a.width));
    const int count = list[0];
    if (count < 0) return;
    if (h == 0 && chunk == 0 && threadIdx.x == 0) a.batch.lengths[s] = a.budget;
    const int part = threadIdx.x % 16;
    for (int n = chunk * kMoveSlots + threadIdx.x / 16; n < min(count, (chunk + 1) * kMoveSlots); n += kMoveThreads / 16) {
        const int to = list[1 + n], from = list[1 + a.width + n];
        const int to_page = page_of(a.cache, a.batch, s, to), from_page = page_of(a.cache, a.batch, s, from);
        if (to_page < 0 || from_page < 0) continue;
        const int64_t x = slot_offset(a.cache, from_page, from) + h * a.cache.head_stride;
        const int64_t y = slot_offset(a.cache, to_page, to) + h * a.cache.head_stride;
        uint16_t* k = static_cast<uint16_t*>(a.cache.k);
        uint16_t* v = static_cast<uint16_t*>(a.cache.v);
        for (int d = 8 * part; d < static_cast<int>(a.cache.head_dim); d += 128) {
            const uint4 kx = *reinterpret_cast<const uint4*>(k + x + d), vx = *reinterpret_cast<const uint4*>(v + x + d);
            *reinterpret_cast<uint4*>(k + y + d) = kx;
            *reinterpret_cast<uint4*>(v + y + d) = vx;
        }
        if (part == 0) {
            const int64_t i = slot_index(a.cache, from_page, h, from), j = slot_index(a.cache, to_page, h, to);
            a.cache.weights[j] = a.cache.weights[i];
            a.cache.positions[j] = a.cache.positions[i];
        }
    }
}

// ---------------------------------------------------------------- launches

bool by_eights(const Rows& x) {
    return reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.row_stride % 8 == 0 && x.head_stride % 8 == 0 &&
           x.head_dim % 8 == 0;
}

// Long steps: as many rows per work-group, four at most, as give every thread a unit (4096 rows of 48 heads: 17.1 us with
// one row, 17.6 with four; 16384 rows 69 and 79). Short ones: one row, its units over up to `tasks` / 256 work-groups, since
// the call's time is the time of one work-group.
struct RowGrid {
    dim3 grid;
    int rows;
};

RowGrid row_grid(uint32_t rows, uint64_t tasks) {
    if (rows >= kComputeUnits * kRotateRows) {
        const uint64_t fit = (kRotateThreads + tasks - 1) / tasks;
        const uint32_t per = static_cast<uint32_t>(fit < kRotateRows ? fit : kRotateRows);
        return {dim3((rows + per - 1) / per), static_cast<int>(per)};
    }
    const uint64_t parts = (tasks + kRotateThreads - 1) / kRotateThreads;
    return {dim3(rows, static_cast<uint32_t>(parts < 64 ? parts : 64)), 1};
}

}  // namespace

hipError_t launch_rotate(const Rotation& r, const Rows& x, const int32_t* positions, const Rows& y, hipStream_t stream) {
    const bool wide = by_eights(x) && by_eights(y) && r.n_rot % 16 == 0;
    const uint64_t units = (r.n_rot / 2 + (x.head_dim - r.n_rot)) / (wide ? 8 : 1);
    const RowGrid g = row_grid(x.rows, x.heads * units);
    // more than the 32 MB of the L2 caches is written past them: 4096 rows of 48 heads of bf16 values 17 us, 23 through them
    const bool past = static_cast<uint64_t>(y.rows) * y.heads * y.head_dim * (y.type == kF32 ? 4 : 2) > (32U << 20);
    return launch(wide ? past ? k_rotate<8, true> : k_rotate<8, false> : k_rotate<1, false>, g.grid, dim3(kRotateThreads),
                  stream, r, x, positions, y, g.rows);
}

hipError_t launch_append(const Rotation* rotation, const Cache& c, const Batch& b, const Rows& k, const Rows& v,
                         const int32_t* positions, hipStream_t stream) {
    const Rotation r = rotation ? *rotation : Rotation{};
    const bool wide = by_eights(k) && by_eights(v) && r.n_rot % 16 == 0;
    const uint64_t units = (r.n_rot / 2 + (k.head_dim - r.n_rot) + v.head_dim) / (wide ? 8 : 1) + 1;
    const RowGrid g = row_grid(k.rows, c.n_head_kv * units);
    return launch(wide ? k_append<8> : k_append<1>, g.grid, dim3(kRotateThreads), stream, r, c, b, k, v, positions, g.rows);
}

namespace {

// Queries (rows times the heads of a K/V head) of a sequence up to which the waves of a work-group divide its keys: 16,
// one tile of scores, and 32 where there are so many positions that the bytes of K and V alone count (21 queries, 32 K/V
// heads of sequences of 30000 positions: 95 us, 116 on tiles; of 4000: 29, 26 on tiles).
uint32_t few_queries(const Cache& c, const Batch& b) {
    return c.head_dim <= 128 && static_cast<uint64_t>(c.n_head_kv) * b.n_seq * b.max_length >= (1U << 19) ? 32 : 16;
}

// How a step's attention is divided: by the most queries that a sequence may have.
struct Tiling {
    uint32_t queries;  // of a work-group
    uint32_t keys;     // that its waves take at a time, all together
    uint64_t groups;   // work-groups per split
};

Tiling tiling(const Cache& c, const Batch& b, uint32_t group) {
    const uint64_t most = static_cast<uint64_t>(b.max_rows) * group;
    Tiling t;
    if (most <= few_queries(c, b)) {
        t.queries = most <= 16 ? 16 : 32;
        t.keys = (c.head_dim > 128 ? kFewWaves<256> : kFewWaves<128>) * kFewKeys;
    } else {
        t.queries = kTileQueries;
        t.keys = c.head_dim <= 128 ? kTileKeys<128> : kTileKeys<256>;
    }
    t.groups = (most + t.queries - 1) / t.queries * c.n_head_kv * b.n_seq;
    return t;
}

template <typename T, int HDP>
hipError_t attend_of(const Attend& a, hipStream_t stream) {
    const int group = static_cast<int>(a.q.heads / a.cache.n_head_kv);
    const Tiling t = tiling(a.cache, a.batch, a.q.heads / a.cache.n_head_kv);
    const uint64_t groups = t.groups * a.splits;
    if (groups > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    const dim3 grid(static_cast<uint32_t>(groups)), few(64 * kFewWaves<HDP>);
    if (t.queries == kTileQueries) return launch(k_attend_tile<T, HDP>, grid, dim3(kTileThreads), stream, a, group);
    if constexpr (HDP <= 128) {
        if (t.queries == 32) return launch(k_attend_few<T, HDP, 2>, grid, few, stream, a, group);
    }
    return launch(k_attend_few<T, HDP, 1>, grid, few, stream, a, group);
}

template <typename T>
hipError_t attend(const Attend& a, hipStream_t stream) {
    if (a.cache.head_dim <= 64) return attend_of<T, 64>(a, stream);
    if (a.cache.head_dim <= 128) return attend_of<T, 128>(a, stream);
    return attend_of<T, 256>(a, stream);
}

}  // namespace

uint32_t attend_splits(const Cache& c, const Batch& b, uint32_t group) {
    const Tiling t = tiling(c, b, group);
    if (t.groups == 0) return 1;
    // Rounds of keys in a row set the time, counted in halves: a work-group's beginning and end take about three halves,
    // the join four (of 256 keys; eight of a tile's 64). Work-groups that run at once: one per compute unit of the
    // few-query form and of head dims above 128, two of the other tiles (two sequences of 18624 positions, 144 queries of
    // 256: 43 us in 64 splits, 56 in the 117 of two rounds). No splits, or so many as fill the chip once, or, of long
    // few-query calls, twice where that costs little, and 128 at most, for the join: the second rounds even out sequences
    // of different lengths (eight rows over up to 32701 positions 104 us, 133 in one round; 32 K/V heads of sequences of
    // 4000, equal: 22 in one, 29 in two short ones).
    const bool few = t.queries != kTileQueries;
    const uint64_t resident = (few || c.head_dim > 128 ? 1 : 2) * kComputeUnits, least = t.queries <= 16 ? 1 : 2;
    if (t.groups >= resident) return 1;
    const uint64_t rounds = (b.max_length + t.keys - 1) / t.keys;
    uint64_t best = 1, cost = 2 * rounds + 3;
    for (uint64_t fill = 1; fill <= (few ? 2 : 1); ++fill) {
        const uint64_t fills = fill * resident / t.groups, wanted = fills < 128 ? fills : 128;
        const uint64_t even = (rounds + wanted - 1) / wanted, per = even > least ? even : least;
        const uint64_t splits = (rounds + per - 1) / per, turns = (t.groups * splits + resident - 1) / resident;
        const uint64_t takes = turns * (2 * per + 3) + (few ? 4 : 8);
        if (splits > 1 && (takes < cost || (best > 1 && per >= 8 && 10 * takes <= 11 * cost))) best = splits, cost = takes;
    }
    return static_cast<uint32_t>(best);
}

hipError_t launch_attend(const Attend& a, hipStream_t stream) {
    const hipError_t e = a.cache.type == kF16 ? attend<_Float16>(a, stream) : attend<__bf16>(a, stream);
    if (e != hipSuccess || a.splits == 1) return e;
    // as many takers as splits, in powers of two, up to a work-group's units
    const uint32_t units = a.cache.head_dim <= 128 ? 16 : 8;
    uint32_t takers = 1;
    while (2 * takers <= a.splits && takers < units) takers *= 2;
    const uint64_t joins = units / takers, all = static_cast<uint64_t>(a.q.rows) * a.q.heads;
    return launch(k_attend_join, dim3(static_cast<uint32_t>((all + joins - 1) / joins)), dim3(kJoinThreads), stream, a,
                  static_cast<int>(takers));
}

namespace {

// Queries of a sequence and K/V head up to which a wave that adds up weights has slots of its own: four tiles of 16, which
// it reads beside its K rows.
constexpr uint32_t kFewWeighed = 64;

// How a step's weights are divided: by the most queries that a sequence may have.
struct WeighTiling {
    bool few;
    int blocks;       // work-groups that a sequence's slots take, per K/V head
    uint64_t groups;  // work-groups per split
};

WeighTiling weigh_tiling(const Cache& c, const Batch& b, uint32_t group) {
    WeighTiling t;
    t.few = static_cast<uint64_t>(b.max_rows) * group <= kFewWeighed;
    const uint32_t slots = kWeighWaves * (t.few ? kFewWeighSlots : 16 * (c.head_dim <= 128 ? kWeighTiles<128> : kWeighTiles<256>));
    t.blocks = static_cast<int>((b.max_length + slots - 1) / slots);
    t.groups = static_cast<uint64_t>(t.blocks) * c.n_head_kv * b.n_seq;
    return t;
}

template <typename T, int HDP>
hipError_t weigh_of(const Weigh& a, hipStream_t stream) {
    const int group = static_cast<int>(a.q.heads / a.cache.n_head_kv);
    const WeighTiling t = weigh_tiling(a.cache, a.batch, a.q.heads / a.cache.n_head_kv);
    const uint64_t groups = t.groups * a.splits;
    if (groups > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    return launch(t.few ? k_weigh_few<T, HDP> : k_weigh_many<T, HDP>, dim3(static_cast<uint32_t>(groups)),
                  dim3(kWeighThreads), stream, a, group, t.blocks);
}

template <typename T>
hipError_t weigh(const Weigh& a, hipStream_t stream) {
    if (a.cache.head_dim <= 64) return weigh_of<T, 64>(a, stream);
    if (a.cache.head_dim <= 128) return weigh_of<T, 128>(a, stream);
    return weigh_of<T, 256>(a, stream);
}

}  // namespace

uint32_t weigh_splits(const Cache& c, const Batch& b, uint32_t group) {
    const WeighTiling t = weigh_tiling(c, b, group);
    if (t.few || t.groups == 0) return 1;
    // two work-groups per compute unit, of four tiles of 64 queries at least
    const uint64_t wanted = (2 * kComputeUnits + t.groups - 1) / t.groups, most = static_cast<uint64_t>(b.max_rows) * group / 256;
    return static_cast<uint32_t>(wanted < most ? wanted : most > 0 ? most : 1);
}

hipError_t launch_weigh(const Weigh& a, hipStream_t stream) {
    const hipError_t e = a.cache.type == kF16 ? weigh<_Float16>(a, stream) : weigh<__bf16>(a, stream);
    if (e != hipSuccess || a.splits == 1) return e;
    const int blocks = static_cast<int>((a.batch.max_length + kWeighThreads - 1) / kWeighThreads);
    const uint64_t groups = static_cast<uint64_t>(blocks) * a.cache.n_head_kv * a.batch.n_seq;
    if (groups > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    return launch(k_weigh_join, dim3(static_cast<uint32_t>(groups)), dim3(kWeighThreads), stream, a, blocks);
}

hipError_t launch_evict(const Evict& a, hipStream_t stream) {
    const uint64_t pairs = static_cast<uint64_t>(a.cache.n_head_kv) * a.batch.n_seq;
    const int chunks = (a.width + kMoveSlots - 1) / kMoveSlots;
    if (pairs * static_cast<uint64_t>(chunks) > 0x7FFFFFFF) return hipErrorInvalidConfiguration;
    // the larger LDS takes a compute unit for one work-group
    const bool few = a.batch.max_length <= kSelectFew;
    const hipError_t e = launch(few ? k_evict_select<kSelectFew, 8> : k_evict_select<kSelectMany, 16>,
                                dim3(static_cast<uint32_t>(pairs)), dim3(kSelectThreads), stream, a);
    if (e != hipSuccess) return e;
    return launch(k_evict_move, dim3(static_cast<uint32_t>(pairs) * chunks), dim3(kMoveThreads), stream, a, chunks);
}

}  // namespace jfh::paged
