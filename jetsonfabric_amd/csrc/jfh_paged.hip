// gfx950 kernels of the paged-cache operators (jfh_paged.hpp).
#include "jfh_paged.hpp"

#include <hip/hip_runtime.h>

#include <type_traits>

namespace jfh::paged {

namespace {

using half8 = _Float16 __attribute__((ext_vector_type(8)));
using bhalf8 = __bf16 __attribute__((ext_vector_type(8)));
using float4v = float __attribute__((ext_vector_type(4)));

enum : uint32_t { kF32 = 1, kF16 = 2, kBF16 = 3 };

template <typename... KArgs, typename... Args>
hipError_t launch(void (*kernel)(KArgs...), dim3 grid, dim3 block, hipStream_t stream, const Args&... args) {
    static_assert((std::is_same_v<KArgs, Args> && ...), "arguments are passed by address");
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

// The one rounding to the output's type, to nearest.
template <int N>
__device__ __forceinline__ void store(void* data, int64_t at, uint32_t type, const float (&x)[N]) {
    if constexpr (N == 8) {
        if (type == kF32) {
            float4v* p = reinterpret_cast<float4v*>(static_cast<float*>(data) + at);
            p[0] = float4v{x[0], x[1], x[2], x[3]};
            p[1] = float4v{x[4], x[5], x[6], x[7]};
        } else if (type == kF16) {
            half8 v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = static_cast<_Float16>(x[i]);
            *reinterpret_cast<half8*>(static_cast<_Float16*>(data) + at) = v;
        } else {
            bhalf8 v;
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = static_cast<__bf16>(x[i]);
            *reinterpret_cast<bhalf8*>(static_cast<__bf16*>(data) + at) = v;
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
template <int N>
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
        store(y, y_at + lo, y_type, a);
        store(y, y_at + hi, y_type, b);
    } else {
        const int d = static_cast<int>(r.n_rot) + (u * N - half);
        float a[N];
        load(x, x_at + d, x_type, a);
        store(y, y_at + d, y_type, a);
    }
}

// Bound by the rows' bytes, one read and one write. A work-group computes the angles of its rows once for all heads;
// a thread owns a unit, so rows may be rotated in place.
template <int N>
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
        rotate_unit<N>(r, cs[row], u, x.data, (row0 + row) * x.row_stride + head * x.head_stride, x.type, y.data,
                       (row0 + row) * y.row_stride + head * y.head_stride, y.type);
    }
}

// New rows into their pages: keys rotated where the step gives a rotation, values as they are, weight 0 and the row's
// position for every K/V head. Rows of no sequence, before slot 0 or on absent pages are not written.
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
        const int slot = span.len - span.rows + (row - span.row0);
        pages[threadIdx.x] = s >= 0 && slot >= 0 ? page_of(c, b, s, slot) : -1;
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
            rotate_unit<N>(r, cs[row], left - head * ku, k.data, (row0 + row) * k.row_stride + head * k.head_stride,
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

bool by_eights(const Rows& x) {
    return reinterpret_cast<uintptr_t>(x.data) % 16 == 0 && x.row_stride % 8 == 0 && x.head_stride % 8 == 0 &&
           x.head_dim % 8 == 0;
}

// Long steps: four rows per work-group, so that 64 pairs' angles are one per thread. Short ones: one row, its units
// over up to `tasks` / 256 work-groups, since the call's time is the time of one work-group.
struct RowGrid {
    dim3 grid;
    int rows;
};

RowGrid row_grid(uint32_t rows, uint64_t tasks) {
    if (rows >= kComputeUnits * kRotateRows) return {dim3((rows + kRotateRows - 1) / kRotateRows), kRotateRows};
    const uint64_t parts = (tasks + kRotateThreads - 1) / kRotateThreads;
    return {dim3(rows, static_cast<uint32_t>(parts < 64 ? parts : 64)), 1};
}

}  // namespace

hipError_t launch_rotate(const Rotation& r, const Rows& x, const int32_t* positions, const Rows& y, hipStream_t stream) {
    const bool wide = by_eights(x) && by_eights(y) && r.n_rot % 16 == 0;
    const uint64_t units = (r.n_rot / 2 + (x.head_dim - r.n_rot)) / (wide ? 8 : 1);
    const RowGrid g = row_grid(x.rows, x.heads * units);
    return launch(wide ? k_rotate<8> : k_rotate<1>, g.grid, dim3(kRotateThreads), stream, r, x, positions, y, g.rows);
}

hipError_t launch_append(const Rotation* rotation, const Cache& c, const Batch& b, const Rows& k, const Rows& v,
                         const int32_t* positions, hipStream_t stream) {
    const Rotation r = rotation ? *rotation : Rotation{};
    const bool wide = by_eights(k) && by_eights(v) && r.n_rot % 16 == 0;
    const uint64_t units = (r.n_rot / 2 + (k.head_dim - r.n_rot) + v.head_dim) / (wide ? 8 : 1) + 1;
    const RowGrid g = row_grid(k.rows, c.n_head_kv * units);
    return launch(wide ? k_append<8> : k_append<1>, g.grid, dim3(kRotateThreads), stream, r, c, b, k, v, positions, g.rows);
}

}  // namespace jfh::paged
