// The common norm of many tensors, and their scaling to at most a given norm (smx_gradient_*).
//
//   norm = sqrt(sum over tensors and values of t^2),   out = t * (norm <= max_norm ? 1 : max_norm / norm)
//
// Squares and sums are float64 whatever the tensors' type: a float32 square leaves the type's range from 1e19 on upwards and below 1e-23. Tensors are cut into
// tiles; the CTAs of the first kernel own consecutive tiles and write one partial sum each, the CTAs of the second one add all of them in the same
// order, so all scale by the same factor and the same call gives the same bits. No atomics, no counters: two calls may share nothing but inputs.
#include "gradients.hpp"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "routing.hpp"

namespace smx {
namespace {

// Bytes bound it: 64,000,000 values of 96 tensors (284 MB) 47 us for the norm and 91 for the scaling, 6.0 and 6.2 TB/s, which walks the tiles backwards since the
// last ones are in L2 still; 407 tensors of 6,000,001 values 18 us for both kernels, 22 a call of a set that is kept (making the set takes the host
// 1.8 us a tensor: 750 us).
constexpr int kThreads = 256, kTileBytes = 16384;
constexpr int kMaxCtas = 8 * 148;                    // of a launch; a constant, so that sizes and sums do not depend on the device

// The tensors of a launch, as kernel arguments: nothing is copied to the device, and a captured launch carries its list along.
struct Tensor { const void* from; void* to; long long count; int first_tile, wide; };     // wide: bit 0 float64, bit 1 both start on 16 bytes
template <int N>
struct TensorList { Tensor tensor[N]; int count, tiles; };
template <int N>
struct ListSize { static constexpr int value = N; };
constexpr int kLargestList = 1000;                   // 32 KB of arguments

// The tensor that holds tile t.
template <int N>
__device__ __forceinline__ int tensor_of(const TensorList<N>& list, int t) {
    int lo = 0, hi = list.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (list.tensor[mid].first_tile <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// The CTA's tiles, tensor by tensor: fn(tensor, first value, values).
template <int N, typename Fn>
__device__ __forceinline__ void for_tiles(const TensorList<N>& list, bool backwards, Fn&& fn) {
    const long long tiles = list.tiles;
    const int begin = static_cast<int>(tiles * blockIdx.x / gridDim.x), end = static_cast<int>(tiles * (blockIdx.x + 1) / gridDim.x);
    if (begin >= end) return;
    const int step = backwards ? -1 : 1;
    int at = tensor_of(list, backwards ? end - 1 : begin);
    for (int t = backwards ? end - 1 : begin; t >= begin && t < end; t += step) {
        while (t < list.tensor[at].first_tile) --at;
        while (at + 1 < list.count && t >= list.tensor[at + 1].first_tile) ++at;
        const Tensor& x = list.tensor[at];
        const int per = (x.wide & 1) ? kTileBytes / 8 : kTileBytes / 4;
        const long long from = static_cast<long long>(t - x.first_tile) * per;
        fn(x, from, static_cast<int>(min(static_cast<long long>(per), x.count - from)));
    }
}

// Sum over the CTA, the same in all threads.
__device__ __forceinline__ double cta_sum(double v, double* shared) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
    if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) s += shared[w];
    return s;
}

template <typename T>
__device__ __forceinline__ double tile_squares(const T* from, int n, bool wide) {
    constexpr int per = 16 / sizeof(T), kUnits = kTileBytes / 16 / kThreads;
    double s = 0.0;
    if (wide) {
        using V = std::conditional_t<sizeof(T) == 4, float4, double2>;
        union { V v; T t[per]; } u[kUnits];
#pragma unroll
        for (int q = 0; q < kUnits; ++q) {
            const int i = (q * kThreads + threadIdx.x) * per;
            u[q].v = V{};
            if (i + per <= n) u[q].v = *reinterpret_cast<const V*>(from + i);
            else
#pragma unroll
                for (int e = 0; e < per; ++e)
                    if (i + e < n) u[q].t[e] = from[i + e];
        }
#pragma unroll
        for (int q = 0; q < kUnits; ++q)
#pragma unroll
            for (int e = 0; e < per; ++e) s = fma(static_cast<double>(u[q].t[e]), static_cast<double>(u[q].t[e]), s);
        return s;
    }
    for (int i = threadIdx.x; i < n; i += kThreads) {
        const double d = from[i];
        s = fma(d, d, s);
    }
    return s;
}

template <int N>
__global__ void __launch_bounds__(kThreads) gradient_norm_kernel(const __grid_constant__ TensorList<N> list, double* __restrict__ partial) {
    __shared__ double shared[kThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the scaling kernel comes in as CTAs of this one end
    double s = 0.0;
    for_tiles(list, false, [&](const Tensor& x, long long from, int n) {
        if (x.wide & 1) s += tile_squares(static_cast<const double*>(x.from) + from, n, (x.wide & 2) != 0);
        else s += tile_squares(static_cast<const float*>(x.from) + from, n, (x.wide & 2) != 0);
    });
    s = cta_sum(s, shared);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// float64 products of float32 values are rounded once, to float32.
template <typename T>
__device__ __forceinline__ void tile_scale(const T* from, T* to, int n, bool wide, double factor) {
    constexpr int per = 16 / sizeof(T), kUnits = kTileBytes / 16 / kThreads;
    if (wide) {
        using V = std::conditional_t<sizeof(T) == 4, float4, double2>;
        union { V v; T t[per]; } u[kUnits];
#pragma unroll
        for (int q = 0; q < kUnits; ++q) {
            const int i = (q * kThreads + threadIdx.x) * per;
            if (i + per <= n) u[q].v = __ldcs(reinterpret_cast<const V*>(from + i));
        }
#pragma unroll
        for (int q = 0; q < kUnits; ++q) {
            const int i = (q * kThreads + threadIdx.x) * per;
            if (i + per <= n) {
#pragma unroll
                for (int e = 0; e < per; ++e) u[q].t[e] = static_cast<T>(static_cast<double>(u[q].t[e]) * factor);
                __stcs(reinterpret_cast<V*>(to + i), u[q].v);
            } else {
                for (int e = 0; e < per; ++e)
                    if (i + e < n) to[i + e] = static_cast<T>(static_cast<double>(from[i + e]) * factor);
            }
        }
        return;
    }
    // Tensors that start anywhere: eight values in flight, since a store holds back the loads behind it, which might read what it writes (in place, 64,000,000
    // float32 values: 255 us one by one, 110 by eights, 74 in units of 16 bytes).
    for (int i0 = threadIdx.x; i0 < n; i0 += 8 * kThreads) {
        T v[8];
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (i0 + q * kThreads < n) v[q] = __ldcs(from + i0 + q * kThreads);
#pragma unroll
        for (int q = 0; q < 8; ++q)
            if (i0 + q * kThreads < n) __stcs(to + i0 + q * kThreads, static_cast<T>(static_cast<double>(v[q]) * factor));
    }
}

__device__ __forceinline__ double norm_of(const double* partial, int partials, double* shared) {
    double s = 0.0;
    for (int i = threadIdx.x; i < partials; i += kThreads) s += partial[i];
    return sqrt(cta_sum(s, shared));
}

// `partial` is written while CTAs of this kernel start: no promise that it is constant.
template <int N>
__global__ void __launch_bounds__(kThreads) gradient_scale_kernel(const __grid_constant__ TensorList<N> list, const double* partial, int partials,
                                                                  double max_norm, double* norm) {
    __shared__ double shared[kThreads / 32];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const double n = norm_of(partial, partials, shared);
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
    // a NaN makes the norm NaN, and that the factor and all values
    const double factor = n <= max_norm ? 1.0 : max_norm / n;
    for_tiles(list, true, [&](const Tensor& x, long long from, int count) {
        if (factor == 1.0 && x.from == x.to) return;
        if (x.wide & 1) tile_scale(static_cast<const double*>(x.from) + from, static_cast<double*>(x.to) + from, count, (x.wide & 2) != 0, factor);
        else tile_scale(static_cast<const float*>(x.from) + from, static_cast<float*>(x.to) + from, count, (x.wide & 2) != 0, factor);
    });
}

__global__ void __launch_bounds__(kThreads) gradient_root_kernel(const double* __restrict__ partial, int partials, double* __restrict__ norm) {
    __shared__ double shared[kThreads / 32];
    const double n = norm_of(partial, partials, shared);
    if (threadIdx.x == 0) *norm = n;
}

void launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
    ++operator_launches;
}

long long tiles_of(const smx_gradient& g) {
    const long long per = g.precision == SMX_FP64 ? kTileBytes / 8 : kTileBytes / 4;
    return (g.count + per - 1) / per;
}

// The list cut into launches: fn(first tensor, one behind the last, tiles).
template <typename Fn>
void for_launches(const smx_gradient* list, int count, Fn&& fn) {
    for (int a = 0; a < count;) {
        long long tiles = 0;
        int b = a;
        while (b < count && b - a < kLargestList && tiles + tiles_of(list[b]) <= INT_MAX) tiles += tiles_of(list[b++]);
        fn(a, b, static_cast<int>(tiles));
        a = b;
    }
}
int grid_of(int tiles) { return std::max(1, std::min(tiles, kMaxCtas)); }

void check_list(const smx_gradient* list, int count) {
    if (count < 0 || (count > 0 && !list)) throw ArgError("smx_gradient: bad list");
    for (int i = 0; i < count; ++i) {
        const smx_gradient& g = list[i];
        if (g.precision != SMX_FP32 && g.precision != SMX_FP64) throw ArgError("smx_gradient: precision must be 32 or 64");
        if (g.count < 0 || g.count > (1LL << 40)) throw ArgError("smx_gradient: bad number of values");
    }
}

template <typename Fn>
void with_list(const smx_gradient* list, int a, int b, int tiles, Fn&& fn) {
    auto fill = [&](auto size) {
        constexpr int N = decltype(size)::value;
        TensorList<N> l;
        l.count = 0;
        l.tiles = tiles;
        int tile = 0;
        for (int i = a; i < b; ++i) {
            const smx_gradient& g = list[i];
            if (g.count == 0) continue;
            Tensor& t = l.tensor[l.count++];
            t.from = g.values; t.to = g.out; t.count = g.count; t.first_tile = tile;
            const bool aligned = ((reinterpret_cast<uintptr_t>(g.values) | reinterpret_cast<uintptr_t>(g.out)) & 15) == 0;
            t.wide = (g.precision == SMX_FP64 ? 1 : 0) | (aligned ? 2 : 0);
            tile += static_cast<int>(tiles_of(g));
        }
        fn(l);
    };
    if (b - a <= 32) fill(ListSize<32>{});
    else if (b - a <= 128) fill(ListSize<128>{});
    else if (b - a <= 512) fill(ListSize<512>{});
    else fill(ListSize<kLargestList>{});
}

}  // namespace

size_t gradient_workspace_bytes(const smx_gradient* list, int count) {
    check_list(list, count);
    size_t partials = 1;
    for_launches(list, count, [&](int, int, int tiles) { partials += grid_of(tiles); });
    return partials * sizeof(double);
}

void gradient_norm_clip(const smx_gradient* list, int count, bool clip, double max_norm, double* norm, void* workspace, size_t workspace_bytes,
                        cudaStream_t stream) {
    check_list(list, count);
    if (!norm && !clip) throw ArgError("smx_gradient_norm: null norm");
    if (clip && !(max_norm >= 0.0)) throw ArgError("smx_gradient_clip: the largest norm must not be negative or NaN");
    for (int i = 0; i < count; ++i) {
        const smx_gradient& g = list[i];
        if (g.count == 0) continue;
        if (!g.values || (clip && !g.out)) throw ArgError("smx_gradient: null pointer");
        check_pointers("smx_gradient", g.precision == SMX_FP64 ? 8 : 4, {g.values, clip ? g.out : nullptr});
    }
    check_pointers("smx_gradient", sizeof(double), {norm, workspace});
    const size_t need = gradient_workspace_bytes(list, count);
    if (workspace_bytes < need || !workspace) throw ArgError("smx_gradient: the workspace is smaller than smx_gradient_workspace_bytes says");
    double* partial = static_cast<double*>(workspace);
    int partials = 0;
    for_launches(list, count, [&](int a, int b, int tiles) {
        if (tiles == 0) return;
        with_list(list, a, b, tiles, [&](const auto& l) {
            const int grid = grid_of(tiles);
            gradient_norm_kernel<<<grid, kThreads, 0, stream>>>(l, partial + partials);
            launched("gradient_norm_kernel");
            partials += grid;
        });
    });
    if (!clip || partials == 0) {
        if (!norm) return;
        gradient_root_kernel<<<1, kThreads, 0, stream>>>(partial, partials, norm);
        launched("gradient_root_kernel");
        return;
    }
    bool first = true;
    for_launches(list, count, [&](int a, int b, int tiles) {
        if (tiles == 0) return;
        with_list(list, a, b, tiles, [&](const auto& l) {
            constexpr int N = sizeof(l.tensor) / sizeof(Tensor);
            chain_launch(Launcher{stream, first}, gradient_scale_kernel<N>, dim3(grid_of(tiles)), kThreads, 0, 1, l, partial, partials, max_norm, first ? norm : nullptr);
            ++operator_launches;
            first = false;
        });
    });
}

}  // namespace smx
