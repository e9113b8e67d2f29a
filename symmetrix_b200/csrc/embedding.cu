// Embeddings (smx_embedding_*): rows of a table named by tokens, weighted and summed, and the gradients of the table and of the weights.
//
//   y[n] = scale sum_s w[n, s] table[ids[n, s]]
//   grad_table[t] = scale sum over pairs (n, s) with ids[n, s] = t of w[n, s] grad_y[n],   grad_w[n, s] = scale <grad_y[n], table[ids[n, s]]>
//
// A pair whose id is no row of the table (negative or too large) counts for nothing. The sums of the table's gradient go over the pairs sorted by
// token (csrc/routing.cu), cut into chunks of equal length: a token's run inside a chunk is one sum; runs that cross chunks leave partial sums,
// which are added in order. No atomics: the same call gives the same bits.
#include "embedding.hpp"

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>

#include "common.cuh"
#include "routing.hpp"

namespace smx {
namespace {

template <typename T> struct Wide;
template <> struct Wide<float> { using type = float4; };
template <> struct Wide<double> { using type = double2; };
template <typename T, typename V>
union Lanes {
    static constexpr int n = sizeof(V) / sizeof(T);
    V v;
    T t[n];
};

__global__ void __launch_bounds__(256) embedding_tokens_kernel(const int* __restrict__ ids, const int* __restrict__ order, long long pairs, int table_rows,
                                                               int* __restrict__ tokens) {
    for (long long p = blockIdx.x * 256LL + threadIdx.x; p < pairs; p += 256LL * gridDim.x) {
        const int t = ids[order[p]];
        tokens[p] = t < 0 || t >= table_rows ? table_rows : t;
    }
}

template <typename T, typename V>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const V* __restrict__ table, long long table_stride, int table_rows, const int* __restrict__ ids,
                                                                long long num_rows, int slots, int units, const T* __restrict__ weights, T scale,
                                                                V* __restrict__ y, long long y_stride) {
    using L = Lanes<T, V>;
    for (long long n = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y; n < num_rows; n += static_cast<long long>(gridDim.x) * blockDim.y) {
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
            L sum{};
            for (int s = 0; s < slots; ++s) {
                const int t = ids[n * slots + s];
                if (t < 0 || t >= table_rows) continue;
                const T w = weights ? scale * weights[n * slots + s] : scale;
                L r;
                r.v = table[t * table_stride + u];
#pragma unroll
                for (int q = 0; q < L::n; ++q) sum.t[q] += w * r.t[q];
            }
            y[n * y_stride + u] = sum.v;
        }
    }
}

// Sums of the runs of a chunk of sorted pairs, kGradThreads units of a row a CTA. parts: [chunk][2][units]: the run that an earlier chunk began, and the
// run that goes on in the next one.
constexpr int kGradThreads = 128, kMaxChunk = 512;
template <typename T, typename V>
__global__ void __launch_bounds__(kGradThreads) embedding_grad_kernel(const V* __restrict__ grad_y, long long grad_y_stride, const int* __restrict__ order,
                                                                      const int* __restrict__ tokens, long long pairs, int slots, int table_rows, int units,
                                                                      const T* __restrict__ weights, T scale, int chunk, V* __restrict__ grad_table,
                                                                      V* __restrict__ parts) {
    using L = Lanes<T, V>;
    constexpr int kAhead = 8;
    __shared__ long long row[kMaxChunk];
    __shared__ T weight[kMaxChunk];
    __shared__ int token[kMaxChunk + 2];                                 // with the neighbours
    const long long begin = static_cast<long long>(blockIdx.x) * chunk;
    const int count = static_cast<int>(min(static_cast<long long>(chunk), pairs - begin));
    for (int i = threadIdx.x; i < count + 2; i += kGradThreads) {
        const long long p = begin + i - 1;
        token[i] = p >= 0 && p < pairs ? tokens[p] : -1;
        if (i >= 1 && i <= count) {
            const int pair = order[p];
            row[i - 1] = pair / slots * grad_y_stride;
            weight[i - 1] = weights ? scale * weights[pair] : scale;
        }
    }
    __syncthreads();
    const int u = blockIdx.y * kGradThreads + threadIdx.x;
    if (u >= units) return;
    L sum{};
    int from = 0;                                                        // where the run at hand began
    for (int i0 = 0; i0 < count; i0 += kAhead) {
        L g[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            g[q].v = V{};
            if (i0 + q < count && token[i0 + q + 1] < table_rows) g[q].v = grad_y[row[i0 + q] + u];
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int i = i0 + q;
            if (i >= count) break;
            const int t = token[i + 1];
            if (t >= table_rows) return;                                 // pairs without a token come last
            const T w = weight[i];
#pragma unroll
            for (int e = 0; e < L::n; ++e) sum.t[e] += w * g[q].t[e];
            if (token[i + 2] == t && i + 1 < count) continue;
            const bool began = from > 0 || token[0] != t, ends = token[i + 2] != t;
            if (began && ends) grad_table[static_cast<long long>(t) * units + u] = sum.v;
            else parts[(2LL * blockIdx.x + (began ? 1 : 0)) * units + u] = sum.v;
            sum = L{};
            from = i + 1;
        }
    }
}

// The runs that cross chunks: the CTAs of the chunk where one begins add its parts in order, four of them side by side.
constexpr int kJoinUnits = 32, kJoinWays = 8;
template <typename T, typename V>
__global__ void __launch_bounds__(kJoinUnits * kJoinWays) embedding_join_kernel(const int* __restrict__ tokens, long long pairs, int table_rows, int units, int chunk,
                                                                                int chunks, const V* __restrict__ parts, V* __restrict__ grad_table) {
    using L = Lanes<T, V>;
    __shared__ V joined[kJoinWays][kJoinUnits];
    const long long begin = static_cast<long long>(blockIdx.x) * chunk, end = begin + chunk;
    if (end >= pairs) return;
    const int t = tokens[end - 1];
    if (t >= table_rows || tokens[end] != t || (begin > 0 && tokens[begin - 1] == t)) return;      // no run, or not its beginning
    int more = 0;                                                        // chunks that go on with it
    for (int c0 = blockIdx.x + 1;; c0 += kJoinUnits * kJoinWays) {
        const int c = c0 + threadIdx.x;
        const int n = __syncthreads_count(c < chunks && tokens[static_cast<long long>(c) * chunk] == t);
        more += n;
        if (n < kJoinUnits * kJoinWays) break;
    }
    const int lane = threadIdx.x % kJoinUnits, way = threadIdx.x / kJoinUnits, u = blockIdx.y * kJoinUnits + lane;
    const int per = (more + 1 + kJoinWays - 1) / kJoinWays, first = way * per, last = min(more + 1, first + per);
    L sum{};
    if (u < units) {
        for (int i0 = first; i0 < last; i0 += 8) {
            L v[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int i = i0 + q;
                v[q].v = i < last ? parts[(2LL * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * units + u] : V{};
            }
#pragma unroll
            for (int q = 0; q < 8; ++q)
#pragma unroll
                for (int e = 0; e < L::n; ++e) sum.t[e] += v[q].t[e];
        }
    }
    joined[way][lane] = sum.v;
    __syncthreads();
    if (way > 0 || u >= units) return;
    for (int w = 1; w < kJoinWays; ++w) {
        L v;
        v.v = joined[w][lane];
#pragma unroll
        for (int e = 0; e < L::n; ++e) sum.t[e] += v.t[e];
    }
    grad_table[static_cast<long long>(t) * units + u] = sum.v;
}

// grad_w: a warp per pair, in sorted order (the table's rows then come from the cache).
template <typename T, typename V>
__global__ void __launch_bounds__(256) embedding_weight_grad_kernel(const V* __restrict__ grad_y, long long grad_y_stride, const V* __restrict__ table,
                                                                    long long table_stride, int table_rows, const int* __restrict__ order,
                                                                    const int* __restrict__ tokens, long long pairs, int slots, int units, T scale,
                                                                    T* __restrict__ grad_weights) {
    using L = Lanes<T, V>;
    const int lane = threadIdx.x & 31;
    for (long long p = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5; p < pairs; p += static_cast<long long>(gridDim.x) * 8) {
        const int pair = order[p], t = tokens[p];
        T dot = T(0);
        if (t < table_rows)
            for (int u = lane; u < units; u += 32) {
                L g, r;
                g.v = grad_y[pair / slots * grad_y_stride + u];
                r.v = table[t * table_stride + u];
#pragma unroll
                for (int e = 0; e < L::n; ++e) dot += g.t[e] * r.t[e];
            }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (lane == 0) grad_weights[pair] = scale * dot;
    }
}

// ------------------------------------------------------------------------------------------- host side
void launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
    ++operator_launches;
}
void check_sizes(const char* what, long num_rows, int slots, int table_rows, long width) {
    if (table_rows < 1 || table_rows > SMX_EMBEDDING_MAX_ROWS)
        throw ArgError(std::string(what) + ": the number of table rows must lie in 1 .. " + std::to_string(SMX_EMBEDDING_MAX_ROWS));
    if (width < 0 || width > INT_MAX) throw ArgError(std::string(what) + ": bad row width");
    route_plan_bytes(num_rows, slots, 1);                                // rows and slots as there
}
void check_stride(const char* what, long stride, long width, long rows, bool written) {
    if (stride < 0 || (written && rows > 1 && stride < width)) throw ArgError(std::string(what) + ": bad row stride");
}
template <typename T>
bool wide_rows(std::initializer_list<const void*> pointers, std::initializer_list<long> strides) {
    constexpr long per = 16 / sizeof(T);
    for (long s : strides) if (s % per != 0) return false;
    for (const void* p : pointers) if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return true;
}
template <typename T, typename Fn>
void by_unit(bool wide, Fn&& fn) {
    if (wide) fn(typename Wide<T>::type{});
    else fn(T{});
}

// Chunks of the sorted pairs: eight CTAs for each of 148 SMs where there are enough pairs (a constant, so that sizes do not depend on the device).
int grad_chunk(long pairs) { return static_cast<int>(std::max(16L, std::min<long>(kMaxChunk, (pairs + 1183) / 1184))); }

}  // namespace

size_t embedding_plan_bytes(long num_rows, int slots, int table_rows) {
    check_sizes("smx_embedding_plan", num_rows, slots, table_rows, 0);
    return token_sort_bytes(num_rows * slots, table_rows);
}
void embedding_plan(const int* ids, long num_rows, int slots, int table_rows, int* order, int* tokens, void* workspace, size_t workspace_bytes,
                    cudaStream_t stream) {
    const size_t need = embedding_plan_bytes(num_rows, slots, table_rows);
    const long pairs = num_rows * slots;
    if (pairs == 0) return;
    if (!ids || !order || !tokens) throw ArgError("smx_embedding_plan: null pointer");
    check_pointers("smx_embedding_plan", sizeof(int), {ids, order, tokens, workspace});
    if (workspace_bytes < need || (need && !workspace)) throw ArgError("smx_embedding_plan: the workspace is smaller than smx_embedding_plan_bytes says");
    token_sort(ids, pairs, table_rows, order, workspace, stream);
    embedding_tokens_kernel<<<static_cast<unsigned>(std::min<long>((pairs + 255) / 256, 8L * sm_count())), 256, 0, stream>>>(ids, order, pairs, table_rows, tokens);
    launched("embedding_tokens_kernel");
}

template <typename T>
void embedding_forward(const T* table, long table_stride, int table_rows, const int* ids, long num_rows, int slots, long width, const T* weights,
                       double scale, T* y, long y_stride, cudaStream_t stream) {
    const char* what = "smx_embedding_forward";
    check_sizes(what, num_rows, slots, table_rows, width);
    check_stride(what, table_stride, width, table_rows, false);
    check_stride(what, y_stride, width, num_rows, true);
    if (num_rows == 0 || width == 0) return;
    if (!table || !ids || !y) throw ArgError("smx_embedding_forward: null pointer");
    check_pointers(what, sizeof(int), {ids});
    check_pointers(what, sizeof(T), {table, weights, y});
    by_unit<T>(wide_rows<T>({table, y}, {table_stride, y_stride, width}), [&](auto unit) {
        using V = decltype(unit);
        constexpr long per = sizeof(V) / sizeof(T);
        unsigned tx = 32;
        while (tx < 256 && tx < width / per) tx *= 2;
        const unsigned ty = 256 / tx;
        const unsigned blocks = static_cast<unsigned>(std::min<long long>((num_rows + ty - 1) / ty, 64LL * sm_count()));
        embedding_forward_kernel<T, V><<<blocks, dim3(tx, ty), 0, stream>>>(reinterpret_cast<const V*>(table), table_stride / per, table_rows, ids, num_rows, slots,
                                                                            static_cast<int>(width / per), weights, static_cast<T>(scale), reinterpret_cast<V*>(y),
                                                                            y_stride / per);
    });
    launched("embedding_forward_kernel");
}

template <typename T>
size_t embedding_backward_bytes(long num_rows, int slots, long width) {
    check_sizes("smx_embedding_backward", num_rows, slots, 1, width);
    const long pairs = num_rows * slots;
    const long chunks = pairs > 0 ? (pairs + grad_chunk(pairs) - 1) / grad_chunk(pairs) : 0;
    return static_cast<size_t>(chunks) * 2 * width * sizeof(T);
}
template <typename T>
void embedding_backward(const T* grad_y, long grad_y_stride, const T* table, long table_stride, int table_rows, const int* order, const int* tokens,
                        long num_rows, int slots, long width, const T* weights, double scale, T* grad_table, T* grad_weights, void* workspace,
                        size_t workspace_bytes, cudaStream_t stream) {
    const char* what = "smx_embedding_backward";
    check_sizes(what, num_rows, slots, table_rows, width);
    check_stride(what, grad_y_stride, width, num_rows, false);
    const long pairs = num_rows * slots;
    check_pointers(what, sizeof(int), {order, tokens});
    check_pointers(what, sizeof(T), {grad_y, table, weights, grad_table, grad_weights});
    if (pairs > 0 && (!order || !tokens || (width > 0 && !grad_y))) throw ArgError("smx_embedding_backward: null pointer");
    if (grad_weights) {
        check_stride(what, table_stride, width, table_rows, false);
        if (pairs > 0 && width > 0 && !table) throw ArgError("smx_embedding_backward: the weights' gradient needs the table");
    }
    if (grad_table) {
        const size_t need = embedding_backward_bytes<T>(num_rows, slots, width);
        if (workspace_bytes < need || (need && !workspace)) throw ArgError("smx_embedding_backward: the workspace is smaller than smx_embedding_backward_bytes says");
        if (reinterpret_cast<uintptr_t>(workspace) & 15) throw ArgError("smx_embedding_backward: the workspace must start on a 16-byte boundary");
        if (width > 65535L * kJoinUnits) throw ArgError("smx_embedding_backward: rows are too wide");
    }
    if (grad_weights && pairs > 0) {
        by_unit<T>(wide_rows<T>({grad_y, table}, {grad_y_stride, table_stride, width}), [&](auto unit) {
            using V = decltype(unit);
            constexpr long per = sizeof(V) / sizeof(T);
            embedding_weight_grad_kernel<T, V><<<static_cast<unsigned>(std::min<long long>((pairs + 7) / 8, 64LL * sm_count())), 256, 0, stream>>>(
                reinterpret_cast<const V*>(grad_y), grad_y_stride / per, reinterpret_cast<const V*>(table), table_stride / per, table_rows, order, tokens, pairs, slots,
                static_cast<int>(width / per), static_cast<T>(scale), grad_weights);
        });
        launched("embedding_weight_grad_kernel");
    }
    if (!grad_table || width == 0) return;
    SMX_CUDA(cudaMemsetAsync(grad_table, 0, static_cast<size_t>(table_rows) * width * sizeof(T), stream));
    if (pairs == 0) return;
    const int chunk = grad_chunk(pairs), chunks = static_cast<int>((pairs + chunk - 1) / chunk);
    by_unit<T>(wide_rows<T>({grad_y, grad_table}, {grad_y_stride, width}), [&](auto unit) {
        using V = decltype(unit);
        constexpr long per = sizeof(V) / sizeof(T);
        const int units = static_cast<int>(width / per);
        const int slabs = (units + kGradThreads - 1) / kGradThreads, joins = (units + kJoinUnits - 1) / kJoinUnits;
        embedding_grad_kernel<T, V><<<dim3(chunks, slabs), kGradThreads, 0, stream>>>(reinterpret_cast<const V*>(grad_y), grad_y_stride / per, order, tokens, pairs,
                                                                                      slots, table_rows, units, weights, static_cast<T>(scale), chunk,
                                                                                      reinterpret_cast<V*>(grad_table), static_cast<V*>(workspace));
        launched("embedding_grad_kernel");
        if (chunks == 1) return;
        embedding_join_kernel<T, V><<<dim3(chunks, joins), kJoinUnits * kJoinWays, 0, stream>>>(tokens, pairs, table_rows, units, chunk, chunks,
                                                                                                static_cast<const V*>(workspace), reinterpret_cast<V*>(grad_table));
        launched("embedding_join_kernel");
    });
}

#define SMX_EMBEDDING_INSTANCE(T)                                                                                                                   \
    template void embedding_forward<T>(const T*, long, int, const int*, long, int, long, const T*, double, T*, long, cudaStream_t);               \
    template size_t embedding_backward_bytes<T>(long, int, long);                                                                                  \
    template void embedding_backward<T>(const T*, long, const T*, long, int, const int*, const int*, long, int, long, const T*, double, T*, T*,   \
                                        void*, size_t, cudaStream_t);
SMX_EMBEDDING_INSTANCE(float)
SMX_EMBEDDING_INSTANCE(double)

}  // namespace smx
