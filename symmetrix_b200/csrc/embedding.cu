// Embeddings (smx_embedding_*): rows of a table named by tokens, weighted and summed, and the gradients of the table and of the weights.
//
//   y[n] = scale sum_s w[n, s] table[ids[n, s]]
//   grad_table[t] = scale sum over pairs (n, s) with ids[n, s] = t of w[n, s] grad_y[n],   grad_w[n, s] = scale <grad_y[n], table[ids[n, s]]>
//
// A pair whose id is no row of the table (negative or too large) counts for nothing. The sums of the table's gradient go over the pairs sorted by
// token (csrc/routing.cu), cut into chunks of equal length: a token's run inside a chunk is one sum, of sums of eight where it is long; runs that cross chunks leave
// partial sums, which are added in order and in 64 bits. So a sum's error does not grow with its length: at most some 90 roundings whatever the number of pairs. No
// atomics: the same call gives the same bits.
#include "embedding.hpp"

#include <algorithm>
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

// blockDim.x threads (up to a warp) along a row, blockDim.y rows at a time; a thread has kAhead units of its row in flight, so that the wait for the id is
// shared among them, and the next row's id is read ahead. 98,304 rows of 512 floats: 34.5 us for 201 MB, 5.8 TB/s (the kernel alone, back to back); with a thread for every unit of
// 16 bytes half as long again, since an id and a weight then are read with each. The reads of the table come from L2 and are as many as the writes.
constexpr int kAhead = 4;
template <typename T, typename V>
__global__ void __launch_bounds__(256) embedding_forward_kernel(const V* __restrict__ table, long long table_stride, int table_rows, const int* __restrict__ ids,
                                                                long long num_rows, int slots, int units, const T* __restrict__ weights, T scale,
                                                                V* __restrict__ y, long long y_stride) {
    using L = Lanes<T, V>;
    const int tx = blockDim.x;
    const long long step = static_cast<long long>(gridDim.x) * blockDim.y;
    long long n = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y;
    int next = n < num_rows ? ids[n * slots] : -1;                       // the first slot's id, read a row ahead
    for (; n < num_rows; n += step) {
        const int first = next;
        if (n + step < num_rows) next = ids[(n + step) * slots];
        for (int u = threadIdx.x; u < units; u += kAhead * tx) {
            L sum[kAhead] = {};
            for (int s = 0; s < slots; ++s) {
                const int t = s == 0 ? first : ids[n * slots + s];
                if (t < 0 || t >= table_rows) continue;
                const T w = weights ? scale * weights[n * slots + s] : scale;
                const V* row = table + t * table_stride + u;
                L r[kAhead];
#pragma unroll
                for (int a = 0; a < kAhead; ++a) {
                    r[a].v = V{};
                    if (u + a * tx < units) r[a].v = row[a * tx];
                }
#pragma unroll
                for (int a = 0; a < kAhead; ++a)
#pragma unroll
                    for (int q = 0; q < L::n; ++q) sum[a].t[q] += w * r[a].t[q];
            }
#pragma unroll
            for (int a = 0; a < kAhead; ++a)
                if (u + a * tx < units) y[n * y_stride + u + a * tx] = sum[a].v;
        }
    }
}

// Sums of the runs of a chunk of sorted pairs, kGradThreads units of a row a CTA. parts: [chunk][2][units]: the run that an earlier chunk began, and the
// run that goes on in the next one. kWeights: the weights' gradients too, since a run's row of the table then is read once. Their sums over the units of a
// CTA go to `dots` [slab][pairs], or straight to the gradient where one CTA has the whole row.
// 49,152 rows of 512 floats, two slots, 1,424 tokens, all of the backward pass: 47 us, of which this kernel 33 for 201 MB of rows, 6.1 TB/s; 64 with a look
// at every pair's token (its instructions bounded it), 56 with the rows copied ahead through shared memory, 50 with eight CTAs of 64 registers an SM.
constexpr int kGradThreads = 128, kMaxChunk = 512, kLoads = 8, kRows = 4;
template <typename T> constexpr int grad_ctas = sizeof(T) == 4 ? 6 : 5;  // of an SM
template <typename T, typename V, bool kWeights>
__global__ void __launch_bounds__(kGradThreads, grad_ctas<T>) embedding_grad_kernel(const V* __restrict__ grad_y, long long grad_y_stride, const V* __restrict__ table,
                                                                      long long table_stride, const int* __restrict__ order, const int* __restrict__ tokens,
                                                                      long long pairs, int slots, int table_rows, int units, const T* __restrict__ weights, T scale,
                                                                      int chunk, V* __restrict__ grad_table, V* __restrict__ parts, T* __restrict__ dots,
                                                                      T* __restrict__ grad_weights) {
    using L = Lanes<T, V>;
    constexpr int kWarps = kGradThreads / 32;
    __shared__ long long row[kMaxChunk];
    __shared__ T weight[kMaxChunk];
    __shared__ int token[kMaxChunk + 2];                                 // with the neighbours
    __shared__ T warp_dot[kWeights ? kWarps : 1][kWeights ? kMaxChunk : 1];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the joining kernel comes in as CTAs of this one end
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long begin = static_cast<long long>(blockIdx.x) * chunk;
    const int count = static_cast<int>(min(static_cast<long long>(chunk), pairs - begin));
    int live = 0;                                                        // pairs without a token come last
    for (int i0 = 0; i0 < count + 2; i0 += kGradThreads) {
        const int i = i0 + threadIdx.x;
        const long long p = begin + i - 1;
        const int t = i < count + 2 && p >= 0 && p < pairs ? tokens[p] : -1;
        if (i < count + 2) token[i] = t;
        const bool in = i >= 1 && i <= count && t < table_rows;
        if (in) {
            const int pair = order[p];
            row[i - 1] = pair / slots * grad_y_stride;
            weight[i - 1] = weights ? scale * weights[pair] : scale;
        }
        live += __syncthreads_count(in);
    }
    const int u = blockIdx.y * kGradThreads + threadIdx.x;
    const bool mine = u < units;
    L sum{}, last{};                                                     // the run at hand; the row of the table of the pair before
    int from = 0, last_token = -1;                                       // where the run began
    auto give = [&](int i, int t) {                                      // the run of token t ends with pair i, or is cut behind it
        const bool began = from > 0 || token[0] != t, ends = token[i + 2] != t;
        if (mine) {
            if (began && ends) grad_table[static_cast<long long>(t) * units + u] = sum.v;
            else parts[(2LL * blockIdx.x + (began ? 1 : 0)) * units + u] = sum.v;
        }
        sum = L{};
        from = i + 1;
    };
    for (int i0 = 0; i0 < live; i0 += kLoads) {
        // One token for all (the pairs are sorted) is what long runs mostly meet: without a look at every pair a batch takes a third of the instructions.
        const int t0 = token[i0 + 1];
        const bool one = i0 + kLoads <= live && token[i0 + kLoads] == t0;
        L g[kLoads];
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
            g[q].v = V{};
            if (mine && i0 + q < live) g[q].v = grad_y[row[i0 + q] + u];
        }
        if constexpr (kWeights) {
            T d[kLoads];
            if (one) {
                if (t0 != last_token && mine) last.v = table[t0 * table_stride + u];
                last_token = t0;
#pragma unroll
                for (int q = 0; q < kLoads; ++q) {
                    d[q] = T(0);
#pragma unroll
                    for (int e = 0; e < L::n; ++e) d[q] += g[q].t[e] * last.t[e];
                }
            } else
#pragma unroll
            for (int q0 = 0; q0 < kLoads; q0 += kRows) {
                L r[kRows];                                              // read where the token changes
#pragma unroll
                for (int q = 0; q < kRows; ++q) {
                    const int i = i0 + q0 + q, t = i < live ? token[i + 1] : last_token;
                    if (t != last_token && mine) last.v = table[t * table_stride + u];
                    last_token = t;
                    r[q] = last;
                }
#pragma unroll
                for (int q = 0; q < kRows; ++q) {
                    d[q0 + q] = T(0);
#pragma unroll
                    for (int e = 0; e < L::n; ++e) d[q0 + q] += g[q0 + q].t[e] * r[q].t[e];
                }
            }
            // eight sums over the warp at once: every step halves the values that a lane carries on
#pragma unroll
            for (int h = kLoads / 2, m = 16; h >= 1; h /= 2, m /= 2)
#pragma unroll
                for (int q = 0; q < h; ++q) {
                    const bool upper = lane & m;
                    const T keep = upper ? d[q + h] : d[q], send = upper ? d[q] : d[q + h];
                    d[q] = keep + __shfl_xor_sync(0xffffffffu, send, m);
                }
            d[0] += __shfl_xor_sync(0xffffffffu, d[0], 2);
            d[0] += __shfl_xor_sync(0xffffffffu, d[0], 1);
            const int i = i0 + (lane >> 2);                              // of the three uppermost bits of the lane's number
            if ((lane & 3) == 0 && i < live) warp_dot[warp][i] = d[0];
        }
        if (!grad_table) continue;
        if (one) {
            L eight{};
#pragma unroll
            for (int q = 0; q < kLoads; ++q) {
                const T w = weight[i0 + q];
#pragma unroll
                for (int e = 0; e < L::n; ++e) eight.t[e] += w * g[q].t[e];
            }
#pragma unroll
            for (int e = 0; e < L::n; ++e) sum.t[e] += eight.t[e];
            const int i = i0 + kLoads - 1;
            if (token[i + 2] != t0 || i + 1 == count) give(i, t0);
            continue;
        }
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
            const int i = i0 + q;
            if (i >= live) break;
            const int t = token[i + 1];
            const T w = weight[i];
#pragma unroll
            for (int e = 0; e < L::n; ++e) sum.t[e] += w * g[q].t[e];
            if (token[i + 2] == t && i + 1 < count) continue;
            give(i, t);
        }
    }
    if constexpr (kWeights) {
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += kGradThreads) {
            T s = T(0);
            if (i < live)
                for (int w = 0; w < kWarps; ++w) s += warp_dot[w][i];
            const int pair = order[begin + i];
            if (gridDim.y == 1) grad_weights[pair] = scale * s;
            else dots[blockIdx.y * pairs + pair] = s;
        }
    }
}
template <typename T>
__global__ void __launch_bounds__(256) embedding_dots_kernel(const T* __restrict__ dots, long long pairs, int slabs, T scale, T* __restrict__ grad_weights) {
    for (long long i = blockIdx.x * 256LL + threadIdx.x; i < pairs; i += 256LL * gridDim.x) {
        double s = 0.0;
        for (int q = 0; q < slabs; ++q) s += dots[q * pairs + i];
        grad_weights[i] = static_cast<T>(scale * s);
    }
}

// The runs that cross chunks: the CTAs of the chunk where one begins add its parts in order, kJoinWays of them side by side. Most CTAs have none; they
// see that from the tokens, before the sums are there. (`parts` is written while CTAs of this kernel start: no promise that it is constant.)
constexpr int kJoinUnits = 32, kJoinWays = 8;
template <typename T, typename V>
__global__ void __launch_bounds__(kJoinUnits * kJoinWays) embedding_join_kernel(const int* __restrict__ tokens, long long pairs, int table_rows, int units, int chunk,
                                                                                int chunks, const V* parts, V* grad_table) {
    using L = Lanes<T, V>;
    __shared__ double joined[kJoinWays][L::n][kJoinUnits];
    const long long begin = static_cast<long long>(blockIdx.x) * chunk, end = begin + chunk;
    int t = table_rows, after = -1, before = -1;
    if (end < pairs) {
        t = tokens[end - 1];
        after = tokens[end];
        if (begin > 0) before = tokens[begin - 1];
    }
    const bool mine = t < table_rows && after == t && before != t;       // a run, and its beginning
    // (one CTA waits in any case, so that this kernel does not end before the one whose sums it reads)
    if (mine || (blockIdx.x == 0 && blockIdx.y == 0)) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (!mine) return;
    int more = 0;                                                        // chunks that go on with it
    for (int c0 = blockIdx.x + 1;; c0 += kJoinUnits * kJoinWays) {
        const int c = c0 + threadIdx.x;
        const int n = __syncthreads_count(c < chunks && tokens[static_cast<long long>(c) * chunk] == t);
        more += n;
        if (n < kJoinUnits * kJoinWays) break;
    }
    const int lane = threadIdx.x % kJoinUnits, way = threadIdx.x / kJoinUnits, u = blockIdx.y * kJoinUnits + lane;
    const int per = (more + 1 + kJoinWays - 1) / kJoinWays, first = way * per, last = min(more + 1, first + per);
    double sum[L::n] = {};
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
                for (int e = 0; e < L::n; ++e) sum[e] += v[q].t[e];
        }
    }
#pragma unroll
    for (int e = 0; e < L::n; ++e) joined[way][e][lane] = sum[e];
    __syncthreads();
    if (way > 0 || u >= units) return;
    L out;
#pragma unroll
    for (int e = 0; e < L::n; ++e) {
        for (int w = 1; w < kJoinWays; ++w) sum[e] += joined[w][e][lane];
        out.t[e] = static_cast<T>(sum[e]);
    }
    grad_table[static_cast<long long>(t) * units + u] = out.v;
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
    if (width < 0 || width > (1L << 30)) throw ArgError(std::string(what) + ": the row width must lie in 0 .. 2^30");         // (so that steps along a row stay ints)
    route_plan_bytes(num_rows, slots, 1);                                // rows and slots as there
}
void check_stride(const char* what, long stride, long width, long rows, bool written) {
    if (stride < 0 || (written && rows > 1 && stride < width)) throw ArgError(std::string(what) + ": bad row stride");
}
// Units of 16 bytes where all rows start on them, single values otherwise (49,152 rows of 512 floats, two slots: lookup 29 and 49 us, backward pass 45 and 94).
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

// Chunks of the sorted pairs: as many CTAs as 148 SMs hold where there are enough pairs (a constant, so that sizes do not depend on the device).
template <typename T>
int grad_chunk(long pairs, long width) {
    constexpr long ctas = 148 * grad_ctas<T>, per = 16 / sizeof(T) * kGradThreads;
    const long slabs = std::max(1L, (width + per - 1) / per);
    return static_cast<int>(std::max(16L, std::min<long>(kMaxChunk, (pairs * slabs + ctas - 1) / ctas)));
}

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
    token_sort(ids, pairs, table_rows, order, tokens, workspace, stream);
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
        unsigned tx = 1;
        while (tx < 32 && kAhead * tx < width / per) tx *= 2;
        const unsigned ty = 256 / tx;
        const unsigned blocks = static_cast<unsigned>(std::min<long long>((num_rows + ty - 1) / ty, 8LL * sm_count()));
        embedding_forward_kernel<T, V><<<blocks, dim3(tx, ty), 0, stream>>>(reinterpret_cast<const V*>(table), table_stride / per, table_rows, ids, num_rows, slots,
                                                                            static_cast<int>(width / per), weights, static_cast<T>(scale), reinterpret_cast<V*>(y),
                                                                            y_stride / per);
    });
    launched("embedding_forward_kernel");
}

namespace {
// Workspace: the parts of runs that cross chunks, and the dots of rows that several CTAs share (single values, if rows start anywhere).
struct Room { size_t parts, dots; };
template <typename T>
Room room(long pairs, long width) {
    const long chunk = grad_chunk<T>(pairs, width), chunks = (pairs + chunk - 1) / chunk, slabs = (width + kGradThreads - 1) / kGradThreads;
    return {(static_cast<size_t>(chunks) * 2 * width * sizeof(T) + 255) / 256 * 256, slabs > 1 ? static_cast<size_t>(slabs) * pairs * sizeof(T) : 0};
}
}  // namespace
template <typename T>
size_t embedding_backward_bytes(long num_rows, int slots, long width) {
    check_sizes("smx_embedding_backward", num_rows, slots, 1, width);
    if (width > 65535L * kJoinUnits) throw ArgError("smx_embedding_backward: the row width must lie in 0 .. 2097120");
    const Room r = room<T>(num_rows * slots, width);
    return r.parts + r.dots;
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
    if (!grad_table && !grad_weights) return;
    const size_t need = embedding_backward_bytes<T>(num_rows, slots, width);                                                  // (which checks the width too)
    if (workspace_bytes < need || (need && !workspace)) throw ArgError("smx_embedding_backward: the workspace is smaller than smx_embedding_backward_bytes says");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) throw ArgError("smx_embedding_backward: the workspace must start on a 16-byte boundary");
    if (grad_table && width > 0) SMX_CUDA(cudaMemsetAsync(grad_table, 0, static_cast<size_t>(table_rows) * width * sizeof(T), stream));
    if (pairs == 0) return;
    if (width == 0) {
        if (grad_weights) SMX_CUDA(cudaMemsetAsync(grad_weights, 0, static_cast<size_t>(pairs) * sizeof(T), stream));
        return;
    }
    T* const dots = reinterpret_cast<T*>(static_cast<char*>(workspace) + room<T>(pairs, width).parts);
    const int chunk = grad_chunk<T>(pairs, width), chunks = static_cast<int>((pairs + chunk - 1) / chunk);
    by_unit<T>(wide_rows<T>({grad_y, grad_table, grad_weights ? table : nullptr}, {grad_y_stride, width, grad_weights ? table_stride : 0}), [&](auto unit) {
        using V = decltype(unit);
        constexpr long per = sizeof(V) / sizeof(T);
        const int units = static_cast<int>(width / per);
        const int slabs = (units + kGradThreads - 1) / kGradThreads, joins = (units + kJoinUnits - 1) / kJoinUnits;
        const auto kernel = grad_weights ? embedding_grad_kernel<T, V, true> : embedding_grad_kernel<T, V, false>;
        kernel<<<dim3(chunks, slabs), kGradThreads, 0, stream>>>(reinterpret_cast<const V*>(grad_y), grad_y_stride / per, reinterpret_cast<const V*>(table),
                                                                 table_stride / per, order, tokens, pairs, slots, table_rows, units, weights, static_cast<T>(scale),
                                                                 chunk, reinterpret_cast<V*>(grad_table), static_cast<V*>(workspace), dots, grad_weights);
        launched("embedding_grad_kernel");
        if (grad_table && chunks > 1) {
            chain_launch(Launcher{stream, true}, embedding_join_kernel<T, V>, dim3(chunks, joins), kJoinUnits * kJoinWays, 0, 1, tokens,
                         static_cast<long long>(pairs), table_rows, units, chunk, chunks, static_cast<const V*>(workspace), reinterpret_cast<V*>(grad_table));
            ++operator_launches;
        }
        if (grad_weights && slabs > 1) {
            embedding_dots_kernel<T><<<static_cast<unsigned>(std::min(8LL * sm_count(), (pairs + 255LL) / 256)), 256, 0, stream>>>(dots, pairs, slabs, static_cast<T>(scale),
                                                                                                                                  grad_weights);
            launched("embedding_dots_kernel");
        }
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
