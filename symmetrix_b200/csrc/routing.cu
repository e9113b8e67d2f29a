// Rows sorted by group and back (smx_route_*): a stable counting sort of the pairs (row, slot) by group, the copy of the rows into that
// order, their weighted sum back, and both gradients. A pair whose id is not a group (negative or too large) is an empty slot: its
// position is -1, nothing of it is read, and it is listed behind the last group.
//
//   order[p] = n * slots + s of the p-th pair;  position[n, s] = p or -1;  offsets[g] = first p of group g, offsets[G] = pairs in groups
//   dispatch          rows[position[n, s]] = x[n]
//   combine           y[n] = base[n] + sum_s w[n, s] rows[position[n, s]], slots in order
//   combine_backward  grad_rows[position[n, s]] = w[n, s] grad_y[n],  grad_w[n, s] = <grad_y[n], rows[position[n, s]]>
//
// The gradient of dispatch is combine without weights. No atomics: the same call gives the same bits.
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>

#include "common.cuh"
#include "routing.hpp"

namespace smx {
namespace {

constexpr int kMaxGroups = SMX_ROUTE_MAX_GROUPS;

// ------------------------------------------------------------------------------------------- plan
// Pairs are counted and ranked by warps that own consecutive pairs: 32 at a time, lanes of equal group found with match_any, one counter
// per (warp, group) in shared memory that only that warp touches. Equal keys therefore keep their order. Latency bounds it: 13.5 us for 7,545
// pairs in one CTA, 6 + 4 + 10 us for the three kernels at 196,608 pairs (2.4 MB).
// kSlots: the keys are the slots of pairs, ids[i] = n * groups + slot (see route_slots).
template <bool kSlots>
__device__ __forceinline__ int route_key(const int* ids, long long i, int groups) {
    const int g = ids[i];
    if (kSlots) return g % groups;
    return (g < 0 || g >= groups) ? groups : g;
}

template <bool kSlots>
__device__ __forceinline__ void route_count(const int* __restrict__ ids, long long begin, long long end, int groups, int* __restrict__ hist) {
    const int lane = threadIdx.x & 31;
    for (long long i0 = begin; i0 < end; i0 += 32) {
        const bool in = i0 + lane < end;
        const int g = in ? route_key<kSlots>(ids, i0 + lane, groups) : groups + 1;
        const unsigned same = __match_any_sync(0xffffffffu, g);
        if (in && lane == __ffs(same) - 1) hist[g] += __popc(same);
        __syncwarp();
    }
}

// `next[g]`: where this warp's next pair of group g goes.
template <bool kSlots>
__device__ __forceinline__ void route_place(const int* __restrict__ ids, long long begin, long long end, int groups, int* __restrict__ next,
                                            int* __restrict__ order, int* __restrict__ position) {
    const int lane = threadIdx.x & 31;
    for (long long i0 = begin; i0 < end; i0 += 32) {
        const bool in = i0 + lane < end;
        const int g = in ? route_key<kSlots>(ids, i0 + lane, groups) : groups + 1;
        const unsigned same = __match_any_sync(0xffffffffu, g);
        int first = 0;
        if (in) first = next[g];
        __syncwarp();
        if (in) {
            const int p = first + __popc(same & ((1u << lane) - 1u));
            order[p] = static_cast<int>(i0 + lane);
            if (!kSlots) position[i0 + lane] = g < groups ? p : -1;
            if (lane == __ffs(same) - 1) next[g] = first + __popc(same);
        }
        __syncwarp();
    }
}

// Exclusive scan of v[0 .. n) in shared memory by the whole CTA (a multiple of 32 threads, at most 1,024); returns nothing, v[n] receives the
// total. `sums` holds 33 ints.
__device__ __forceinline__ void cta_scan(int* v, int n, int* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    const int per = (n + static_cast<int>(blockDim.x) - 1) / static_cast<int>(blockDim.x);
    const int begin = min(n, static_cast<int>(threadIdx.x) * per), end = min(n, begin + per);
    int mine = 0;
    for (int i = begin; i < end; ++i) mine += v[i];
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += up;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int s = lane < warps ? sums[lane] : 0, t = s;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, t, d);
            if (lane >= d) t += up;
        }
        sums[lane] = t - s;
        if (lane == 31) sums[32] = t;
    }
    __syncthreads();
    int run = sums[warp] + incl - mine;
    for (int i = begin; i < end; ++i) { const int c = v[i]; v[i] = run; run += c; }
    if (threadIdx.x == 0) v[n] = sums[32];
    __syncthreads();
}

// Few pairs: one CTA does all three steps.
constexpr int kSmallPlanThreads = 1024, kSmallPlanPairs = 8192;
template <bool kSlots>
__global__ void __launch_bounds__(kSmallPlanThreads) route_plan_small_kernel(const int* __restrict__ ids, int pairs, int groups, int warps_used,
                                                                             int* __restrict__ order, int* __restrict__ position,
                                                                             int* __restrict__ offsets) {
    extern __shared__ int route_smem[];
    __shared__ int sums[33];
    const int bins = groups + 1, warp = threadIdx.x >> 5;
    int* total = route_smem;                    // bins + 1
    int* hist = route_smem + bins + 1;          // [warps_used][bins]
    for (int i = threadIdx.x; i < warps_used * bins; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    const int per = ((pairs + warps_used - 1) / warps_used + 31) & ~31;
    const int begin = min(pairs, warp * per), end = min(pairs, begin + per);
    if (warp < warps_used) route_count<kSlots>(ids, begin, end, groups, hist + warp * bins);
    __syncthreads();
    for (int g = threadIdx.x; g < bins; g += blockDim.x) {
        int run = 0;
        for (int w = 0; w < warps_used; ++w) { const int c = hist[w * bins + g]; hist[w * bins + g] = run; run += c; }
        total[g] = run;
    }
    __syncthreads();
    cta_scan(total, bins, sums);
    for (int g = threadIdx.x; g < bins; g += blockDim.x) {
        if (!kSlots) offsets[g] = total[g];     // bins = groups + 1 entries: the start of the empty slots is the end of the groups
        for (int w = 0; w < warps_used; ++w) hist[w * bins + g] += total[g];
    }
    __syncthreads();
    if (warp < warps_used) route_place<kSlots>(ids, begin, end, groups, hist + warp * bins, order, position);
}

// Many pairs: counts per chunk, a scan over the chunks of every group, then the ranks. chunk_hist is [bins][chunks].
constexpr int kPlanWarps = 8, kPlanThreads = 32 * kPlanWarps, kPlanChunk = 2048;
template <bool kSlots>
__global__ void __launch_bounds__(kPlanThreads) route_count_kernel(const int* __restrict__ ids, long long pairs, int groups, int chunks,
                                                                   int* __restrict__ chunk_hist) {
    extern __shared__ int route_smem[];
    const int bins = groups + 1, warp = threadIdx.x >> 5;
    for (int i = threadIdx.x; i < kPlanWarps * bins; i += kPlanThreads) route_smem[i] = 0;
    __syncthreads();
    constexpr int per = kPlanChunk / kPlanWarps;
    const long long begin = min(pairs, static_cast<long long>(blockIdx.x) * kPlanChunk + warp * per), end = min(pairs, begin + per);
    route_count<kSlots>(ids, begin, end, groups, route_smem + warp * bins);
    __syncthreads();
    for (int g = threadIdx.x; g < bins; g += kPlanThreads) {
        int sum = 0;
        for (int w = 0; w < kPlanWarps; ++w) sum += route_smem[w * bins + g];
        chunk_hist[static_cast<long long>(g) * chunks + blockIdx.x] = sum;
    }
}
__global__ void __launch_bounds__(256) route_scan_kernel(int bins, int chunks, int* __restrict__ chunk_hist, int* __restrict__ total) {
    const int lane = threadIdx.x & 31;
    const int g = (blockIdx.x * 256 + threadIdx.x) >> 5;
    if (g >= bins) return;
    int* row = chunk_hist + static_cast<long long>(g) * chunks;
    int run = 0;
    for (int c0 = 0; c0 < chunks; c0 += 32) {
        const int v = c0 + lane < chunks ? row[c0 + lane] : 0;
        int incl = v;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += up;
        }
        if (c0 + lane < chunks) row[c0 + lane] = run + incl - v;
        run += __shfl_sync(0xffffffffu, incl, 31);
    }
    if (lane == 0) total[g] = run;
}
template <bool kSlots>
__global__ void __launch_bounds__(kPlanThreads) route_place_kernel(const int* __restrict__ ids, long long pairs, int groups, int chunks,
                                                                   const int* __restrict__ chunk_prefix, const int* __restrict__ total,
                                                                   int* __restrict__ order, int* __restrict__ position, int* __restrict__ offsets) {
    extern __shared__ int route_smem[];
    __shared__ int sums[33];
    const int bins = groups + 1, warp = threadIdx.x >> 5;
    int* start = route_smem;                    // bins + 1
    int* hist = route_smem + bins + 1;
    for (int i = threadIdx.x; i < kPlanWarps * bins; i += kPlanThreads) hist[i] = 0;
    for (int g = threadIdx.x; g < bins; g += kPlanThreads) start[g] = total[g];
    __syncthreads();
    cta_scan(start, bins, sums);
    constexpr int per = kPlanChunk / kPlanWarps;
    const long long begin = min(pairs, static_cast<long long>(blockIdx.x) * kPlanChunk + warp * per), end = min(pairs, begin + per);
    route_count<kSlots>(ids, begin, end, groups, hist + warp * bins);
    __syncthreads();
    for (int g = threadIdx.x; g < bins; g += kPlanThreads) {
        if (!kSlots && blockIdx.x == 0) offsets[g] = start[g];
        int run = start[g] + chunk_prefix[static_cast<long long>(g) * chunks + blockIdx.x];
        for (int w = 0; w < kPlanWarps; ++w) { const int c = hist[w * bins + g]; hist[w * bins + g] = run; run += c; }
    }
    __syncthreads();
    route_place<kSlots>(ids, begin, end, groups, hist + warp * bins, order, position);
}

// Where group g begins among slot s's places (sorted positions, ascending; runs of num_rows): a warp each, cutting the run into 33 pieces per step.
__global__ void __launch_bounds__(256) route_slot_offsets_kernel(const int* __restrict__ places, int num_rows, int slots, const int* __restrict__ offsets,
                                                                 int groups, int* __restrict__ slot_offsets) {
    const int t = (blockIdx.x * 256 + threadIdx.x) >> 5, lane = threadIdx.x & 31;
    if (t >= slots * (groups + 1)) return;
    const int* run = places + static_cast<long long>(t / (groups + 1)) * num_rows;
    const int bound = offsets[t % (groups + 1)];
    long long lo = 0, hi = num_rows;                 // the answer lies in lo .. hi
    while (lo < hi) {
        const long long at = lo + (hi - lo) * (lane + 1) / 33;                  // ascending, below hi
        const int below = __popc(__ballot_sync(0xffffffffu, run[at] < bound));  // a prefix of the lanes
        const long long next = __shfl_sync(0xffffffffu, at, below & 31), last = __shfl_sync(0xffffffffu, at, below ? below - 1 : 0);
        if (below < 32) hi = next;
        if (below) lo = last + 1;
    }
    if (lane == 0) slot_offsets[t] = static_cast<int>(lo);
}

// ------------------------------------------------------------------------------------------- rows
// A row is walked in units of V: 16 bytes where every row starts on such a boundary, else single values.
template <typename T> struct Wide;
template <> struct Wide<float> { using type = float4; };
template <> struct Wide<double> { using type = double2; };
template <typename T, typename V>
union Lanes {
    static constexpr int n = sizeof(V) / sizeof(T);
    V v;
    T t[n];
};

// CTA: blockDim.x threads along a row, blockDim.y rows at a time. 98,304 rows of 512 floats into two slots: 94 us for
// 604 MB, 6.4 TB/s, the copy rate of the memory.
template <typename V>
__global__ void __launch_bounds__(256) route_dispatch_kernel(const V* __restrict__ x, long long x_stride, long long num_rows, int slots, int units,
                                                             const int* __restrict__ position, const int* __restrict__ offsets, int groups,
                                                             V* __restrict__ rows, int zero_tail) {
    for (long long n = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y; n < num_rows; n += static_cast<long long>(gridDim.x) * blockDim.y) {
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
            const V v = x[n * x_stride + u];
            for (int s = 0; s < slots; ++s) {
                const int p = position[n * slots + s];
                if (p >= 0) rows[static_cast<long long>(p) * units + u] = v;
            }
        }
    }
    if (!zero_tail) return;
    const V zero{};
    for (long long p = offsets[groups] + static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y; p < num_rows * slots;
         p += static_cast<long long>(gridDim.x) * blockDim.y)
        for (int u = threadIdx.x; u < units; u += blockDim.x) rows[p * units + u] = zero;
}

// Bound by HBM; 98,304 rows of 512 floats, two slots and a base: 131 us for 805 MB, 6.2 TB/s.
template <typename T, typename V>
__global__ void __launch_bounds__(256) route_combine_kernel(const V* __restrict__ rows, const int* __restrict__ position, long long num_rows, int slots,
                                                            int units, const T* __restrict__ weights, const V* base, long long base_stride, V* y,
                                                            long long y_stride) {
    using L = Lanes<T, V>;
    for (long long n = static_cast<long long>(blockIdx.x) * blockDim.y + threadIdx.y; n < num_rows; n += static_cast<long long>(gridDim.x) * blockDim.y) {
        for (int u = threadIdx.x; u < units; u += blockDim.x) {
            L sum{};
            if (base) sum.v = base[n * base_stride + u];
            for (int s = 0; s < slots; ++s) {
                const int p = position[n * slots + s];
                if (p < 0) continue;
                L r;
                r.v = rows[static_cast<long long>(p) * units + u];
                const T w = weights ? weights[n * slots + s] : T(1);
#pragma unroll
                for (int q = 0; q < L::n; ++q) sum.t[q] += w * r.t[q];
            }
            y[n * y_stride + u] = sum.v;
        }
    }
}

// A warp per row, or a CTA (kWarps = 8) where there are too few rows to fill the GPU with warps; the row's gradient is read once for up to
// kSlotBlock slots. 49,152 rows of 512 floats, two slots, with the weights' gradient: 89 us for 503 MB, 5.7 TB/s; 1,029 rows of
// 2,304 doubles, three slots: 24 us by CTAs.
constexpr int kSlotBlock = 4;
template <typename T, typename V, int kWarps>
__global__ void __launch_bounds__(256) route_combine_backward_kernel(const V* __restrict__ grad_y, long long grad_y_stride, const V* __restrict__ rows,
                                                                     const int* __restrict__ position, const int* __restrict__ offsets, int groups,
                                                                     long long num_rows, int slots, int units, const T* __restrict__ weights,
                                                                     V* __restrict__ grad_rows, T* __restrict__ grad_weights, int zero_tail) {
    using L = Lanes<T, V>;
    constexpr int kLanes = 32 * kWarps;
    __shared__ T parts[kWarps][kSlotBlock];
    const int lane = threadIdx.x % kLanes;
    const long long warp = (static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x) / kLanes, warps = static_cast<long long>(gridDim.x) * blockDim.x / kLanes;
    for (long long n = warp; n < num_rows; n += warps) {
        for (int s0 = 0; s0 < slots; s0 += kSlotBlock) {
            int p[kSlotBlock];
            T w[kSlotBlock], dot[kSlotBlock];
#pragma unroll
            for (int q = 0; q < kSlotBlock; ++q) {
                p[q] = s0 + q < slots ? position[n * slots + s0 + q] : -1;
                w[q] = p[q] >= 0 ? (weights ? weights[n * slots + s0 + q] : T(1)) : T(0);
                dot[q] = T(0);
            }
            for (int u = lane; u < units; u += kLanes) {
                L g;
                g.v = grad_y[n * grad_y_stride + u];
#pragma unroll
                for (int q = 0; q < kSlotBlock; ++q) {
                    if (p[q] < 0) continue;
                    if (grad_weights) {
                        L r;
                        r.v = rows[static_cast<long long>(p[q]) * units + u];
#pragma unroll
                        for (int e = 0; e < L::n; ++e) dot[q] += g.t[e] * r.t[e];
                    }
                    L out;
#pragma unroll
                    for (int e = 0; e < L::n; ++e) out.t[e] = w[q] * g.t[e];
                    grad_rows[static_cast<long long>(p[q]) * units + u] = out.v;
                }
            }
            if (grad_weights) {
#pragma unroll
                for (int q = 0; q < kSlotBlock; ++q) {
#pragma unroll
                    for (int d = 16; d > 0; d >>= 1) dot[q] += __shfl_xor_sync(0xffffffffu, dot[q], d);
                    if (kWarps == 1 && lane == 0 && s0 + q < slots) grad_weights[n * slots + s0 + q] = dot[q];
                    if (kWarps > 1 && (lane & 31) == 0) parts[lane >> 5][q] = dot[q];
                }
                if constexpr (kWarps > 1) {
                    __syncthreads();
                    if (lane < kSlotBlock && s0 + lane < slots) {
                        T sum = T(0);
                        for (int w = 0; w < kWarps; ++w) sum += parts[w][lane];
                        grad_weights[n * slots + s0 + lane] = sum;
                    }
                    __syncthreads();
                }
            }
        }
    }
    if (!zero_tail) return;
    const V zero{};
    for (long long p = offsets[groups] + warp; p < num_rows * slots; p += warps)
        for (int u = lane; u < units; u += kLanes) grad_rows[p * units + u] = zero;
}

// ------------------------------------------------------------------------------------------- host side
void check_sizes(const char* what, long num_rows, int slots, int num_groups) {
    if (num_rows < 0) throw ArgError(std::string(what) + ": negative number of rows");
    if (slots < 1 || slots > SMX_ROUTE_MAX_SLOTS) throw ArgError(std::string(what) + ": slots must lie in 1 .. " + std::to_string(SMX_ROUTE_MAX_SLOTS));
    if (num_groups < 1 || num_groups > kMaxGroups) throw ArgError(std::string(what) + ": the number of groups must lie in 1 .. " + std::to_string(kMaxGroups));
    if (num_rows > (INT_MAX - kPlanChunk) / slots) throw ArgError(std::string(what) + ": rows x slots exceeds the range of 32-bit positions");
}
void check_width(const char* what, long width, long stride) {
    if (width < 0 || width > INT_MAX) throw ArgError(std::string(what) + ": bad row width");
    if (stride < 0) throw ArgError(std::string(what) + ": negative row stride");
}

template <typename T>
bool wide_rows(std::initializer_list<const void*> pointers, std::initializer_list<long> strides) {
    constexpr long per = 16 / sizeof(T);
    for (long s : strides) if (s % per != 0) return false;
    for (const void* p : pointers) if (reinterpret_cast<uintptr_t>(p) & 15) return false;
    return true;
}

struct RowGrid { dim3 grid, block; };
RowGrid row_grid(long num_rows, long units) {
    unsigned tx = 32;
    while (tx < 256 && tx < units) tx *= 2;
    const unsigned ty = 256 / tx;
    const long long blocks = (num_rows + ty - 1) / ty;
    return {dim3(static_cast<unsigned>(std::max(1LL, std::min<long long>(blocks, 64LL * sm_count())))), dim3(tx, ty)};
}

}  // namespace
void check_pointers(const char* what, size_t bytes, std::initializer_list<const void*> pointers) {
    for (const void* p : pointers)
        if (reinterpret_cast<uintptr_t>(p) % bytes) throw ArgError(std::string(what) + ": an array does not start on a multiple of its elements' size");
}
namespace {

void launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
    ++operator_launches;
}

}  // namespace

thread_local long operator_launches = 0;

int sm_count() {
    static std::atomic<int> count[64];
    int dev = 0;
    SMX_CUDA(cudaGetDevice(&dev));
    const int known = dev < 64 ? count[dev].load(std::memory_order_relaxed) : 0;
    if (known) return known;
    int n = 0;
    SMX_CUDA(cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev));
    if (dev < 64) count[dev].store(n, std::memory_order_relaxed);
    return n;
}
bool first_on_device(std::atomic<bool> (&done)[64]) {
    int dev = 0;
    SMX_CUDA(cudaGetDevice(&dev));
    return dev >= 64 || !done[dev].load(std::memory_order_acquire);
}
void mark_on_device(std::atomic<bool> (&done)[64]) {
    int dev = 0;
    SMX_CUDA(cudaGetDevice(&dev));
    if (dev < 64) done[dev].store(true, std::memory_order_release);
}

size_t route_plan_bytes(long num_rows, int slots, int num_groups) {
    check_sizes("smx_route_plan", num_rows, slots, num_groups);
    const long long pairs = static_cast<long long>(num_rows) * slots;
    if (pairs <= kSmallPlanPairs) return 0;
    const long long chunks = (pairs + kPlanChunk - 1) / kPlanChunk;
    return static_cast<size_t>((num_groups + 1) * (chunks + 1) * sizeof(int));
}

namespace {
template <bool kSlots>
void counting_sort(const int* ids, long long pairs, int num_groups, int* order, int* position, int* offsets, void* workspace, cudaStream_t stream) {
    const int bins = num_groups + 1;
    if (pairs <= kSmallPlanPairs) {
        // a warp for every 32 pairs, as far as their counters fit into 128 KB
        int warps = static_cast<int>(std::min<long long>(32, std::max<long long>(1, (pairs + 31) / 32)));
        while (warps > 1 && (warps + 1) * bins > 32768) warps /= 2;
        const int smem = ((warps + 1) * bins + 1) * static_cast<int>(sizeof(int));
        static std::atomic<bool> done[64];
        // beyond 48 KB a launch has to be allowed, and the kernel's own arrays (the sums of its scan) count too
        if (smem > 47 * 1024 && first_on_device(done)) {
            SMX_CUDA(cudaFuncSetAttribute(route_plan_small_kernel<kSlots>, cudaFuncAttributeMaxDynamicSharedMemorySize, 160 * 1024));
            mark_on_device(done);
        }
        const int threads = std::max(128, 32 * warps);
        route_plan_small_kernel<kSlots><<<1, threads, smem, stream>>>(ids, static_cast<int>(pairs), num_groups, warps, order, position, offsets);
        launched("route_plan_small_kernel");
        return;
    }
    const int chunks = static_cast<int>((pairs + kPlanChunk - 1) / kPlanChunk);
    int* hist = static_cast<int*>(workspace);
    int* total = hist + static_cast<size_t>(bins) * chunks;
    const int smem = kPlanWarps * bins * static_cast<int>(sizeof(int));
    route_count_kernel<kSlots><<<chunks, kPlanThreads, smem, stream>>>(ids, pairs, num_groups, chunks, hist);
    launched("route_count_kernel");
    route_scan_kernel<<<(bins * 32 + 255) / 256, 256, 0, stream>>>(bins, chunks, hist, total);
    launched("route_scan_kernel");
    route_place_kernel<kSlots><<<chunks, kPlanThreads, smem + (bins + 1) * static_cast<int>(sizeof(int)), stream>>>(ids, pairs, num_groups, chunks, hist, total,
                                                                                                                   order, position, offsets);
    launched("route_place_kernel");
}
}  // namespace

void route_plan(const int* ids, long num_rows, int slots, int num_groups, int* order, int* position, int* offsets, void* workspace,
                size_t workspace_bytes, cudaStream_t stream) {
    const size_t need = route_plan_bytes(num_rows, slots, num_groups);
    check_pointers("smx_route_plan", sizeof(int), {ids, order, position, offsets, workspace});
    const long long pairs = static_cast<long long>(num_rows) * slots;
    if (!offsets || (pairs > 0 && (!ids || !order || !position))) throw ArgError("smx_route_plan: null pointer");
    if (workspace_bytes < need || (need && !workspace)) throw ArgError("smx_route_plan: the workspace is smaller than smx_route_plan_bytes says");
    counting_sort<false>(ids, pairs, num_groups, order, position, offsets, workspace, stream);
}

size_t route_slots_bytes(long num_rows, int slots) { return route_plan_bytes(num_rows * slots, 1, slots); }
void route_slots(const int* order, long num_rows, int slots, const int* offsets, int num_groups, int* places, int* slot_offsets, void* workspace,
                 cudaStream_t stream) {
    counting_sort<true>(order, static_cast<long long>(num_rows) * slots, slots, places, nullptr, nullptr, workspace, stream);
    const int n = slots * (num_groups + 1);
    route_slot_offsets_kernel<<<(n + 7) / 8, 256, 0, stream>>>(places, static_cast<int>(num_rows), slots, offsets, num_groups, slot_offsets);
    launched("route_slot_offsets_kernel");
}

template <typename T>
void route_dispatch(const T* x, long x_stride, long num_rows, int slots, long width, const int* position, const int* offsets, int num_groups,
                    T* rows, bool zero_tail, cudaStream_t stream) {
    check_sizes("smx_route_dispatch", num_rows, slots, num_groups);
    check_width("smx_route_dispatch", width, x_stride);
    if (num_rows == 0 || width == 0) return;
    if (!x || !position || !offsets || !rows) throw ArgError("smx_route_dispatch: null pointer");
    check_pointers("smx_route_dispatch", sizeof(int), {position, offsets});
    check_pointers("smx_route_dispatch", sizeof(T), {x, rows});
    auto go = [&](auto unit) {
        using V = decltype(unit);
        constexpr long per = sizeof(V) / sizeof(T);
        const RowGrid g = row_grid(num_rows, width / per);
        route_dispatch_kernel<V><<<g.grid, g.block, 0, stream>>>(reinterpret_cast<const V*>(x), x_stride / per, num_rows, slots, static_cast<int>(width / per),
                                                                 position, offsets, num_groups, reinterpret_cast<V*>(rows), zero_tail ? 1 : 0);
    };
    if (wide_rows<T>({x, rows}, {x_stride, width})) go(typename Wide<T>::type{});
    else go(T{});
    launched("route_dispatch_kernel");
}

template <typename T>
void route_combine(const T* rows, const int* position, long num_rows, int slots, long width, const T* weights, const T* base, long base_stride,
                   T* y, long y_stride, cudaStream_t stream) {
    check_sizes("smx_route_combine", num_rows, slots, 1);
    check_width("smx_route_combine", width, base ? base_stride : 0);
    check_width("smx_route_combine", width, y_stride);
    if (num_rows == 0 || width == 0) return;
    if (!rows || !position || !y) throw ArgError("smx_route_combine: null pointer");
    check_pointers("smx_route_combine", sizeof(int), {position});
    check_pointers("smx_route_combine", sizeof(T), {rows, weights, base, y});
    if (y_stride < width && num_rows > 1) throw ArgError("smx_route_combine: the output's rows overlap");
    if (!base) base_stride = 0;
    auto go = [&](auto unit) {
        using V = decltype(unit);
        constexpr long per = sizeof(V) / sizeof(T);
        const RowGrid g = row_grid(num_rows, width / per);
        route_combine_kernel<T, V><<<g.grid, g.block, 0, stream>>>(reinterpret_cast<const V*>(rows), position, num_rows, slots, static_cast<int>(width / per),
                                                                   weights, reinterpret_cast<const V*>(base), base_stride / per, reinterpret_cast<V*>(y),
                                                                   y_stride / per);
    };
    if (wide_rows<T>({rows, base, y}, {width, base_stride, y_stride})) go(typename Wide<T>::type{});
    else go(T{});
    launched("route_combine_kernel");
}

template <typename T>
void route_combine_backward(const T* grad_y, long grad_y_stride, const T* rows, const int* position, const int* offsets, int num_groups,
                            long num_rows, int slots, long width, const T* weights, T* grad_rows, T* grad_weights, bool zero_tail,
                            cudaStream_t stream) {
    check_sizes("smx_route_combine_backward", num_rows, slots, num_groups);
    check_width("smx_route_combine_backward", width, grad_y_stride);
    if (num_rows == 0) return;
    if (!position || !offsets || (width > 0 && (!grad_y || !grad_rows || (grad_weights && !rows)))) throw ArgError("smx_route_combine_backward: null pointer");
    check_pointers("smx_route_combine_backward", sizeof(int), {position, offsets});
    check_pointers("smx_route_combine_backward", sizeof(T), {grad_y, rows, weights, grad_rows, grad_weights});
    auto go = [&](auto unit) {
        using V = decltype(unit);
        constexpr long per = sizeof(V) / sizeof(T);
        // CTAs of eight rows leave SMs without one below 8 x 4 x SMs rows
        const bool few = num_rows < 32LL * sm_count() && width / per > 64;
        const auto kernel = few ? route_combine_backward_kernel<T, V, 8> : route_combine_backward_kernel<T, V, 1>;
        const unsigned grid = static_cast<unsigned>(std::max<long long>(1, std::min<long long>(few ? num_rows : (num_rows + 7) / 8, 64LL * sm_count())));
        kernel<<<grid, 256, 0, stream>>>(reinterpret_cast<const V*>(grad_y), grad_y_stride / per, reinterpret_cast<const V*>(rows), position, offsets,
                                         num_groups, num_rows, slots, static_cast<int>(width / per), weights, reinterpret_cast<V*>(grad_rows),
                                         grad_weights, zero_tail ? 1 : 0);
    };
    if (wide_rows<T>({grad_y, rows, grad_rows}, {grad_y_stride, width})) go(typename Wide<T>::type{});
    else go(T{});
    launched("route_combine_backward_kernel");
}

#define SMX_ROUTE_INSTANCE(T)                                                                                                                       \
    template void route_dispatch<T>(const T*, long, long, int, long, const int*, const int*, int, T*, bool, cudaStream_t);                         \
    template void route_combine<T>(const T*, const int*, long, int, long, const T*, const T*, long, T*, long, cudaStream_t);                       \
    template void route_combine_backward<T>(const T*, long, const T*, const int*, const int*, int, long, int, long, const T*, T*, T*, bool, cudaStream_t);
SMX_ROUTE_INSTANCE(float)
SMX_ROUTE_INSTANCE(double)

}  // namespace smx
