// Linears of all degrees with low-rank adapters of many requests beside the shared weights (smx_adapter_*).
//
// A row is (atom n, component m of degree l). With slots s, group g = g(n, s), mixing weight w = w[n, s]:
//   forward   t = x A_g,  y = x W + sum_s w t B_g
//   backward  h = gy B_g^T,  gx = gy W^T + sum_s w h A_g^T,  gA_g = sum w x^T h,  gB_g = sum w t^T gy,  gw = sum_(l, m) <t, h>
// The backward pass to x is the forward pass with the transposed matrices, so one kernel does both.
//
// Rows are taken in the order of the routing (csrc/routing.cu), in tiles that never mix groups. With one slot a row belongs to one tile: the
// tile's kernel makes the shared product, its own adapter's and their sum, so x is read and y is written once. With more slots the plan is split
// by slot: the first slot's pass is that of one slot, the others' add their products to the rows it wrote, in slot order (a row is in one
// tile of a slot's pass, so nothing races). Sums over rows (gA, gB) are split into chunks of a fixed number of rows, whose partial sums are added in order: no atomics.
#include "adapters.hpp"

#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "routing.hpp"
#include "row_tiles.cuh"

namespace smx {
namespace {

constexpr int kMaxDegrees = SMX_ADAPTER_MAX_DEGREES, kMaxRank = SMX_ADAPTER_MAX_RANK;

// One pass over the rows, in either direction: out rows = in rows . W + weight (in rows . first_g) . second_g, degree by degree.
template <typename T>
struct PassDegree {
    int comps, Kd, Nc;
    long long in_off, out_off;
    const T* W; const T* first; const T* second;     // in the kernels' layouts; W null: no shared weights
    long long first_group, second_group;             // values from adapter to adapter
    T* hidden;                                       // [pairs * comps][rank] in sorted order, or null
};
template <typename T>
struct Pass {
    PassDegree<T> degree[kMaxDegrees];
    int rank, groups, slots;
    long long pairs;                                 // places in all
    const int* order; const int* offsets;
    const int* places;                               // of a slot (csrc/routing.hpp), with its offsets; null: the plan itself
    const T* weights;
    const T* in; long long in_stride;
    T* out; long long out_stride;                    // null: only the hidden rows
    int add;           // to `out`, instead of writing it
    int tail;          // the rows without a group are a last group of their own
    int* status;       // null, or where a wait that ran out is reported (float32; the float64 kernels have no waits of the kind)
    int expire_polls;  // test switch of those waits
};

// ------------------------------------------------------------------------------------------- gradients of the adapters
// part[chunk][k][r] = sum over the chunk's rows of a[row][k] weight[row] h[row][r]; a is x with h = gy B^T, or gy with h = x A. A chunk has 512 rows,
// fewer where those would leave SMs idle (818 atoms of 2 slots and 26 channels, rank 55: 23 us with 64 rows, 118 with 512).
constexpr int kGradChunk = 512;
template <typename T>
struct GradProblem {
    int comps, Kd;
    const T* a; long long a_stride, a_off;
    const T* hidden;                             // [pairs * comps][rank], not weighted
    T* part;                                     // [chunks][Kd][rank]
    T* grad; long long g_group, g_k, g_r;        // gA: [group][k][r], gB: [group][r][k]
};
template <typename T>
struct GradPass {
    GradProblem<T> problem[2 * kMaxDegrees];
    int rank, groups, slots, chunk;
    long long pairs;
    const int* order; const int* offsets;
    const T* weights;
};

// grad of group blockIdx.x: its chunks added in order (none: zero).
template <typename T>
__global__ void __launch_bounds__(256) adapter_grad_sum_kernel(const __grid_constant__ GradPass<T> pass) {
    const GradProblem<T>& d = pass.problem[blockIdx.z];
    const int g = blockIdx.x, R = pass.rank;
    __shared__ long long sh[2];
    if (threadIdx.x < 32) {
        long long before = 0;
        for (int q = threadIdx.x; q < g; q += 32)
            before += (static_cast<long long>(pass.offsets[q + 1] - pass.offsets[q]) * d.comps + pass.chunk - 1) / pass.chunk;
#pragma unroll
        for (int s = 16; s > 0; s >>= 1) before += __shfl_xor_sync(0xffffffffu, before, s);
        if (threadIdx.x == 0) {
            sh[0] = before;
            sh[1] = (static_cast<long long>(pass.offsets[g + 1] - pass.offsets[g]) * d.comps + pass.chunk - 1) / pass.chunk;
        }
    }
    __syncthreads();
    const long long c0 = sh[0], chunks = sh[1];
    const long long size = static_cast<long long>(d.Kd) * R;
    for (long long i = static_cast<long long>(blockIdx.y) * 256 + threadIdx.x; i < size; i += 256LL * gridDim.y) {
        T s = T(0);
        const T* part = d.part + c0 * size + i;
        for (long long c = 0; c < chunks; c += 8) {                // eight loads in flight, added in order
            T v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = c + u < chunks ? part[(c + u) * size] : T(0);
#pragma unroll
            for (int u = 0; u < 8; ++u) s += v[u];
        }
        d.grad[g * d.g_group + (i / R) * d.g_k + (i % R) * d.g_r] = s;
    }
}

// gw of every pair: a warp adds the products of both hidden rows over components, degree after degree. Empty slots get zero.
template <typename T>
struct WeightGrad {
    const T* t[kMaxDegrees]; const T* h[kMaxDegrees];
    int comps[kMaxDegrees];
    int degrees, rank;
    long long pairs;
    const int* position;
    T* grad;
};
template <typename T>
__global__ void __launch_bounds__(256) adapter_weight_grad_kernel(const __grid_constant__ WeightGrad<T> a) {
    const int lane = threadIdx.x & 31;
    for (long long i = (static_cast<long long>(blockIdx.x) * 256 + threadIdx.x) >> 5; i < a.pairs; i += (static_cast<long long>(gridDim.x) * 256) >> 5) {
        const int p = a.position[i];
        T s = T(0);
        if (p >= 0)
            for (int d = 0; d < a.degrees; ++d) {
                const int n = a.comps[d] * a.rank;
                const T* t = a.t[d] + static_cast<long long>(p) * n;
                const T* h = a.h[d] + static_cast<long long>(p) * n;
                for (int q = lane; q < n; q += 32) s += t[q] * h[q];
            }
#pragma unroll
        for (int w = 16; w > 0; w >>= 1) s += __shfl_xor_sync(0xffffffffu, s, w);
        if (lane == 0) a.grad[i] = s;
    }
}

}  // namespace
}  // namespace smx

#include "adapters_f32.cuh"
#include "adapters_f64.cuh"

namespace smx {
namespace {

// ------------------------------------------------------------------------------------------- host side
void launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
    ++operator_launches;
}

struct Widths { long in = 0, out = 0; long long comps = 0; };
Widths widths(const smx_adapter_linear& c) {
    Widths w;
    for (int d = 0; d < c.num_degrees; ++d) {
        w.in += static_cast<long>(c.degrees[d].components) * c.degrees[d].in_channels;
        w.out += static_cast<long>(c.degrees[d].components) * c.degrees[d].out_channels;
        w.comps += c.degrees[d].components;
    }
    return w;
}

void check_call(const smx_adapter_linear& c) {
    if (c.precision != SMX_FP32 && c.precision != SMX_FP64) throw ArgError("smx_adapter: precision must be 32 or 64");
    if (c.num_degrees < 1 || c.num_degrees > kMaxDegrees) throw ArgError("smx_adapter: the number of degrees must lie in 1 .. " + std::to_string(kMaxDegrees));
    if (c.rank < 1 || c.rank > kMaxRank) throw ArgError("smx_adapter: the rank must lie in 1 .. " + std::to_string(kMaxRank));
    route_plan_bytes(c.num_rows, c.slots, c.num_groups);       // sizes shared with the routing
    for (int d = 0; d < c.num_degrees; ++d) {
        const smx_adapter_degree& g = c.degrees[d];
        if (g.components < 1 || g.components > 1024 || g.in_channels < 1 || g.out_channels < 1 || g.in_channels > (1 << 20) || g.out_channels > (1 << 20))
            throw ArgError("smx_adapter: a degree needs 1 .. 1024 components and 1 .. 1048576 channels");
    }
}
// buffers whose layout is the library's own are read and written in 16-byte pieces
void check_aligned(const smx_adapter_linear& c) {
    for (const void* p : {static_cast<const void*>(c.tiles), static_cast<const void*>(c.hidden), static_cast<const void*>(c.workspace)})
        if (reinterpret_cast<uintptr_t>(p) & 15) throw ArgError("smx_adapter: tiles, hidden and workspace must start on 16-byte boundaries");
}
void check_plan(const smx_adapter_linear& c) {
    check_call(c);
    if (!c.tiles) throw ArgError("smx_adapter: null tiles");
    check_aligned(c);
    if (!c.offsets || (c.num_rows > 0 && (!c.order || !c.position))) throw ArgError("smx_adapter: null plan");
    check_pointers("smx_adapter", sizeof(int), {c.order, c.position, c.offsets, c.status});
    const size_t value = c.precision == SMX_FP32 ? sizeof(float) : sizeof(double);
    check_pointers("smx_adapter", value, {c.x, c.y, c.grad_y, c.grad_x, c.weights, c.grad_weights});
    for (int d = 0; d < c.num_degrees; ++d) check_pointers("smx_adapter", value, {c.degrees[d].grad_down, c.degrees[d].grad_up});
}

void check_rows(const char* what, const void* p, long stride, long width, long rows, bool written) {
    if (rows > 0 && !p) throw ArgError(std::string("smx_adapter: null ") + what);
    if (stride < 0 || (written && rows > 1 && stride < width)) throw ArgError(std::string("smx_adapter: bad row stride of ") + what);
}

// Workspace: the plan by slots (several slots), hidden rows of both directions and partial sums (backward); parts start on 256 bytes.
struct Workspace {
    char* base;
    size_t used = 0;
    template <typename T>
    T* take(size_t n) {
        T* p = base ? reinterpret_cast<T*>(base + used) : nullptr;
        used += (n * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

int grad_chunk(const smx_adapter_linear& c) {
    const int cols = c.precision == SMX_FP64 ? kDpGradK : 128;           // inner indices of a CTA
    int chunk = kGradChunk;
    for (; chunk > 64; chunk /= 2) {
        long long ctas = 0;
        for (int d = 0; d < c.num_degrees; ++d) {
            const smx_adapter_degree& g = c.degrees[d];
            ctas += (static_cast<long long>(c.num_rows) * c.slots * g.components / chunk) * ((g.in_channels + cols - 1) / cols + (g.out_channels + cols - 1) / cols);
        }
        if (ctas >= 296) break;                                          // two per SM; a constant, so that sizes do not depend on the device
    }
    return chunk;
}
long long grad_chunks(const smx_adapter_linear& c, int comps) {
    return static_cast<long long>(c.num_rows) * c.slots * comps / grad_chunk(c) + c.num_groups;
}

template <typename T>
struct Buffers {
    T* back_hidden = nullptr; T* hidden = nullptr; T* parts[2 * kMaxDegrees] = {};
    int* places = nullptr; int* slot_offsets = nullptr; void* scratch = nullptr;
    size_t bytes = 0;
};
template <typename T>
Buffers<T> lay_out(const smx_adapter_linear& c, bool backward) {
    Buffers<T> b;
    Workspace ws{static_cast<char*>(c.workspace)};
    const Widths w = widths(c);
    const size_t pairs = static_cast<size_t>(c.num_rows) * c.slots;
    if (c.slots > 1) {
        b.places = ws.take<int>(pairs);
        b.slot_offsets = ws.take<int>(static_cast<size_t>(c.slots) * (c.num_groups + 1));
        b.scratch = ws.take<char>(route_slots_bytes(c.num_rows, c.slots));
    }
    if (backward) {
        b.back_hidden = ws.take<T>(pairs * w.comps * c.rank);
        if (!c.hidden) b.hidden = ws.take<T>(pairs * w.comps * c.rank);
        for (int d = 0; d < c.num_degrees; ++d) {
            b.parts[2 * d] = ws.take<T>(static_cast<size_t>(grad_chunks(c, c.degrees[d].components)) * c.degrees[d].in_channels * c.rank);
            b.parts[2 * d + 1] = ws.take<T>(static_cast<size_t>(grad_chunks(c, c.degrees[d].components)) * c.degrees[d].out_channels * c.rank);
        }
    }
    b.bytes = ws.used;
    return b;
}

// The matrices of a degree inside `tiles`, for both directions (index 1: transposed): float32 as operand images, float64 with aligned rows.
struct Matrices {
    const void *shared[2], *down[2], *up[2];
    size_t down_group[2], up_group[2];           // values from adapter to adapter
};
template <typename T>
size_t tile_layout(const smx_adapter_linear& c, Matrices (&m)[kMaxDegrees]) {
    Workspace ws{static_cast<char*>(c.tiles)};
    const int Rp = padded_rank(c.rank);
    for (int d = 0; d < c.num_degrees; ++d) {
        const smx_adapter_degree& g = c.degrees[d];
        for (int back = 0; back < 2; ++back) {
            // `down` is the first factor forward and the second one backward, `up` the other way round
            const int K = back ? g.out_channels : g.in_channels, N = back ? g.in_channels : g.out_channels;
            if (sizeof(T) == 8) {
                const size_t first = static_cast<size_t>(K) * even(c.rank), second = static_cast<size_t>(c.rank) * even(N);
                m[d].shared[back] = g.shared ? ws.take<T>(static_cast<size_t>(K) * even(N)) : nullptr;
                m[d].down_group[back] = back ? second : first;
                m[d].up_group[back] = back ? first : second;
                m[d].down[back] = ws.take<T>(m[d].down_group[back] * c.num_groups);
                m[d].up[back] = ws.take<T>(m[d].up_group[back] * c.num_groups);
                continue;
            }
            const size_t tile = 2 * kTsTileBytes / sizeof(float);
            const size_t first = static_cast<size_t>(ts_chunks(K)) * 2 * Rp * kTsChunk, second = static_cast<size_t>(ts_blocks(N)) * ts_chunks(Rp) * tile;
            m[d].shared[back] = g.shared ? ws.take<T>(static_cast<size_t>(ts_blocks(N)) * ts_chunks(K) * tile) : nullptr;
            m[d].down_group[back] = back ? second : first;
            m[d].up_group[back] = back ? first : second;
            m[d].down[back] = ws.take<T>(m[d].down_group[back] * c.num_groups);
            m[d].up[back] = ws.take<T>(m[d].up_group[back] * c.num_groups);
        }
    }
    return ws.used;
}

void prepare(const smx_adapter_linear& c, int parts) {
    Matrices m[kMaxDegrees];
    const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
    for (int d = 0; d < c.num_degrees; ++d) {
        check_pointers("smx_adapter_prepare", c.precision == SMX_FP32 ? sizeof(float) : sizeof(double), {(parts & SMX_ADAPTER_SHARED) ? c.degrees[d].shared : nullptr,
                       (parts & SMX_ADAPTER_MATRICES) ? c.degrees[d].down : nullptr, (parts & SMX_ADAPTER_MATRICES) ? c.degrees[d].up : nullptr});
        if ((parts & SMX_ADAPTER_MATRICES) && (!c.degrees[d].down || !c.degrees[d].up)) throw ArgError("smx_adapter_prepare: null matrix");
    }
    int n = 0;
    long long most = 0;
    if (c.precision == SMX_FP64) {
        tile_layout<double>(c, m);
        DoubleList list{};
        auto add = [&](const void* src, const void* dst, int groups, long long group_stride, int K, long long k_stride, int N, long long n_stride) {
            DoubleSegment& s = list.segment[n++];
            s.src = static_cast<const double*>(src); s.dst = static_cast<double*>(const_cast<void*>(dst));
            s.groups = groups; s.group_stride = group_stride; s.K = K; s.k_stride = k_stride; s.N = N; s.n_stride = n_stride; s.ld = even(N);
            most = std::max(most, static_cast<long long>(groups) * K * s.ld);
        };
        const int R = c.rank;
        for (int d = 0; d < c.num_degrees; ++d) {
            const smx_adapter_degree& g = c.degrees[d];
            const int I = g.in_channels, O = g.out_channels;
            if ((parts & SMX_ADAPTER_SHARED) && g.shared) {
                add(g.shared, m[d].shared[0], 1, 0, I, O, O, 1);
                add(g.shared, m[d].shared[1], 1, 0, O, 1, I, O);
            }
            if (parts & SMX_ADAPTER_MATRICES) {
                const long long down = static_cast<long long>(I) * R, up = static_cast<long long>(R) * O;
                add(g.down, m[d].down[0], c.num_groups, down, I, R, R, 1);
                add(g.up, m[d].up[0], c.num_groups, up, R, O, O, 1);
                add(g.up, m[d].up[1], c.num_groups, up, O, 1, R, O);
                add(g.down, m[d].down[1], c.num_groups, down, R, 1, I, R);
            }
        }
        if (!n) return;
        adapter_layout_kernel<<<dim3(static_cast<unsigned>(std::min<long long>(1024, (most + 255) / 256)), n), 256, 0, stream>>>(list);
        launched("adapter_layout_kernel");
        return;
    }
    tile_layout<float>(c, m);
    ImageList list{};
    auto add = [&](const void* src, const void* dst, int groups, long long group_stride, int K, long long k_stride, int N, long long n_stride, int rows) {
        ImageSegment& s = list.segment[n++];
        s.src = static_cast<const float*>(src); s.dst = static_cast<float*>(const_cast<void*>(dst));
        s.groups = groups; s.group_stride = group_stride; s.K = K; s.k_stride = k_stride; s.N = N; s.n_stride = n_stride;
        s.rows = rows; s.blocks = (N + rows - 1) / rows; s.chunks = ts_chunks(K);
        most = std::max(most, static_cast<long long>(groups) * s.blocks * s.chunks * rows * 8);
    };
    const int R = c.rank, Rp = padded_rank(R);
    for (int d = 0; d < c.num_degrees; ++d) {
        const smx_adapter_degree& g = c.degrees[d];
        const int I = g.in_channels, O = g.out_channels;
        if ((parts & SMX_ADAPTER_SHARED) && g.shared) {
            add(g.shared, m[d].shared[0], 1, 0, I, O, O, 1, 128);
            add(g.shared, m[d].shared[1], 1, 0, O, 1, I, O, 128);
        }
        if (parts & SMX_ADAPTER_MATRICES) {
            const long long down = static_cast<long long>(I) * R, up = static_cast<long long>(R) * O;
            add(g.down, m[d].down[0], c.num_groups, down, I, R, R, 1, Rp);
            add(g.up, m[d].up[0], c.num_groups, up, R, O, O, 1, 128);
            add(g.up, m[d].up[1], c.num_groups, up, O, 1, R, O, Rp);
            add(g.down, m[d].down[1], c.num_groups, down, R, 1, I, R, 128);
        }
    }
    if (!n) return;
    adapter_image_kernel<<<dim3(static_cast<unsigned>(std::min<long long>(1024, (most + 255) / 256)), n), 256, 0, stream>>>(list);
    launched("adapter_image_kernel");
}

template <typename T>
Pass<T> make_pass(const smx_adapter_linear& c, bool transposed, T* hidden) {
    Pass<T> p{};
    Matrices m[kMaxDegrees];
    tile_layout<T>(c, m);
    long long in_off = 0, out_off = 0;
    const size_t pairs = static_cast<size_t>(c.num_rows) * c.slots;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_adapter_degree& g = c.degrees[q];
        PassDegree<T>& d = p.degree[q];
        d.comps = g.components;
        d.in_off = in_off; d.out_off = out_off;
        d.Kd = transposed ? g.out_channels : g.in_channels;
        d.Nc = transposed ? g.in_channels : g.out_channels;
        const int back = transposed ? 1 : 0;
        d.W = static_cast<const T*>(m[q].shared[back]);
        d.first = static_cast<const T*>(transposed ? m[q].up[1] : m[q].down[0]);
        d.second = static_cast<const T*>(transposed ? m[q].down[1] : m[q].up[0]);
        d.first_group = static_cast<long long>(transposed ? m[q].up_group[1] : m[q].down_group[0]);
        d.second_group = static_cast<long long>(transposed ? m[q].down_group[1] : m[q].up_group[0]);
        d.hidden = hidden;
        if (hidden) hidden += pairs * g.components * c.rank;
        in_off += static_cast<long long>(g.components) * d.Kd;
        out_off += static_cast<long long>(g.components) * d.Nc;
    }
    p.rank = c.rank; p.groups = c.num_groups; p.slots = c.slots;
    p.pairs = static_cast<long long>(pairs);
    p.order = c.order; p.offsets = c.offsets;
    p.weights = static_cast<const T*>(c.weights);
    return p;
}

template <int HP, bool kWide>
void launch_ts(const TsPass& t, long long tiles, cudaStream_t stream) {
    using L = TsPassLayout<HP, kWide>;
    const auto kernel = adapter_pass_f32_kernel<HP, kWide>;
    // the warps' shares of registers are drawn from what the launch gives: fewer than planned and they would wait for ever
    static std::atomic<bool> done[64];
    if (first_on_device(done)) {
        cudaFuncAttributes a{};
        SMX_CUDA(cudaFuncGetAttributes(&a, kernel));
        if (a.numRegs < kTsRegsLaunch) throw CudaError("adapter_pass_f32_kernel was built with too few registers");
        SMX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem));
        mark_on_device(done);
    }
    kernel<<<static_cast<unsigned>(std::min<long long>(tiles, sm_count())), kTsPassThreads, L::smem, stream>>>(t);
    launched("adapter_pass_f32_kernel");
}
void launch_pass(const smx_adapter_linear& c, bool transposed, const Pass<float>& p, int degrees, cudaStream_t stream) {
    TsPass t{};
    long long tiles = 0;
    for (int q = 0; q < degrees; ++q) {
        const PassDegree<float>& d = p.degree[q];
        TsDegree& e = t.degree[q];
        e.comps = d.comps; e.Kd = d.Kd; e.Nc = d.Nc; e.in_off = d.in_off; e.out_off = d.out_off; e.hidden = d.hidden;
        e.W = d.W; e.first = d.first; e.first_group = d.first_group; e.second = d.second; e.second_group = d.second_group;
        tiles += (p.pairs * d.comps / kTsRows + p.groups + 1) * (p.out ? ts_blocks(d.Nc) : 1);
    }
    t.degrees = degrees; t.rank = p.rank; t.groups = p.groups; t.slots = p.slots; t.pairs = p.pairs;
    t.order = p.order; t.offsets = p.offsets; t.places = p.places; t.weights = p.weights; t.in = p.in; t.in_stride = p.in_stride; t.out = p.out; t.out_stride = p.out_stride;
    t.add = p.add; t.tail = p.tail; t.status = p.status; t.expire_polls = p.expire_polls;
    if (tiles > INT_MAX - 4096) throw ArgError("smx_adapter: too many rows");
    bool bare = false;
    for (int q = 0; q < degrees; ++q) bare = bare || !p.degree[q].W;
    if (bare && p.out && p.tail) {
        const Widths w = widths(c);
        adapter_zero_rows_kernel<<<static_cast<unsigned>(std::min<long long>(p.pairs, 8LL * sm_count())), 256, 0, stream>>>(
            p.offsets, p.groups, p.pairs, p.order, p.places, p.slots, p.out, p.out_stride, static_cast<int>(transposed ? w.in : w.out));
        launched("adapter_zero_rows_kernel");
    }
    bool wide = ((static_cast<unsigned long long>(p.out_stride) * 4u | reinterpret_cast<uintptr_t>(p.out)) & 31) == 0;
    for (int q = 0; q < degrees; ++q) wide = wide && p.degree[q].out_off % 8 == 0 && p.degree[q].Nc % 64 == 0;
    auto by_rank = [&](auto w) {
        constexpr bool kWide = decltype(w)::value;
        if (padded_rank(p.rank) == 16) launch_ts<1, kWide>(t, tiles, stream);
        else if (padded_rank(p.rank) == 32) launch_ts<2, kWide>(t, tiles, stream);
        else if (padded_rank(p.rank) == 48) launch_ts<3, kWide>(t, tiles, stream);
        else launch_ts<4, kWide>(t, tiles, stream);
    };
    if (wide || !p.out) by_rank(std::true_type{});
    else by_rank(std::false_type{});
}

// float64: tiles of 64 x 64, or of 16 x 32 while those leave SMs idle.
template <int BM, int BN, int WM, int WN, int NR, int ST>
void launch_dp(const DpPass& t, long long tiles, cudaStream_t stream) {
    using L = DpLayout<BM, BN, NR, ST>;
    if (tiles > INT_MAX) throw ArgError("smx_adapter: too many rows");
    const auto kernel = adapter_pass_f64_kernel<BM, BN, WM, WN, NR, ST>;
    static std::atomic<bool> done[64];
    if (first_on_device(done)) {
        SMX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem));
        mark_on_device(done);
    }
    kernel<<<static_cast<unsigned>(tiles), kDpThreads, L::smem, stream>>>(t);
    launched("adapter_pass_f64_kernel");
}
void launch_pass(const smx_adapter_linear&, bool, const Pass<double>& p, int degrees, cudaStream_t stream) {
    DpPass t{};
    for (int q = 0; q < degrees; ++q) {
        const PassDegree<double>& d = p.degree[q];
        DpDegree& e = t.degree[q];
        e.comps = d.comps; e.Kd = d.Kd; e.Nc = d.Nc; e.ldw = even(d.Nc); e.in_off = d.in_off; e.out_off = d.out_off; e.hidden = d.hidden;
        if (!p.out) e.ldw = 0;
        e.W = d.W; e.first = d.first; e.first_group = d.first_group; e.second = d.second; e.second_group = d.second_group;
    }
    t.degrees = degrees; t.rank = p.rank; t.groups = p.groups; t.slots = p.slots; t.pairs = p.pairs;
    t.order = p.order; t.offsets = p.offsets; t.places = p.places; t.weights = p.weights; t.in = p.in; t.in_stride = p.in_stride; t.out = p.out; t.out_stride = p.out_stride;
    t.add = p.add; t.tail = p.tail;
    auto tiles = [&](int BM, int BN) {
        long long n = 0;
        for (int q = 0; q < degrees; ++q) {
            const bool all = !p.out || (t.whole && !p.degree[q].W);          // one CTA makes all blocks of columns
            n += (p.pairs * p.degree[q].comps / BM + p.groups + 1) * (all ? 1 : (p.degree[q].Nc + BN - 1) / BN);
        }
        return n;
    };
    auto by_rank = [&](auto nr) {
        constexpr int NR = decltype(nr)::value;
        t.whole = 1;
        if (tiles(64, 64) > 2LL * sm_count()) { launch_dp<64, 64, 2, 2, NR, 2>(t, tiles(64, 64), stream); return; }
        t.whole = tiles(16, 32) > 2LL * sm_count();
        launch_dp<16, 32, 1, 4, NR, 4>(t, tiles(16, 32), stream);
    };
    if (p.rank <= 8) by_rank(std::integral_constant<int, 1>{});
    else if (p.rank <= 16) by_rank(std::integral_constant<int, 2>{});
    else if (p.rank <= 32) by_rank(std::integral_constant<int, 4>{});
    else by_rank(std::integral_constant<int, 8>{});
}

void launch_grads(const GradPass<double>& gp, int problems, cudaStream_t stream) {
    DpGrad t{};
    long long ctas = 0;
    for (int q = 0; q < problems; ++q) {
        t.problem[q] = gp.problem[q];
        ctas += (gp.pairs * gp.problem[q].comps / gp.chunk + gp.groups) * ((gp.problem[q].Kd + kDpGradK - 1) / kDpGradK);
    }
    t.problems = problems; t.rank = gp.rank; t.groups = gp.groups; t.slots = gp.slots; t.chunk = gp.chunk; t.pairs = gp.pairs;
    t.order = gp.order; t.offsets = gp.offsets; t.weights = gp.weights;
    if (ctas > INT_MAX) throw ArgError("smx_adapter: too many rows");
    const auto kernel = gp.rank <= 8 ? adapter_grad_f64_kernel<1> : gp.rank <= 16 ? adapter_grad_f64_kernel<2> : gp.rank <= 32 ? adapter_grad_f64_kernel<4> : adapter_grad_f64_kernel<8>;
    kernel<<<static_cast<unsigned>(ctas), kDpThreads, 0, stream>>>(t);
    launched("adapter_grad_f64_kernel");
}
void launch_grads(const GradPass<float>& gp, int problems, cudaStream_t stream) {
    TsGrad t{};
    long long ctas = 0;
    for (int q = 0; q < problems; ++q) {
        t.problem[q] = gp.problem[q];
        ctas += (gp.pairs * gp.problem[q].comps / gp.chunk + gp.groups) * ts_blocks(gp.problem[q].Kd);
    }
    t.problems = problems; t.rank = gp.rank; t.groups = gp.groups; t.slots = gp.slots; t.chunk = gp.chunk; t.pairs = gp.pairs;
    t.order = gp.order; t.offsets = gp.offsets; t.weights = gp.weights;
    if (ctas > INT_MAX) throw ArgError("smx_adapter: too many rows");
    const int NH = padded_rank(gp.rank) / 16;
    static std::atomic<bool> done[64];
    if (first_on_device(done)) {
        for (const auto kern : {adapter_grad_f32_kernel<1>, adapter_grad_f32_kernel<2>, adapter_grad_f32_kernel<3>, adapter_grad_f32_kernel<4>})
            SMX_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kGradChunk * 64 * static_cast<int>(sizeof(float))));
        mark_on_device(done);
    }
    const auto kernel = NH == 1 ? adapter_grad_f32_kernel<1> : NH == 2 ? adapter_grad_f32_kernel<2> : NH == 3 ? adapter_grad_f32_kernel<3> : adapter_grad_f32_kernel<4>;
    kernel<<<static_cast<unsigned>(ctas), kTsThreads, std::max(gp.chunk, 128) * 16 * NH * static_cast<int>(sizeof(float)), stream>>>(t);
    launched("adapter_grad_f32_kernel");
}

// out = in W + adapters, in either direction; `hidden` (may be null) receives in . first of every pair. Without `out` that is all.
template <typename T>
void run_pass(const smx_adapter_linear& c, bool transposed, const T* in, long in_stride, T* out, long out_stride, T* hidden, const Buffers<T>& b,
              int expire_polls) {
    if (c.num_rows == 0) return;
    const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
    Pass<T> p = make_pass<T>(c, transposed, hidden);
    p.in = in; p.in_stride = in_stride;
    p.status = c.status; p.expire_polls = expire_polls;
    if (!out) {
        for (int d = 0; d < c.num_degrees; ++d) { p.degree[d].W = nullptr; p.degree[d].Nc = 1; }      // one (unused) block of columns
        launch_pass(c, transposed, p, c.num_degrees, stream);
        return;
    }
    p.out = out; p.out_stride = out_stride; p.tail = 1;
    if (c.slots > 1) route_slots(c.order, c.num_rows, c.slots, c.offsets, c.num_groups, b.places, b.slot_offsets, b.scratch, stream);
    for (int s = 0; s < c.slots; ++s) {
        if (c.slots > 1) {
            p.places = b.places + static_cast<size_t>(s) * c.num_rows;
            p.offsets = b.slot_offsets + static_cast<size_t>(s) * (c.num_groups + 1);
            p.pairs = c.num_rows;
        }
        launch_pass(c, transposed, p, c.num_degrees, stream);
        p.add = 1; p.tail = 0;
        for (int d = 0; d < c.num_degrees; ++d) p.degree[d].W = nullptr;
    }
}

template <typename T>
void forward(const smx_adapter_linear& c, int expire_polls) {
    const Buffers<T> b = lay_out<T>(c, false);
    if (c.workspace_bytes < 0 || static_cast<size_t>(c.workspace_bytes) < b.bytes || (b.bytes && !c.workspace))
        throw ArgError("smx_adapter_forward: the workspace is smaller than smx_adapter_workspace_bytes says");
    const Widths w = widths(c);
    check_rows("x", c.x, c.x_stride, w.in, c.num_rows, false);
    check_rows("y", c.y, c.y_stride, w.out, c.num_rows, true);
    run_pass<T>(c, false, static_cast<const T*>(c.x), c.x_stride, static_cast<T*>(c.y), c.y_stride, static_cast<T*>(c.hidden), b, expire_polls);
}

template <typename T>
void backward(const smx_adapter_linear& c, int expire_polls) {
    const Buffers<T> b = lay_out<T>(c, true);
    if (c.workspace_bytes < 0 || static_cast<size_t>(c.workspace_bytes) < b.bytes || (b.bytes && !c.workspace))
        throw ArgError("smx_adapter_backward: the workspace is smaller than smx_adapter_workspace_bytes says");
    const Widths w = widths(c);
    check_rows("grad_y", c.grad_y, c.grad_y_stride, w.out, c.num_rows, false);
    if (c.grad_x) check_rows("grad_x", c.grad_x, c.grad_x_stride, w.in, c.num_rows, true);
    bool adapters = false;
    for (int d = 0; d < c.num_degrees; ++d) {
        const bool any = c.degrees[d].grad_down || c.degrees[d].grad_up;
        if (any && !(c.degrees[d].grad_down && c.degrees[d].grad_up)) throw ArgError("smx_adapter_backward: grad_down and grad_up come together");
        if (d > 0 && any != adapters) throw ArgError("smx_adapter_backward: the adapters' gradients are wanted for all degrees or none");
        adapters = any;
    }
    const bool hidden_needed = adapters || c.grad_weights;
    if (!hidden_needed && !c.grad_x) return;
    if (adapters || (c.grad_weights && !c.hidden)) check_rows("x", c.x, c.x_stride, w.in, c.num_rows, false);
    const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
    const size_t pairs = static_cast<size_t>(c.num_rows) * c.slots;
    const T* x = static_cast<const T*>(c.x);
    const T* gy = static_cast<const T*>(c.grad_y);
    run_pass<T>(c, true, gy, c.grad_y_stride, static_cast<T*>(c.grad_x), c.grad_x_stride, b.back_hidden, b, expire_polls);
    if (!hidden_needed) return;
    const T* hidden = static_cast<const T*>(c.hidden);
    if (!hidden) {
        run_pass<T>(c, false, x, c.x_stride, nullptr, 0, b.hidden, b, expire_polls);
        hidden = b.hidden;
    }
    GradPass<T> gp{};
    gp.rank = c.rank; gp.groups = c.num_groups; gp.slots = c.slots; gp.chunk = grad_chunk(c); gp.pairs = static_cast<long long>(pairs);
    gp.order = c.order; gp.offsets = c.offsets; gp.weights = static_cast<const T*>(c.weights);
    WeightGrad<T> wg{};
    long long in_off = 0, out_off = 0, hid_off = 0;
    int cols = 0;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_adapter_degree& g = c.degrees[q];
        GradProblem<T>&a = gp.problem[2 * q], &u = gp.problem[2 * q + 1];
        const long long I = g.in_channels, O = g.out_channels, R = c.rank;
        a.comps = u.comps = g.components;
        a.Kd = g.in_channels; u.Kd = g.out_channels;
        a.a = x; a.a_stride = c.x_stride; a.a_off = in_off; a.hidden = b.back_hidden + hid_off;
        u.a = gy; u.a_stride = c.grad_y_stride; u.a_off = out_off; u.hidden = hidden + hid_off;
        a.part = b.parts[2 * q]; u.part = b.parts[2 * q + 1];
        a.grad = static_cast<T*>(g.grad_down); a.g_group = I * R; a.g_k = R; a.g_r = 1;
        u.grad = static_cast<T*>(g.grad_up); u.g_group = R * O; u.g_k = 1; u.g_r = O;
        wg.t[q] = hidden + hid_off; wg.h[q] = b.back_hidden + hid_off; wg.comps[q] = g.components;
        in_off += g.components * I; out_off += g.components * O; hid_off += static_cast<long long>(pairs) * g.components * R;
        cols = std::max(cols, std::max(g.in_channels, g.out_channels));
    }
    if (adapters) {
        if (pairs > 0) {
            launch_grads(gp, 2 * c.num_degrees, stream);
        }
        const int slabs = static_cast<int>(std::min<long long>(64, (static_cast<long long>(cols) * c.rank + 255) / 256));
        adapter_grad_sum_kernel<T><<<dim3(c.num_groups, slabs, 2 * c.num_degrees), 256, 0, stream>>>(gp);
        launched("adapter_grad_sum_kernel");
    }
    if (c.grad_weights && pairs > 0) {
        wg.degrees = c.num_degrees; wg.rank = c.rank; wg.pairs = static_cast<long long>(pairs); wg.position = c.position;
        wg.grad = static_cast<T*>(c.grad_weights);
        adapter_weight_grad_kernel<T><<<static_cast<unsigned>(std::min<long long>((wg.pairs + 7) / 8, 148 * 32)), 256, 0, stream>>>(wg);
        launched("adapter_weight_grad_kernel");
    }
}

}  // namespace

size_t adapter_hidden_elements(const smx_adapter_linear& c) {
    check_call(c);
    return static_cast<size_t>(c.num_rows) * c.slots * widths(c).comps * c.rank;
}
size_t adapter_workspace_bytes(const smx_adapter_linear& c, bool backward) {
    check_call(c);
    smx_adapter_linear empty = c;
    empty.workspace = nullptr;
    return c.precision == SMX_FP32 ? lay_out<float>(empty, backward).bytes : lay_out<double>(empty, backward).bytes;
}
size_t adapter_tiles_bytes(const smx_adapter_linear& c) {
    check_call(c);
    smx_adapter_linear empty = c;
    empty.tiles = nullptr;
    Matrices m[kMaxDegrees];
    return c.precision == SMX_FP32 ? tile_layout<float>(empty, m) : tile_layout<double>(empty, m);
}
void adapter_prepare(const smx_adapter_linear& c, int parts) {
    check_call(c);
    if (!c.tiles) throw ArgError("smx_adapter_prepare: null tiles");
    check_aligned(c);
    if (parts & ~(SMX_ADAPTER_SHARED | SMX_ADAPTER_MATRICES)) throw ArgError("smx_adapter_prepare: unknown part");
    prepare(c, parts);
}
void adapter_forward(const smx_adapter_linear& c, int expire_polls) {
    check_plan(c);
    if (c.precision == SMX_FP32) forward<float>(c, expire_polls);
    else forward<double>(c, expire_polls);
}
void adapter_backward(const smx_adapter_linear& c, int expire_polls) {
    check_plan(c);
    if (c.precision == SMX_FP32) backward<float>(c, expire_polls);
    else backward<double>(c, expire_polls);
}

}  // namespace smx
