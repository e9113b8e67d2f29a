// Linears of routed rows, each group with matrices of its own (smx_grouped_*).
//
// Rows are sorted by group (csrc/routing.cu); those of group g begin at offsets[g]. A row holds, degree after degree, `components` rows of
// in_channels values. With W_g of the degree [in][out]:
//   forward   y = x W_g          backward   gx = gy W_g^T,  gW_g = sum over the group's rows and their components of x^T gy
#include "grouped.hpp"

#include <cuda_runtime.h>

#include <algorithm>
#include <atomic>
#include <climits>
#include <cstdint>
#include <type_traits>

#include "common.cuh"
#include "routing.hpp"

namespace smx {
namespace {

constexpr int kMaxDegrees = SMX_GROUPED_MAX_DEGREES;

}  // namespace
}  // namespace smx

#include "grouped_f32.cuh"
#include "grouped_f64.cuh"

namespace smx {
namespace {

// ------------------------------------------------------------------------------------------- host side
void launched(const char* what) {
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) throw CudaError(std::string(what) + ": " + cudaGetErrorString(e));
    ++operator_launches;
}

struct Widths { long in = 0, out = 0; };
Widths widths(const smx_grouped_linear& c) {
    Widths w;
    for (int d = 0; d < c.num_degrees; ++d) {
        w.in += static_cast<long>(c.degrees[d].components) * c.degrees[d].in_channels;
        w.out += static_cast<long>(c.degrees[d].components) * c.degrees[d].out_channels;
    }
    return w;
}

void check_call(const smx_grouped_linear& c) {
    if (c.precision != SMX_FP32 && c.precision != SMX_FP64) throw ArgError("smx_grouped: precision must be 32 or 64");
    if (c.num_degrees < 1 || c.num_degrees > kMaxDegrees) throw ArgError("smx_grouped: the number of degrees must lie in 1 .. " + std::to_string(kMaxDegrees));
    route_plan_bytes(c.num_rows, 1, c.num_groups);             // sizes shared with the routing
    for (int d = 0; d < c.num_degrees; ++d) {
        const smx_grouped_degree& g = c.degrees[d];
        if (g.components < 1 || g.components > 1024 || g.in_channels < 1 || g.out_channels < 1 || g.in_channels > (1 << 20) || g.out_channels > (1 << 20))
            throw ArgError("smx_grouped: a degree needs 1 .. 1024 components and 1 .. 1048576 channels");
    }
}
void check_plan(const smx_grouped_linear& c) {
    check_call(c);
    if (!c.offsets) throw ArgError("smx_grouped: null plan");
    if (reinterpret_cast<uintptr_t>(c.workspace) & 31) throw ArgError("smx_grouped: the workspace must start on a 32-byte boundary");
    check_pointers("smx_grouped", sizeof(int), {c.offsets, c.status});
    const size_t value = c.precision == SMX_FP32 ? sizeof(float) : sizeof(double);
    check_pointers("smx_grouped", value, {c.x, c.y, c.grad_y, c.grad_x});
    for (int d = 0; d < c.num_degrees; ++d) check_pointers("smx_grouped", value, {c.degrees[d].weight, c.degrees[d].grad_weight});
}
void check_rows(const char* what, const void* p, long stride, long width, long rows, bool written) {
    if (rows > 0 && !p) throw ArgError(std::string("smx_grouped: null ") + what);
    if (stride < 0 || (written && rows > 1 && stride < width)) throw ArgError(std::string("smx_grouped: bad row stride of ") + what);
}
void check_weights(const smx_grouped_linear& c) {
    for (int d = 0; d < c.num_degrees; ++d)
        if (!c.degrees[d].weight) throw ArgError("smx_grouped: null weight");
}

// What a call allocates nothing for: the partial sums of the matrices' gradients. Their chunks of rows are as long as leaves four tiles for each of 148
// SMs (a constant, so that sizes and sums do not depend on the device), and 4,096 rows at most: longer float32 sums lose more, and joining them costs little beside the
// products (98,304 atoms, seven components, 2,048 x 2,048: 2.8 GB of sums, joined in 1.7 of 41 ms).
int grad_chunk(const smx_grouped_linear& c) {
    const int tile = c.precision == SMX_FP32 ? 128 : 64;
    long long steps = 0;
    for (int d = 0; d < c.num_degrees; ++d) {
        const smx_grouped_degree& g = c.degrees[d];
        steps += (c.num_rows * static_cast<long long>(g.components) + 63) / 64 * ((g.in_channels + tile - 1) / tile) * ((g.out_channels + tile - 1) / tile);
    }
    return 64 * static_cast<int>(std::max(2LL, std::min(64LL, (steps + 591) / 592)));
}
size_t part_values(const smx_grouped_linear& c, int d) {
    const smx_grouped_degree& g = c.degrees[d];
    // a group with several chunks has one more at most than its rows fill
    const long long whole = c.num_rows * static_cast<long long>(g.components) / grad_chunk(c), parts = whole + std::min<long long>(c.num_groups, whole);
    return static_cast<size_t>((parts * g.in_channels * g.out_channels + 63) / 64 * 64);
}

// Gradients of groups with several sums: added in order, by eights and those in 64 bits (a long list loses no more than eight roundings; conversions of every sum would
// take another 7 us of the case below), in units V of 16 bytes where all matrices allow it (sums of 8,001 atoms in two slots behind the tensor
// product, 41 MB: 12.5 us; value by value half as long again).
template <typename V>
struct JoinPass {
    struct { int comps; long long size; const V* part; V* grad; } degree[kMaxDegrees];     // size: units of a matrix
    int chunk; const int* offsets;
};
template <typename T, typename V>
__global__ void __launch_bounds__(256) grouped_join_kernel(const __grid_constant__ JoinPass<V> pass) {
    constexpr int per = sizeof(V) / sizeof(T);
    union Unit { V v; T t[per]; };
    const auto& d = pass.degree[blockIdx.z];
    __shared__ int first, sums;
    const int g = blockIdx.x;
    auto sums_of = [&](int q) { return static_cast<int>((static_cast<long long>(pass.offsets[q + 1] - pass.offsets[q]) * d.comps + pass.chunk - 1) / pass.chunk); };
    if (threadIdx.x < 32) {
        int before = 0;
        for (int q = threadIdx.x; q < g; q += 32) {
            const int n = sums_of(q);
            before += n > 1 ? n : 0;
        }
        before = __reduce_add_sync(0xffffffffu, before);
        if (threadIdx.x == 0) { first = before; sums = sums_of(g); }
    }
    __syncthreads();
    const int n = sums;
    if (n <= 1) return;
    for (long long i = blockIdx.y * 256LL + threadIdx.x; i < d.size; i += 256LL * gridDim.y) {
        const V* part = d.part + first * d.size + i;
        double s[per] = {};
        for (int c = 0; c < n; c += 8) {                                 // eight loads in flight, added in order
            Unit v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u].v = c + u < n ? part[(c + u) * d.size] : V{};
            Unit eight{};
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < per; ++e) eight.t[e] += v[u].t[e];
#pragma unroll
            for (int e = 0; e < per; ++e) s[e] += eight.t[e];
        }
        Unit out;
#pragma unroll
        for (int e = 0; e < per; ++e) out.t[e] = static_cast<T>(s[e]);
        d.grad[g * d.size + i] = out.v;
    }
}
template <typename T, typename V>
void join_units(const smx_grouped_linear& c) {
    JoinPass<V> p{};
    const T* part = static_cast<const T*>(c.workspace);
    long long most = 0;
    bool split = false;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_grouped_degree& g = c.degrees[q];
        auto& d = p.degree[q];
        d.comps = g.components;
        d.size = static_cast<long long>(g.in_channels) * g.out_channels * sizeof(T) / sizeof(V);
        d.part = reinterpret_cast<const V*>(part);
        d.grad = static_cast<V*>(g.grad_weight);
        part += part_values(c, q);
        split = split || part_values(c, q) > 0;
        most = std::max(most, d.size);
    }
    if (!split) return;
    p.chunk = grad_chunk(c); p.offsets = c.offsets;
    grouped_join_kernel<T, V><<<dim3(c.num_groups, static_cast<unsigned>(std::min(64LL, (most + 255) / 256)), c.num_degrees), 256, 0,
                             static_cast<cudaStream_t>(c.stream)>>>(p);
    launched("grouped_join_kernel");
}
template <typename T>
void join(const smx_grouped_linear& c) {
    using V = std::conditional_t<sizeof(T) == 4, float4, double2>;
    bool wide = true;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_grouped_degree& g = c.degrees[q];
        wide = wide && static_cast<long long>(g.in_channels) * g.out_channels * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(g.grad_weight) & 15) == 0;
    }
    if (wide) join_units<T, V>(c);
    else join_units<T, T>(c);
}

template <int kMode, bool kWide>
void launch_gs(const GsPass& p, long long tiles, const Launcher& on) {
    const auto kernel = grouped_f32_kernel<kMode, kWide>;
    // The warps' shares of registers are drawn from what the launch gives: fewer than planned and they would wait for ever. What the kernel's own arrays
    // leave of the shared memory starts on a multiple of 1,024 bytes.
    static std::atomic<bool> done[64];
    static std::atomic<int> smem{0};
    if (first_on_device(done)) {
        cudaFuncAttributes a{};
        SMX_CUDA(cudaFuncGetAttributes(&a, kernel));
        if (a.numRegs < kGsRegsLaunch) throw CudaError("grouped_f32_kernel was built with too few registers");
        const int own = static_cast<int>(a.sharedSizeBytes), bytes = GsLayout<kWide>::bytes + std::min(1024, GsLayout<kWide>::largest);
        if (own > 2048) throw CudaError("grouped_f32_kernel was built with too much shared memory");
        SMX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
        smem.store(bytes, std::memory_order_relaxed);
        mark_on_device(done);
    }
    if (tiles > INT_MAX) throw ArgError("smx_grouped: too many rows");
    chain_launch(on, kernel, dim3(static_cast<unsigned>(std::min<long long>(tiles, sm_count()))), kGsThreads, smem.load(std::memory_order_relaxed), 1, p);
    ++operator_launches;
}

GsPass gs_pass(const smx_grouped_linear& c, bool transposed) {
    GsPass p{};
    long long in_off = 0, out_off = 0;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_grouped_degree& g = c.degrees[q];
        GsDegree& d = p.degree[q];
        d.comps = g.components;
        d.K = transposed ? g.out_channels : g.in_channels;
        d.N = transposed ? g.in_channels : g.out_channels;
        d.a_off = in_off; d.b_off = out_off;
        d.w = static_cast<const float*>(g.weight);
        in_off += static_cast<long long>(d.comps) * d.K;
        out_off += static_cast<long long>(d.comps) * d.N;
    }
    p.degrees = c.num_degrees; p.groups = c.num_groups; p.rows = c.num_rows; p.offsets = c.offsets;
    p.out_width = out_off;
    p.status = c.status; p.expire_polls = c.expire_polls;
    return p;
}

void rows_f32(const smx_grouped_linear& c, bool transposed) {
    GsPass p = gs_pass(c, transposed);
    p.a = static_cast<const float*>(transposed ? c.grad_y : c.x); p.a_stride = transposed ? c.grad_y_stride : c.x_stride;
    p.out = static_cast<float*>(transposed ? c.grad_x : c.y); p.out_stride = transposed ? c.grad_x_stride : c.y_stride;
    p.zero_tail = transposed || c.zero_tail;
    long long tiles = 0;
    // whole sectors are written straight from registers (98,304 atoms of 89 elements 92 us, 156 through shared memory, as other widths and starts have to go)
    bool wide = ((static_cast<unsigned long long>(p.out_stride) * 4u | reinterpret_cast<uintptr_t>(p.out)) & 31) == 0;
    for (int q = 0; q < p.degrees; ++q) {
        const GsDegree& d = p.degree[q];
        tiles += (c.num_rows * d.comps / 128 + c.num_groups) * ((d.N + 127) / 128);
        wide = wide && d.b_off % 8 == 0 && d.N % 8 == 0;
    }
    const Launcher on{static_cast<cudaStream_t>(c.stream), false};
    if (transposed) {
        if (wide) launch_gs<kGsBackward, true>(p, tiles, on);
        else launch_gs<kGsBackward, false>(p, tiles, on);
    } else {
        if (wide) launch_gs<kGsForward, true>(p, tiles, on);
        else launch_gs<kGsForward, false>(p, tiles, on);
    }
}

// `behind_rows`: right behind the rows' pass of the same call
void gradient_f32(const smx_grouped_linear& c, bool behind_rows) {
    GsPass p = gs_pass(c, false);
    p.a = static_cast<const float*>(c.x); p.a_stride = c.x_stride;
    p.b = static_cast<const float*>(c.grad_y); p.b_stride = c.grad_y_stride;
    p.chunk = grad_chunk(c);
    float* part = static_cast<float*>(c.workspace);
    long long tiles = 0;
    bool wide = true;
    for (int q = 0; q < p.degrees; ++q) {
        GsDegree& d = p.degree[q];
        d.grad = static_cast<float*>(c.degrees[q].grad_weight);
        d.part = part;
        part += part_values(c, q);
        tiles += (c.num_rows * d.comps / p.chunk + c.num_groups) * ((d.N + 127) / 128) * ((d.K + 127) / 128);
        wide = wide && d.N % 8 == 0 && (reinterpret_cast<uintptr_t>(d.grad) & 31) == 0;
    }
    const Launcher on{static_cast<cudaStream_t>(c.stream), behind_rows};
    if (wide) launch_gs<kGsGradient, true>(p, tiles, on);
    else launch_gs<kGsGradient, false>(p, tiles, on);
    join<float>(c);
}

// float64: tiles of 64 x 64, or of 16 x 32 while those leave SMs idle. 300 atoms of three groups (scalars and vectors, 128 x 128) 16.4 us with tiles of 64 x 64,
// 10.2 with 16 x 32; 4,001 atoms of eight 30.7 and 34.8; 20,000 atoms of 16 groups behind two and three paths 223 and 297.
template <int kMode, int BM, int BN, int WM, int WN, int ST>
void launch_gd(const GdPass& p, long long tiles, const Launcher& on) {
    using L = GdLayout<kMode, BM, BN, ST>;
    if (tiles > INT_MAX) throw ArgError("smx_grouped: too many rows");
    const auto kernel = grouped_f64_kernel<kMode, BM, BN, WM, WN, ST>;
    static std::atomic<bool> done[64];
    if (first_on_device(done)) {
        SMX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::smem));
        mark_on_device(done);
    }
    chain_launch(on, kernel, dim3(static_cast<unsigned>(tiles)), kGdThreads, L::smem, 1, p);
    ++operator_launches;
}
template <int kMode>
void launch_gd(const GdPass& p, const Launcher& on) {
    auto tiles = [&](int BM, int BN) {
        long long n = 0;
        for (int q = 0; q < p.degrees; ++q) {
            const GdDegree& d = p.degree[q];
            if (kMode == kGsGradient) n += (p.rows * d.comps / p.chunk + p.groups) * ((d.K + BM - 1) / BM) * ((d.N + BN - 1) / BN);
            else n += (p.rows * d.comps / BM + p.groups) * ((d.N + BN - 1) / BN);
        }
        return n;
    };
    if (tiles(64, 64) > 2LL * sm_count()) launch_gd<kMode, 64, 64, 2, 2, 2>(p, tiles(64, 64), on);
    else launch_gd<kMode, 16, 32, 1, 4, 4>(p, tiles(16, 32), on);
}

GdPass gd_pass(const smx_grouped_linear& c, bool transposed) {
    GdPass p{};
    long long in_off = 0, out_off = 0;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_grouped_degree& g = c.degrees[q];
        GdDegree& d = p.degree[q];
        d.comps = g.components;
        d.K = transposed ? g.out_channels : g.in_channels;
        d.N = transposed ? g.in_channels : g.out_channels;
        d.a_off = in_off; d.b_off = out_off;
        d.w = static_cast<const double*>(g.weight);
        in_off += static_cast<long long>(d.comps) * d.K;
        out_off += static_cast<long long>(d.comps) * d.N;
    }
    p.degrees = c.num_degrees; p.groups = c.num_groups; p.rows = c.num_rows; p.offsets = c.offsets;
    p.out_width = out_off;
    return p;
}

void rows_f64(const smx_grouped_linear& c, bool transposed) {
    GdPass p = gd_pass(c, transposed);
    p.a = static_cast<const double*>(transposed ? c.grad_y : c.x); p.a_stride = transposed ? c.grad_y_stride : c.x_stride;
    p.out = static_cast<double*>(transposed ? c.grad_x : c.y); p.out_stride = transposed ? c.grad_x_stride : c.y_stride;
    p.zero_tail = transposed || c.zero_tail;
    const Launcher on{static_cast<cudaStream_t>(c.stream), false};
    if (transposed) launch_gd<kGsBackward>(p, on);
    else launch_gd<kGsForward>(p, on);
}

void gradient_f64(const smx_grouped_linear& c, bool behind_rows) {
    GdPass p = gd_pass(c, false);
    p.a = static_cast<const double*>(c.x); p.a_stride = c.x_stride;
    p.b = static_cast<const double*>(c.grad_y); p.b_stride = c.grad_y_stride;
    p.chunk = grad_chunk(c);
    double* part = static_cast<double*>(c.workspace);
    for (int q = 0; q < p.degrees; ++q) {
        GdDegree& d = p.degree[q];
        d.grad = static_cast<double*>(c.degrees[q].grad_weight);
        d.part = part;
        part += part_values(c, q);
    }
    launch_gd<kGsGradient>(p, Launcher{static_cast<cudaStream_t>(c.stream), behind_rows});
    join<double>(c);
}

template <typename T>
void rows_pass(const smx_grouped_linear& c, bool transposed) {
    if (c.num_rows == 0) return;
    if (sizeof(T) == 4) rows_f32(c, transposed);
    else rows_f64(c, transposed);
}

template <typename T>
void forward(const smx_grouped_linear& c) {
    const Widths w = widths(c);
    check_rows("x", c.x, c.x_stride, w.in, c.num_rows, false);
    check_rows("y", c.y, c.y_stride, w.out, c.num_rows, true);
    check_weights(c);
    rows_pass<T>(c, false);
}

template <typename T>
void backward(const smx_grouped_linear& c) {
    const Widths w = widths(c);
    check_rows("grad_y", c.grad_y, c.grad_y_stride, w.out, c.num_rows, false);
    bool matrices = false;
    for (int d = 0; d < c.num_degrees; ++d) {
        const bool any = c.degrees[d].grad_weight != nullptr;
        if (d > 0 && any != matrices) throw ArgError("smx_grouped_backward: the matrices' gradients are wanted for all degrees or none");
        matrices = any;
    }
    if (c.grad_x) {
        check_rows("grad_x", c.grad_x, c.grad_x_stride, w.in, c.num_rows, true);
        check_weights(c);
    }
    if (matrices) check_rows("x", c.x, c.x_stride, w.in, c.num_rows, false);
    if (matrices) {
        const size_t need = grouped_workspace_bytes(c, true);
        if (c.workspace_bytes < 0 || static_cast<size_t>(c.workspace_bytes) < need || (need && !c.workspace))
            throw ArgError("smx_grouped_backward: the workspace is smaller than smx_grouped_workspace_bytes says");
    }
    if (c.grad_x) rows_pass<T>(c, true);
    if (!matrices) return;
    const bool behind_rows = c.grad_x && c.num_rows > 0;
    if (sizeof(T) == 4) gradient_f32(c, behind_rows);
    else gradient_f64(c, behind_rows);
}

}  // namespace

size_t grouped_workspace_bytes(const smx_grouped_linear& c, bool backward) {
    check_call(c);
    if (!backward) return 0;
    size_t values = 0;
    for (int d = 0; d < c.num_degrees; ++d) values += part_values(c, d);
    return values * (c.precision == SMX_FP32 ? sizeof(float) : sizeof(double));
}
void grouped_forward(const smx_grouped_linear& c) {
    check_plan(c);
    if (c.precision == SMX_FP32) forward<float>(c);
    else forward<double>(c);
}
void grouped_backward(const smx_grouped_linear& c) {
    check_plan(c);
    if (c.precision == SMX_FP32) backward<float>(c);
    else backward<double>(c);
}

}  // namespace smx
