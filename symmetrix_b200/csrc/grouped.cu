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

#include "common.cuh"
#include "routing.hpp"
#include "row_tiles.cuh"

namespace smx {
namespace {

constexpr int kMaxDegrees = SMX_GROUPED_MAX_DEGREES;

// out[row][n] = sum_k in[row][k] W_g[k * w_k + n * w_n]
template <typename T>
struct RowsDegree { int comps, K, N; long long in_off, out_off; const T* w; long long w_group, w_k, w_n; };
template <typename T>
struct RowsPass {
    RowsDegree<T> degree[kMaxDegrees];
    int degrees, groups; long long rows; const int* offsets;
    const T* in; long long in_stride; T* out; long long out_stride;
    int zero_tail, out_width;
};

constexpr int kTile = 64, kStep = 16;
template <typename T>
__global__ void __launch_bounds__(256) grouped_rows_kernel(const __grid_constant__ RowsPass<T> pass) {
    __shared__ T as[kStep][kTile + 1], bs[kStep][kTile + 1];
    __shared__ TileRows tile;
    __shared__ int which, block;
    const int tid = threadIdx.x;
    if (tid < 32) {
        long long at = blockIdx.x, tiles = 0;
        TileRows t{};
        int hit = -1, b = 0;
        for (int q = 0; q < pass.degrees && hit < 0; ++q) {
            const int blocks = (pass.degree[q].N + kTile - 1) / kTile;
            if (find_tile(pass.offsets, pass.groups, false, pass.rows, pass.degree[q].comps, kTile, at / blocks, t, tiles)) { hit = q; b = static_cast<int>(at % blocks); }
            else at -= tiles * blocks;
        }
        if (tid == 0) { which = hit; block = b; tile = t; }
    }
    if (pass.zero_tail)
        for (long long p = pass.offsets[pass.groups] + blockIdx.x; p < pass.rows; p += gridDim.x)
            for (int c = tid; c < pass.out_width; c += 256) pass.out[p * pass.out_stride + c] = T(0);
    __syncthreads();
    if (which < 0) return;
    const RowsDegree<T>& d = pass.degree[which];
    const T* w = d.w + tile.group * d.w_group;
    const int col0 = block * kTile, ty = tid / 16, tx = tid % 16;
    auto row_at = [&](long long r, long long stride, long long off, int width) {
        const long long q = tile.row0 + r;
        return (tile.first_pair + q / d.comps) * stride + off + q % d.comps * width;
    };
    T acc[4][4] = {};
    for (int k0 = 0; k0 < d.K; k0 += kStep) {
        for (int i = tid; i < kTile * kStep; i += 256) {
            const int r = i / kStep, k = i % kStep;
            as[k][r] = r < tile.rows && k0 + k < d.K ? pass.in[row_at(r, pass.in_stride, d.in_off, d.K) + k0 + k] : T(0);
            const int n = i % kTile, kb = i / kTile;
            bs[kb][n] = col0 + n < d.N && k0 + kb < d.K ? w[(k0 + kb) * d.w_k + (col0 + n) * d.w_n] : T(0);
        }
        __syncthreads();
        for (int k = 0; k < kStep; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] += as[k][ty + 16 * i] * bs[k][tx + 16 * j];
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = ty + 16 * i;
        if (r >= tile.rows) continue;
        const long long to = row_at(r, pass.out_stride, d.out_off, d.N) + col0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (col0 + tx + 16 * j < d.N) pass.out[to + tx + 16 * j] = acc[i][j];
    }
}

// grad_w[g][k][n] = sum over the group's rows of x[row][k] gy[row][n]
template <typename T>
struct GradDegree { int comps, K, N; long long x_off, y_off; T* grad; };
template <typename T>
struct GradPass {
    GradDegree<T> degree[kMaxDegrees];
    int groups; const int* offsets;
    const T* x; long long x_stride; const T* gy; long long gy_stride;
};
template <typename T>
__global__ void __launch_bounds__(256) grouped_grad_kernel(const __grid_constant__ GradPass<T> pass) {
    __shared__ T as[kStep][kTile + 1], bs[kStep][kTile + 1];
    const GradDegree<T>& d = pass.degree[blockIdx.z];
    const int blocks = (d.N + kTile - 1) / kTile, tiles = blocks * ((d.K + kTile - 1) / kTile);
    const int tid = threadIdx.x, ty = tid / 16, tx = tid % 16, g = blockIdx.x;
    const long long first = pass.offsets[g], rows = (pass.offsets[g + 1] - first) * d.comps;
    for (int t = blockIdx.y; t < tiles; t += gridDim.y) {
        const int k0 = t / blocks * kTile, n0 = t % blocks * kTile;
        T acc[4][4] = {};
        for (long long r0 = 0; r0 < rows; r0 += kStep) {
            for (int i = tid; i < kTile * kStep; i += 256) {
                const int c = i % kTile, r = i / kTile;
                const long long q = r0 + r, p = first + q / d.comps, m = q % d.comps;
                as[r][c] = q < rows && k0 + c < d.K ? pass.x[p * pass.x_stride + d.x_off + m * d.K + k0 + c] : T(0);
                bs[r][c] = q < rows && n0 + c < d.N ? pass.gy[p * pass.gy_stride + d.y_off + m * d.N + n0 + c] : T(0);
            }
            __syncthreads();
            for (int r = 0; r < kStep; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[i][j] += as[r][ty + 16 * i] * bs[r][tx + 16 * j];
            __syncthreads();
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = k0 + ty + 16 * i, n = n0 + tx + 16 * j;
                if (k < d.K && n < d.N) d.grad[(static_cast<long long>(g) * d.K + k) * d.N + n] = acc[i][j];
            }
    }
}

}  // namespace
}  // namespace smx

#include "grouped_f32.cuh"

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
// SMs (a constant, so that sizes and sums do not depend on the device); a group with several chunks has less than twice as many as its rows fill.
int grad_chunk(const smx_grouped_linear& c) {
    long long steps = 0;
    for (int d = 0; d < c.num_degrees; ++d) {
        const smx_grouped_degree& g = c.degrees[d];
        steps += (c.num_rows * static_cast<long long>(g.components) + 63) / 64 * ((g.in_channels + 127) / 128) * ((g.out_channels + 127) / 128);
    }
    return 64 * static_cast<int>(std::max(2LL, std::min(64LL, (steps + 591) / 592)));
}
size_t part_values(const smx_grouped_linear& c, int d) {
    const smx_grouped_degree& g = c.degrees[d];
    const long long parts = 2 * (c.num_rows * static_cast<long long>(g.components) / grad_chunk(c));
    return static_cast<size_t>((parts * g.in_channels * g.out_channels + 63) / 64 * 64);
}

template <int kMode, bool kWide>
void launch_gs(const GsPass& p, long long tiles, cudaStream_t stream) {
    const auto kernel = grouped_f32_kernel<kMode, kWide>;
    // the warps' shares of registers are drawn from what the launch gives: fewer than planned and they would wait for ever
    static std::atomic<bool> done[64];
    if (first_on_device(done)) {
        cudaFuncAttributes a{};
        SMX_CUDA(cudaFuncGetAttributes(&a, kernel));
        if (a.numRegs < kGsRegsLaunch) throw CudaError("grouped_f32_kernel was built with too few registers");
        SMX_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, GsLayout<kMode, kWide>::smem));
        mark_on_device(done);
    }
    kernel<<<static_cast<unsigned>(std::min<long long>(tiles, sm_count())), kGsThreads, GsLayout<kMode, kWide>::smem, stream>>>(p);
    launched("grouped_f32_kernel");
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
    p.out_width = static_cast<int>(out_off);
    p.status = c.status; p.expire_polls = c.expire_polls;
    return p;
}

void rows_f32(const smx_grouped_linear& c, bool transposed) {
    GsPass p = gs_pass(c, transposed);
    p.a = static_cast<const float*>(transposed ? c.grad_y : c.x); p.a_stride = transposed ? c.grad_y_stride : c.x_stride;
    p.out = static_cast<float*>(transposed ? c.grad_x : c.y); p.out_stride = transposed ? c.grad_x_stride : c.y_stride;
    p.zero_tail = transposed || c.zero_tail;
    long long tiles = 0;
    bool wide = ((static_cast<unsigned long long>(p.out_stride) * 4u | reinterpret_cast<uintptr_t>(p.out)) & 31) == 0;
    for (int q = 0; q < p.degrees; ++q) {
        const GsDegree& d = p.degree[q];
        tiles += (c.num_rows * d.comps / 128 + c.num_groups) * ((d.N + 127) / 128);
        wide = wide && d.b_off % 8 == 0 && d.N % 64 == 0;
    }
    if (tiles > INT_MAX) throw ArgError("smx_grouped: too many rows");
    const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
    if (transposed) {
        if (wide) launch_gs<kGsBackward, true>(p, tiles, stream);
        else launch_gs<kGsBackward, false>(p, tiles, stream);
    } else {
        if (wide) launch_gs<kGsForward, true>(p, tiles, stream);
        else launch_gs<kGsForward, false>(p, tiles, stream);
    }
}

void gradient_f32(const smx_grouped_linear& c) {
    GsPass p = gs_pass(c, false);
    p.a = static_cast<const float*>(c.x); p.a_stride = c.x_stride;
    p.b = static_cast<const float*>(c.grad_y); p.b_stride = c.grad_y_stride;
    p.chunk = grad_chunk(c);
    float* part = static_cast<float*>(c.workspace);
    long long tiles = 0, most = 0;
    bool wide = true, split = false;
    for (int q = 0; q < p.degrees; ++q) {
        GsDegree& d = p.degree[q];
        d.grad = static_cast<float*>(c.degrees[q].grad_weight);
        d.part = part;
        part += part_values(c, q);
        split = split || part_values(c, q) > 0;
        tiles += (c.num_rows * d.comps / p.chunk + c.num_groups) * ((d.N + 127) / 128) * ((d.K + 127) / 128);
        most = std::max(most, static_cast<long long>(d.K) * d.N);
        wide = wide && d.N % 64 == 0 && (reinterpret_cast<uintptr_t>(d.grad) & 31) == 0;
    }
    if (tiles > INT_MAX) throw ArgError("smx_grouped: too many rows");
    const cudaStream_t stream = static_cast<cudaStream_t>(c.stream);
    if (wide) launch_gs<kGsGradient, true>(p, tiles, stream);
    else launch_gs<kGsGradient, false>(p, tiles, stream);
    if (!split) return;
    grouped_join_kernel<<<dim3(c.num_groups, static_cast<unsigned>(std::min(64LL, (most + 255) / 256)), c.num_degrees), 256, 0, stream>>>(p);
    launched("grouped_join_kernel");
}

template <typename T>
void rows_pass(const smx_grouped_linear& c, bool transposed) {
    if (c.num_rows == 0) return;
    if (sizeof(T) == 4) return rows_f32(c, transposed);
    RowsPass<T> p{};
    long long in_off = 0, out_off = 0, tiles = 0;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_grouped_degree& g = c.degrees[q];
        RowsDegree<T>& d = p.degree[q];
        d.comps = g.components;
        d.K = transposed ? g.out_channels : g.in_channels;
        d.N = transposed ? g.in_channels : g.out_channels;
        d.in_off = in_off; d.out_off = out_off;
        d.w = static_cast<const T*>(g.weight);
        d.w_group = static_cast<long long>(g.in_channels) * g.out_channels;
        d.w_k = transposed ? 1 : g.out_channels;
        d.w_n = transposed ? g.out_channels : 1;
        in_off += static_cast<long long>(d.comps) * d.K;
        out_off += static_cast<long long>(d.comps) * d.N;
        tiles += (c.num_rows * d.comps / kTile + c.num_groups) * ((d.N + kTile - 1) / kTile);
    }
    p.degrees = c.num_degrees; p.groups = c.num_groups; p.rows = c.num_rows; p.offsets = c.offsets;
    p.in = static_cast<const T*>(transposed ? c.grad_y : c.x); p.in_stride = transposed ? c.grad_y_stride : c.x_stride;
    p.out = static_cast<T*>(transposed ? c.grad_x : c.y); p.out_stride = transposed ? c.grad_x_stride : c.y_stride;
    p.zero_tail = transposed || c.zero_tail;
    p.out_width = static_cast<int>(out_off);
    if (tiles > INT_MAX) throw ArgError("smx_grouped: too many rows");
    grouped_rows_kernel<T><<<static_cast<unsigned>(tiles), 256, 0, static_cast<cudaStream_t>(c.stream)>>>(p);
    launched("grouped_rows_kernel");
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
    if (sizeof(T) == 4) return gradient_f32(c);
    GradPass<T> p{};
    long long x_off = 0, y_off = 0;
    for (int q = 0; q < c.num_degrees; ++q) {
        const smx_grouped_degree& g = c.degrees[q];
        GradDegree<T>& d = p.degree[q];
        d.comps = g.components; d.K = g.in_channels; d.N = g.out_channels; d.x_off = x_off; d.y_off = y_off;
        d.grad = static_cast<T*>(g.grad_weight);
        x_off += static_cast<long long>(d.comps) * d.K;
        y_off += static_cast<long long>(d.comps) * d.N;
    }
    p.groups = c.num_groups; p.offsets = c.offsets;
    p.x = static_cast<const T*>(c.x); p.x_stride = c.x_stride; p.gy = static_cast<const T*>(c.grad_y); p.gy_stride = c.grad_y_stride;
    grouped_grad_kernel<T><<<dim3(c.num_groups, 64, c.num_degrees), 256, 0, static_cast<cudaStream_t>(c.stream)>>>(p);
    launched("grouped_grad_kernel");
}

}  // namespace

size_t grouped_workspace_bytes(const smx_grouped_linear& c, bool backward) {
    check_call(c);
    if (!backward || c.precision == SMX_FP64) return 0;
    size_t values = 0;
    for (int d = 0; d < c.num_degrees; ++d) values += part_values(c, d);
    return values * sizeof(float);
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
