// float64 kernel of the linears of routed rows on the double-precision tensor cores (mma.sync.m8n8k4; the 5th-generation instruction has no
// float64 kind), included by grouped.cu. As in float32 one kernel makes all three products, D [BM x BN] += A [BM x inner] B [inner x BN]:
//   forward    D = rows of y        A = rows of x                 B = W_g
//   backward   D = rows of grad_x   A = rows of grad_y            B = W_g^T
//   gradient   D = rows of grad_W   A = x^T (inner: rows)         B = grad_y (inner: rows)
#pragma once

#include <type_traits>

#include "gemm_tcgen05.cuh"

namespace smx {
namespace {

struct GdDegree {
    int comps, K, N;                 // rows passes: inner values and columns; gradient: rows and columns of the matrices
    long long a_off, b_off;          // of `a`; of `out`, or in the gradient of `b`
    const double* w;
    double* grad; double* part;      // gradient: the result, and partial sums of groups with several sums
};
struct GdPass {
    GdDegree degree[SMX_GROUPED_MAX_DEGREES];
    int degrees, groups, zero_tail;
    long long out_width;
    int chunk;                       // gradient: rows of a sum
    long long rows;
    const int* offsets;
    const double* a; long long a_stride;
    const double* b; long long b_stride;
    double* out; long long out_stride;
};

__device__ __forceinline__ void gd_copy8(double* smem, const double* gmem, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(bytes) : "memory");
}

constexpr int kGdThreads = 128, kGdStep = 16;
// Strides of 4 mod 16 doubles: fragments are read without conflicts. kAcross: the tile holds inner values by rows ([inner][BM or BN]), else rows of inner values.
template <int kWidth, bool kAcross>
struct GdTile {
    static constexpr int stride = kAcross ? kWidth + 4 : kGdStep + 4;
    static constexpr int doubles = kAcross ? kGdStep * stride : kWidth * stride;
    static __device__ __forceinline__ int at(int i, int k) { return kAcross ? k * stride + i : i * stride + k; }
};
template <int kMode, int BM, int BN, int ST>
struct GdLayout {
    using A = GdTile<BM, kMode == kGsGradient>;
    using B = GdTile<BN, kMode != kGsBackward>;
    static constexpr int stage = A::doubles + B::doubles, smem = ST * stage * 8;
};

// The tile-th tile of a pass: degrees, groups, row tiles or sums, then blocks of D. Called by a warp.
struct GdWork { int degree, group, block, mtile, rows, inner, runs, part, comp0; long long first_pair, row0; };   // gradient: from first_pair, comp0 on
template <int kMode>
__device__ __forceinline__ bool gd_find(const GdPass& p, int BM, int BN, long long tile, GdWork& w) {
    const int lane = threadIdx.x & 31;
    for (int q = 0; q < p.degrees; ++q) {
        const GdDegree& d = p.degree[q];
        const int blocks = (d.N + BN - 1) / BN, plane = kMode == kGsGradient ? blocks * ((d.K + BM - 1) / BM) : blocks;
        long long run = 0, parts = 0;
        for (int g0 = 0; g0 < p.groups; g0 += 32) {
            const int g = g0 + lane;
            long long first = 0, rows = 0, runs = 0;
            if (g < p.groups) {
                first = p.offsets[g];
                const long long count = p.offsets[g + 1] - first;
                rows = count * d.comps;
                runs = kMode == kGsGradient ? max(1LL, (rows + p.chunk - 1) / p.chunk) : (rows + BM - 1) / BM;      // a group without rows gets its zeros
            }
            const long long split = kMode == kGsGradient && runs > 1 ? runs : 0;
            long long incl = runs * plane, incl_parts = split;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, incl, s), up_parts = __shfl_up_sync(0xffffffffu, incl_parts, s);
                if (lane >= s) { incl += up; incl_parts += up_parts; }
            }
            const long long begin = run + incl - runs * plane;
            const unsigned hit = __ballot_sync(0xffffffffu, tile >= begin && tile < run + incl);
            if (hit) {
                const int src = __ffs(hit) - 1;
                const int local = static_cast<int>(tile - __shfl_sync(0xffffffffu, begin, src)), at = local / plane, in_plane = local - at * plane;
                rows = __shfl_sync(0xffffffffu, rows, src);
                w.degree = q; w.group = g0 + src;
                w.runs = static_cast<int>(__shfl_sync(0xffffffffu, runs, src));
                w.part = static_cast<int>(parts + __shfl_sync(0xffffffffu, incl_parts - split, src)) + at;
                w.first_pair = __shfl_sync(0xffffffffu, first, src);
                w.mtile = in_plane / blocks;
                w.block = in_plane - w.mtile * blocks;
                w.row0 = static_cast<long long>(at) * (kMode == kGsGradient ? p.chunk : BM);
                const long long left = rows - w.row0;
                if (kMode == kGsGradient) {
                    w.inner = static_cast<int>(min(static_cast<long long>(p.chunk), left));
                    w.first_pair += w.row0 / d.comps;
                    w.comp0 = static_cast<int>(w.row0 % d.comps);
                    w.rows = min(BM, d.K - BM * w.mtile);
                } else {
                    w.inner = d.K;
                    w.rows = static_cast<int>(min(static_cast<long long>(BM), left));
                }
                return true;
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
            parts += __shfl_sync(0xffffffffu, incl_parts, 31);
        }
        tile -= run;
    }
    return false;
}

// A CTA of four warps (WM x WN) makes a tile from ST stages of 16 inner values in flight. The double-precision tensor pipe bounds large calls: 20,000 atoms of 16
// groups, 7.2 GFLOP, 223 us, 32 TFLOP/s of 36. Calls of a few hundred tiles are a chain of copies and products a tile: 1,029 atoms, 131 x 97 (0.24 GFLOP, rows of
// odd length in copies of 8 bytes), 25 us forward; neither tiles of 32 x 64, eight warps a tile, a third stage nor leaving out the blocks behind a tile's end shorten
// that by more than a tenth, and all of them cost large calls 3 to 15 %.
template <int kMode, int BM, int BN, int WM, int WN, int ST>
__global__ void __launch_bounds__(kGdThreads) grouped_f64_kernel(const __grid_constant__ GdPass pass) {
    using L = GdLayout<kMode, BM, BN, ST>;
    using TA = typename L::A;
    using TB = typename L::B;
    constexpr int MB = BM / WM / 8, NB = BN / WN / 8;
    constexpr bool kRows = kMode != kGsGradient;
    static_assert(WM * WN == 4, "four warps");
    extern __shared__ __align__(16) double gd_smem[];
    __shared__ long long a_base[kRows ? BM : 1], out_base[kRows ? BM : 1];
    __shared__ GdWork work;
    __shared__ int found;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp / WN, wn = warp % WN;
    // The gradient reads nothing that the rows' pass before it writes: its CTAs come in as that one's end (one of them waits, so that it does not end first).
    if (kMode == kGsBackward) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (kMode == kGsGradient && blockIdx.x == gridDim.x - 1) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) {
        GdWork w{};
        const bool hit = gd_find<kMode>(pass, BM, BN, blockIdx.x, w);
        if (lane == 0) { work = w; found = hit; }
    }
    if (kRows && pass.zero_tail)
        for (long long p = pass.offsets[pass.groups] + blockIdx.x; p < pass.rows; p += gridDim.x)
            for (long long c = tid; c < pass.out_width; c += kGdThreads) pass.out[p * pass.out_stride + c] = 0.0;
    __syncthreads();
    if (!found) return;
    const GdDegree& d = pass.degree[work.degree];
    const int rows = work.rows, inner = work.inner, col0 = BN * work.block, cols = min(BN, d.N - col0);
    if constexpr (kRows) {
        for (int i = tid; i < BM; i += kGdThreads) {
            const long long r = work.row0 + i, ahead = r / d.comps, m = r - ahead * d.comps, pair = work.first_pair + ahead;
            a_base[i] = i < rows ? pair * pass.a_stride + d.a_off + m * d.K : -1;
            out_base[i] = i < rows ? pair * pass.out_stride + d.b_off + m * d.N + col0 : -1;
        }
        __syncthreads();
    }
    const double* const matrix = d.w + static_cast<long long>(work.group) * d.K * d.N;
    // 16 bytes at a time where all rows start on such a boundary
    const bool wide_a = ((pass.a_stride | d.a_off | d.K) & 1) == 0 && (reinterpret_cast<uintptr_t>(pass.a) & 15) == 0;
    const bool wide_b = kMode == kGsGradient ? ((pass.b_stride | d.b_off | d.N) & 1) == 0 && (reinterpret_cast<uintptr_t>(pass.b) & 15) == 0
                                             : ((kMode == kGsForward ? d.N : d.K) & 1) == 0 && (reinterpret_cast<uintptr_t>(d.w) & 15) == 0;
    // Where inner value k of the gradient's operands begins. (comp0 + k lies below 2^13, where the quotient by a reciprocal is exact.)
    const float reciprocal = 1.f / d.comps;
    auto inner_row = [&](int k, long long stride, int width) {
        const int r = work.comp0 + k, ahead = __float2int_rd((r + 0.5f) * reciprocal);
        return (work.first_pair + ahead) * stride + static_cast<long long>(r - ahead * d.comps) * width;
    };
    auto issue = [&](int chunk) {
        double* const As = gd_smem + (chunk % ST) * L::stage;
        double* const Bs = As + TA::doubles;
        const int k0 = chunk * kGdStep;
        auto copies = [&](bool wide, auto&& fn) {        // fn(values of a copy, copy to, from, offset, whether there is anything)
            if (wide) fn(std::integral_constant<int, 2>{}, [](double* to, const double* base, long long from, bool in) { cp_async16(to, base + (in ? from : 0), in ? 16 : 0); });
            else fn(std::integral_constant<int, 1>{}, [](double* to, const double* base, long long from, bool in) { gd_copy8(to, base + (in ? from : 0), in ? 8 : 0); });
        };
        copies(wide_a, [&](auto values, auto copy) {
            constexpr int per = decltype(values)::value, n = (kRows ? kGdStep : BM) / per;
            const int m0 = BM * work.mtile;
#pragma unroll 4
            for (int i = tid; i < BM * kGdStep / per; i += kGdThreads) {
                if constexpr (kRows) {
                    const int r = i / n, k = (i % n) * per;
                    copy(As + TA::at(r, k), pass.a, a_base[r] + k0 + k, a_base[r] >= 0 && k0 + k < inner);
                } else {
                    const int k = i / n, c = (i % n) * per;
                    const bool in = k0 + k < inner && m0 + c < d.K;
                    copy(As + TA::at(c, k), pass.a, inner_row(k0 + k, pass.a_stride, d.K) + d.a_off + m0 + c, in);
                }
            }
        });
        copies(wide_b, [&](auto values, auto copy) {
            constexpr int per = decltype(values)::value, n = (kMode == kGsBackward ? kGdStep : BN) / per;
#pragma unroll 4
            for (int i = tid; i < BN * kGdStep / per; i += kGdThreads) {
                if constexpr (kMode == kGsBackward) {
                    const int c = i / n, k = (i % n) * per;
                    copy(Bs + TB::at(c, k), matrix, static_cast<long long>(col0 + c) * d.K + k0 + k, c < cols && k0 + k < inner);
                } else {
                    const int k = i / n, c = (i % n) * per;
                    const bool in = k0 + k < inner && c < cols;
                    if constexpr (kMode == kGsForward) copy(Bs + TB::at(c, k), matrix, static_cast<long long>(k0 + k) * d.N + col0 + c, in);
                    else copy(Bs + TB::at(c, k), pass.b, inner_row(k0 + k, pass.b_stride, d.N) + d.b_off + col0 + c, in);
                }
            }
        });
    };
    const int chunks = (inner + kGdStep - 1) / kGdStep;
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) {
        if (s < chunks) issue(s);
        cp_async_commit();
    }
    double acc[MB][NB][2];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NB; ++j) acc[i][j][0] = acc[i][j][1] = 0.0;
    const int fr = lane >> 2, fk = lane & 3;
    for (int t = 0; t < chunks; ++t) {
        cp_async_wait<ST - 2>();
        __syncthreads();                                 // chunk t is there, and the stage of chunk t - 1 has been read
        if (t + ST - 1 < chunks) issue(t + ST - 1);
        cp_async_commit();
        const double* const As = gd_smem + (t % ST) * L::stage;
        const double* const Bs = As + TA::doubles;
#pragma unroll
        for (int kk = 0; kk < kGdStep; kk += 4) {
            double a[MB], b[NB];
#pragma unroll
            for (int i = 0; i < MB; ++i) a[i] = As[TA::at(wm * MB * 8 + i * 8 + fr, kk + fk)];
#pragma unroll
            for (int j = 0; j < NB; ++j) b[j] = Bs[TB::at(wn * NB * 8 + j * 8 + fr, kk + fk)];
#pragma unroll
            for (int i = 0; i < MB; ++i)
#pragma unroll
                for (int j = 0; j < NB; ++j) dmma_m8n8k4(acc[i][j][0], acc[i][j][1], a[i], b[j]);
        }
    }
    double* out = pass.out;
    bool out_wide;
    if constexpr (kRows) {
        out_wide = ((pass.out_stride | d.b_off | d.N) & 1) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    } else {
        out = (work.runs == 1 ? d.grad + static_cast<long long>(work.group) * d.K * d.N : d.part + static_cast<long long>(work.part) * d.K * d.N) +
              static_cast<long long>(BM) * work.mtile * d.N + col0;
        out_wide = (d.N & 1) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0;
    }
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const int r = wm * MB * 8 + i * 8 + fr;
        if (r >= rows) continue;
        double* const to_row = out + (kRows ? out_base[kRows ? r : 0] : static_cast<long long>(r) * d.N);
#pragma unroll
        for (int j = 0; j < NB; ++j) {
            const int c = wn * NB * 8 + 8 * j + 2 * fk;
            if (out_wide && c < cols) {
                *reinterpret_cast<double2*>(to_row + c) = make_double2(acc[i][j][0], acc[i][j][1]);
            } else {
                if (c < cols) to_row[c] = acc[i][j][0];
                if (c + 1 < cols) to_row[c + 1] = acc[i][j][1];
            }
        }
    }
}

}  // namespace
}  // namespace smx
