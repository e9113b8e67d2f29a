// float64 kernels of the linears with adapters on the double-precision tensor cores (mma.sync.m8n8k4; the 5th-generation instruction has
// no float64 kind), included by adapters.cu after adapters_f32.cuh (gemm helpers).
#pragma once

namespace smx {
namespace {

// Matrices of both directions are kept with rows that start on 16-byte boundaries: [k][even(n)] each, see DoubleSegment.
inline int even(int n) { return (n + 1) & ~1; }
struct DoubleSegment {
    const double* src; double* dst;
    long long group_stride, k_stride, n_stride;
    int groups, K, N, ld;
};
struct DoubleList {
    DoubleSegment segment[6 * SMX_ADAPTER_MAX_DEGREES];
};
__global__ void __launch_bounds__(256) adapter_layout_kernel(const __grid_constant__ DoubleList list) {
    const DoubleSegment& s = list.segment[blockIdx.y];
    const long long total = static_cast<long long>(s.groups) * s.K * s.ld;
    for (long long t = blockIdx.x * 256LL + threadIdx.x; t < total; t += 256LL * gridDim.x) {
        const int n = static_cast<int>(t % s.ld);
        const long long u = t / s.ld;
        s.dst[t] = n < s.N ? s.src[u / s.K * s.group_stride + u % s.K * s.k_stride + n * s.n_stride] : 0.0;
    }
}

struct DpDegree {
    int comps, Kd, Nc, ldw;                      // ldw: leading dimension of W and second_g
    long long in_off, out_off;
    const double* W;
    const double* first; long long first_group;  // leading dimension even(rank)
    const double* second; long long second_group;
    double* hidden;
};
struct DpPass {
    DpDegree degree[SMX_ADAPTER_MAX_DEGREES];
    int degrees, rank, groups, slots;
    long long pairs;
    const int* order; const int* offsets; const int* places;
    const double* weights;
    const double* in; long long in_stride;
    double* out; long long out_stride;
    int add, tail;                               // as in Pass
    int whole;                                   // a CTA makes all blocks of columns of a tile without shared weights
};

__device__ __forceinline__ void dp_copy16(double* smem, const double* gmem, int bytes) { cp_async16(smem, gmem, bytes); }
__device__ __forceinline__ void dp_copy8(double* smem, const double* gmem, int bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(smem_u32(smem)), "l"(gmem), "r"(bytes) : "memory");
}

constexpr int kDpThreads = 128, kDpBK = 16, kDpSA = kDpBK + 4;       // strides of 4 mod 16 doubles: fragment reads without conflicts
template <int BM, int BN, int NR, int ST>
struct DpLayout {
    static constexpr int SB = BN + 4, SF = 8 * NR + 4;
    static constexpr int stage = BM * kDpSA + kDpBK * SB + kDpBK * SF;
    static constexpr int smem = (ST * stage + BM * SF + 8 * NR * SB) * 8;
};

// A CTA of four warps (WM x WN) makes BM rows x BN columns of one degree and adapter: in . W and in . first_g from the same row fragments (the warps of
// a row of warps share the inner values of the latter among them and add up through shared memory), then the weighted hidden rows times
// second_g on top. ST stages of 16 inner values are in flight. NR: hidden columns / 8.
// A tile without shared weights makes its blocks of columns one after another from one hidden tile, unless its CTAs are few (11,772 rows of 256
// channels, rank 4: 31 us, and 116 with a CTA for every block). Measured with shared weights: 80,120 rows of 128 channels, rank 8: 140 us, 19 TFLOP/s;
// 28,260 of rank 32: 137 us. The double-precision pipes bound it, with the waits of tiles that run in less than two full rounds of the SMs.
template <int BM, int BN, int WM, int WN, int NR, int ST>
__global__ void __launch_bounds__(kDpThreads) adapter_pass_f64_kernel(const __grid_constant__ DpPass pass) {
    using L = DpLayout<BM, BN, NR, ST>;
    constexpr int MB = BM / WM / 8, NB = BN / WN / 8, SA = kDpSA, SB = L::SB, SF = L::SF;
    static_assert(WM * WN == 4 && 4 % WN == 0, "four warps");
    extern __shared__ __align__(16) double dp_smem[];
    __shared__ long long in_base[BM], out_base[BM], hid_row[BM];
    __shared__ double weight[BM];
    __shared__ TileRows tile;
    __shared__ int which, col_block;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wm = warp / WN, wn = warp % WN;
    if (warp == 0) {
        int hit = -1, cb = 0;
        TileRows t{};
        long long at = blockIdx.x;
        for (int q = 0; q < pass.degrees && hit < 0; ++q) {
            const DpDegree& d = pass.degree[q];
            const int blocks = pass.out && (!pass.whole || d.W) ? (d.Nc + BN - 1) / BN : 1;
            const long long row_tile = at / blocks;
            long long tiles;
            if (find_tile(pass.offsets, pass.groups, pass.tail != 0, pass.pairs, d.comps, BM, row_tile, t, tiles)) { hit = q; cb = static_cast<int>(at % blocks); }
            else at -= tiles * blocks;
        }
        if (lane == 0) { which = hit; col_block = cb; tile = t; }
    }
    __syncthreads();
    if (which < 0) return;
    const DpDegree& d = pass.degree[which];
    const int rows = static_cast<int>(tile.rows), g = tile.group, R = pass.rank, ldf = (R + 1) & ~1;
    int col0 = col_block * BN;
    const bool adapter = g < pass.groups, shared = d.W && pass.out;
    for (int i = tid; i < BM; i += kDpThreads) {
        long long ib = -1, ob = -1, hr = 0;
        double w = 1.0;
        if (i < rows) {
            const long long r = tile.row0 + i, listed = tile.first_pair + r / d.comps, p = pass.places ? pass.places[listed] : listed;
            const int m = static_cast<int>(r % d.comps);
            const int pair = pass.order[p];
            const long long n = pair / pass.slots;
            ib = n * pass.in_stride + d.in_off + static_cast<long long>(m) * d.Kd;
            ob = n * pass.out_stride + d.out_off + static_cast<long long>(m) * d.Nc;
            hr = p * d.comps + m;
            if (adapter && pass.weights) w = pass.weights[pair];
        }
        in_base[i] = ib; out_base[i] = ob; hid_row[i] = hr; weight[i] = w;
    }
    double* const Hs = dp_smem + ST * L::stage;          // [BM][SF] hidden rows
    double* const S2 = Hs + BM * SF;                     // [8 NR][SB] second_g
    const bool wide = ((pass.in_stride | d.in_off | d.Kd) & 1) == 0 && (reinterpret_cast<uintptr_t>(pass.in) & 15) == 0;
    const double* const first = adapter ? d.first + g * d.first_group : nullptr;
    __syncthreads();

    auto issue = [&](int chunk) {
        double* As = dp_smem + (chunk % ST) * L::stage;
        double* Bs = As + BM * SA;
        double* Fs = Bs + kDpBK * SB;
        const int k0 = chunk * kDpBK;
        if (wide) {
            for (int i = tid; i < BM * (kDpBK / 2); i += kDpThreads) {
                const int r = i / (kDpBK / 2), k = (i % (kDpBK / 2)) * 2;
                const int bytes = in_base[r] >= 0 && k0 + k < d.Kd ? 16 : 0;
                dp_copy16(As + r * SA + k, pass.in + (bytes ? in_base[r] + k0 + k : 0), bytes);
            }
        } else {
            for (int i = tid; i < BM * kDpBK; i += kDpThreads) {
                const int r = i / kDpBK, k = i % kDpBK;
                const int bytes = in_base[r] >= 0 && k0 + k < d.Kd ? 8 : 0;
                dp_copy8(As + r * SA + k, pass.in + (bytes ? in_base[r] + k0 + k : 0), bytes);
            }
        }
        if (shared)
            for (int i = tid; i < kDpBK * (BN / 2); i += kDpThreads) {
                const int k = i / (BN / 2), c = (i % (BN / 2)) * 2;
                const int bytes = k0 + k < d.Kd && col0 + c < d.ldw ? 16 : 0;
                dp_copy16(Bs + k * SB + c, d.W + (bytes ? static_cast<long long>(k0 + k) * d.ldw + col0 + c : 0), bytes);
            }
        if (adapter)
            for (int i = tid; i < kDpBK * 4 * NR; i += kDpThreads) {
                const int k = i / (4 * NR), c = (i % (4 * NR)) * 2;
                const int bytes = k0 + k < d.Kd && c < ldf ? 16 : 0;
                dp_copy16(Fs + k * SF + c, first + (bytes ? static_cast<long long>(k0 + k) * ldf + c : 0), bytes);
            }
    };
    const int chunks = adapter || shared ? (d.Kd + kDpBK - 1) / kDpBK : 0;
    auto copy_second = [&]() {
        const double* second = d.second + g * d.second_group;
        for (int i = tid; i < 8 * NR * (BN / 2); i += kDpThreads) {
            const int r = i / (BN / 2), c = (i % (BN / 2)) * 2;
            const int bytes = r < R && col0 + c < d.ldw ? 16 : 0;
            dp_copy16(S2 + r * SB + c, second + (bytes ? static_cast<long long>(r) * d.ldw + col0 + c : 0), bytes);
        }
    };
    if (adapter && pass.out) copy_second();
#pragma unroll
    for (int s = 0; s < ST - 1; ++s) {
        if (s < chunks) issue(s);
        cp_async_commit();
    }
    double acc[MB][NB][2], hid[MB][NR][2];
    const int fr = lane >> 2, fk = lane & 3;
    const bool out_wide = ((pass.out_stride | d.out_off | d.Nc) & 1) == 0 && (reinterpret_cast<uintptr_t>(pass.out) & 15) == 0;
    auto begin_sums = [&]() {                            // from zero, or from what the earlier slots left
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const long long ob = pass.add ? out_base[wm * MB * 8 + i * 8 + fr] : -1;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int c = col0 + wn * NB * 8 + 8 * j + 2 * fk;
                const double* from = pass.out + ob + c;
                double2 v = make_double2(0.0, 0.0);
                if (ob >= 0 && out_wide && c < d.Nc) {
                    v = *reinterpret_cast<const double2*>(from);
                } else if (ob >= 0) {
                    if (c < d.Nc) v.x = from[0];
                    if (c + 1 < d.Nc) v.y = from[1];
                }
                acc[i][j][0] = v.x; acc[i][j][1] = v.y;
            }
        }
    };
    begin_sums();
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
        for (int j = 0; j < NR; ++j) hid[i][j][0] = hid[i][j][1] = 0.0;
    for (int t = 0; t < chunks; ++t) {
        cp_async_wait<ST - 2>();
        __syncthreads();                                 // chunk t is there, and the stage of chunk t - 1 has been read
        if (t + ST - 1 < chunks) issue(t + ST - 1);
        cp_async_commit();
        const double* As = dp_smem + (t % ST) * L::stage + (wm * MB * 8 + fr) * SA + fk;
        const double* Bs = dp_smem + (t % ST) * L::stage + BM * SA;
        const double* Fs = Bs + kDpBK * SB + fk * SF + fr;
        Bs += fk * SB + wn * NB * 8 + fr;
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            double a[MB];
#pragma unroll
            for (int i = 0; i < MB; ++i) a[i] = As[i * 8 * SA + 4 * kk];
            if (shared) {
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const double b = Bs[4 * kk * SB + 8 * j];
#pragma unroll
                    for (int i = 0; i < MB; ++i) dmma_m8n8k4(acc[i][j][0], acc[i][j][1], a[i], b);
                }
            }
            if (adapter && kk % WN == wn) {
#pragma unroll
                for (int j = 0; j < NR; ++j) {
                    const double b = Fs[4 * kk * SF + 8 * j];
#pragma unroll
                    for (int i = 0; i < MB; ++i) dmma_m8n8k4(hid[i][j][0], hid[i][j][1], a[i], b);
                }
            }
        }
    }
    if (adapter) {
        cp_async_wait<0>();
#pragma unroll
        for (int turn = 0; turn < WN; ++turn) {
            if (wn == turn) {
#pragma unroll
                for (int i = 0; i < MB; ++i)
#pragma unroll
                    for (int j = 0; j < NR; ++j)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            double* h = Hs + (wm * MB * 8 + i * 8 + fr) * SF + 8 * j + 2 * fk + e;
                            *h = turn == 0 ? hid[i][j][e] : *h + hid[i][j][e];
                        }
            }
            __syncthreads();
        }
        for (int i = tid; i < rows * R; i += kDpThreads) {
            const int r = i / R, c = i - r * R;
            const double h = Hs[r * SF + c];
            if (d.hidden && col_block == 0) d.hidden[hid_row[r] * R + c] = h;
            Hs[r * SF + c] = h * weight[r];
        }
        // the columns that fill the rank up to four: zeros times the row, so NaN where it holds an infinity, and the rows of second_g they meet are zeros
        const int pad = -R & 3;
        for (int i = tid; i < rows * pad; i += kDpThreads) Hs[i / pad * SF + R + i % pad] = 0.0;
        if (!pass.out) return;
        __syncthreads();
    }
    const int end = pass.whole && !d.W ? d.Nc : min(d.Nc, col0 + BN);
    for (;;) {
        if (adapter)
#pragma unroll 2
        for (int r0 = 0; r0 < R; r0 += 4) {
            double a[MB];
#pragma unroll
            for (int i = 0; i < MB; ++i) a[i] = Hs[(wm * MB * 8 + i * 8 + fr) * SF + r0 + fk];
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const double b = S2[(r0 + fk) * SB + wn * NB * 8 + 8 * j + fr];
#pragma unroll
                for (int i = 0; i < MB; ++i) dmma_m8n8k4(acc[i][j][0], acc[i][j][1], a[i], b);
            }
        }
#pragma unroll
        for (int i = 0; i < MB; ++i) {
            const long long ob = out_base[wm * MB * 8 + i * 8 + fr];
            if (ob < 0) continue;
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int c = col0 + wn * NB * 8 + 8 * j + 2 * fk;
                double* to = pass.out + ob + c;
                if (out_wide && c < d.Nc) {
                    *reinterpret_cast<double2*>(to) = make_double2(acc[i][j][0], acc[i][j][1]);
                } else {
                    if (c < d.Nc) to[0] = acc[i][j][0];
                    if (c + 1 < d.Nc) to[1] = acc[i][j][1];
                }
            }
        }
        col0 += BN;
        if (col0 >= end) break;
        // the next block of columns of a tile without shared weights
        __syncthreads();
        if (adapter) copy_second();
        cp_async_commit();
        begin_sums();
        cp_async_wait<0>();
        __syncthreads();
    }
}

// part[chunk][k][r] = sum over the chunk's rows of a[row][k] (weight h)[row][r], as in adapter_grad_f32_kernel. A CTA has 64 inner indices k, a warp 16
// of them and all hidden columns; 16 rows a step, double-buffered.
struct DpGrad {
    GradProblem<double> problem[2 * SMX_ADAPTER_MAX_DEGREES];
    int problems, rank, groups, slots, chunk;
    long long pairs;
    const int* order; const int* offsets;
    const double* weights;
};
constexpr int kDpGradK = 64, kDpGradSA = kDpGradK + 4, kDpGradRows = 16;
template <int NR>
__global__ void __launch_bounds__(kDpThreads) adapter_grad_f64_kernel(const __grid_constant__ DpGrad pass) {
    constexpr int SF = 8 * NR + 4;
    __shared__ __align__(16) double As[2][kDpGradRows * kDpGradSA];
    __shared__ __align__(16) double Hs[2][kDpGradRows * SF];
    __shared__ long long a_base[kGradChunk];
    __shared__ double row_weight[kGradChunk];
    __shared__ TileRows tile;
    __shared__ int which, k_block;
    __shared__ long long chunk_index;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (warp == 0) {
        long long t = blockIdx.x, tiles = 0;
        TileRows rows{};
        int hit = -1, kb = 0;
        for (int q = 0; q < pass.problems; ++q) {
            const int blocks = (pass.problem[q].Kd + kDpGradK - 1) / kDpGradK;
            if (find_tile(pass.offsets, pass.groups, false, pass.pairs, pass.problem[q].comps, pass.chunk, t / blocks, rows, tiles)) {
                hit = q; kb = static_cast<int>(t % blocks); t /= blocks;
                break;
            }
            t -= tiles * blocks;
        }
        if (lane == 0) { which = hit; k_block = kb; chunk_index = t; tile = rows; }
    }
    __syncthreads();
    if (which < 0) return;
    const GradProblem<double>& d = pass.problem[which];
    const int R = pass.rank, rows = static_cast<int>(tile.rows), k0 = k_block * kDpGradK;
    for (int i = tid; i < pass.chunk; i += kDpThreads) {
        long long base = -1;
        double w = 0.0;
        if (i < rows) {
            const long long r = tile.row0 + i;
            const int pair = pass.order[tile.first_pair + r / d.comps];
            base = static_cast<long long>(pair / pass.slots) * d.a_stride + d.a_off + (r % d.comps) * d.Kd + k0;
            w = pass.weights ? pass.weights[pair] : 1.0;
        }
        a_base[i] = base;
        row_weight[i] = w;
    }
    __syncthreads();
    const bool wide = ((d.a_stride | d.a_off | d.Kd) & 1) == 0 && (reinterpret_cast<uintptr_t>(d.a) & 15) == 0;
    const double* hidden = d.hidden + (tile.first_pair * d.comps + tile.row0) * R;
    const int left = d.Kd - k0;
    auto issue = [&](int s) {
        const int r0 = s * kDpGradRows;
        if (wide) {
            for (int i = tid; i < kDpGradRows * (kDpGradK / 2); i += kDpThreads) {
                const int r = i / (kDpGradK / 2), k = (i % (kDpGradK / 2)) * 2;
                const int bytes = r0 + r < rows && k < left ? 16 : 0;
                dp_copy16(&As[s & 1][r * kDpGradSA + k], d.a + (bytes ? a_base[r0 + r] + k : 0), bytes);
            }
        } else {
            for (int i = tid; i < kDpGradRows * kDpGradK; i += kDpThreads) {
                const int r = i / kDpGradK, k = i % kDpGradK;
                const int bytes = r0 + r < rows && k < left ? 8 : 0;
                dp_copy8(&As[s & 1][r * kDpGradSA + k], d.a + (bytes ? a_base[r0 + r] + k : 0), bytes);
            }
        }
        for (int i = tid; i < kDpGradRows * 8 * NR; i += kDpThreads) {
            const int r = i / (8 * NR), c = i % (8 * NR);
            const int bytes = r0 + r < rows && c < R ? 8 : 0;
            dp_copy8(&Hs[s & 1][r * SF + c], hidden + (bytes ? static_cast<long long>(r0 + r) * R + c : 0), bytes);
        }
        cp_async_commit();
    };
    double acc[2][NR][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < NR; ++j) acc[i][j][0] = acc[i][j][1] = 0.0;
    const int steps = (rows + kDpGradRows - 1) / kDpGradRows, fr = lane >> 2, fk = lane & 3;
    issue(0);
    for (int s = 0; s < steps; ++s) {
        if (s + 1 < steps) { issue(s + 1); cp_async_wait<1>(); }
        else cp_async_wait<0>();
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < kDpGradRows; kk += 4) {
            double a[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) a[i] = As[s & 1][(kk + fk) * kDpGradSA + warp * 16 + i * 8 + fr];
            const double w = row_weight[s * kDpGradRows + kk + fk];
#pragma unroll
            for (int j = 0; j < NR; ++j) {
                const double b = w * Hs[s & 1][(kk + fk) * SF + 8 * j + fr];
#pragma unroll
                for (int i = 0; i < 2; ++i) dmma_m8n8k4(acc[i][j][0], acc[i][j][1], a[i], b);
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int k = k0 + warp * 16 + i * 8 + fr;
        if (k >= d.Kd) continue;
        double* to = d.part + (chunk_index * d.Kd + k) * R;
#pragma unroll
        for (int j = 0; j < NR; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (8 * j + 2 * fk + e < R) to[8 * j + 2 * fk + e] = acc[i][j][e];
    }
}

}  // namespace
}  // namespace smx
