// float32 kernels of the linears with adapters on the 5th-generation tensor cores (tcgen05.mma kind::tf32), included by adapters.cu.
//
// float32 accuracy comes from operands x = hi + lo, both rounded to TF32's 11 bits: lo hi + hi lo + hi hi per product (3xTF32).
// The row operand goes through registers anyway to be split, so it is stored to tensor memory (a thread owns a row, a column holds
// one inner value) and read from there by the matrix instruction; shared memory holds the weights only.
#pragma once

#include "gemm_tcgen05.cuh"

namespace smx {
namespace {

constexpr int kTsRows = 128, kTsThreads = 128, kTsChunk = 32;              // rows and inner values of a step
constexpr int kTsTileBytes = 128 * kTsChunk * 4;                           // 128 columns x 32 inner values
constexpr int kTsSlot = 192;                                               // TMEM: D and hidden columns 0 .. 191, row operand 192 .. 255
constexpr int kTsColumns = 256;

inline int padded_rank(int rank) { return (rank + 15) & ~15; }
inline int ts_chunks(int k) { return (k + kTsChunk - 1) / kTsChunk; }
inline int ts_blocks(int n) { return (n + 127) / 128; }

__device__ __forceinline__ void ts_split(float x, float& hi, float& lo) {
    hi = __uint_as_float(to_tf32(x));
    lo = __uint_as_float(to_tf32(x - hi));
}

__device__ __forceinline__ void ts_store32(uint32_t taddr, const float (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
        "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]),
        "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]),
        "f"(v[30]), "f"(v[31])
        : "memory");
}
__device__ __forceinline__ void ts_store16(uint32_t taddr, const float (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
        "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
        ::"r"(taddr), "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
        "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
        : "memory");
}
__device__ __forceinline__ void ts_load16(uint32_t taddr, float (&v)[16]) {
    uint32_t u[16];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]), "=r"(u[9]),
          "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int q = 0; q < 16; ++q) v[q] = __uint_as_float(u[q]);
}
// D (+)= A B with A in tensor memory and B in shared memory
__device__ __forceinline__ void ts_mma(uint32_t d, uint32_t a, uint64_t b_desc, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t"
        ".reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], %2, %3, p;\n\t"
        "}\n" ::"r"(d), "r"(a), "l"(b_desc), "r"(idesc), "r"(accumulate ? 1u : 0u)
        : "memory");
}
// D = F32, A = B = TF32, both K-major, M = 128, N = n (a multiple of 16)
__device__ __forceinline__ uint32_t ts_idesc(int n) {
    return (1u << 4) | (2u << 7) | (2u << 10) | (static_cast<uint32_t>(n >> 3) << 17) | ((128u >> 4) << 24);
}
// The products of one chunk of `steps` x 8 inner values: row operand hi at column a_hi, lo at a_lo; weights hi at b, lo at b + b_lo bytes.
__device__ __forceinline__ void ts_chunk(uint32_t d, uint32_t a_hi, uint32_t a_lo, uint32_t b_hi, uint32_t b_lo, uint32_t idesc, int steps, bool accumulate) {
    for (int ks = 0; ks < steps; ++ks) {
        ts_mma(d, a_lo + 8 * ks, tc5_smem_desc(b_hi + 32 * ks), idesc, accumulate || ks > 0);
        ts_mma(d, a_hi + 8 * ks, tc5_smem_desc(b_lo + 32 * ks), idesc, true);
        ts_mma(d, a_hi + 8 * ks, tc5_smem_desc(b_hi + 32 * ks), idesc, true);
    }
}
__device__ __forceinline__ void ts_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void ts_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ts_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void ts_wait_store() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// ------------------------------------------------------------------------------------------- operand images
// A matrix as the matrix instruction reads it: [group][column block][chunk][hi, lo][rows][32], rows = columns of the matrix, 128-byte
// swizzle. `rows` of a block is 128, or the padded rank for the first factor of an adapter.
struct ImageSegment {
    const float* src; float* dst;
    long long group_stride, k_stride, n_stride;
    int groups, K, N, rows, blocks, chunks;
};
struct ImageList {
    ImageSegment segment[6 * SMX_ADAPTER_MAX_DEGREES];
};
__global__ void __launch_bounds__(256) adapter_image_kernel(const __grid_constant__ ImageList list) {
    const ImageSegment& s = list.segment[blockIdx.y];
    const long long total = static_cast<long long>(s.groups) * s.blocks * s.chunks * s.rows * 8;
    for (long long t = blockIdx.x * 256LL + threadIdx.x; t < total; t += 256LL * gridDim.x) {
        const int c4 = static_cast<int>(t & 7);
        const long long u = t >> 3;
        const int row = static_cast<int>(u % s.rows);
        const long long tile = u / s.rows;                       // (group * blocks + block) * chunks + chunk
        const int chunk = static_cast<int>(tile % s.chunks);
        const long long gb = tile / s.chunks;
        const int block = static_cast<int>(gb % s.blocks);
        const float* src = s.src + (gb / s.blocks) * s.group_stride;
        const int n = block * s.rows + row;
        float hi[4], lo[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int k = chunk * kTsChunk + c4 * 4 + q;
            ts_split(k < s.K && n < s.N ? src[k * s.k_stride + n * s.n_stride] : 0.f, hi[q], lo[q]);
        }
        float* dst = s.dst + tile * 2 * s.rows * kTsChunk;
        const int off = tc5_swizzled_group(row, c4) >> 2;
        *reinterpret_cast<float4*>(dst + off) = make_float4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<float4*>(dst + s.rows * kTsChunk + off) = make_float4(lo[0], lo[1], lo[2], lo[3]);
    }
}

// ------------------------------------------------------------------------------------------- one direction of the linear
struct TsDegree {
    int comps, Kd, Nc;
    long long in_off, out_off;
    const float* W;                              // images; null: no shared weights
    const float* first; long long first_group;   // floats from adapter to adapter
    const float* second; long long second_group;
    float* hidden;
};
struct TsPass {
    TsDegree degree[SMX_ADAPTER_MAX_DEGREES];
    int degrees, rank, groups, slots;
    long long num_rows, pairs;
    const int* order; const int* offsets;
    const float* weights;
    const float* in; long long in_stride;
    float* out; long long out_stride;
    int sorted, out_sorted, tail;                // as in Pass
};
struct TsWork { int degree, block; TileRows rows; };

// The t-th tile of the pass: degrees, then groups, then row tiles, then column blocks (so that a row tile's blocks run side by side and
// its rows come from L2 after the first). Called by one warp.
__device__ __forceinline__ bool ts_find(const TsPass& p, long long t, TsWork& w) {
    for (int q = 0; q < p.degrees; ++q) {
        const TsDegree& d = p.degree[q];
        const int blocks = p.out ? (d.Nc + 127) / 128 : 1;
        long long tiles;
        if (p.sorted) {
            if (find_tile(p.offsets, p.groups, p.tail != 0, p.pairs, d.comps, kTsRows, t / blocks, w.rows, tiles)) {
                w.degree = q; w.block = static_cast<int>(t % blocks);
                return true;
            }
        } else {
            const long long all = p.num_rows * d.comps;
            tiles = (all + kTsRows - 1) / kTsRows;
            if (t / blocks < tiles) {
                w.degree = q; w.block = static_cast<int>(t % blocks);
                w.rows.group = p.groups; w.rows.first_pair = 0; w.rows.row0 = t / blocks * kTsRows;
                w.rows.rows = min(static_cast<long long>(kTsRows), all - w.rows.row0);
                return true;
            }
        }
        t -= tiles * blocks;
    }
    return false;
}

// 32 inner values of a row from k0 on, zero beyond the row's end.
__device__ __forceinline__ void ts_load_chunk(const float* row, int k0, int Kd, int align, float (&v)[32]) {
    if (row && k0 + 32 <= Kd && align >= 4) {
        if (align >= 8) {
#pragma unroll
            for (int q = 0; q < 4; ++q)
                asm volatile("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                             : "=f"(v[8 * q]), "=f"(v[8 * q + 1]), "=f"(v[8 * q + 2]), "=f"(v[8 * q + 3]), "=f"(v[8 * q + 4]), "=f"(v[8 * q + 5]),
                               "=f"(v[8 * q + 6]), "=f"(v[8 * q + 7])
                             : "l"(row + k0 + 8 * q));
        } else {
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float4 f = __ldg(reinterpret_cast<const float4*>(row + k0) + q);
                v[4 * q] = f.x; v[4 * q + 1] = f.y; v[4 * q + 2] = f.z; v[4 * q + 3] = f.w;
            }
        }
    } else {
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] = row && k0 + q < Kd ? __ldg(row + k0 + q) : 0.f;
    }
}

// A CTA of 128 threads makes a tile of 128 rows x 128 columns, two CTAs to an SM (256 TMEM columns each). A thread owns a row: it loads 32
// of its values ahead, splits the previous 32 and stores them to tensor memory; thread 0 issues the products with [W | first_g] (one
// instruction for the shared and the hidden columns), whose images arrive by bulk copies two chunks ahead. Then every thread takes its hidden
// row out of tensor memory, keeps it if wanted, weights and splits it in place, and the products with second_g are added to the tile.
// Waits are bounded; a tile whose wait runs out is filled with NaN.
__global__ void __launch_bounds__(kTsThreads, 2) adapter_pass_f32_kernel(const __grid_constant__ TsPass pass) {
    extern __shared__ unsigned char ts_smem_raw[];
    __shared__ __align__(8) unsigned long long mma_bar, b_bar[2];
    __shared__ uint32_t tmem_slot;
    __shared__ long long out_base[kTsRows];
    __shared__ TsWork shared_work;
    __shared__ int found, failed;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (warp == 0) {
        TsWork w{};
        const bool ok = ts_find(pass, blockIdx.x, w);
        if (lane == 0) { shared_work = w; found = ok ? 1 : 0; failed = 0; }
    }
    __syncthreads();
    if (!found) return;
    const TsDegree& d = pass.degree[shared_work.degree];
    const int g = shared_work.rows.group, rows = static_cast<int>(shared_work.rows.rows), block = shared_work.block;
    const bool adapter = g < pass.groups, outputs = pass.out != nullptr;
    const int R = pass.rank, Rp = (R + 15) & ~15, col0 = block * 128;
    const int NB = outputs ? min(128, (d.Nc - col0 + 15) & ~15) : 0;        // columns of the tile
    const int main_cols = d.W && outputs ? NB : 0;
    const int first_rows = adapter ? Rp : 0;
    const int hid_col = main_cols ? main_cols : 128;                        // TMEM column of the hidden values
    const int nx = (d.Kd + kTsChunk - 1) / kTsChunk, ne = adapter && outputs ? (Rp + 31) / 32 : 0;

    if (!adapter && !main_cols) {                    // no product at all: zeros
        if (tid < rows) {
            const long long r = shared_work.rows.row0 + tid, p = shared_work.rows.first_pair + r / d.comps;
            const long long n = pass.sorted ? pass.order[p] / pass.slots : p;
            float* to = pass.out + (pass.out_sorted ? p : n) * pass.out_stride + d.out_off + (r % d.comps) * d.Nc;
            for (int c = col0; c < min(d.Nc, col0 + 128); ++c) to[c] = 0.f;
        }
        return;
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTsColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    const float* in_row = nullptr;
    float weight = 1.f;
    long long hid_row = 0;
    {
        long long ob = -1;
        if (tid < rows) {
            const long long r = shared_work.rows.row0 + tid, p = shared_work.rows.first_pair + r / d.comps;
            const int m = static_cast<int>(r % d.comps);
            const long long pair = pass.sorted ? pass.order[p] : p, n = pass.sorted ? pair / pass.slots : p;
            in_row = pass.in + n * pass.in_stride + d.in_off + static_cast<long long>(m) * d.Kd;
            ob = (pass.out_sorted ? p : n) * pass.out_stride + d.out_off + static_cast<long long>(m) * d.Nc;
            hid_row = p * d.comps + m;
            if (adapter && pass.weights) weight = pass.weights[pair];
        }
        out_base[tid] = ob;
    }
    // values every row of the pass is aligned to: 8 (32-byte loads), 4 or fewer
    const unsigned long long bits = static_cast<unsigned long long>(pass.in_stride | d.in_off | d.Kd) * 4u | reinterpret_cast<uintptr_t>(pass.in);
    const int align = (bits & 31) == 0 ? 8 : (bits & 15) == 0 ? 4 : 1;

    unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ts_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    const uint32_t stage_bytes = (128u + Rp) * 256u;
    auto copy_chunk = [&](int j) {        // thread 0
        unsigned char* s = stages + (j & 1) * stage_bytes;
        unsigned long long* bar = &b_bar[j & 1];
        if (j < nx) {
            const uint32_t half = (main_cols + first_rows) * 128u;
            mbar_expect_tx(bar, 2 * half);
            if (main_cols) {
                const float* w = d.W + (static_cast<long long>(block) * nx + j) * (2 * kTsTileBytes / 4);
                bulk_copy_g2s(s, w, main_cols * 128u, bar);
                bulk_copy_g2s(s + half, w + kTsTileBytes / 4, main_cols * 128u, bar);
            }
            if (first_rows) {
                const float* f = d.first + g * d.first_group + static_cast<long long>(j) * 2 * Rp * kTsChunk;
                bulk_copy_g2s(s + main_cols * 128u, f, Rp * 128u, bar);
                bulk_copy_g2s(s + half + main_cols * 128u, f + Rp * kTsChunk, Rp * 128u, bar);
            }
        } else {
            const uint32_t half = NB * 128u;
            mbar_expect_tx(bar, 2 * half);
            const float* f = d.second + g * d.second_group + (static_cast<long long>(block) * ((Rp + 31) / 32) + (j - nx)) * (2 * kTsTileBytes / 4);
            bulk_copy_g2s(s, f, half, bar);
            bulk_copy_g2s(s + half, f + kTsTileBytes / 4, half, bar);
        }
    };
    if (tid == 0) {
        mbar_init(&mma_bar, 1);
        mbar_init(&b_bar[0], 1);
        mbar_init(&b_bar[1], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        copy_chunk(0);
        if (nx + ne > 1) copy_chunk(1);
    }
    ts_fence_before();
    __syncthreads();
    ts_fence_after();
    const uint32_t tmem = tmem_slot, lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    int copied = nx + ne > 1 ? 2 : 1, seen = 0;      // thread 0: chunks whose copies were issued, and waited for
    auto waited = [&](bool ok) { if (!ok) atomicMax(&failed, 1); };
    auto issue = [&](int j, bool accumulate) {       // thread 0: the products of chunk j
        waited(mbar_wait(&b_bar[j & 1], (j >> 1) & 1));
        seen = j + 1;
        if (*reinterpret_cast<volatile int*>(&failed)) return;
        ts_fence_after();
        const uint32_t b = smem_u32(stages + (j & 1) * stage_bytes);
        if (j < nx) {
            const int n = main_cols + first_rows;
            ts_chunk(tmem + (main_cols ? 0 : 128), tmem + kTsSlot, tmem + kTsSlot + 32, b, b + n * 128u, ts_idesc(n), 4, accumulate);
        } else {
            const int e = j - nx;
            ts_chunk(tmem, tmem + hid_col + 32 * e, tmem + kTsSlot + 32 * e, b, b + NB * 128u, ts_idesc(NB), min(4, Rp / 8 - 4 * e), accumulate);
        }
    };

    float cur[32], next[32];
    ts_load_chunk(in_row, 0, d.Kd, align, cur);
    auto step = [&](int j, float (&v)[32]) {
        if (j > 0) {
            if (!*reinterpret_cast<volatile int*>(&failed)) waited(mbar_wait(&mma_bar, (j - 1) & 1));
            ts_fence_after();
            if (tid == 0 && j + 1 < nx + ne && !*reinterpret_cast<volatile int*>(&failed)) { copy_chunk(j + 1); copied = j + 2; }
        }
        float lo[32];
#pragma unroll
        for (int q = 0; q < 32; ++q) ts_split(v[q], v[q], lo[q]);
        ts_store32(lanes + kTsSlot, v);
        ts_store32(lanes + kTsSlot + 32, lo);
        if (j + 2 < nx) ts_load_chunk(in_row, (j + 2) * kTsChunk, d.Kd, align, v);
        ts_wait_store();
        ts_fence_before();
        __syncthreads();
        if (tid == 0 && !*reinterpret_cast<volatile int*>(&failed)) {
            issue(j, j > 0);
            ts_commit(&mma_bar);
        }
    };
    if (nx > 1) ts_load_chunk(in_row, kTsChunk, d.Kd, align, next);
    for (int j = 0; j < nx; j += 2) {
        step(j, cur);
        if (j + 1 < nx) step(j + 1, next);
    }
    __syncthreads();                                 // `failed` as thread 0 left it
    if (!*reinterpret_cast<volatile int*>(&failed)) waited(mbar_wait(&mma_bar, (nx - 1) & 1));
    ts_fence_after();
    if (adapter) {
        if (tid == 0 && nx + 1 < nx + ne && !*reinterpret_cast<volatile int*>(&failed)) { copy_chunk(nx + 1); copied = nx + 2; }
        for (int r0 = 0; r0 < Rp; r0 += 16) {
            float h[16], lo[16];
            ts_load16(lanes + hid_col + r0, h);
            if (d.hidden && block == 0 && tid < rows) {
                float* to = d.hidden + hid_row * R + r0;
                if ((R & 3) == 0) {
#pragma unroll
                    for (int q = 0; q < 16; q += 4)
                        if (r0 + q < R) *reinterpret_cast<float4*>(to + q) = make_float4(h[q], h[q + 1], h[q + 2], h[q + 3]);
                } else {
#pragma unroll
                    for (int q = 0; q < 16; ++q)
                        if (r0 + q < R) to[q] = h[q];
                }
            }
            if (!ne) continue;
#pragma unroll
            for (int q = 0; q < 16; ++q) ts_split(weight * h[q], h[q], lo[q]);
            ts_store16(lanes + hid_col + r0, h);
            ts_store16(lanes + kTsSlot + r0, lo);
        }
        if (ne) {
            ts_wait_store();
            ts_fence_before();
            __syncthreads();
            if (tid == 0 && !*reinterpret_cast<volatile int*>(&failed)) {
                for (int e = 0; e < ne; ++e) issue(nx + e, main_cols > 0 || e > 0);
                ts_commit(&mma_bar);
            }
            __syncthreads();
            if (!*reinterpret_cast<volatile int*>(&failed)) waited(mbar_wait(&mma_bar, nx & 1));
            ts_fence_after();
        }
    }
    __syncthreads();
    const bool bad = *reinterpret_cast<volatile int*>(&failed) != 0;
    if (bad && tid == 0)                             // copies that may be in flight get one more bounded wait before their memory is given back
        for (int j = seen; j < copied; ++j) mbar_wait(&b_bar[j & 1], (j >> 1) & 1);
    if (outputs) {
        // a thread's row leaves through the idle stages so that a store instruction writes whole rows (16-byte groups XOR-ed with the row)
        float* stage = reinterpret_cast<float*>(stages) + warp * (32 * 128);
        if (bad) __syncthreads();
        for (int cc = 0; cc < NB; cc += 16) {
            float v[16];
            ts_load16(lanes + cc, v);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int grp = cc / 4 + j;
                const float4 f = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                *reinterpret_cast<float4*>(stage + lane * 128 + ((grp ^ lane) << 2)) = bad ? make_float4(NAN, NAN, NAN, NAN) : f;
            }
        }
        __syncwarp();
        const unsigned long long obits = static_cast<unsigned long long>(pass.out_stride | d.out_off | d.Nc) * 4u | reinterpret_cast<uintptr_t>(pass.out);
        const bool wide = (obits & 15) == 0;
        const int col = col0 + lane * 4;
        if (lane * 4 < NB)
#pragma unroll 4
            for (int r = 0; r < 32; ++r) {
                const long long ob = out_base[warp * 32 + r];
                if (ob < 0) continue;
                const float4 o = *reinterpret_cast<const float4*>(stage + r * 128 + ((lane ^ r) << 2));
                float* dst = pass.out + ob + col;
                if (wide && col + 3 < d.Nc) {
                    *reinterpret_cast<float4*>(dst) = o;
                } else {
                    const float ov[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
                    for (int q = 0; q < 4; ++q)
                        if (col + q < d.Nc) dst[q] = ov[q];
                }
            }
    } else if (bad && adapter && d.hidden && tid < rows) {
        for (int q = 0; q < R; ++q) d.hidden[hid_row * R + q] = NAN;
    }
    ts_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTsColumns) : "memory");
}

// ------------------------------------------------------------------------------------------- gradients of the adapters
struct TsGrad {
    GradProblem<float> problem[2 * SMX_ADAPTER_MAX_DEGREES];
    int problems, rank, groups, slots;
    long long pairs;
    const int* order; const int* offsets;
    const float* weights;
};

// part[chunk][k][r] as in adapter_grad_kernel: D[k, r] = sum over rows a[row][k] (w h)[row][r]. A thread owns an inner index k of 128 and
// loads a[row][k] of 32 rows (a warp reads 128 consecutive bytes of each), which is the row operand's transpose for nothing; the hidden values
// are split into shared memory. One accumulator of at most 64 columns: four CTAs to an SM.
constexpr int kTsGradColumns = 128, kTsGradSlot = 64;
__global__ void __launch_bounds__(kTsThreads, 4) adapter_grad_f32_kernel(const __grid_constant__ TsGrad pass) {
    extern __shared__ unsigned char ts_smem_raw[];
    __shared__ __align__(8) unsigned long long mma_bar;
    __shared__ uint32_t tmem_slot;
    __shared__ long long a_base[kGradChunk];
    __shared__ float row_weight[kGradChunk];
    __shared__ TileRows tile;
    __shared__ int which, found, failed, k_block;
    __shared__ long long chunk_index;
    const int tid = threadIdx.x, warp = tid >> 5;
    if (warp == 0) {
        long long t = blockIdx.x, tiles = 0;
        TileRows rows{};
        int hit = -1, kb = 0;
        for (int q = 0; q < pass.problems; ++q) {
            const int blocks = (pass.problem[q].Kd + 127) / 128;
            if (find_tile(pass.offsets, pass.groups, false, pass.pairs, pass.problem[q].comps, kGradChunk, t / blocks, rows, tiles)) {
                hit = q; kb = static_cast<int>(t % blocks); t /= blocks;
                break;
            }
            t -= tiles * blocks;
        }
        if (tid == 0) { which = hit; found = hit >= 0; k_block = kb; chunk_index = t; tile = rows; failed = 0; }
    }
    __syncthreads();
    if (!found) return;
    const GradProblem<float>& d = pass.problem[which];
    const int R = pass.rank, Rp = (R + 15) & ~15, rows = static_cast<int>(tile.rows), k = k_block * 128 + tid;
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(kTsGradColumns) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    for (int i = tid; i < kGradChunk; i += kTsThreads) {
        long long base = -1;
        float w = 0.f;
        if (i < rows) {
            const long long r = tile.row0 + i;
            const int pair = pass.order[tile.first_pair + r / d.comps];
            base = static_cast<long long>(pair / pass.slots) * d.a_stride + d.a_off + (r % d.comps) * d.Kd;
            w = pass.weights ? pass.weights[pair] : 1.f;
        }
        a_base[i] = base;
        row_weight[i] = w;
    }
    unsigned char* B = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ts_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    for (int i = tid; i < Rp * 16; i += kTsThreads) reinterpret_cast<float4*>(B)[i] = make_float4(0.f, 0.f, 0.f, 0.f);      // padding rows stay zero
    if (tid == 0) {
        mbar_init(&mma_bar, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    ts_fence_before();
    __syncthreads();
    ts_fence_after();
    const uint32_t tmem = tmem_slot, lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    const float* hidden = d.hidden + (tile.first_pair * d.comps + tile.row0) * R;
    const int hid_values = 32 * R;
    float a[32], h[16];
    auto load = [&](int s) {
#pragma unroll
        for (int q = 0; q < 32; ++q) {
            const int i = s * 32 + q;
            a[q] = i < rows && k < d.Kd ? __ldg(d.a + a_base[i] + k) : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int e = tid + q * kTsThreads;
            h[q] = e < hid_values && s * 32 + e / R < rows ? __ldg(hidden + static_cast<long long>(s) * hid_values + e) * row_weight[s * 32 + e / R] : 0.f;
        }
    };
    const int steps = (rows + 31) / 32;
    load(0);
    for (int s = 0; s < steps; ++s) {
        if (s > 0) {
            if (!*reinterpret_cast<volatile int*>(&failed) && !mbar_wait(&mma_bar, (s - 1) & 1)) atomicMax(&failed, 1);
            ts_fence_after();
        }
        float lo[32];
#pragma unroll
        for (int q = 0; q < 32; ++q) ts_split(a[q], a[q], lo[q]);
        ts_store32(lanes + kTsGradSlot, a);
        ts_store32(lanes + kTsGradSlot + 32, lo);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
            const int e = tid + q * kTsThreads;
            if (e < hid_values) {
                const int i = e / R, r = e % R;
                float hi, l;
                ts_split(h[q], hi, l);
                const int off = tc5_swizzled_group(r, i >> 2) + (i & 3) * 4;
                *reinterpret_cast<float*>(B + off) = hi;
                *reinterpret_cast<float*>(B + Rp * 128 + off) = l;
            }
        }
        if (s + 1 < steps) load(s + 1);
        ts_wait_store();
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        ts_fence_before();
        __syncthreads();
        if (tid == 0 && !*reinterpret_cast<volatile int*>(&failed)) {
            ts_fence_after();
            const uint32_t b = smem_u32(B);
            ts_chunk(tmem, tmem + kTsGradSlot, tmem + kTsGradSlot + 32, b, b + Rp * 128, ts_idesc(Rp), 4, s > 0);
            ts_commit(&mma_bar);
        }
    }
    __syncthreads();
    if (!*reinterpret_cast<volatile int*>(&failed) && !mbar_wait(&mma_bar, (steps - 1) & 1)) atomicMax(&failed, 1);
    __syncthreads();
    ts_fence_after();
    const bool bad = *reinterpret_cast<volatile int*>(&failed) != 0;
    for (int r0 = 0; r0 < Rp; r0 += 16) {
        float v[16];
        ts_load16(lanes + r0, v);
        if (k < d.Kd) {
            float* to = d.part + (chunk_index * d.Kd + k) * R + r0;
#pragma unroll
            for (int q = 0; q < 16; ++q)
                if (r0 + q < R) to[q] = bad ? NAN : v[q];
        }
    }
    ts_fence_before();
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTsGradColumns) : "memory");
}

}  // namespace
}  // namespace smx
