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

inline int padded_rank(int rank) { return (rank + 15) & ~15; }
inline int ts_chunks(int k) { return (k + kTsChunk - 1) / kTsChunk; }
inline int ts_blocks(int n) { return (n + 127) / 128; }

// x = hi + lo, both rounded to TF32's 11 bits (half away from zero; as integers, since conversions run at a quarter of the rate). Bits below
// those must be zero: left in, they cost more than the tensor core's cut of its operands explains (6.6e-7 instead of 2.5e-7 in the sums over rows).
// The addition to the bits carries out of the mantissa of a NaN (all bits set is what the GPU's own arithmetic makes) and leaves zero in both parts; 0 x
// puts a NaN, or what an infinity makes one of, back into hi and changes nothing else.
__device__ __forceinline__ float ts_round(float x) { return __uint_as_float((__float_as_uint(x) + 0x1000u) & kTc5HiMask); }
__device__ __forceinline__ void ts_split(float x, float& hi, float& lo) {
    const float head = ts_round(x);
    hi = __fmaf_rn(x, 0.f, head);
    lo = ts_round(x - head);
}
__device__ __forceinline__ float ts_largest(float a, float b, float c) {
    float m;
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(a), "f"(b), "f"(c));
    return m;
}
// 16 values of a row. A NaN or an infinity among them makes the row's products NaN whichever it is, so the first head tells of all (at 98,304 atoms, 128
// channels, rank 32 162 us, with 0 x for each value 163 and without any 161; lo cut instead of rounded keeps NaN at 160, but the cuts add up: 4.29e-7 instead of
// 4.17e-7 off in the norm at 64 channels, rank 4).
__device__ __forceinline__ void ts_split_row(float (&v)[16], float (&lo)[16]) {
    float most[5];
#pragma unroll
    for (int e = 0; e < 5; ++e) most[e] = ts_largest(v[3 * e], v[3 * e + 1], v[3 * e + 2]);
    const float m = ts_largest(ts_largest(most[0], most[1], most[2]), ts_largest(most[3], most[4], v[15]), 0.f);
#pragma unroll
    for (int e = 0; e < 16; ++e) {
        const float head = ts_round(v[e]);
        lo[e] = ts_round(v[e] - head);
        v[e] = head;
    }
    v[0] = __fmaf_rn(m, 0.f, v[0]);
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
__device__ __forceinline__ void ts_load32(uint32_t taddr, float (&v)[32]) {
    uint32_t u[32];
    tc5_ld32(taddr, u);
#pragma unroll
    for (int q = 0; q < 32; ++q) v[q] = __uint_as_float(u[q]);
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
// The products of one chunk of `steps` x 8 inner values: row operand hi at column a_hi, lo at a_lo; weights hi at b_hi, lo at b_lo. The
// remainders' products come first, while the sum is small: the tensor core cuts its sums, so an addition costs up to 2^-23 of the sum.
// Descriptors of one step ahead are 32 bytes on, two units of their address field.
__device__ __forceinline__ void ts_chunk(uint32_t d, uint32_t a_hi, uint32_t a_lo, uint32_t b_hi, uint32_t b_lo, uint32_t idesc, int steps, bool accumulate) {
    const uint64_t hi = tc5_smem_desc(b_hi), lo = tc5_smem_desc(b_lo);
#pragma unroll 1
    for (int ks = 0; ks < steps; ++ks) {
        ts_mma(d, a_lo + 8 * ks, hi + 2 * ks, idesc, accumulate || ks > 0);
        ts_mma(d, a_hi + 8 * ks, lo + 2 * ks, idesc, true);
    }
#pragma unroll 1
    for (int ks = 0; ks < steps; ++ks) ts_mma(d, a_hi + 8 * ks, hi + 2 * ks, idesc, true);
}
__device__ __forceinline__ void ts_commit(unsigned long long* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// A value that is the same in all lanes, known to be so by the compiler: it can live in the uniform registers that the instructions issued by one lane
// take their operands from.
__device__ __forceinline__ int ts_uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ bool ts_elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
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
    long long pairs;
    const int* order; const int* offsets; const int* places;
    const float* weights;
    const float* in; long long in_stride;
    float* out; long long out_stride;
    int add, tail;                               // as in Pass
    int* status;                                 // null, or receives kTsStatusWait if a wait runs out
    int expire_polls;                            // test switch, zero in normal operation: every CTA loses its weights behind the first chunk and gives up
                                                 // after this many polls
};
constexpr int kTsStatusWait = 7;
struct TsWork { int index, degree, block, found; TileRows rows; };

// The tiles of a pass one after the other: degrees, then groups, then row tiles, then column blocks (so that a row tile's blocks run side by
// side and its rows come from L2 after the first). A cursor remembers the 32 groups it stands at; `t` may only grow. Called by one warp.
struct TsCursor {
    int q = 0, g0 = 0;
    int before = 0, run = 0;                     // work items before degree q, row tiles of degree q before group g0 (the host keeps them below 2^31)
    __device__ __forceinline__ bool find(const TsPass& p, int t, TsWork& w) {
        const int lane = threadIdx.x & 31;
        w.found = 0;
        w.index = t;
        while (q < p.degrees) {
            const TsDegree& d = p.degree[q];
            const int blocks = p.out ? (d.Nc + 127) / 128 : 1;
            const int tile = (t - before) / blocks, g = g0 + lane;
            int first = 0, count = 0;            // places of the group
            if (g < p.groups || (g == p.groups && p.tail)) {
                first = p.offsets[g];
                count = (g < p.groups ? p.offsets[g + 1] : static_cast<int>(p.pairs)) - first;
            }
            const int tiles = static_cast<int>((static_cast<long long>(count) * d.comps + kTsRows - 1) / kTsRows);
            int incl = tiles;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, incl, s);
                if (lane >= s) incl += up;
            }
            const int begin = run + incl - tiles;
            const unsigned hit = __ballot_sync(0xffffffffu, tile >= begin && tile < begin + tiles);
            if (hit) {
                const int src = __ffs(hit) - 1;
                w.found = 1; w.degree = q; w.block = t - before - tile * blocks;
                w.rows.group = g0 + src;
                w.rows.first_pair = __shfl_sync(0xffffffffu, first, src);
                w.rows.row0 = static_cast<long long>(tile - __shfl_sync(0xffffffffu, begin, src)) * kTsRows;
                w.rows.rows = min(static_cast<long long>(kTsRows), static_cast<long long>(__shfl_sync(0xffffffffu, count, src)) * d.comps - w.rows.row0);
                return true;
            }
            run += __shfl_sync(0xffffffffu, incl, 31);
            g0 += 32;
            if (g0 > p.groups) { before += run * blocks; ++q; g0 = 0; run = 0; }
        }
        return false;
    }
};

// What a tile consists of: `nx` chunks of 32 inner values into [shared | hidden] columns, two of them to a partial sum (`sums`), then `rounds` of
// 32 hidden values into the tile.
struct TsShape {
    int group, rows, col0, cols, main_cols, hid_col, nx, sums, rounds;
    bool adapter;
};
__device__ __forceinline__ TsShape ts_shape(const TsPass& p, const TsWork& w) {
    const TsDegree& d = p.degree[w.degree];
    TsShape s;
    s.group = w.rows.group;
    s.rows = static_cast<int>(w.rows.rows);
    s.col0 = w.block * 128;
    s.adapter = s.group < p.groups;
    s.cols = p.out ? min(128, (d.Nc - s.col0 + 15) & ~15) : 0;
    s.main_cols = d.W ? s.cols : 0;
    s.hid_col = s.main_cols ? s.main_cols : 128;
    s.nx = s.adapter || s.main_cols ? (d.Kd + kTsChunk - 1) / kTsChunk : 0;      // neither: nothing but zeros
    s.sums = (s.nx + 1) / 2;
    s.rounds = s.adapter && p.out ? (p.rank + 31) / 32 : 0;
    return s;
}

// One value into the tile (and its hidden rows, where it writes them), by `count` threads.
__device__ __forceinline__ void ts_fill(const TsPass& p, const TsWork& w, int thread, int count, float value) {
    const TsDegree& d = p.degree[w.degree];
    const TsShape s = ts_shape(p, w);
    for (int i = thread; i < s.rows; i += count) {
        const long long r = w.rows.row0 + i, at = w.rows.first_pair + r / d.comps, m = r % d.comps;
        const long long place = p.places ? p.places[at] : at, n = p.order[place] / p.slots;
        if (p.out)
            for (int c = s.col0; c < min(d.Nc, s.col0 + 128); ++c) p.out[n * p.out_stride + d.out_off + m * d.Nc + c] = value;
        if (s.adapter && d.hidden && w.block == 0)
            for (int q = 0; q < p.rank; ++q) d.hidden[(place * d.comps + m) * p.rank + q] = value;
    }
}

// Waits of the pass kernel: bounded by guard[1] polls, and given up at once when another one ran out (guard[0]).
__device__ __forceinline__ bool ts_try(uint32_t addr, unsigned parity) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(addr), "r"(parity) : "memory");
    return done != 0;
}
__device__ __forceinline__ bool ts_wait(unsigned long long* bar, unsigned parity, int* guard) {
    const uint32_t addr = smem_u32(bar);
#pragma unroll 1
    for (unsigned spin = 0; !ts_try(addr, parity); ++spin) {
        if ((spin & 63u) != 63u) continue;
        if (*reinterpret_cast<volatile int*>(guard)) return false;
        if (spin >= static_cast<unsigned>(guard[1])) { atomicExch(guard, 1); return false; }
    }
    return true;
}
__device__ __forceinline__ bool ts_wait_warp(unsigned long long* bar, unsigned parity, int* guard) {
    return __all_sync(0xffffffffu, ts_wait(bar, parity, guard));
}
// All warps of the pass kernel, each from the end of its own part.
__device__ __forceinline__ void ts_meet() {
    __syncwarp();
    ts_fence_before();
    asm volatile("bar.sync 1, 512;" ::: "memory");
}
template <int N> __device__ __forceinline__ void ts_registers_more() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void ts_registers_less() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Rows without a group where a linear has no shared weights for them.
__global__ void __launch_bounds__(256) adapter_zero_rows_kernel(const int* __restrict__ offsets, int groups, long long rows, const int* __restrict__ order,
                                                                const int* __restrict__ places, int slots, float* __restrict__ out, long long stride, int width) {
    for (long long p = offsets[groups] + blockIdx.x; p < rows; p += gridDim.x) {
        const long long n = order[places ? places[p] : p] / slots;
        for (int c = threadIdx.x; c < width; c += 256) out[n * stride + c] = 0.f;
    }
}

__device__ __forceinline__ void cp_async4(void* smem, const void* gmem) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(smem)), "l"(gmem) : "memory");
}

__device__ __forceinline__ void ts_bulk(uint32_t to, const float* from, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

// One persistent CTA per SM walks tiles of 128 rows x 128 columns; its warps are specialised, so that the parts of neighbouring tiles overlap:
//   warp 0      weight images: bulk copies of a chunk's [W | first_g] tiles, or of a round's second_g tiles, into a ring of stages; a stage
//               is these tiles in shared memory and 32 values of the rows in tensor memory, with one barrier for both
//   warp 1      the products (one thread)
//   warp 2      finds the tiles and looks up their atoms and weights (a ring, ahead of all others)
//   warps 4-7   rows: a warp copies 32 values of each of its 32 rows asynchronously, 16 bytes a lane (4 where rows start on no 16-byte boundary),
//               row_stages - 1 chunks ahead; a thread splits those of its row and stores them to the tensor memory's row operand. (Loads and stores by
//               the thread that owns a row touch 32 rows an instruction; a bulk copy takes 70 cycles to issue; one warp that copied for all
//               four took longer than the products: 184 us instead of 160 at 98,304 atoms.)
//   warps 8-15  a thread adds half of its row's partial sums of every 64 inner values in registers (the tensor core cuts its sums instead of
//               rounding them: a single sum over 128 inner values was off five times as far as float32) and writes its half of the row
//               while the products of the next tile run
// TMEM: two partial sums of 128 + Rp columns, taken in turn, and the stages' row operands of 64. The hidden row of a tile is weighted, split and
// stored into the hidden columns of its last two sums (head in the last one's, remainder in the other's); the products with second_g go on
// top of the last sum, which is read after them.
// Every wait is bounded; if one runs out, the CTA gives up, fills its remaining tiles with NaN, reports it to `status` and ends when its copies and
// products in flight have.
constexpr int kTsPassThreads = 512;                                          // as in ts_meet
constexpr int kTsRowPitch = kTsChunk + 4;                                     // floats: threads that read their rows 16 bytes at a time hit all banks
constexpr int kTsOutPitch = 17;                                               // floats of a row in the way out of rows that are not aligned
constexpr int kTsRegsControl = 72, kTsRegsRows = 120, kTsRegsSums = 160, kTsRegsLaunch = 128;
static_assert(kTsRegsControl + kTsRegsRows + 2 * kTsRegsSums <= 4 * kTsRegsLaunch, "the registers of the launch are shared out");
// HP: hidden columns / 16. kWide: every row's half of a tile starts on 32 bytes and is 64 columns long, so nothing is staged on its way out and the
// rows have five stages instead of four (161 .. 165 us instead of 167 at 98,304 atoms, 128 channels, rank 32).
template <int HP, bool kWide>
struct TsPassLayout {
    static constexpr int row_stages = kWide ? 5 : 4;
    // Tiles in the ring. Where tiles have one chunk each (up to 32 inner values), the row warps ask for tile i + row_stages - 1 before they are
    // done with tile i, so the ring holds all of i .. i + row_stages - 1: a shorter one would put the former into the place of the latter, and both
    // sides would wait for each other.
    static constexpr int work_ring = row_stages;
    static_assert(work_ring >= row_stages, "the rows' copies run row_stages - 1 tiles ahead of the tile that is given back last");
    static constexpr int Rp = 16 * HP, sum_cols = 128 + Rp, stages = HP > 2 ? 2 : 3;
    static constexpr int slot0 = 2 * sum_cols;
    static constexpr uint32_t stage_bytes = sum_cols * 256u;
    static constexpr int row_floats = kTsRows * kTsRowPitch;
    static constexpr int smem = stages * static_cast<int>(stage_bytes) + (row_stages * row_floats + (kWide ? 0 : 8 * 32 * kTsOutPitch)) * 4 + 1024;
    static_assert(slot0 + 64 * stages <= 512, "tensor memory has 512 columns");
    static constexpr int fixed_smem = work_ring * (kTsRows * 22 + 64) + 256;  // the ring (work_* below) and the barriers
    static_assert(smem + fixed_smem <= 227 * 1024, "shared memory of one CTA per SM");
};

template <int HP, bool kWide>
__global__ void __launch_bounds__(kTsPassThreads, 1) adapter_pass_f32_kernel(const __grid_constant__ TsPass pass) {
    using L = TsPassLayout<HP, kWide>;
    constexpr int NS = L::stages, RS = L::row_stages, kRing = L::work_ring;
    extern __shared__ unsigned char ts_smem_raw[];
    __shared__ __align__(8) unsigned long long work_full[kRing], work_free[kRing], full[NS], free[NS], d_full[2], d_free[2], t_full, t_done, drained;
    __shared__ TsWork work[kRing];
    __shared__ long long work_in[kRing][kTsRows];                                          // where its rows start in `in`;
    __shared__ int work_atom[kRing][kTsRows], work_place[kRing][kTsRows];                  // their atoms, sorted positions
    __shared__ short work_comp[kRing][kTsRows];                                            // and components
    __shared__ float work_weight[kRing][kTsRows];
    __shared__ uint32_t tmem_slot;
    __shared__ int guard[2];                                                               // a wait ran out; polls of a wait
    __shared__ int copies, row_uses[4];                                                    // chunks copied, operands of every row warp
    const int warp = ts_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    unsigned char* stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(ts_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* row_stages = reinterpret_cast<float*>(stages + NS * L::stage_bytes);
    if (threadIdx.x == 0) {
        guard[0] = 0;
        guard[1] = pass.expire_polls > 0 ? pass.expire_polls : static_cast<int>(kMbarSpinLimit);
        copies = 0;
        for (int q = 0; q < kRing; ++q) { mbar_init(&work_full[q], 1); mbar_init(&work_free[q], 14); }
        for (int q = 0; q < NS; ++q) { mbar_init(&full[q], 5); mbar_init(&free[q], 1); }
        for (int q = 0; q < 2; ++q) { mbar_init(&d_full[q], 1); mbar_init(&d_free[q], 8); }
        mbar_init(&t_full, 8);
        mbar_init(&t_done, 1);
        mbar_init(&drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    ts_fence_before();
    __syncthreads();
    ts_fence_after();
    const uint32_t tmem = tmem_slot;

    if (warp < 4) {
        ts_registers_less<kTsRegsControl>();
        if (warp == 2) {
            TsCursor cursor;
            int t = blockIdx.x;
            for (int i = 0;; ++i) {
                const int slot = i % kRing;
                if (i >= kRing && !ts_wait_warp(&work_free[slot], (i / kRing - 1) & 1, guard)) break;
                TsWork w{};
                while (cursor.find(pass, t, w)) {
                    t += gridDim.x;
                    if (ts_shape(pass, w).nx > 0) break;                 // no shared weights and no adapter: adapter_zero_rows_kernel's
                }
                if (w.found) {
                    const TsDegree& d = pass.degree[w.degree];
                    const int comps = d.comps;
                    const long long q0 = w.rows.row0 < (1LL << 31) ? static_cast<int>(w.rows.row0) / comps : w.rows.row0 / comps;
                    const int p0 = static_cast<int>(w.rows.first_pair + q0), m0 = static_cast<int>(w.rows.row0 - q0 * comps);
                    const bool weighted = w.rows.group < pass.groups && pass.weights;
#pragma unroll 2
                    for (int at = lane; at < kTsRows; at += 32) {
                        const bool live = at < w.rows.rows;
                        const int ahead = (m0 + at) / comps, comp = live ? m0 + at - ahead * comps : 0, listed = live ? p0 + ahead : p0;
                        const int place = pass.places ? pass.places[listed] : listed, pair = pass.order[place], atom = pass.slots > 1 ? pair / pass.slots : pair;
                        work_in[slot][at] = atom * pass.in_stride + d.in_off + comp * d.Kd;
                        work_atom[slot][at] = atom;
                        work_place[slot][at] = place;
                        work_comp[slot][at] = static_cast<short>(comp);
                        work_weight[slot][at] = weighted ? pass.weights[pair] : 1.f;
                    }
                }
                if (lane == 0) work[slot] = w;
                __syncwarp();
                if (lane == 0) mbar_arrive(&work_full[slot]);
                if (!w.found) break;
            }
        } else if (warp == 0 && lane == 0) {
            int n = 0, st = 0;                                           // chunks copied so far, stage of the next one
            unsigned round = 1;                                          // parity of the stage's last use but one
            bool ok = true;
            const uint32_t base = smem_u32(stages);
            // one chunk: `rows_a` rows of a 128-column tile and then `rows_b` of a hidden tile, heads and remainders
            auto copy = [&](const float* a, uint32_t rows_a, const float* b, uint32_t rows_b) {
                if (pass.expire_polls > 0 && n > 0) { ok = false; return; }
                if (n >= NS && !ts_wait(&free[st], round, guard)) { ok = false; return; }
                const uint32_t bar = smem_u32(&full[st]), to = base + st * L::stage_bytes, half = (rows_a + rows_b) * 128u;
                asm volatile("{\n\t.reg .b64 t;\n\tmbarrier.arrive.expect_tx.shared::cta.b64 t, [%0], %1;\n\t}" ::"r"(bar), "r"(2 * half) : "memory");
                if (rows_a) {
                    ts_bulk(to, a, rows_a * 128u, bar);
                    ts_bulk(to + half, a + kTsTileBytes / 4, rows_a * 128u, bar);
                }
                if (rows_b) {
                    ts_bulk(to + rows_a * 128u, b, rows_b * 128u, bar);
                    ts_bulk(to + half + rows_a * 128u, b + L::Rp * kTsChunk, rows_b * 128u, bar);
                }
                ++n;
                if (++st == NS) { st = 0; round ^= 1u; }
            };
            for (int i = 0; ok; ++i) {
                const int slot = i % kRing;
                ok = ts_wait(&work_full[slot], (i / kRing) & 1, guard);
                if (!ok) break;
                const TsWork w = work[slot];
                mbar_arrive(&work_free[slot]);
                if (!w.found) break;
                const TsShape s = ts_shape(pass, w);
                const TsDegree& d = pass.degree[w.degree];
                const float* shared = d.W + static_cast<long long>(w.block) * s.nx * (2 * kTsTileBytes / 4);
                const float* first = d.first + s.group * d.first_group;
                const float* second = d.second + s.group * d.second_group + static_cast<long long>(w.block) * s.rounds * (2 * kTsTileBytes / 4);
#pragma unroll 1
                for (int j = 0; j < s.nx + s.rounds && ok; ++j) {
                    if (j < s.nx) {
                        copy(shared, s.main_cols, first, s.adapter ? L::Rp : 0);
                        shared += 2 * kTsTileBytes / 4;
                        first += 2 * L::Rp * kTsChunk;
                    } else {
                        copy(second, s.cols, nullptr, 0);
                        second += 2 * kTsTileBytes / 4;
                    }
                }
            }
            copies = n;
        } else if (warp == 1) {
            int st = 0, sum = 0, nd = 0;                                 // stage and partial sum in turn, with the parity of their next and last use
            unsigned st_par = 0, sum_par = 1, hid_par = 0;
            bool ok = true;
            const bool leader = ts_elect();
            const uint32_t base = smem_u32(stages), t0 = ts_uniform(tmem);
            for (int i = 0; ok; ++i) {
                const int slot = i % kRing;
                ok = ts_wait_warp(&work_full[slot], (i / kRing) & 1, guard);
                if (!ok) break;
                const TsWork w = work[slot];
                __syncwarp();
                if (leader) mbar_arrive(&work_free[slot]);
                if (!ts_uniform(w.found)) break;
                const TsShape s = ts_shape(pass, w);
                const int nx = ts_uniform(s.nx), items = nx + ts_uniform(s.rounds), main_cols = ts_uniform(s.main_cols), out_cols = ts_uniform(s.cols),
                          in_cols = main_cols + ts_uniform(s.adapter ? L::Rp : 0), hid_col = ts_uniform(s.hid_col);
                // chunks of inner values, then rounds of hidden values on top of the last sum: one piece of code, which stays in the instruction cache
#pragma unroll 1
                for (int j = 0; j < items; ++j) {
                    const bool inner = j < nx;
                    const int e = j - nx;
                    int cols, steps = 4;
                    uint32_t d, hi, lo;
                    bool add;
                    if (inner) {
                        if ((j & 1) == 0 && nd >= 2) ok = ts_wait_warp(&d_free[sum], sum_par, guard);
                        cols = in_cols;
                        d = t0 + sum * L::sum_cols + (main_cols ? 0 : 128);
                        hi = t0 + L::slot0 + 64 * st;
                        lo = hi + 32;
                        add = (j & 1) != 0;
                    } else {
                        if (e == 0) ok = ts_wait_warp(&t_full, hid_par, guard);
                        cols = out_cols;
                        steps = min(4, L::Rp / 8 - 4 * e);
                        d = t0 + (sum ^ 1) * L::sum_cols;
                        hi = d + hid_col + 32 * e;
                        lo = t0 + sum * L::sum_cols + hid_col + 32 * e;
                        add = main_cols > 0 || e > 0;
                    }
                    ok = ok && ts_wait_warp(&full[st], st_par, guard);
                    if (!ok) break;
                    ts_fence_after();
                    const uint32_t b = base + st * L::stage_bytes;
                    const bool last_sum = inner && ((j & 1) != 0 || j + 1 == nx), last_round = !inner && j + 1 == items;
                    if (leader) {
                        ts_chunk(d, hi, lo, b, b + cols * 128u, ts_idesc(cols), steps, add);
                        ts_commit(&free[st]);
                        if (last_sum) ts_commit(&d_full[sum]);
                        if (last_round) ts_commit(&t_done);
                    }
                    __syncwarp();
                    if (++st == NS) { st = 0; st_par ^= 1u; }
                    if (last_sum) {
                        ++nd;
                        sum ^= 1;
                        if (sum == 0) sum_par ^= 1u;
                    }
                    if (last_round) hid_par ^= 1u;
                }
            }
        }
        ts_meet();
        if (guard[0]) {
            // what was started ends before the CTA does: products read its shared and tensor memory, copies write into the former
            if (warp == 1) {
                if (ts_elect()) ts_commit(&drained);
                __syncwarp();
                mbar_wait(&drained, 0);
            } else if (warp == 0 && lane == 0) {
                // the last chunks' barriers, with the arrivals that row warps still owed them
                for (int q = max(0, copies - NS); q < copies; ++q) {
                    for (int w = 0; w < 4; ++w)
                        if (row_uses[w] <= q) mbar_arrive(&full[q % NS]);
                    mbar_wait(&full[q % NS], (q / NS) & 1);
                }
                if (pass.status) atomicMax(pass.status, kTsStatusWait);
            }
        }
    } else if (warp < 8) {
        ts_registers_less<kTsRegsRows>();
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int tid = threadIdx.x & 127, first = tid & ~31;            // the warp's rows are its own: no barrier but the work's
        float* const rows_at = row_stages + first * kTsRowPitch;
        int op = 0, na = 0, xs = 0;                  // operand stage and row stage in turn, operands so far
        unsigned op_par = 1;                         // parity of the operand stage's last use
        bool ok = true;
        // copies run row_stages - 1 chunks ahead of what is split, across tiles
        int ahead_tile = 0, ahead = 0, ahead_nx = 0, ahead_slot = 0, ahead_Kd = 0, ahead_rows = 0;
        bool more = true, wide = false;
        const float* from = nullptr;
        auto copy_next = [&](int stage) {
            if (more && ahead == ahead_nx) {
                ahead_slot = ahead_tile % kRing;
                if (!ts_wait_warp(&work_full[ahead_slot], (ahead_tile / kRing) & 1, guard)) {
                    ok = more = false;
                } else {
                    const TsWork& w = work[ahead_slot];
                    more = w.found != 0;
                    if (more) {
                        const TsDegree& d = pass.degree[w.degree];
                        const unsigned long long bits = static_cast<unsigned long long>(pass.in_stride | d.in_off | d.Kd) * 4u | reinterpret_cast<uintptr_t>(pass.in);
                        wide = (bits & 15) == 0;
                        ahead = 0; ahead_Kd = d.Kd; ahead_nx = (d.Kd + kTsChunk - 1) / kTsChunk;
                        ahead_rows = min(32, static_cast<int>(w.rows.rows) - first);
                        from = pass.in;
                        ++ahead_tile;
                    }
                }
            }
            if (more) {
                float* to = rows_at + stage * L::row_floats;
                const long long* where = work_in[ahead_slot] + first;
                const int left = min(kTsChunk, ahead_Kd - ahead * kTsChunk);
                if (wide) {                          // four rows an instruction, 16 bytes a lane
                    const int c = (lane & 7) * 4;
                    if (c < left)
#pragma unroll 4
                        for (int r = lane >> 3; r < ahead_rows; r += 4) cp_async16(to + r * kTsRowPitch + c, from + where[r] + c, 16);
                } else if (lane < left) {
#pragma unroll 4
                    for (int r = 0; r < ahead_rows; ++r) cp_async4(to + r * kTsRowPitch + lane, from + where[r] + lane);
                }
                from += kTsChunk;
                ++ahead;
            }
            cp_async_commit();
        };
        for (int q = 0; q < RS - 1; ++q) copy_next(q);
        for (int i = 0; ok; ++i) {
            const int slot = i % kRing;
            if (!ts_wait_warp(&work_full[slot], (i / kRing) & 1, guard)) break;
            const TsWork w = work[slot];
            if (!w.found) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&work_free[slot]);
                break;
            }
            const TsShape s = ts_shape(pass, w);
            const int Kd = pass.degree[w.degree].Kd;
            const bool live = tid < s.rows;
            for (int j = 0; j < s.nx + s.rounds; ++j) {
                const bool inner = j < s.nx;
                if (inner) {
                    cp_async_wait<RS - 2>();
                    __syncwarp();                    // the chunk is there for all lanes, and all have read the one before
                    copy_next(xs == 0 ? RS - 1 : xs - 1);
                    if (!ok) break;
                }
                if (na >= NS && !ts_wait_warp(&free[op], op_par, guard)) { ok = false; break; }
                ++na;
                unsigned long long* const bar = &full[op];
                const uint32_t to = lanes + L::slot0 + 64 * op;
                if (++op == NS) { op = 0; op_par ^= 1u; }
                if (!inner) {                        // a round of hidden values has the stage's weights, not its row operand
                    if (lane == 0) mbar_arrive(bar);
                    continue;
                }
                ts_fence_after();
                const float* row = row_stages + xs * L::row_floats + tid * kTsRowPitch;
                if (++xs == RS) xs = 0;
                const int good = live ? Kd - j * kTsChunk : 0;           // what the stage holds behind the tile's or the row's end is no value
#pragma unroll 1
                for (int q = 0; q < kTsChunk; q += 16) {
                    float v[16], lo[16];
#pragma unroll
                    for (int e = 0; e < 16; e += 4) {
                        const float4 f = *reinterpret_cast<const float4*>(row + q + e);
                        v[e] = f.x; v[e + 1] = f.y; v[e + 2] = f.z; v[e + 3] = f.w;
                    }
                    if (good < q + 16)
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[e] = q + e < good ? v[e] : 0.f;
                    ts_split_row(v, lo);
                    ts_store16(to + q, v);
                    ts_store16(to + 32 + q, lo);
                }
                ts_wait_store();
                ts_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(bar);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&work_free[slot]);
        }
        asm volatile("cp.async.wait_all;" ::: "memory");                 // none may be in flight when the CTA ends
        if (lane == 0) row_uses[warp & 3] = na;
        ts_meet();
    } else {
        ts_registers_more<kTsRegsSums>();
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int tid = threadIdx.x & 127, half = (warp - 8) >> 2, R = pass.rank;
        constexpr int kLower = (HP + 1) / 2;         // blocks of 16 hidden columns of the lower half; the upper half has the others
        const int hid0 = half ? kLower : 0, hid_blocks = half ? HP - kLower : kLower;
        float* const out_stage = row_stages + RS * L::row_floats + (warp - 8) * 32 * kTsOutPitch;
        const unsigned long long out_bits = static_cast<unsigned long long>(pass.out_stride) * 4u | reinterpret_cast<uintptr_t>(pass.out);
        int nd = 0, nt = 0, i = 0;                   // partial sums and hidden rows used so far, tiles
        bool ok = true;
        TsWork w{};
        long long out_at = 0;
        int place = 0, comp = 0;
        float weight = 1.f;
        auto next_work = [&]() {
            const int slot = i % kRing;
            if (!ts_wait_warp(&work_full[slot], (i / kRing) & 1, guard)) { ok = false; return; }
            w = work[slot];
            const int atom = work_atom[slot][tid];
            place = work_place[slot][tid];
            comp = work_comp[slot][tid];
            weight = work_weight[slot][tid];
            __syncwarp();
            if (lane == 0) mbar_arrive(&work_free[slot]);
            const TsDegree& d = pass.degree[w.degree];
            out_at = atom * pass.out_stride + d.out_off + static_cast<long long>(comp) * d.Nc;
            ++i;
        };
        next_work();
        int at_hand = blockIdx.x;              // for the tiles to give up
        while (ok && w.found) {
            at_hand = w.index;
            const TsShape s = ts_shape(pass, w);
            const TsDegree& d = pass.degree[w.degree];
            const float mix = weight;
            const bool live = tid < s.rows;
            float* out_row = nullptr;
            float* hid_row = nullptr;
            if (live && pass.out) out_row = pass.out + out_at + s.col0 + 64 * half;
            if (live && s.adapter && d.hidden && w.block == 0) hid_row = d.hidden + (static_cast<long long>(place) * d.comps + comp) * R + 16 * hid0;
            const int left = d.Nc - s.col0 - 64 * half;                  // columns of this half that exist
            const bool out_wide = kWide ? left >= 64 : left >= 64 && ((out_bits | 4u * static_cast<unsigned>(d.out_off | d.Nc)) & 31) == 0;
            float sum[64], hid[16 * kLower];
#pragma unroll
            for (int q = 0; q < 64; ++q) sum[q] = 0.f;
            if (pass.add) {
                // what the earlier slots left comes in while the products run
                if (out_wide) {
                    if (out_row)
#pragma unroll
                        for (int q = 0; q < 64; q += 8)
                            asm volatile("ld.global.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];" : "=f"(sum[q]), "=f"(sum[q + 1]), "=f"(sum[q + 2]), "=f"(sum[q + 3]),
                                         "=f"(sum[q + 4]), "=f"(sum[q + 5]), "=f"(sum[q + 6]), "=f"(sum[q + 7]) : "l"(out_row + q) : "memory");
                } else if constexpr (!kWide) {
                    const unsigned long long mine = reinterpret_cast<unsigned long long>(out_row);
#pragma unroll
                    for (int c0 = 0; c0 < 64; c0 += 16) {
                        if (c0 >= left) continue;
                        const int c = c0 + (lane & 15);
                        float v[16];
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, mine, 2 * r + (lane >> 4)));
                            v[r] = from && c < left ? from[c] : 0.f;
                        }
                        __syncwarp();
#pragma unroll
                        for (int r = 0; r < 16; ++r) out_stage[(2 * r + (lane >> 4)) * kTsOutPitch + (lane & 15)] = v[r];
                        __syncwarp();
#pragma unroll
                        for (int q = 0; q < 16; ++q) sum[c0 + q] = out_stage[lane * kTsOutPitch + q];
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < 16 * kLower; ++q) hid[q] = 0.f;
            auto add_columns = [&](uint32_t from, int cols) {            // of [0, cols) those of this half
#pragma unroll
                for (int cc = 0; cc < 2; ++cc)
                    if (64 * half + 32 * cc < cols) {                    // 16 columns of a last, odd block may be another's: never used
                        float v[32];
                        ts_load32(from + 64 * half + 32 * cc, v);
#pragma unroll
                        for (int q = 0; q < 32; ++q) sum[32 * cc + q] += v[q];
                    }
            };
            auto release = [&](int use) {
                ts_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&d_free[use & 1]);
            };
            // with rounds, the last sum's shared columns are read at the end, and the last two are given back there
            const int stay = s.rounds > 0 ? s.sums - 1 : s.sums, kept = s.rounds > 0 ? min(2, s.sums) : 0;
            for (int j = 0; j < s.sums; ++j, ++nd) {
                if (!ts_wait_warp(&d_full[nd & 1], (nd >> 1) & 1, guard)) { ok = false; break; }
                ts_fence_after();
                const uint32_t from = lanes + (nd & 1) * L::sum_cols;
                if (s.adapter)
#pragma unroll
                    for (int cc = 0; cc < kLower; ++cc)
                        if (cc < hid_blocks) {
                            float v[16];
                            ts_load16(from + s.hid_col + 16 * (hid0 + cc), v);
#pragma unroll
                            for (int q = 0; q < 16; ++q) hid[16 * cc + q] += v[q];
                        }
                if (j < stay) add_columns(from, s.main_cols);
                if (j < s.sums - kept) release(nd);
            }
            if (!ok) break;
            if (s.rounds > 0) {
                // the halves read and store hidden blocks of their own; where the tile has one sum, the other partial sum is the previous tile's, which
                // the other half's warp may still be reading
                if (s.sums == 1 && nd > 1 && !ts_wait_warp(&d_free[nd & 1], ((nd - 2) >> 1) & 1, guard)) { ok = false; break; }
                const uint32_t hi_at = lanes + ((nd - 1) & 1) * L::sum_cols + s.hid_col, lo_at = lanes + (nd & 1) * L::sum_cols + s.hid_col;
#pragma unroll
                for (int cc = 0; cc < kLower; ++cc)
                    if (cc < hid_blocks) {
                        float hi[16], lo[16];
#pragma unroll
                        for (int q = 0; q < 16; ++q) ts_split(mix * hid[16 * cc + q], hi[q], lo[q]);
                        ts_store16(hi_at + 16 * (hid0 + cc), hi);
                        ts_store16(lo_at + 16 * (hid0 + cc), lo);
                    }
                ts_wait_store();
                ts_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&t_full);
            }
            if (hid_row) {
                const int n = min(16 * hid_blocks, R - 16 * hid0);
#pragma unroll
                for (int q = 0; q < 16 * kLower; q += 4) {
                    if ((R & 3) == 0) {
                        if (q < n) *reinterpret_cast<float4*>(hid_row + q) = make_float4(hid[q], hid[q + 1], hid[q + 2], hid[q + 3]);
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            if (q + e < n) hid_row[q + e] = hid[q + e];
                    }
                }
            }
            if (s.rounds > 0) {
                if (!ts_wait_warp(&t_done, nt & 1, guard)) { ok = false; break; }
                ++nt;
                ts_fence_after();
                if (kept == 2) release(nd - 2);
                add_columns(lanes + ((nd - 1) & 1) * L::sum_cols, s.cols);
                release(nd - 1);
            }
            next_work();
            if (!ok) break;
            if (out_wide) {
                if (out_row)
#pragma unroll
                    for (int q = 0; q < 64; q += 8)
                        asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(out_row + q), "f"(sum[q]), "f"(sum[q + 1]), "f"(sum[q + 2]),
                                     "f"(sum[q + 3]), "f"(sum[q + 4]), "f"(sum[q + 5]), "f"(sum[q + 6]), "f"(sum[q + 7]) : "memory");
            } else if (!kWide && pass.out) {
                // 16 columns of the warp's rows at a time through shared memory, so that a store touches two rows instead of 32
                const unsigned long long mine = reinterpret_cast<unsigned long long>(out_row);
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 16) {
                    if (c0 >= left) continue;
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 16; ++q) out_stage[lane * kTsOutPitch + q] = sum[c0 + q];
                    __syncwarp();
                    const int c = c0 + (lane & 15);
#pragma unroll 4
                    for (int r = lane >> 4; r < 32; r += 2) {
                        float* to = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, mine, r));
                        if (to && c < left) to[c] = out_stage[r * kTsOutPitch + (c - c0)];
                    }
                }
                __syncwarp();
            }
        }
        if (!ok) {
            // NaN into the tile at hand and all that would have followed
            TsCursor cursor;
            TsWork lost{};
            for (int t = at_hand; cursor.find(pass, t, lost); t += gridDim.x) ts_fill(pass, lost, tid, 128, NAN);
        }
        ts_meet();
    }
    __syncthreads();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------------------------------- gradients of the adapters
struct TsGrad {
    GradProblem<float> problem[2 * SMX_ADAPTER_MAX_DEGREES];
    int problems, rank, groups, slots, chunk;
    long long pairs;
    const int* order; const int* offsets;
    const float* weights;
};

// part[chunk][k][r] = sum over the chunk's rows of (weight a)[row][k] h[row][r] on the FMA pipes, two hidden columns an instruction. The chunk's
// hidden rows are copied to shared memory once; then every warp walks its rows by itself, a lane with four inner indices and 16 hidden columns
// (the warps of a CTA share out first the hidden columns, then the rows), four rows ahead. On the tensor cores a product with 16 columns
// takes as long as one with 96, and the rows would have to be turned and split: 177 us where this takes 92 (8,001 atoms behind the tensor
// product, rank 16; FMA pipes 40 % busy, issue slots 44 %).
template <int NH>                                    // hidden columns / 16
__global__ void __launch_bounds__(kTsThreads, NH == 4 ? 3 : 4) adapter_grad_f32_kernel(const __grid_constant__ TsGrad pass) {
    constexpr int Rp = 16 * NH, kPer = 4, kCols = 32 * kPer, kAhead = 4;               // inner indices of a lane, of the CTA
    constexpr int kRowWarps = NH == 1 ? 4 : NH == 2 ? 2 : 1;                             // warps that share the rows of 16 hidden columns
    extern __shared__ __align__(16) unsigned char ts_smem_raw[];
    float* const hs = reinterpret_cast<float*>(ts_smem_raw);                             // [chunk][Rp], afterwards the warps' sums [Rp][kCols]
    __shared__ long long a_base[kGradChunk];
    __shared__ float row_weight[kGradChunk];
    __shared__ TileRows tile;
    __shared__ int which, k_block;
    __shared__ long long chunk_index;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, col16 = 16 * (warp / kRowWarps);
    if (warp == 0) {
        long long t = blockIdx.x, tiles = 0;
        TileRows rows{};
        int hit = -1, kb = 0;
        for (int q = 0; q < pass.problems; ++q) {
            const int blocks = (pass.problem[q].Kd + kCols - 1) / kCols;
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
    const GradProblem<float>& d = pass.problem[which];
    const int R = pass.rank, rows = static_cast<int>(tile.rows), k = k_block * kCols + kPer * lane, left = d.Kd - k;
    const float* hidden = d.hidden + (tile.first_pair * d.comps + tile.row0) * R;
    if ((R & 3) == 0) {                              // rows of hidden values follow one another: 16 bytes at a time
        for (int i = tid; i < rows * (Rp / 4); i += kTsThreads) {
            const int r = i / (Rp / 4), c = (i % (Rp / 4)) * 4;
            cp_async16(hs + r * Rp + c, hidden + (c < R ? r * R + c : 0), c < R ? 16 : 0);
        }
    } else {
        for (int i = tid; i < rows * Rp; i += kTsThreads) {
            const int r = i / Rp, c = i % Rp;
            if (c < R) cp_async4(hs + i, hidden + r * R + c);
            else hs[i] = 0.f;
        }
    }
    cp_async_commit();
    const long long q0 = tile.row0 / d.comps;
    const int m0 = static_cast<int>(tile.row0 - q0 * d.comps);
    for (int i = tid; i < rows; i += kTsThreads) {
        const int ahead = (m0 + i) / d.comps, pair = pass.order[tile.first_pair + q0 + ahead];
        a_base[i] = static_cast<long long>(pair / pass.slots) * d.a_stride + d.a_off + static_cast<long long>(m0 + i - ahead * d.comps) * d.Kd;
        row_weight[i] = pass.weights ? pass.weights[pair] : 1.f;
    }
    const bool wide = ((d.a_stride | d.a_off | d.Kd) & (kPer - 1)) == 0 && (reinterpret_cast<uintptr_t>(d.a) & (4 * kPer - 1)) == 0;
    unsigned long long acc[kPer][8];                 // pairs of hidden columns
#pragma unroll
    for (int q = 0; q < kPer; ++q)
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[q][j] = 0ull;
    cp_async_wait<0>();
    __syncthreads();
    auto load = [&](int r0, float (&a)[kAhead][kPer]) {          // rows r0, r0 + kRowWarps, ..
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = r0 + kRowWarps * u;
            const float* src = r < rows ? d.a + a_base[r] + k : nullptr;
            if (wide) {
                const float4 f = src && left > 0 ? __ldg(reinterpret_cast<const float4*>(src)) : make_float4(0.f, 0.f, 0.f, 0.f);
                a[u][0] = f.x; a[u][1] = f.y; a[u][2] = f.z; a[u][3] = f.w;
            } else {
#pragma unroll
                for (int q = 0; q < kPer; ++q) a[u][q] = src && q < left ? __ldg(src + q) : 0.f;
            }
        }
    };
    auto add = [&](int r0, const float (&a)[kAhead][kPer]) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int r = r0 + kRowWarps * u;
            if (r >= rows) break;
            const ulonglong2* h = reinterpret_cast<const ulonglong2*>(hs + r * Rp + col16);
            const float w = row_weight[r];
            unsigned long long twice[kPer];
#pragma unroll
            for (int q = 0; q < kPer; ++q) asm("mov.b64 %0, {%1, %1};" : "=l"(twice[q]) : "f"(w * a[u][q]));
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const ulonglong2 two = h[j];
#pragma unroll
                for (int q = 0; q < kPer; ++q) {
                    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[q][2 * j]) : "l"(twice[q]), "l"(two.x));
                    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc[q][2 * j + 1]) : "l"(twice[q]), "l"(two.y));
                }
            }
        }
    };
    float a0[kAhead][kPer], a1[kAhead][kPer];
    const bool idle = col16 >= Rp;                   // three blocks of hidden columns leave a warp without one
    const int first_row = idle ? rows : warp % kRowWarps;
    load(first_row, a0);
#pragma unroll 1
    for (int r0 = first_row; r0 < rows; r0 += 2 * kRowWarps * kAhead) {
        load(r0 + kRowWarps * kAhead, a1);
        add(r0, a0);
        load(r0 + 2 * kRowWarps * kAhead, a0);
        add(r0 + kRowWarps * kAhead, a1);
    }
    // the warps' sums in turn
    float* const joined = hs;
    for (int turn = 0; turn < kRowWarps; ++turn) {
        __syncthreads();
        if (idle || warp % kRowWarps != turn) continue;
#pragma unroll
        for (int q = 0; q < kPer; ++q)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                float x, y;
                asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(acc[q][j]));
                float* to = joined + (col16 + 2 * j) * kCols + kPer * lane + q;
                to[0] = turn ? to[0] + x : x;
                to[kCols] = turn ? to[kCols] + y : y;
            }
    }
    __syncthreads();
    for (int i = tid; i < kCols * R; i += kTsThreads) {
        const int kk = i / R, r = i - kk * R;
        if (k_block * kCols + kk < d.Kd) d.part[(chunk_index * d.Kd + k_block * kCols) * R + i] = joined[r * kCols + kk];
    }
}

}  // namespace
}  // namespace smx
