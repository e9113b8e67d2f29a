// float32 kernel of the linears of routed rows on the 5th-generation tensor cores (tcgen05.mma kind::tf32), included by grouped.cu.
//
// One kernel makes all three products, as D [128 rows x 128 columns] += A [128 x inner] B [inner x 128]:
//   forward    D = rows of y        A = rows of x                 B = W_g
//   backward   D = rows of grad_x   A = rows of grad_y            B = W_g^T
//   gradient   D = rows of grad_W   A = x^T (inner: rows)         B = grad_y (inner: rows)
// float32 accuracy comes from operands v = hi + lo of 11 bits each: lo hi + hi lo + hi hi per product (3xTF32). Both operands are read as they are and
// split on their way: A, a thread per row, to tensor memory; B, a thread per column, to shared memory in the layout of the instruction. There is
// no prepared copy of the matrices: training changes them in every step, and few rows per group read them once.
#pragma once

#include "tcgen05_ops.cuh"

namespace smx {
namespace {

enum GsMode { kGsForward, kGsBackward, kGsGradient };
constexpr int kGsThreads = 1024, kGsChunk = 64, kGsStages = 2, kGsRing = 8;   // inner values of a step; stages of A and of B; tiles in the ring
constexpr int kGsPartBytes = 128 * 32 * 4, kGsHalfBytes = 2 * kGsPartBytes, kGsStageBytes = 2 * kGsHalfBytes;     // B: 32 inner values; hi or lo; both
constexpr int kGsOutPitch = 17;                                              // floats of a row on its way out of rows that are not aligned
constexpr int kGsStatusWait = 8;
// the warps' shares of the registers, by fours: control, A, sums, B, copies
constexpr int kGsRegsLaunch = 64, kGsRegsControl = 40, kGsRegsOperand = 56, kGsRegsSums = 96, kGsRegsCopies = 56;
static_assert(kGsRegsControl + 4 * kGsRegsOperand + 2 * kGsRegsSums + kGsRegsCopies <= 8 * kGsRegsLaunch, "the registers of the launch are shared out");

struct GsDegree {
    int comps, K, N;                 // rows passes: inner values and columns; gradient: rows and columns of the matrices
    long long a_off, b_off;          // of `a`; of `out`, or in the gradient of `b`
    const float* w;                  // the matrices
    float* grad; float* part;        // gradient: the result, and partial sums of groups with several chunks of rows
};
struct GsPass {
    GsDegree degree[SMX_GROUPED_MAX_DEGREES];
    int degrees, groups, zero_tail;
    long long out_width;
    int chunk;                       // gradient: rows of a tile's sum, a multiple of kGsChunk
    long long rows;
    const int* offsets;
    const float* a; long long a_stride;
    const float* b; long long b_stride;
    float* out; long long out_stride;
    int* status;                     // null, or receives kGsStatusWait if a wait runs out
    int expire_polls;                // test switch, zero in normal operation: every CTA loses its B behind the first chunk and gives up after this many polls
};
// A tile of D. `fresh`: its B is not the one before's; `last`: the next tile's is another one.
struct GsWork {
    int found, degree, tile, group, block, mtile, rows, inner, chunks, fresh, last, first_pair;
    long long row0;
    float* out;                      // gradient
};

template <int kMode>
__device__ __forceinline__ bool gs_resident(const GsDegree& d) { return kMode != kGsGradient && d.K <= kGsChunk * kGsStages; }
template <int kMode>
__device__ __forceinline__ int gs_plane(const GsDegree& d) {             // tiles of a group's D that share its rows
    const int blocks = (d.N + 127) / 128;
    return kMode == kGsGradient ? blocks * ((d.K + 127) / 128) : blocks;
}
template <int kMode>
__device__ __forceinline__ int gs_runs(const GsPass& p, const GsDegree& d, long long count) {        // row tiles of a group, or chunks of its rows
    const long long rows = count * d.comps;
    if (kMode == kGsGradient) return max(1, static_cast<int>((rows + p.chunk - 1) / p.chunk));          // a group without rows gets its zeros
    return static_cast<int>((rows + 127) / 128);
}

// The CTA's tiles, the same share of all steps for each (a sum of the gradient counts as a whole chunk, whatever the group's rows): lane q holds begin and end among the tiles of
// degree q. Called by a warp.
template <int kMode>
__device__ __forceinline__ void gs_share(const GsPass& p, int& begin, int& end) {
    const int lane = threadIdx.x & 31;
    long long total = 0, before = 0;
    int mine = 0;
    auto cost_of = [&](const GsDegree& d) { return (kMode == kGsGradient ? p.chunk / kGsChunk : (d.K + kGsChunk - 1) / kGsChunk) + 2; };
    for (int q = 0; q < p.degrees; ++q) {
        const GsDegree& d = p.degree[q];
        int n = 0;
        for (int g = lane; g < p.groups; g += 32) n += gs_runs<kMode>(p, d, p.offsets[g + 1] - p.offsets[g]);
        n = __reduce_add_sync(0xffffffffu, n) * gs_plane<kMode>(d);
        if (lane == q) { mine = n; before = total; }
        total += static_cast<long long>(n) * cost_of(d);
    }
    begin = end = 0;
    if (lane < p.degrees) {
        const long long cost = cost_of(p.degree[lane]);
        auto cut = [&](long long at) { return static_cast<int>(min(static_cast<long long>(mine), max(0LL, (at - before + cost - 1) / cost))); };
        begin = cut(total * blockIdx.x / gridDim.x);
        end = cut(total * (blockIdx.x + 1) / gridDim.x);
    }
}

// Finds the tiles of a degree in ascending order: groups, then where a tile's B stays for the next ones column blocks and row tiles, else row tiles and
// column blocks (neighbours then read the same rows).
// The bounds of 32 groups stay in a warp's registers: read and added up for every tile, they would take as long as the products of a short one.
struct GsCursor {
    int q = -1, g0 = 0, run = 0, parts = 0;          // tiles and partial sums of the groups before g0
    int end = 0, first, count, runs, begin, part;    // tiles up to the last of the 32 groups; the lane's group
    template <int kMode>
    __device__ __forceinline__ void look(const GsPass& p, const GsDegree& d) {
        const int lane = threadIdx.x & 31, g = g0 + lane;
        first = count = runs = 0;
        if (g < p.groups) {
            first = p.offsets[g];
            count = p.offsets[g + 1] - first;
            runs = gs_runs<kMode>(p, d, count);
        }
        const int mine = runs * gs_plane<kMode>(d), split = kMode == kGsGradient && runs > 1 ? runs : 0;
        int incl = mine, incl_parts = split;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, s);
            if (lane >= s) incl += up;
            if (kMode == kGsGradient) {
                const int up_parts = __shfl_up_sync(0xffffffffu, incl_parts, s);
                if (lane >= s) incl_parts += up_parts;
            }
        }
        begin = run + incl - mine;
        part = parts + incl_parts - split;
        end = run + __shfl_sync(0xffffffffu, incl, 31);
        parts += __shfl_sync(0xffffffffu, incl_parts, 31);
    }
    template <int kMode>
    __device__ __forceinline__ bool find(const GsPass& p, int degree, int t, GsWork& w) {
        const GsDegree& d = p.degree[degree];
        if (degree != q) {
            q = degree;
            g0 = run = parts = 0;
            look<kMode>(p, d);
        }
        while (t >= end) {
            g0 += 32;
            run = end;
            if (g0 >= p.groups) { w.found = 0; return false; }
            look<kMode>(p, d);
        }
        const int src = __ffs(__ballot_sync(0xffffffffu, t >= begin && t < begin + runs * gs_plane<kMode>(d))) - 1;
        const int local = t - __shfl_sync(0xffffffffu, begin, src), group_runs = __shfl_sync(0xffffffffu, runs, src);
        const long long rows = static_cast<long long>(__shfl_sync(0xffffffffu, count, src)) * d.comps;
        const int blocks = (d.N + 127) / 128;
        w.found = 1; w.degree = q; w.tile = t; w.group = g0 + src;
        w.first_pair = __shfl_sync(0xffffffffu, first, src);
        w.fresh = w.last = 1;
        if (kMode == kGsGradient) {
            const int plane = gs_plane<kMode>(d), at = local / plane, in_plane = local - at * plane;
            w.mtile = in_plane / blocks;
            w.block = in_plane - w.mtile * blocks;
            w.row0 = static_cast<long long>(at) * p.chunk;
            w.rows = min(128, d.K - 128 * w.mtile);
            w.inner = static_cast<int>(min(static_cast<long long>(p.chunk), rows - w.row0));
            const long long place = __shfl_sync(0xffffffffu, part, src) + at;
            float* to = group_runs == 1 ? d.grad + static_cast<long long>(w.group) * d.K * d.N : d.part + place * d.K * d.N;
            w.out = to + 128LL * w.mtile * d.N + 128 * w.block;
        } else {
            int at = local;
            w.block = 0;
            if (gs_resident<kMode>(d)) {
                if (blocks > 1) {
                    w.block = local / group_runs;
                    at = local - w.block * group_runs;
                }
                w.last = at + 1 == group_runs;
            } else if (blocks > 1) {
                at = local / blocks;
                w.block = local - at * blocks;
            }
            w.mtile = 0;
            w.row0 = static_cast<long long>(at) * 128;
            w.rows = static_cast<int>(min(128LL, rows - w.row0));
            w.inner = d.K;
        }
        w.chunks = (w.inner + kGsChunk - 1) / kGsChunk;
        return true;
    }
};

// Where row i of D of a rows pass is: the row of the arrays (a pair of the plan) and its component.
__device__ __forceinline__ void gs_row(const GsWork& w, int comps, int i, int& pair, int& comp) {
    const long long r = w.row0 + i;
    const long long ahead = r < (1LL << 31) ? static_cast<int>(r) / comps : r / comps;
    pair = w.first_pair + static_cast<int>(ahead);
    comp = static_cast<int>(r - ahead * comps);
}

// Tiles of 32 x 32 values on their way from global memory to the registers of an operand warp, through 4 KB of shared memory each. A row of the array is a
// line of 128 bytes there. kInner: rows are inner values, and a lane owns a column; else a lane owns a row, and its 16-byte pieces are permuted by the row.
template <bool kInner>
struct GsTile {
    static __device__ __forceinline__ int place(int r, int c) { return 32 * r + (kInner ? c : ((((c >> 2) ^ r) & 7) << 2) + (c & 3)); }
    // `rows` x `cols` of the tile exist. at(u): where row lane / 8 + 4 u begins, if `wide` (four rows an instruction, 16 bytes a lane); row_at(r): row r
    template <typename At, typename RowAt>
    static __device__ __forceinline__ void copy(float* buffer, const float* base, int rows, int cols, bool wide, At&& at, RowAt&& row_at) {
        const int lane = threadIdx.x & 31;
        if (wide) {
            const int c = (lane & 7) * 4;
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const int r = (lane >> 3) + 4 * u;
                const long long from = at(u);
                if (r < rows && c < cols) cp_async16(buffer + place(r, c), base + from + c, 16);
            }
        } else {
#pragma unroll 2
            for (int r = 0; r < 32; ++r) {
                const long long from = row_at(r);
                if (r < rows && lane < cols) cp_async4(buffer + place(r, lane), base + from + lane);
            }
        }
    }
    // the lane's values, zero where the tile has none
    static __device__ __forceinline__ void read(const float* buffer, int rows, int cols, float (&v)[32]) {
        const int lane = threadIdx.x & 31;
        if (kInner) {
#pragma unroll
            for (int r = 0; r < 32; ++r) v[r] = buffer[32 * r + lane];
        } else {
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
                const float4 f = *reinterpret_cast<const float4*>(buffer + place(lane, c));
                v[c] = f.x; v[c + 1] = f.y; v[c + 2] = f.z; v[c + 3] = f.w;
            }
        }
        const int good = kInner ? (lane < cols ? rows : 0) : (lane < rows ? cols : 0);
        if (good < 32)
#pragma unroll
            for (int e = 0; e < 32; ++e) v[e] = e < good ? v[e] : 0.f;
    }
};
// Arrives when the thread's copies so far have.
__device__ __forceinline__ void gs_arrive_behind_copies(unsigned long long* bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// NaN into a warp's part of a tile, 32 rows of 64 columns.
template <int kMode>
__device__ __forceinline__ void gs_lose(const GsPass& p, const GsWork& w, int row0, int col0) {
    const GsDegree& d = p.degree[w.degree];
    const int cols = min(col0 + 64, d.N - 128 * w.block);
    for (int i = row0; i < min(row0 + 32, w.rows); ++i) {
        float* to = w.out + static_cast<long long>(i) * d.N;
        if (kMode != kGsGradient) {
            int pair, comp;
            gs_row(w, d.comps, i, pair, comp);
            to = p.out + pair * p.out_stride + d.b_off + static_cast<long long>(comp) * d.N + 128 * w.block;
        }
        for (int c = col0 + (threadIdx.x & 31); c < cols; c += 32) to[c] = NAN;
    }
}

// hi of 11 bits, rounded; lo cut to 11 bits: the bits of its tail are the only loss, 2^-23 of the value at most. NaN stays NaN in one of the two, an
// infinity leaves a NaN in lo.
__device__ __forceinline__ void gs_split(float v, float& hi, float& lo) {
    hi = ts_round(v);
    lo = __uint_as_float(__float_as_uint(v - hi) & kTc5HiMask);
}

// Two by two blocks of eight values are turned between a lane and the one kLane on: the lower one gets both first blocks, the upper one both second ones.
template <int kLane>
__device__ __forceinline__ void gs_turn(float* first, float* second) {
    const bool upper = threadIdx.x & kLane;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float got = __shfl_xor_sync(0xffffffffu, upper ? first[e] : second[e], kLane);
        if (upper) first[e] = got;
        else second[e] = got;
    }
}

__device__ __forceinline__ void gs_meet() {
    __syncwarp();
    ts_fence_before();
    asm volatile("bar.sync 1, 1024;" ::: "memory");
}

// D of one step, its inner values 8 at a time. The remainders' products come first, while the sum is small: the tensor core cuts its sums, so an addition
// costs up to 2^-23 of the sum. Descriptors of one step ahead are 32 bytes on, two units of their address field; 32 inner values make a part of B.
__device__ __forceinline__ void gs_products(uint32_t d, uint32_t a_hi, uint32_t a_lo, uint32_t b, uint32_t idesc, int steps) {
    const uint64_t hi = tc5_smem_desc(b), lo = tc5_smem_desc(b + kGsHalfBytes);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (k >= steps) break;
        const int at = (k >> 2) * (kGsPartBytes >> 4) + (k & 3) * 2;
        ts_mma(d, a_lo + 8 * k, hi + at, idesc, k > 0);
        ts_mma(d, a_hi + 8 * k, lo + at, idesc, true);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        if (k >= steps) break;
        ts_mma(d, a_hi + 8 * k, hi + (k >> 2) * (kGsPartBytes >> 4) + (k & 3) * 2, idesc, true);
    }
}

// kWide: every row of a tile of the output starts on 32 bytes, and its columns are a multiple of eight.
template <bool kWide>
struct GsLayout {
    static constexpr int raw_a = kWide ? 2 : 1;                                                            // tiles that an A warp's rows have room for
    static constexpr int raw_at = kGsStages * kGsStageBytes, tile_floats = 32 * 32;
    static constexpr int out_at = raw_at + 8 * (raw_a + 1) * tile_floats * 4;
    static constexpr int bytes = out_at + (kWide ? 0 : 8 * 32 * kGsOutPitch * 4);
    static constexpr int largest = 227 * 1024 - 2048 - bytes;                                              // what the kernel's own arrays may take, with the alignment
    static_assert(largest >= 1024, "shared memory of one CTA per SM");
};

// One persistent CTA per SM walks its share of the tiles, 64 inner values a step; its warps are specialised, so that the parts of neighbouring tiles overlap:
//   warp 0        the products (one thread)
//   warp 1        finds the tiles (a ring, ahead of all others)
//   warps 2, 3    zeros into the rows behind the last group
//   warps 4-11    A, 32 rows of 32 inner values a warp, split and stored to tensor memory
//   warps 12-19   a thread adds half of its row's partial sums of every step in registers (the tensor core cuts its sums instead of rounding them: one
//                 sum over 128 inner values is off five times as far as float32) and writes its half of the row
//   warps 20-27   B, 32 columns of 32 inner values a warp, split and stored to shared memory; where a matrix has up to 128 inner values it stays for all
//                 row tiles of its group
//   warps 28-31   copies for both: a copy takes the time that memory needs for it to be issued (200 to 300 cycles for 512 bytes), and operand warps
//                 that issued their own waited for that 2,000 to 2,900 of 4,300 cycles a step
// TMEM: two stages of a partial sum of 128 columns and 128 of A (hi, lo), taken in turn. A hand-over costs its warps some hundred cycles: with steps of
// 32 inner values and half the warps for A and B the products waited two thirds of the time (98,304 atoms of 89 elements 127 us).
// 98,304 atoms of 89 elements, scalars and vectors, 128 x 128 (414 MB): 92 us, 4.5 TB/s, 140 TFLOP/s. 8,001 atoms in two slots behind the tensor product, 21 GFLOP each:
// forward 154 us, the rows' gradient 127, the matrices' 155 with their joins (166 to 136 TFLOP/s; three tf32 products of them could reach 272). A step takes some 4,000 cycles, 1,536
// of them the products': its warps issue in 53 to 57 % of the cycles (splitting, copies and sums, some 300 instructions a warp and step), the data pipe of shared memory
// is 41 % busy beside the reads of the products, and each of the five hand-overs between warps costs some hundred cycles. A step takes as long where B stays (44 an SM in the 92 us)
// as where it is copied and split every time (68 in the 154), so what bounds it is the loop over a stage of tensor memory: A is stored behind its last products, and the products wait for
// all sixteen warps of A and of the sums.
// Every wait is bounded; if one runs out, the CTA gives up, fills its remaining tiles with NaN, reports it to `status` and ends when its products
// and copies in flight have.
template <int kMode, bool kWide>
__global__ void __launch_bounds__(kGsThreads, 1) grouped_f32_kernel(const __grid_constant__ GsPass pass) {
    using L = GsLayout<kWide>;
    constexpr bool kRows = kMode != kGsGradient;
    constexpr int kRawA = L::raw_a;
    extern __shared__ unsigned char gs_smem_raw[];
    // ready: a stage of A is there and its partial sum has been read; done: its products are; raw_*: tiles of the operand warps, A's first
    __shared__ __align__(8) unsigned long long work_full[kGsRing], work_free[kGsRing], ready[kGsStages], done[kGsStages], b_full[kGsStages], b_free[kGsStages],
        raw_full[8 * (kRawA + 1)], raw_free[8 * (kRawA + 1)];
    __shared__ GsWork work[kGsRing];
    __shared__ uint32_t tmem_slot;
    __shared__ int guard[2];                                                             // a wait ran out; polls of a wait
    const int warp = ts_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    unsigned char* const stages = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(gs_smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
    float* const raw = reinterpret_cast<float*>(stages + L::raw_at);
    if (threadIdx.x == 0) {
        guard[0] = 0;
        guard[1] = pass.expire_polls > 0 ? pass.expire_polls : static_cast<int>(kMbarSpinLimit);
        for (int q = 0; q < kGsRing; ++q) { mbar_init(&work_full[q], 1); mbar_init(&work_free[q], 29); }
        for (int q = 0; q < kGsStages; ++q) { mbar_init(&ready[q], 16); mbar_init(&done[q], 1); mbar_init(&b_full[q], 8); mbar_init(&b_free[q], 1); }
        for (int q = 0; q < 8 * (kRawA + 1); ++q) { mbar_init(&raw_full[q], 32); mbar_init(&raw_free[q], 1); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    // The gradient reads nothing that the rows' pass before it writes: its CTAs come in as that one's end.
    if (kMode == kGsBackward) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    ts_fence_before();
    __syncthreads();
    ts_fence_after();
    const uint32_t tmem = tmem_slot, a_at = tmem + 256;

    if (warp < 4) {
        ts_registers_less<kGsRegsControl>();
        if (warp == 0) {
            int na = 0, nb = 0, base_b = 0, freed = 0;               // stages of A (and partial sums) and of B used so far; B's first one of the tile; those given back
            bool ok = true;
            const bool leader = ts_elect();
            const uint32_t b_at = smem_u32(stages);
            for (int i = 0; ok; ++i) {
                const int slot = i % kGsRing;
                ok = ts_wait_warp(&work_full[slot], (i / kGsRing) & 1, guard);
                if (!ok) break;
                const GsWork& w = work[slot];
                const int found = ts_uniform(w.found), chunks = ts_uniform(w.chunks), fresh = ts_uniform(w.fresh), last = ts_uniform(w.last), inner = ts_uniform(w.inner);
                const int cols = found ? ts_uniform(min(128, (pass.degree[w.degree].N - 128 * w.block + 15) & ~15)) : 0;
                __syncwarp();
                if (leader) mbar_arrive(&work_free[slot]);
                if (!found) break;
                if (fresh) { base_b = nb; nb += chunks; }
#pragma unroll 1
                for (int j = 0; j < chunks; ++j, ++na) {
                    const int st = na % kGsStages, n = base_b + j, bs = n % kGsStages;
                    ok = ts_wait_warp(&ready[st], (na / kGsStages) & 1, guard);
                    if (fresh) ok = ok && ts_wait_warp(&b_full[bs], (n / kGsStages) & 1, guard);
                    if (!ok) break;
                    ts_fence_after();
                    const uint32_t hi = ts_uniform(a_at + 128 * st), b = ts_uniform(b_at + bs * kGsStageBytes), d = ts_uniform(tmem + 128 * st);
                    if (leader) {
                        gs_products(d, hi, hi + 64, b, ts_idesc(cols), min(8, (inner - kGsChunk * j + 7) / 8));
                        if (last) ts_commit(&b_free[bs]);
                        ts_commit(&done[st]);
                    }
                    __syncwarp();
                    if (last) freed = n + 1;
                }
            }
            // What was started ends, and what it arrives at is told, before the CTA ends: products read its shared and tensor memory, and nobody else waits for the last
            // stages of B.
            for (int q = max(0, na - kGsStages); q < na; ++q) mbar_wait(&done[q % kGsStages], (q / kGsStages) & 1);
            for (int q = max(0, freed - kGsStages); q < freed; ++q) mbar_wait(&b_free[q % kGsStages], (q / kGsStages) & 1);
        } else if (warp == 1) {
            GsCursor cursor;
            int begin, end, i = 0, last_degree = -1, last_group = 0, last_block = 0;
            gs_share<kMode>(pass, begin, end);
            bool ok = true;
            for (int q = 0; q <= pass.degrees && ok; ++q) {
                const int t0 = q < pass.degrees ? __shfl_sync(0xffffffffu, begin, q) : 0, t1 = q < pass.degrees ? __shfl_sync(0xffffffffu, end, q) : 1;
                for (int t = t0; t < t1 && ok; ++t, ++i) {
                    const int slot = i % kGsRing;
                    GsWork w{};
                    if (q < pass.degrees) {
                        cursor.find<kMode>(pass, q, t, w);
                        if (gs_resident<kMode>(pass.degree[q])) {
                            w.fresh = w.degree != last_degree || w.group != last_group || w.block != last_block;
                            w.last = w.last || t + 1 == t1;
                        }
                        last_degree = w.degree; last_group = w.group; last_block = w.block;
                    }
                    if (i >= kGsRing && !ts_wait_warp(&work_free[slot], (i / kGsRing - 1) & 1, guard)) { ok = false; break; }
                    if (lane == 0) work[slot] = w;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&work_full[slot]);
                }
            }
        } else if (kRows && pass.zero_tail) {
            for (long long p = pass.offsets[pass.groups] + 2LL * blockIdx.x + (warp - 2); p < pass.rows; p += 2LL * gridDim.x)
                for (long long c = lane; c < pass.out_width; c += 32) pass.out[p * pass.out_stride + c] = 0.f;
        }
        gs_meet();
        if (guard[0] && threadIdx.x == 0 && pass.status) atomicMax(pass.status, kGsStatusWait);
    } else if (warp < 12) {
        ts_registers_less<kGsRegsOperand>();
        const uint32_t lanes = a_at + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int tid = threadIdx.x & 127, first = tid & ~31, k_part = 32 * ((warp - 4) >> 2);   // the warp's rows and inner values are its own
        int na = 0;
        bool ok = true;
        auto free_stage = [&]() { return na < kGsStages || ts_wait_warp(&done[na % kGsStages], (na / kGsStages - 1) & 1, guard); };
        auto give = [&]() {
            ts_wait_store();
            ts_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ready[na % kGsStages]);
            ++na;
        };
        auto put16 = [&](int q, float (&v)[16]) {
            float hi[16];
            const uint32_t to = lanes + 128 * (na % kGsStages) + k_part + q;
#pragma unroll
            for (int e = 0; e < 16; ++e) { float lo; gs_split(v[e], hi[e], lo); v[e] = lo; }
            ts_store16(to, hi);
            ts_store16(to + 64, v);
        };
        const int mine = warp - 4;                                       // tiles mine, mine + 8
        for (int i = 0; ok; ++i) {
            const int slot = i % kGsRing;
            if (!ts_wait_warp(&work_full[slot], (i / kGsRing) & 1, guard)) break;
            const int found = work[slot].found, chunks = work[slot].chunks, inner = work[slot].inner, owned = min(32, work[slot].rows - first);
            __syncwarp();
            if (lane == 0) mbar_arrive(&work_free[slot]);
            if (!found) break;
#pragma unroll 1
            for (int j = 0; j < chunks; ++j) {
                const int left = inner - j * kGsChunk - k_part, place = mine + 8 * (na % kRawA);
                if (!ts_wait_warp(&raw_full[place], (na / kRawA) & 1, guard)) { ok = false; break; }
                float v[32];
                if (kRows) GsTile<false>::read(raw + place * L::tile_floats, owned, left, v);
                else GsTile<true>::read(raw + place * L::tile_floats, left, owned, v);
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_free[place]);
                if (!free_stage()) { ok = false; break; }
                ts_fence_after();
#pragma unroll
                for (int q = 0; q < 32; q += 16) {
                    float part[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) part[e] = v[q + e];
                    put16(q, part);
                }
                give();
            }
        }
        gs_meet();
    } else if (warp >= 28) {
        ts_registers_less<kGsRegsCopies>();
        // Rows 32 q .. of A and columns 32 q .. of B, for the operand warps q and q + 4 of each.
        const int q = warp - 28, first = 32 * q;
        int na = 0, nb = 0;                                              // steps so far, and those with a B of their own
        bool ok = true;
        for (int i = 0; ok; ++i) {
            const int slot = i % kGsRing;
            if (!ts_wait_warp(&work_full[slot], (i / kGsRing) & 1, guard)) break;
            const GsWork& w = work[slot];
            const int found = w.found, chunks = w.chunks, inner = w.inner, degree = w.degree, fresh = w.fresh;
            const int owned_a = min(32, w.rows - first);
            int comp = 0, pair = 0, owned_b = 0;
            const float *a_base = nullptr, *b_base = nullptr;
            long long mine = 0;                                          // rows passes: where the lane's row of A begins
            if (found) {
                const GsDegree& d = pass.degree[degree];
                owned_b = min(32, d.N - 128 * w.block - first);
                gs_row(w, d.comps, kRows ? first + lane : lane, pair, comp);
                const float* matrix = d.w + static_cast<long long>(w.group) * d.K * d.N;
                if (kRows) {
                    mine = pair * pass.a_stride + static_cast<long long>(comp) * d.K;
                    a_base = pass.a + d.a_off;
                    b_base = kMode == kGsForward ? matrix + 128 * w.block + first : matrix + static_cast<long long>(128 * w.block + first) * d.K;
                } else {
                    a_base = pass.a + d.a_off + 128 * w.mtile + first;
                    b_base = pass.b + d.b_off + 128 * w.block + first;
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&work_free[slot]);
            if (!found) break;
            const GsDegree& d = pass.degree[degree];
            const bool wide_a = ((static_cast<unsigned long long>(pass.a_stride | d.a_off | d.K) * 4u | reinterpret_cast<uintptr_t>(pass.a)) & 15) == 0;
            const bool wide_b = kMode == kGsGradient ? ((static_cast<unsigned long long>(pass.b_stride | d.b_off | d.N) * 4u | reinterpret_cast<uintptr_t>(pass.b)) & 15) == 0
                                                     : ((static_cast<unsigned long long>(kMode == kGsForward ? d.N : d.K) * 4u | reinterpret_cast<uintptr_t>(d.w)) & 15) == 0;
            const int comps_more = 32 % d.comps, pairs_more = 32 / d.comps;
            auto shared_row = [&](long long v) { return [v](int r) { return __shfl_sync(0xffffffffu, v, r); }; };
            auto place_of = [&](int part, int n, int room) { return q + 4 * part + 8 * (n % room); };
#pragma unroll 1
            for (int j = 0; j < chunks && ok; ++j, ++na) {
#pragma unroll 1
                for (int part = 0; part < 2; ++part) {
                    const int k = j * kGsChunk + 32 * part, left = inner - k;
                    {
                        const int place = place_of(part, na, kRawA);
                        if (na >= kRawA && !ts_wait_warp(&raw_free[place], (na / kRawA - 1) & 1, guard)) { ok = false; break; }
                        float* const to = raw + place * L::tile_floats;
                        if constexpr (kRows) {
                            const auto row = shared_row(mine);
                            GsTile<false>::copy(to, a_base + k, owned_a, left, wide_a, [&](int u) { return row((lane >> 3) + 4 * u); }, row);
                        } else {
                            const auto row = shared_row(pair * pass.a_stride + static_cast<long long>(comp) * d.K);
                            GsTile<true>::copy(to, a_base, left, owned_a, wide_a, [&](int u) { return row((lane >> 3) + 4 * u); }, row);
                        }
                        gs_arrive_behind_copies(&raw_full[place]);
                    }
                    if (fresh) {
                        const int place = 8 * kRawA + q + 4 * part;
                        if (nb > 0 && !ts_wait_warp(&raw_free[place], (nb - 1) & 1, guard)) { ok = false; break; }
                        float* const to = raw + place * L::tile_floats;
                        if constexpr (kMode == kGsForward) {
                            const long long step = d.N;
                            GsTile<true>::copy(to, b_base + k * step, left, owned_b, wide_b, [&](int u) { return ((lane >> 3) + 4 * u) * step; }, [&](int r) { return r * step; });
                        } else if constexpr (kMode == kGsBackward) {
                            const long long step = d.K;
                            GsTile<false>::copy(to, b_base + k, owned_b, left, wide_b, [&](int u) { return ((lane >> 3) + 4 * u) * step; }, [&](int r) { return r * step; });
                        } else {
                            const auto row = shared_row(pair * pass.b_stride + static_cast<long long>(comp) * d.N);
                            GsTile<true>::copy(to, b_base, left, owned_b, wide_b, [&](int u) { return row((lane >> 3) + 4 * u); }, row);
                        }
                        gs_arrive_behind_copies(&raw_full[place]);
                    }
                    if (!kRows) {
                        comp += comps_more; pair += pairs_more;
                        if (comp >= d.comps) { comp -= d.comps; ++pair; }
                    }
                }
                if (fresh) ++nb;
            }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");                 // none may be in flight when the CTA ends
        gs_meet();
    } else if (warp >= 20) {
        ts_registers_less<kGsRegsOperand>();
        const int first = 32 * (warp & 3), part = (warp - 20) >> 2, k_part = 32 * part;          // the warp's columns and inner values are its own
        const int place = 8 * kRawA + warp - 20;
        int nb = 0;
        bool ok = true;
        for (int i = 0; ok; ++i) {
            const int slot = i % kGsRing;
            if (!ts_wait_warp(&work_full[slot], (i / kGsRing) & 1, guard)) break;
            const GsWork& w = work[slot];
            const int found = w.found, chunks = w.fresh ? w.chunks : 0, inner = w.inner;
            const int left = found ? min(128, pass.degree[w.degree].N - 128 * w.block) : 0, cols = ((left + 15) & ~15) - first, owned = min(32, left - first);
            __syncwarp();
            if (lane == 0) mbar_arrive(&work_free[slot]);
            if (!found) break;
#pragma unroll 1
            for (int j = 0; j < chunks; ++j) {
                const int good = inner - j * kGsChunk - k_part;
                if (!ts_wait_warp(&raw_full[place], nb & 1, guard)) { ok = false; break; }
                float v[32];
                if (kMode == kGsBackward) GsTile<false>::read(raw + place * L::tile_floats, owned, good, v);
                else GsTile<true>::read(raw + place * L::tile_floats, good, owned, v);
                __syncwarp();
                if (lane == 0) mbar_arrive(&raw_free[place]);
                const int bs = nb % kGsStages;
                if (pass.expire_polls > 0 && nb > 0) { ok = false; break; }
                if (nb >= kGsStages && !ts_wait_warp(&b_free[bs], (nb / kGsStages - 1) & 1, guard)) { ok = false; break; }
                unsigned char* const to = stages + bs * kGsStageBytes + part * kGsPartBytes;
                if (lane < cols) {
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        float4 hi, lo;
                        gs_split(v[4 * c], hi.x, lo.x);
                        gs_split(v[4 * c + 1], hi.y, lo.y);
                        gs_split(v[4 * c + 2], hi.z, lo.z);
                        gs_split(v[4 * c + 3], hi.w, lo.w);
                        const int off = tc5_swizzled_group(first + lane, c);
                        *reinterpret_cast<float4*>(to + off) = hi;
                        *reinterpret_cast<float4*>(to + kGsHalfBytes + off) = lo;
                    }
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&b_full[bs]);
                ++nb;
            }
        }
        gs_meet();
    } else {
        ts_registers_more<kGsRegsSums>();
        const uint32_t lanes = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const int tid = threadIdx.x & 127, half = (warp - 12) >> 2;
        float* const out_stage = reinterpret_cast<float*>(stages + L::out_at) + (warp - 12) * 32 * kGsOutPitch;
        int nd = 0, at_degree = 0, at_tile = 0;      // the tile at hand, for a CTA that gives up (0, 0: none yet)
        if (lane < kGsStages) mbar_arrive(&ready[lane]);                 // the first two sums have nothing to wait for
        bool ok = true;
        for (int i = 0;; ++i) {
            const int slot = i % kGsRing;
            ok = ts_wait_warp(&work_full[slot], (i / kGsRing) & 1, guard);
            if (!ok) break;
            const int found = work[slot].found, chunks = work[slot].chunks, rows = work[slot].rows;
            float* out_row = nullptr;
            int left = 0;
            if (found) {
                const GsWork& w = work[slot];
                const GsDegree& d = pass.degree[w.degree];
                at_degree = w.degree; at_tile = w.tile;
                left = d.N - 128 * w.block - 64 * half;                  // columns of this half that exist
                if (tid < rows) {
                    if (kRows) {
                        int pair, comp;
                        gs_row(w, d.comps, tid, pair, comp);
                        out_row = pass.out + pair * pass.out_stride + d.b_off + static_cast<long long>(comp) * d.N + 128 * w.block + 64 * half;
                    } else {
                        out_row = w.out + static_cast<long long>(tid) * d.N + 64 * half;
                    }
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&work_free[slot]);
            if (!found) break;
            float sum[64];
#pragma unroll
            for (int q = 0; q < 64; ++q) sum[q] = 0.f;
            for (int j = 0; j < chunks; ++j, ++nd) {
                if (!ts_wait_warp(&done[nd & 1], (nd >> 1) & 1, guard)) { ok = false; break; }
                ts_fence_after();
                const uint32_t from = lanes + (nd & 1) * 128 + 64 * half;
#pragma unroll
                for (int c = 0; c < 64; c += 16)
                    if (c < left) {                                      // what a last, odd block holds behind the columns is never written
                        float v[16];
                        ts_load16(from + c, v);
#pragma unroll
                        for (int q = 0; q < 16; ++q) sum[c + q] += v[q];
                    }
                ts_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&ready[nd & 1]);                  // for the step after the next one
            }
            if (!ok) break;
            if (kWide) {
                // Four lanes share out their rows' lines, so that a store touches eight lines instead of 32.
                const unsigned long long mine = reinterpret_cast<unsigned long long>(out_row);
                float* rows_of[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) rows_of[i] = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, mine, (lane & ~3) + i)) + 8 * (lane & 3);
                const unsigned there = __ballot_sync(0xffffffffu, mine != 0) >> (lane & ~3);
#pragma unroll
                for (int c = 0; c < 64; c += 32)
                    if (c < left) {
                        gs_turn<1>(sum + c, sum + c + 8);
                        gs_turn<1>(sum + c + 16, sum + c + 24);
                        gs_turn<2>(sum + c, sum + c + 16);
                        gs_turn<2>(sum + c + 8, sum + c + 24);
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float* v = sum + c + 8 * i;
                            if (((there >> i) & 1u) && c + 8 * (lane & 3) < left)
                                asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(rows_of[i] + c), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                                             "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]) : "memory");
                        }
                    }
            } else {
                // 16 columns of the warp's rows at a time through shared memory, so that a store touches two rows instead of 32
                const unsigned long long mine = reinterpret_cast<unsigned long long>(out_row);
#pragma unroll
                for (int c0 = 0; c0 < 64; c0 += 16) {
                    if (c0 >= left) continue;
                    __syncwarp();
#pragma unroll
                    for (int q = 0; q < 16; ++q) out_stage[lane * kGsOutPitch + q] = sum[c0 + q];
                    __syncwarp();
                    const int c = c0 + (lane & 15);
#pragma unroll 4
                    for (int r = lane >> 4; r < 32; r += 2) {
                        float* to = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, mine, r));
                        if (to && c < left) to[c] = out_stage[r * kGsOutPitch + (c - c0)];
                    }
                }
                __syncwarp();
            }
        }
        if (!ok) {
            // NaN into the warp's part of the tile at hand and of all that would have followed
            GsCursor cursor;
            GsWork lost{};
            int begin, end;
            gs_share<kMode>(pass, begin, end);
            for (int q = 0; q < pass.degrees; ++q) {
                const int t0 = __shfl_sync(0xffffffffu, begin, q), t1 = __shfl_sync(0xffffffffu, end, q);
                for (int t = t0; t < t1; ++t)
                    if ((q > at_degree || (q == at_degree && t >= at_tile)) && cursor.find<kMode>(pass, q, t, lost))
                        gs_lose<kMode>(pass, lost, tid & ~31, 64 * half);
            }
        }
        gs_meet();
    }
    __syncthreads();
    // (one CTA waits for that pass, so that this kernel does not end before it)
    if (kMode == kGsGradient && blockIdx.x == 0) asm volatile("griddepcontrol.wait;" ::: "memory");
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace
}  // namespace smx
