// Products of a few rows with matrices of 4-bit weights, one scale (and zero point) per group of input columns: the
// experts' products of a decode batch (declared in include/moe_fp8_b200.h).
//
//   y[r, n] = sum over k of (code[n, k] - zero[n, k / G]) * scale[n, k / G] * x[r, k]
//
// What bounds it is the stream of the codes out of HBM: a weight is half a byte and meets at most eight rows per read.
// The codes are read in the operator's own layout, two per byte, row by row.  One persistent CTA per SM takes a contiguous
// range of 16-row weight tiles and keeps the next ones on their way into a ring of shared-memory stages (one TMA box per
// tile, requested as soon as all warps have read the stage that it replaces); sixteen warps split a tile's K range and
// multiply with mma.sync (m16n8k16: the weights are the 16-row operand, up to eight rows of x the other one).  tcgen05 has nothing to give here: its M of 128
// would need a dequantised copy of the weights in shared memory or TMEM, and the tensor pipe is far from busy.
//
// The order of K inside a tile is free as long as both operands agree.  A thread's 32-bit word of codes holds the
// columns 8t .. 8t+7 of a 32-column block (t = lane % 4), and the pairs (0,4) (1,5) (2,6) (3,7) fall out of it with a shift
// and a mask each; x is held in registers in that order, loaded once per run of tiles of one expert.
// code - zero is exact in bf16 and fp16; the products are summed in fp32, scaled per 32 columns in fp32, and rounded once.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "call_checks.cuh"
#include "ptx.cuh"

namespace moe {
int encode_tensor_map(void* out_map, const void* base, bool bytes, int rank, const uint64_t* dims, const uint64_t* strides,
                      const uint32_t* box, bool swizzled);

namespace {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kLoadWarp = kWarps - 1;         // also requests the stages
constexpr int kTileRows = 16;                 // weight rows of a tile
constexpr int kRowsOfX = 8;                   // rows of x that share a read of the weights
constexpr int kMaxBlocks = 16;                // 32-column blocks of a warp
constexpr int kMaxK = 8192;
constexpr int kMaxStages = 8;
constexpr uint32_t kSwizzleAtom = 1024;        // what the swizzle repeats after
constexpr int kMaxExperts = MOE_FP8_B200_PLAN_MAX_EXPERTS;
constexpr int kChunkTiles = 8;                // see Run
constexpr size_t kSharedLimit = 227 * 1024;

struct MatvecArgs {
    const uint8_t* x;
    long long x_stride;        // bytes
    int x_rows, x_wide;        // rows that exist; 16-byte loads allowed
    int by_token, top_k;       // x has a row per token: that of row r is row_pair[r] / top_k
    const uint8_t* scales;     // 16-bit
    const uint8_t* zeros;      // or null: 8
    uint8_t* out;
    long long out_stride;
    int E, N, K, group_shift;  // group = 32 << group_shift columns
    const int *expert_offset, *expert_count, *row_pair;   // null: one matrix, `rows` rows
    int rows;                  // rows of out
    int split, stages;         // warps that share a tile; ring
    // A stage: the codes of its tiles, then their scales, then their zero points.  A tile's codes are `chunks` pieces of 128
    // bytes (256 columns) of its sixteen rows, in the 128-byte swizzle (16-byte unit index XOR row mod 8).
    int chunks, whole;             // whole: a row is a multiple of 128 bytes, one box takes a tile
    int scale_bytes, zero_bytes;   // pitch of a row's scales and zero points
    int scale_box, zero_box;       // they come as boxes, else (rows of no multiple of 16 bytes) as they lie
    int scale_at, zero_at, stage_bytes;
};

// The weights as TMA sees them: gated ones as two halves of n / 2 rows, of which a tile takes the same eight.
struct alignas(64) MatvecMaps {
    CUtensorMap codes, scales, zeros;
};

// Tiles of weights that meet the same rows of x one after the other.
struct Run {
    int expert, x_tile, tile, count;
};

struct Shared {
    int abort;
    int warp_sum[32];
    int first[kMaxExperts + 1];   // tiles of x rows in front of expert e
    alignas(8) uint64_t full_bar[kMaxStages];
    long long load_unit;          // what the load warp requests next: tiles load_done .. of the run, then this unit on
    Run load_run;
    int load_done;
    alignas(16) float part[2][kWarps][128];
};


// Work is laid out expert by expert.  An expert with more than eight rows meets its weights once per eight of them, in
// chunks of kChunkTiles tiles, so that the second read of a chunk finds it in L2 (148 CTAs x 8 tiles x 57 KB = 68 MB).
__device__ __forceinline__ Run run_at(const Shared& sh, const MatvecArgs& a, long long unit, long long end, int tiles)
{
    const int at = (int)(unit / tiles);
    int lo = 0, hi = a.E - 1;   // last expert with first[e] <= at
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if (sh.first[mid] <= at) lo = mid; else hi = mid - 1;
    }
    const int x_tiles = sh.first[lo + 1] - sh.first[lo];
    const long long within = unit - (long long)sh.first[lo] * tiles;
    const int chunk_tiles = x_tiles == 1 ? tiles : kChunkTiles;
    const long long chunk_units = (long long)chunk_tiles * x_tiles;
    const int chunk = (int)(within / chunk_units), rem = (int)(within - chunk * chunk_units);
    const int here = min(chunk_tiles, tiles - chunk * chunk_tiles);
    Run r;
    r.expert = lo;
    r.x_tile = rem / here;
    r.tile = chunk * chunk_tiles + rem % here;
    r.count = (int)min((long long)(here - rem % here), end - unit);
    return r;
}

__device__ __forceinline__ void box_load_5d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int row, int half, int chunk,
                                            int expert) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6, %7}], "
                 "[%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(row), "r"(half), "r"(chunk), "r"(expert)
                 : "memory");
}
__device__ __forceinline__ void box_load_4d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int row, int half,
                                            int expert) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(row), "r"(half), "r"(expert)
                 : "memory");
}
// (a & mask) | b in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t mask, uint32_t b) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(d) : "r"(a), "r"(mask), "r"(b));
    return d;
}
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

template <typename T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
    static __device__ __forceinline__ void mma(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    }
    // two equal values 128 + zero
    static __device__ __forceinline__ uint32_t offset(uint32_t zero) { return 0x43004300u + zero * 0x00010001u; }
    // Codes (0,4) (1,5) (2,6) (3,7) of a word minus the zero point: 0x4300 | code is 128 + code, exactly.
    static __device__ __forceinline__ void decode(uint32_t w, uint32_t off, uint32_t (&q)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = and_or(w >> (4 * i), 0x000f000fu, 0x43004300u);
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(q[i]) : "r"(v), "r"(off));
        }
    }
    static __device__ __forceinline__ float scale(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }
    static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Half2<__half> {
    static __device__ __forceinline__ void mma(float (&d)[4], const float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                               uint32_t a3, uint32_t b0, uint32_t b1) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%10, %11, %12, %13};"
            : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
    }
    // two equal values 1024 + zero
    static __device__ __forceinline__ uint32_t offset(uint32_t zero) { return 0x64006400u + zero * 0x00010001u; }
    // 0x6400 | code is 1024 + code, exactly; with the code four bits higher it is 1024 + 16 code, of which 1/16 is 64 + code.
    static __device__ __forceinline__ void decode(uint32_t w, uint32_t off, uint32_t (&q)[4]) {
        uint32_t neg;   // -(64 + zero)
        asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(neg) : "r"(0x63806380u), "r"(off));   // 960 - (1024 + zero)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t s = w >> (8 * i);
            const uint32_t lo = and_or(s, 0x000f000fu, 0x64006400u), hi = and_or(s, 0x00f000f0u, 0x64006400u);
            asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(q[2 * i]) : "r"(lo), "r"(off));
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(q[2 * i + 1]) : "r"(hi), "r"(0x2c002c00u), "r"(neg));
        }
    }
    static __device__ __forceinline__ float scale(uint16_t bits) { return __half2float(__ushort_as_half(bits)); }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};

// A thread's part of a tile in shared memory (bytes into the ring).  A warp takes every split-th pair of 32-column blocks,
// so that its pairs lie at one distance: split / 4 chunks.
struct TileView {
    const uint8_t* ring;
    int even, odd;     // its word of the first pair's two blocks in weight row g; row g + 8 lies 1024 bytes further
    int scales, zeros; // its row's scale and zero point of the first pair; row g + 8's lie scale_rows, zero_rows further
    int scale_rows, zero_rows;
    int pair_step, scale_step, zero_step;
    int last_scale, last_zero;   // of the row: a pair's second block may lie behind the last column, where x is zero
};

// COUNT pairs of blocks from pair FIRST on, in one stretch without a branch, so that their loads, conversions and matrix
// instructions overlap.  The products of a pair are summed in fp32 by the matrix instructions, one scale at a time
// (FINE: two scales in a pair).
template <typename H, bool FINE, bool ZEROS, int FIRST, int COUNT, int BLOCKS>
__device__ __forceinline__ void multiply_pairs(float (&acc)[4], const uint32_t (&xr)[BLOCKS][4], const TileView& v)
{
    constexpr int kScales = FINE ? 2 : 1, kBlocks = 2 / kScales;   // scales of a pair, blocks of a scale
    uint32_t w0[2 * COUNT], w1[2 * COUNT];
#pragma unroll
    for (int p = 0; p < COUNT; ++p) {
        const int at = (FIRST + p) * v.pair_step;
        w0[2 * p] = *reinterpret_cast<const uint32_t*>(v.ring + v.even + at);
        w1[2 * p] = *reinterpret_cast<const uint32_t*>(v.ring + v.even + at + 1024);
        w0[2 * p + 1] = *reinterpret_cast<const uint32_t*>(v.ring + v.odd + at);
        w1[2 * p + 1] = *reinterpret_cast<const uint32_t*>(v.ring + v.odd + at + 1024);
    }
#pragma unroll
    for (int p = 0; p < COUNT; ++p)
#pragma unroll
        for (int i = 0; i < kScales; ++i) {
            int sa = v.scales + (FIRST + p) * v.scale_step, za = v.zeros + (FIRST + p) * v.zero_step;
            if (i) {
                sa = min(sa + 2, v.last_scale);
                za = min(za + 1, v.last_zero);
            }
            const float s0 = H::scale(*reinterpret_cast<const uint16_t*>(v.ring + sa));
            const float s1 = H::scale(*reinterpret_cast<const uint16_t*>(v.ring + sa + v.scale_rows));
            const uint32_t off0 = H::offset(ZEROS ? v.ring[za] : 8u), off1 = H::offset(ZEROS ? v.ring[za + v.zero_rows] : 8u);
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int j = 2 * p + i * kBlocks; j < 2 * p + (i + 1) * kBlocks; ++j) {
                uint32_t q0[4], q1[4];
                H::decode(w0[j], off0, q0);
                H::decode(w1[j], off1, q1);
                H::mma(c, c, q0[0], q1[0], q0[1], q1[1], xr[2 * FIRST + j][0], xr[2 * FIRST + j][1]);
                H::mma(c, c, q0[2], q1[2], q0[3], q1[3], xr[2 * FIRST + j][2], xr[2 * FIRST + j][3]);
            }
            acc[0] = fmaf(s0, c[0], acc[0]);
            acc[1] = fmaf(s0, c[1], acc[1]);
            acc[2] = fmaf(s1, c[2], acc[2]);
            acc[3] = fmaf(s1, c[3], acc[3]);
        }
}

template <typename H, bool FINE, bool ZEROS, int FIRST, int BLOCKS>
__device__ __forceinline__ void multiply_from(float (&acc)[4], const uint32_t (&xr)[BLOCKS][4], const TileView& v, int pairs)
{
    if constexpr (2 * FIRST < BLOCKS) {
        if (pairs >= FIRST + 2) {
            multiply_pairs<H, FINE, ZEROS, FIRST, 2>(acc, xr, v);
            multiply_from<H, FINE, ZEROS, FIRST + 2>(acc, xr, v, pairs);
        } else if (pairs > FIRST) {
            multiply_pairs<H, FINE, ZEROS, FIRST, 1>(acc, xr, v);
        }
    }
}

template <typename T, bool GATED, bool FINE, bool ZEROS>
__global__ void __launch_bounds__(kThreads, 1) matvec4_kernel(const MatvecArgs a, const __grid_constant__ MatvecMaps maps)
{
    extern __shared__ uint8_t pool[];
    __shared__ Shared sh;
    typedef Half2<T> H;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint8_t* const ring = pool + (0u - smem_u32(pool)) % kSwizzleAtom;
    const uint32_t ring0 = smem_u32(ring);
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        sh.abort = 0;
        for (int i = 0; i < a.stages; ++i) mbar_init(smem_u32(&sh.full_bar[i]), 1);
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();

    // tiles of x rows per expert, summed up
    if (a.expert_count) {
        int run = 0;
        for (int e0 = 0; e0 < a.E; e0 += kThreads) {
            const int e = e0 + threadIdx.x;
            int n = 0;
            if (e < a.E) {
                const int off = a.expert_offset[e], count = a.expert_count[e];
                if (off >= 0 && count > 0 && off < a.rows) n = (min(count, a.rows - off) + kRowsOfX - 1) / kRowsOfX;
            }
            int upto = n;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(~0u, upto, d);
                if (lane >= d) upto += v;
            }
            if (lane == 31) sh.warp_sum[warp] = upto;
            __syncthreads();
            int total = 0;
            for (int w = 0; w < kWarps; ++w) {
                if (w < warp) upto += sh.warp_sum[w];
                total += sh.warp_sum[w];
            }
            if (e < a.E) sh.first[e] = run + upto - n;
            run += total;
            __syncthreads();
        }
        if (threadIdx.x == 0) sh.first[a.E] = run;
    } else if (threadIdx.x == 0) {
        sh.first[0] = 0;
        sh.first[1] = (a.rows + kRowsOfX - 1) / kRowsOfX;
    }
    __syncthreads();

    const int tiles = a.N / kTileRows, per_stage = kWarps / a.split, groups = a.K >> (5 + a.group_shift);
    const long long units = (long long)sh.first[a.E] * tiles;
    const long long begin = units * blockIdx.x / gridDim.x, end = units * (blockIdx.x + 1) / gridDim.x;

    // Requests one stage: one weight row per lane, then the scales and zero points.  Only the load warp calls it.
    auto request_stage = [&](int slot) {
        if (sh.load_done == sh.load_run.count) {
            const long long u = sh.load_unit;
            if (u >= end) return;
            const Run next = run_at(sh, a, u, end, tiles);
            __syncwarp();
            if (lane == 0) {
                sh.load_run = next;
                sh.load_unit = u + next.count;
                sh.load_done = 0;
            }
            __syncwarp();
        }
        const Run r = sh.load_run;
        const int t0 = sh.load_done, n = min(per_stage, r.count - t0);
        const uint32_t bar = smem_u32(&sh.full_bar[slot]), dst = ring0 + slot * a.stage_bytes;
        __syncwarp();
        if (lane == 0) {
            sh.load_done = t0 + n;
            const int codes = a.chunks * 128, scales = a.scale_box ? a.scale_bytes : groups * 2, zeros = a.zero_box ? a.zero_bytes : groups;
            mbar_expect_tx(bar, (uint32_t)(n * kTileRows) * (uint32_t)(codes + scales + (ZEROS ? zeros : 0)));
        }
        __syncwarp();
        const int rows = GATED ? kTileRows / 2 : kTileRows;
        // a tile's scales where they are no box: as they lie, in two halves if gated
        auto copy_side = [&](const uint8_t* src, int bytes, int tile, uint32_t to) {
            for (int half = 0; half < (GATED ? 2 : 1); ++half)
                bulk_load(to + half * rows * bytes, src + ((long long)r.expert * a.N + half * (a.N / 2) + tile * rows) * bytes,
                          rows * bytes, bar);
        };
        const int boxes = a.whole ? 1 : a.chunks;
        for (int i = lane; i < n * boxes; i += 32) {
            const int m = i / boxes, c = i - m * boxes;
            box_load_5d(dst + (m * a.chunks + c) * 2048, &maps.codes, bar, a.whole ? 0 : c * 128, (r.tile + t0 + m) * rows, 0, 0, r.expert);
        }
        for (int m = lane; m < n; m += 32) {
            const int tile = r.tile + t0 + m;
            const uint32_t to = dst + a.scale_at + m * kTileRows * a.scale_bytes;
            if (a.scale_box) box_load_4d(to, &maps.scales, bar, 0, tile * rows, 0, r.expert);
            else copy_side(a.scales, groups * 2, tile, to);
            if (ZEROS) {
                const uint32_t zero_to = dst + a.zero_at + m * kTileRows * a.zero_bytes;
                if (a.zero_box) box_load_4d(zero_to, &maps.zeros, bar, 0, tile * rows, 0, r.expert);
                else copy_side(a.zeros, groups, tile, zero_to);
            }
        }
    };
    if (warp == kLoadWarp) {
        if (lane == 0) {
            prefetch_tmap(&maps.codes);
            sh.load_unit = begin;
            sh.load_done = sh.load_run.count = 0;
        }
        __syncwarp();
        for (int i = 0; i < a.stages; ++i) request_stage(i);
    }

    // `split` warps share a tile's K range, tile m of the stage belongs to warps [m * split, (m + 1) * split)
    const int member = warp % a.split, of_stage = warp / a.split;
    // every split-th pair of 32-column blocks; the last pair of an odd number of blocks has its second block's x zero
    const int all_pairs = (a.K + 63) / 64, pairs = (all_pairs - member + a.split - 1) / a.split;
    const int g = lane / 4, t = lane % 4;
    TileView view;
    {
        const int unit = 2 * member % 8;   // 16-byte unit of the first pair's first block in its chunk
        const int row = of_stage * kTileRows + g, group = member * 2 >> a.group_shift;
        const int chunk = (of_stage * a.chunks + member / 4) * 2048 + g * 128 + 4 * t;
        view.ring = ring;
        view.even = chunk + ((unit ^ g) << 4);
        view.odd = chunk + (((unit + 1) ^ g) << 4);
        view.scales = a.scale_at + row * a.scale_bytes + 2 * group;
        view.zeros = a.zero_at + row * a.zero_bytes + group;
        view.scale_rows = 8 * a.scale_bytes;
        view.zero_rows = 8 * a.zero_bytes;
        view.pair_step = a.split * 512;
        view.zero_step = a.split * 2 >> a.group_shift;
        view.scale_step = 2 * view.zero_step;
        view.last_scale = a.scale_at + row * a.scale_bytes + 2 * (groups - 1);
        view.last_zero = a.zero_at + row * a.zero_bytes + groups - 1;
    }
    uint32_t xr[kMaxBlocks][4];
    int it = 0;
    bool ok = true;
    for (long long u = begin; u < end;) {
        const Run r = run_at(sh, a, u, end, tiles);
        u += r.count;
        // rows of x of this run, in the order the codes come out of a word
        const int row0 = (a.expert_count ? a.expert_offset[r.expert] : 0) + r.x_tile * kRowsOfX;
        const int rows = min(kRowsOfX, (a.expert_count ? min(a.expert_count[r.expert], a.rows - a.expert_offset[r.expert]) : a.rows) -
                                           r.x_tile * kRowsOfX);
        {
            int src = row0 + min(g, rows - 1);
            if (a.by_token) src = a.row_pair[src] / a.top_k;
            src = min(max(src, 0), a.x_rows - 1);
            const uint8_t* xp = a.x + src * a.x_stride + (member * 64 + 8 * t) * 2;
#pragma unroll
            for (int j = 0; j < kMaxBlocks; ++j) {
                uint32_t v[4] = {0, 0, 0, 0};
                const int block = 2 * (member + j / 2 * a.split) + j % 2, at = (block - 2 * member) * 64;
                if (block * 32 < a.K) {
                    if (a.x_wide) {
                        const uint4 q = *reinterpret_cast<const uint4*>(xp + at);
                        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
                    } else {
                        const uint16_t* h = reinterpret_cast<const uint16_t*>(xp + at);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
                    }
                }
                xr[j][0] = __byte_perm(v[0], v[2], 0x5410);   // (0, 4)
                xr[j][1] = __byte_perm(v[0], v[2], 0x7632);   // (1, 5)
                xr[j][2] = __byte_perm(v[1], v[3], 0x5410);   // (2, 6)
                xr[j][3] = __byte_perm(v[1], v[3], 0x7632);   // (3, 7)
            }
        }
        for (int t0 = 0; t0 < r.count; t0 += per_stage, ++it) {
            const int slot = it % a.stages, n = min(per_stage, r.count - t0);
            ok = mbar_wait(smem_u32(&sh.full_bar[slot]), (it / a.stages) & 1, &sh.abort) && ok;
            float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (of_stage < n && ok) {
                TileView v = view;
                const int stage = slot * a.stage_bytes;
                v.even += stage;
                v.odd += stage;
                v.scales += stage;
                v.zeros += stage;
                v.last_scale += stage;
                v.last_zero += stage;
                multiply_from<H, FINE, ZEROS, 0>(acc, xr, v, pairs);
            }
            // the tile's partial sums meet (two buffers, so one barrier per stage), and the stage has been read
            float(*part)[128] = sh.part[it & 1];
#pragma unroll
            for (int i = 0; i < 4; ++i) part[warp][i * 32 + lane] = acc[i];
            __syncthreads();
            if (warp == kLoadWarp && ok) request_stage(slot);
            // 128 results per tile, added up by the warps in turn: thread (i, lane) has row g + 8 (i / 2), x row 2t + i % 2
            const int first = (it * 4) % kWarps;
            for (int v = (warp + kWarps - first) % kWarps; v < n * 4; v += kWarps) {
                const int m = v / 4, i = v % 4;
                if (GATED && i >= 2) continue;
                float y = 0.0f, gate = 0.0f;
                for (int k = 0; k < a.split; ++k) {
                    y += part[m * a.split + k][i * 32 + lane];
                    if (GATED) gate += part[m * a.split + k][(i + 2) * 32 + lane];
                }
                const int xrow = 2 * t + (i & 1);
                if (xrow < rows) {
                    if (GATED) y = gate / (1.0f + __expf(-gate)) * y;
                    if (!ok) y = __int_as_float(0x7fc00000);   // a load that never came
                    const int tile = r.tile + t0 + m;
                    const int col = GATED ? tile * 8 + g : tile * kTileRows + g + 8 * (i / 2);
                    reinterpret_cast<T*>(a.out + (row0 + xrow) * a.out_stride)[col] = H::round(y);
                }
            }
        }
    }
}

}  // namespace
}  // namespace moe

using namespace moe;

namespace {

template <typename T, bool GATED, bool FINE, bool ZEROS>
cudaError_t launch_form(const MatvecArgs& a, const MatvecMaps& maps, int sms, cudaStream_t stream)
{
    const size_t smem = (size_t)a.stages * a.stage_bytes + kSwizzleAtom;
    const auto kernel = matvec4_kernel<T, GATED, FINE, ZEROS>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_after(kernel, dim3(sms), dim3(kThreads), smem, 1, stream, a, maps);
}

template <typename T, bool GATED>
cudaError_t launch_groups(const MatvecArgs& a, const MatvecMaps& maps, int sms, cudaStream_t stream)
{
    const bool zeros = a.zeros != nullptr;
    if (a.group_shift == 0)
        return zeros ? launch_form<T, GATED, true, true>(a, maps, sms, stream) : launch_form<T, GATED, true, false>(a, maps, sms, stream);
    return zeros ? launch_form<T, GATED, false, true>(a, maps, sms, stream) : launch_form<T, GATED, false, false>(a, maps, sms, stream);
}

template <typename T>
cudaError_t launch_matvec(const MatvecArgs& a, const MatvecMaps& maps, bool gated, int sms, cudaStream_t stream)
{
    return gated ? launch_groups<T, true>(a, maps, sms, stream) : launch_groups<T, false>(a, maps, sms, stream);
}

// A weight tensor [E, n, row_bytes] as boxes of a tile's sixteen rows (gated: eight of each half) and `box_bytes` of each;
// codes: in chunks of 128 bytes, all of a row's in one box if the row is a whole number of them.
int encode_weights(CUtensorMap& map, const void* base, const MatvecArgs& a, bool gated, int row_bytes, int box_bytes, bool codes)
{
    const uint64_t row = (uint64_t)row_bytes, half = (uint64_t)a.N / 2 * row, expert = (uint64_t)a.N * row;
    const uint64_t rows = gated ? a.N / 2 : a.N, halves = gated ? 2 : 1, E = (uint64_t)a.E;
    const uint32_t box_rows = gated ? 8 : 16, box_halves = gated ? 2 : 1;
    if (!codes) {   // scales, zero points: bytes or 16-bit values
        const int size = base == a.zeros ? 1 : 2;
        const uint64_t dims[4] = {row / size, rows, halves, E}, strides[3] = {row, half, expert};
        const uint32_t box[4] = {(uint32_t)(box_bytes / size), box_rows, box_halves, 1};
        return encode_tensor_map(&map, base, size == 1, 4, dims, strides, box, false);
    }
    const uint64_t dims[5] = {a.whole ? 128 : row, rows, halves, a.whole ? row / 128 : 1, E}, strides[4] = {row, half, 128, expert};
    const uint32_t box[5] = {128, box_rows, box_halves, a.whole ? (uint32_t)a.chunks : 1, 1};
    return encode_tensor_map(&map, base, true, 5, dims, strides, box, true);
}

}  // namespace

extern "C" int moe_fp8_b200_matvec_w4(const void* x, int64_t x_stride, int by_token, const moe_fp8_b200_w4* w, int gated, void* out,
                                      int64_t out_stride, int dtype, const moe_fp8_b200_plan* plan, int num_rows, void* stream,
                                      char* err, size_t err_len)
{
    auto bad = [&](auto... v) { return refuse(err, err_len, MOE_FP8_B200_ERR_INVALID_ARGUMENT, v...); };
    if (!w) return bad("w is NULL");
    if (dtype != MOE_FP8_B200_BF16 && dtype != MOE_FP8_B200_FP16) return bad("x must be bf16 or fp16, got row type %d", dtype);
    if (w->group != 32 && w->group != 64 && w->group != 128) return bad("group must be 32, 64 or 128, got %d", w->group);
    if (w->k < w->group || w->k > kMaxK || w->k % w->group)
        return bad("k must be a multiple of the group of %d in [%d, %d], got %d", w->group, w->group, kMaxK, w->k);
    if (w->n < kTileRows || w->n > (1 << 20) || w->n % kTileRows) return bad("n must be a multiple of 16 in [16, 2^20], got %d", w->n);
    const int groups = w->k / w->group;
    if (gated && w->zeros && groups % 2) return bad("gated weights with zero points need an even number of groups, got %d", groups);
    if (w->num_experts < 1 || w->num_experts > kMaxExperts) return bad("num_experts %d is not in 1 .. %d", w->num_experts, kMaxExperts);
    int64_t rows = num_rows;
    if (plan) {
        if (plan->num_experts != w->num_experts)
            return bad("the plan has %d experts, the weights %d", plan->num_experts, w->num_experts);
        rows = moe_fp8_b200_plan_rows(plan->num_tokens, plan->top_k, plan->num_experts, plan->align);
        if (rows < 0) return bad("plan sizes out of range");
    } else if (w->num_experts != 1 || by_token) {
        return bad("weights of several experts and rows by token need a plan");
    }
    if (rows < 0) return bad("num_rows %d < 0", num_rows);
    if (rows == 0) return MOE_FP8_B200_OK;
    int dev = 0, sms = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e != cudaSuccess) return refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "current device: %s", cudaGetErrorString(e));
    struct { const char* name; const void* p; size_t align; bool wanted; } tensors[] = {
        {"x", x, 2, true}, {"codes", w->codes, 16, true}, {"scales", w->scales, 16, true}, {"zeros", w->zeros, 16, w->zeros != nullptr},
        {"out", out, 2, true}, {"expert_offset", plan ? plan->expert_offset : nullptr, 4, plan != nullptr},
        {"expert_count", plan ? plan->expert_count : nullptr, 4, plan != nullptr},
        {"row_pair", plan ? plan->row_pair : nullptr, 4, plan && by_token}};
    for (const auto& t : tensors) {
        if (!t.wanted) continue;
        if (!t.p) return bad("%s is NULL", t.name);
        if ((uintptr_t)t.p % t.align) return bad("%s must be %d-byte aligned", t.name, (int)t.align);
        if (!memory_of_device(t.p, dev))
            return bad("%s does not live on the current CUDA device (make the tensors' GPU current before the call)", t.name);
    }
    const int64_t columns = gated ? w->n / 2 : w->n, x_rows = by_token ? plan->num_tokens : rows;
    if (x_stride < 0 || x_stride > ((int64_t)1 << 40) || out_stride > ((int64_t)1 << 40)) return bad("a row stride is out of range");
    if (rows > 1 && out_stride < columns) return bad("out: rows of %lld elements overlap at a stride of %lld", (long long)columns, (long long)out_stride);
    const Extent eo = {"out", out, rows, columns * 2, out_stride * 2}, ex = {"x", x, x_rows, (int64_t)w->k * 2, x_stride * 2};
    const int64_t all = (int64_t)w->num_experts * w->n;
    const Extent inputs[] = {ex, {"codes", w->codes, 1, all * (w->k / 2), 0}, {"scales", w->scales, 1, all * groups * 2, 0},
                             {"zeros", w->zeros, 1, all * groups, 0}};
    for (const Extent& in : inputs)
        if (share_memory(eo, in)) return bad("out and %s share memory", in.name);

    MatvecArgs a = {};
    a.x = static_cast<const uint8_t*>(x);
    a.x_stride = x_stride * 2;
    a.x_rows = (int)x_rows;
    a.x_wide = (((uintptr_t)x | (uintptr_t)(x_rows > 1 ? a.x_stride : 0)) & 15u) == 0;
    a.by_token = by_token ? 1 : 0;
    a.scales = static_cast<const uint8_t*>(w->scales);
    a.zeros = w->zeros;
    a.out = static_cast<uint8_t*>(out);
    a.out_stride = out_stride * 2;
    a.E = w->num_experts;
    a.N = w->n;
    a.K = w->k;
    a.group_shift = w->group == 32 ? 0 : w->group == 64 ? 1 : 2;
    a.rows = (int)rows;
    if (plan) {
        a.top_k = plan->top_k;
        a.expert_offset = plan->expert_offset;
        a.expert_count = plan->expert_count;
        a.row_pair = plan->row_pair;
    }
    // a warp holds at most kMaxBlocks blocks of x
    a.split = w->k <= 32 * kMaxBlocks * 4 ? 4 : w->k <= 32 * kMaxBlocks * 8 ? 8 : 16;
    a.chunks = (w->k / 2 + 127) / 128;
    a.whole = w->k % 256 == 0;
    // Scales and zero points come as boxes a little wider than their rows: eight rows start in different groups of four banks
    // if their pitch is an odd number of 16-byte units (a box has at most 256 values; K = 8192 with groups of 32 has that many)
    auto pitch = [](int bytes, int most) { return bytes % 32 || bytes >= most ? bytes : bytes + 16; };
    const int per_stage = kWarps / a.split;
    a.scale_box = groups * 2 % 16 == 0;
    a.zero_box = groups % 16 == 0;
    a.scale_bytes = a.scale_box ? pitch(groups * 2, 512) : groups * 2;
    a.zero_bytes = a.zero_box ? pitch(groups, 256) : groups;
    a.scale_at = per_stage * a.chunks * 2048;
    a.zero_at = (a.scale_at + per_stage * kTileRows * a.scale_bytes + 127) / 128 * 128;
    a.stage_bytes = (a.zero_at + (w->zeros ? per_stage * kTileRows * a.zero_bytes : 0) + 1023) / 1024 * 1024;
    a.stages = (int)((kSharedLimit - sizeof(Shared) - kSwizzleAtom - 256) / a.stage_bytes);
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    MatvecMaps maps = {};
    int r = encode_weights(maps.codes, w->codes, a, gated != 0, w->k / 2, 128, true);
    if (r == 0 && a.scale_box) r = encode_weights(maps.scales, w->scales, a, gated != 0, groups * 2, a.scale_bytes, false);
    if (r == 0 && w->zeros && a.zero_box) r = encode_weights(maps.zeros, w->zeros, a, gated != 0, groups, a.zero_bytes, false);
    if (r != 0) return refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "cuTensorMapEncodeTiled(weights) failed: %d", r);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    e = dtype == MOE_FP8_B200_BF16 ? launch_matvec<__nv_bfloat16>(a, maps, gated != 0, sms, s)
                                    : launch_matvec<__half>(a, maps, gated != 0, sms, s);
    return e == cudaSuccess ? MOE_FP8_B200_OK : refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
}
