// Products of a few rows with matrices of 4-bit weights, one scale (and zero point) per group of input columns: the
// experts' products of a decode batch (declared in include/moe_fp8_b200.h).
//
//   y[r, n] = sum over k of (code[n, k] - zero[n, k / G]) * scale[n, k / G] * x[r, k]
//
// What bounds it is the stream of the codes out of HBM: a weight is half a byte and meets at most eight rows per read.
// The codes are read in the operator's own layout, two per byte, row by row.  One persistent CTA per SM takes a contiguous
// range of 16-row weight tiles and keeps the next ones on their way into a ring of shared-memory stages (one untiled bulk
// copy per weight row, requested by one warp as soon as all have read the stage that it replaces); sixteen warps split a
// tile's K range and multiply with mma.sync (m16n8k16: the weights are the 16-row operand, up to eight rows of x the other
// one).  tcgen05 has nothing to give here: its M of 128
// would need a dequantised copy of the weights in shared memory or TMEM, and the tensor pipe is far from busy.
//
// The order of K inside a tile is free as long as both operands agree.  A thread's 32-bit word of codes holds the
// columns 8t .. 8t+7 of a 32-column block (t = lane % 4), and the pairs (0,4) (1,5) (2,6) (3,7) fall out of it with a shift
// and a mask each; x is held in registers in that order, loaded once per run of tiles of one expert.
// code - zero is exact in bf16 and fp16; the products are summed in fp32, scaled per 32 columns in fp32, and rounded once.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "call_checks.cuh"
#include "ptx.cuh"

namespace moe {
namespace {

constexpr int kWarps = 16;
constexpr int kThreads = kWarps * 32;
constexpr int kLoadWarp = kWarps - 1;         // also requests the stages
constexpr int kTileRows = 16;                 // weight rows of a tile
constexpr int kRowsOfX = 8;                   // rows of x that share a read of the weights
constexpr int kMaxBlocks = 16;                // 32-column blocks of a warp
constexpr int kMaxK = 8192;
constexpr int kMaxStages = 8;
constexpr int kMaxExperts = MOE_FP8_B200_PLAN_MAX_EXPERTS;
constexpr int kChunkTiles = 8;                // see Run
constexpr size_t kSharedLimit = 227 * 1024;

struct MatvecArgs {
    const uint8_t* x;
    long long x_stride;        // bytes
    int x_rows, x_wide;        // rows that exist; 16-byte loads allowed
    int by_token, top_k;       // x has a row per token: that of row r is row_pair[r] / top_k
    const uint8_t* codes;
    const uint8_t* scales;     // 16-bit
    const uint8_t* zeros;      // or null: 8
    uint8_t* out;
    long long out_stride;
    int E, N, K, group_shift;  // group = 32 << group_shift columns
    const int *expert_offset, *expert_count, *row_pair;   // null: one matrix, `rows` rows
    int rows;                  // rows of out
    int split, stages;         // warps that share a tile; ring
    int row_bytes, stage_bytes, scale_at, zero_at;   // layout of a stage
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

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar)
                 : "memory");
}

template <typename T> struct Half2;
template <> struct Half2<__nv_bfloat16> {
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
    // two equal values 128 + zero
    static __device__ __forceinline__ uint32_t offset(uint32_t zero) { return 0x43004300u + zero * 0x00010001u; }
    // Codes (0,4) (1,5) (2,6) (3,7) of a word minus the zero point: 0x4300 | code is 128 + code, exactly.
    static __device__ __forceinline__ void decode(uint32_t w, uint32_t off, uint32_t (&q)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t v = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(q[i]) : "r"(v), "r"(off));
        }
    }
    static __device__ __forceinline__ float scale(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }
    static __device__ __forceinline__ __nv_bfloat16 round(float v) { return __float2bfloat16_rn(v); }
};
template <> struct Half2<__half> {
    static __device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                               uint32_t b1) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                     "{%0, %1, %2, %3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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
            const uint32_t lo = (s & 0x000f000fu) | 0x64006400u, hi = (s & 0x00f000f0u) | 0x64006400u;
            asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(q[2 * i]) : "r"(lo), "r"(off));
            asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(q[2 * i + 1]) : "r"(hi), "r"(0x2c002c00u), "r"(neg));
        }
    }
    static __device__ __forceinline__ float scale(uint16_t bits) { return __half2float(__ushort_as_half(bits)); }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ uint32_t lds32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint16_t lds16(uint32_t addr) {
    uint16_t v;
    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(addr));
    return v;
}
__device__ __forceinline__ uint32_t lds8(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared.u8 %0, [%1];" : "=r"(v) : "r"(addr));
    return v;
}

template <typename T, bool GATED>
__global__ void __launch_bounds__(kThreads, 1) matvec4_kernel(const MatvecArgs a)
{
    extern __shared__ __align__(128) uint8_t ring[];
    __shared__ Shared sh;
    typedef Half2<T> H;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
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
        const int line = a.K / 2;
        __syncwarp();
        if (lane == 0) {
            sh.load_done = t0 + n;
            mbar_expect_tx(bar, (uint32_t)(n * kTileRows) * (uint32_t)(line + groups * (a.zeros ? 3 : 2)));
        }
        __syncwarp();
        const long long row0 = (long long)r.expert * a.N;
        for (int i = lane; i < n * kTileRows; i += 32) {
            const int tile = r.tile + t0 + i / kTileRows, j = i % kTileRows;
            const long long row = row0 + (GATED ? (j < 8 ? 0 : a.N / 2 - 8) + tile * 8 + j : tile * kTileRows + j);
            bulk_load(dst + i * a.row_bytes, a.codes + row * line, line, bar);
        }
        // a tile's scales are contiguous, or two halves of eight rows
        constexpr int kPieces = GATED ? 2 : 1, kPieceRows = kTileRows / kPieces;
        for (int i = lane; i < n * kPieces; i += 32) {
            const int tile = r.tile + t0 + i / kPieces, half = i % kPieces;
            const long long row = row0 + (GATED ? half * (a.N / 2) + tile * 8 : tile * kTileRows);
            bulk_load(dst + a.scale_at + i * kPieceRows * groups * 2, a.scales + row * groups * 2, kPieceRows * groups * 2, bar);
            if (a.zeros)
                bulk_load(dst + a.zero_at + i * kPieceRows * groups, a.zeros + row * groups, kPieceRows * groups, bar);
        }
    };
    if (warp == kLoadWarp) {
        if (lane == 0) {
            sh.load_unit = begin;
            sh.load_done = sh.load_run.count = 0;
        }
        __syncwarp();
        for (int i = 0; i < a.stages; ++i) request_stage(i);
    }

    // `split` warps share a tile's K range, tile m of the stage belongs to warps [m * split, (m + 1) * split)
    const int member = warp % a.split, of_stage = warp / a.split;
    const int blocks = a.K / 32;
    const int b0 = blocks * member / a.split, nb = blocks * (member + 1) / a.split - b0;
    const int g = lane / 4, t = lane % 4;
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
            const uint8_t* xp = a.x + src * a.x_stride + (b0 * 32 + 8 * t) * 2;
#pragma unroll
            for (int j = 0; j < kMaxBlocks; ++j)
                if (j < nb) {
                    uint32_t v[4];
                    if (a.x_wide) {
                        const uint4 q = *reinterpret_cast<const uint4*>(xp + j * 64);
                        v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
                    } else {
                        const uint16_t* h = reinterpret_cast<const uint16_t*>(xp + j * 64);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
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
                const uint32_t stage = ring0 + slot * a.stage_bytes;
                const uint32_t w0 = stage + (of_stage * kTileRows + g) * a.row_bytes + 16 * b0 + 4 * t, w1 = w0 + 8 * a.row_bytes;
                const int line0 = (of_stage * kTileRows + g) * groups, line1 = line0 + 8 * groups;
#pragma unroll
                for (int j = 0; j < kMaxBlocks; ++j)
                    if (j < nb) {
                        const int group = (b0 + j) >> a.group_shift;
                        const uint32_t z0 = a.zeros ? lds8(stage + a.zero_at + line0 + group) : 8u;
                        const uint32_t z1 = a.zeros ? lds8(stage + a.zero_at + line1 + group) : 8u;
                        const float s0 = H::scale(lds16(stage + a.scale_at + 2 * (line0 + group)));
                        const float s1 = H::scale(lds16(stage + a.scale_at + 2 * (line1 + group)));
                        uint32_t q0[4], q1[4];
                        H::decode(lds32(w0 + 16 * j), H::offset(z0), q0);
                        H::decode(lds32(w1 + 16 * j), H::offset(z1), q1);
                        float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        H::mma(c, q0[0], q1[0], q0[1], q1[1], xr[j][0], xr[j][1]);
                        H::mma(c, q0[2], q1[2], q0[3], q1[3], xr[j][2], xr[j][3]);
                        acc[0] = fmaf(s0, c[0], acc[0]);
                        acc[1] = fmaf(s0, c[1], acc[1]);
                        acc[2] = fmaf(s1, c[2], acc[2]);
                        acc[3] = fmaf(s1, c[3], acc[3]);
                    }
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

template <typename T>
cudaError_t launch_matvec(const MatvecArgs& a, bool gated, int sms, cudaStream_t stream)
{
    const size_t smem = (size_t)a.stages * a.stage_bytes;
    auto kernel = gated ? matvec4_kernel<T, true> : matvec4_kernel<T, false>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e != cudaSuccess) return e;
    return launch_after(kernel, dim3(sms), dim3(kThreads), smem, 1, stream, a);
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
    a.codes = static_cast<const uint8_t*>(w->codes);
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
    // eight weight rows start in different groups of four banks if a row is an odd number of 16-byte pieces long
    a.row_bytes = w->k / 2 + (w->k / 32 % 2 ? 0 : 16);
    const int stage_rows = kWarps / a.split * kTileRows;
    a.scale_at = stage_rows * a.row_bytes;
    a.zero_at = a.scale_at + stage_rows * groups * 2;
    a.stage_bytes = (a.zero_at + (w->zeros ? stage_rows * groups : 0) + 127) / 128 * 128;
    a.stages = (int)((kSharedLimit - sizeof(Shared) - 256) / a.stage_bytes);
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    e = dtype == MOE_FP8_B200_BF16 ? launch_matvec<__nv_bfloat16>(a, gated != 0, sms, s) : launch_matvec<__half>(a, gated != 0, sms, s);
    return e == cudaSuccess ? MOE_FP8_B200_OK : refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
}
