// Products of a few rows with matrices of 4-bit weights, one scale (and zero point) per group of input columns: the
// experts' products of a decode batch (declared in include/moe_fp8_b200.h).
//
//   y[r, n] = sum over k of (code[n, k] - zero[n, k / G]) * scale[n, k / G] * x[r, k]
//
// What bounds it is the stream of the codes out of HBM: a weight is half a byte and meets at most eight rows per read.
// The codes are read in the operator's own layout, two per byte, row by row.  One persistent CTA per SM takes a contiguous
// range of 16-row weight tiles.  One warp keeps the next ones on their way into a ring of shared-memory stages (one TMA box
// per tile), sixteen warps split a tile's K range and multiply with mma.sync (the weights are the 16-row operand, the rows
// of x the 8-column one), and three warps add up the sixteen's partial sums and store the results, so that the sixteen go
// on with the next stage.
// tcgen05 has nothing to give here: its M of 128 would need a converted copy of the weights in shared memory or TMEM, and
// the tensor pipe is far from busy.
//
// What the SM has to do per byte of codes decides whether the stream runs at full rate (at 6.4 TB/s an SM gets 46 codes a
// clock).  Two forms of the product:
//
// * Up to four rows of x (two with zero points), by integers (m16n8k32, s8).  A code becomes a signed byte with a shift and a mask per four:
//   (code - 8) * 16 sits in the upper half of a byte already, once its top bit is flipped; with zero points the code stays
//   in the lower half and a second product takes the zero point off.  x is split, per row and warp, into four signed
//   bytes of a 31-bit fixed-point number below the power of two above its largest value: four columns of the product per row, so
//   two rows per instruction.  Such a number is x itself for all values down to 2^-23 of that power (fp16: 2^-20); where a smaller
//   one is not, the warp takes the other form, since it would be lost where a weight of zero meets the largest value.
//   The sums of a scale's products are exact integers, and become floats by starting from the bit pattern of 1.5 * 2^23 times a
//   power of two, which brings them below 1/8, so that their products with any scales stay within fp32.
// * More rows, or a row with an infinity, a NaN or values too far apart, in the type itself (m16n8k16): 0x4300 | code is 128 + code in
//   bf16 (0x6400 | code is 1024 + code in fp16), exactly, and so is the difference to 128 + zero.  11 (9) operations
//   per eight codes instead of 3.
//
// Either way the products are exact and summed exactly or in fp32, scaled in fp32 per 32 or 64 columns, and rounded once.
// The order of K inside a block of 32 columns is free as long as both operands agree: a thread's 32-bit word of codes
// holds the columns 8t .. 8t+7 (t = lane % 4), and x is held in registers in the order they fall out of it.
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

constexpr int kWarps = 16;                    // that multiply
constexpr int kLoadWarp = kWarps;             // requests the stages
constexpr int kSumWarps = 3;                  // add up the partial sums
constexpr int kThreads = (kWarps + 1 + kSumWarps) * 32;
// Registers: 640 threads x 96 at launch = 512 x 112 + 128 x 32.
constexpr int kLaunchRegisters = 96, kMultiplyRegisters = 112, kOtherRegisters = 32;
static_assert(kThreads * kLaunchRegisters == kWarps * 32 * kMultiplyRegisters + (1 + kSumWarps) * 32 * kOtherRegisters, "registers");
constexpr int kTileRows = 16;                 // weight rows of a tile
constexpr int kRowsOfX = 8;                   // rows of x that share a read of the weights
constexpr int kMaxBlocks = 16;                // 32-column blocks of a warp
// Rows of x up to which the product goes by integers.  57344 x 7168 (212 MB), us by integers / in the type: 1 and 2 rows 51 / 62,
// 3 and 4 rows 57 / 63, in fp16 59 / 60; groups of 32: 2 rows 57 / 70, in fp16 4 rows 65 / 64.  With zero points 2 rows 59 / 65,
// with groups of 32 as well 65 / 70, but 4 rows 69 / 64 and 86 / 75: there an instruction per zero point adds up.
__host__ __device__ constexpr int few_rows(bool zeros) { return zeros ? 2 : 4; }
constexpr int kMaxK = 8192;
constexpr int kMaxRows = 1 << 21;              // whatever a plan says, the sums over its experts stay within 32 bits
constexpr int kMaxStages = 4;
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
    int E, N, K, group, gated;
    const int *expert_offset, *expert_count, *row_pair;   // null: one matrix, `rows` rows
    int rows;                  // rows of out
    unsigned share_step;       // 2^32 / CTAs
    int prefetch;              // x is small enough to be asked into L2 first
    int stages;                // of the ring
    // A stage: the codes of 16 / SPLIT tiles, then their scales, then their zero points.  A tile's codes are `chunks` pieces of
    // 128 bytes (256 columns) of its sixteen rows, in the 128-byte swizzle (16-byte unit index XOR row mod 8).
    int chunks, whole;             // whole: a row is a multiple of 128 bytes, one box takes a tile
    int scale_step;                // scales from a pair of a warp to its next
    int scale_bytes, zero_bytes;   // pitch of a row's scales and zero points
    int scale_box, zero_box;       // they come as boxes, else (rows of no multiple of 16 bytes) as they lie
    int scale_at, zero_at, stage_bytes;
    unsigned tile_bytes;           // that arrive per tile
};

// The weights as TMA sees them: gated ones as two halves of n / 2 rows, of which a tile takes the same eight.
struct alignas(64) MatvecMaps {
    CUtensorMap codes, scales, zeros;
};

// Tiles of weights that meet the same rows of x one after the other.
struct Run {
    int expert, x_tile, tile, count;
};

// What a stage holds: `tiles` tiles from `tile` on, for `rows` rows of x and out from `row` on.  No tiles: the end.
struct StageInfo {
    int row, rows, tile, tiles;
};
// The load warp is at most kMaxStages ahead of the multiplying warps, and those two ahead of the adding ones.
constexpr int kStageInfos = 8;

struct Shared {
    int abort;
    int2 warp_sum[kThreads / 32];
    alignas(8) uint64_t full_bar[kMaxStages];  // a stage's bytes are there
    alignas(8) uint64_t empty_bar[kMaxStages]; // all multiplying warps have read it
    alignas(8) uint64_t done_bar[2];           // their partial sums are there, in the buffer of the stage's parity
    alignas(8) uint64_t free_bar[2];           // and have been added up
    alignas(16) StageInfo info[kStageInfos];
    StageInfo start;                           // the first run's rows, before its weights are there
    unsigned begin, end;                       // this CTA's units
    int unit[kWarps][kRowsOfX];                // of a multiplying warp's rows of x: a factor's bits (load_values) or a power (load_digits)
    alignas(16) float part[2][kWarps][128];
};

constexpr size_t kDynamicLimit = kSharedLimit - sizeof(Shared) - 256;

// What the CTAs know of the experts' rows, behind the ring: [E + 1] each.
struct Experts {
    int* first;    // tiles of x rows in front of expert e
    int* cost;     // and what they cost
    int2* rows;    // its first row, and how many
};
size_t experts_bytes(int E) { return ((size_t)(E + 1) * 16 + 127) / 128 * 128; }

__device__ __forceinline__ int last_at_or_below(const int* sums, int n, unsigned at) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) / 2;
        if ((unsigned)sums[mid] <= at) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Tiles of up to eight rows, and what they cost: the figures at few_rows, of bf16 in groups of 128 without zero points, less what a
// call costs besides.  Other forms' ratios differ by a tenth or two, which only makes the shares less even.
constexpr int kTwoCost = 7, kFewCost = 8, kManyCost = 9;
__device__ __forceinline__ int2 x_tiles_of(int rows, bool zeros) {
    const int full = rows / kRowsOfX, rest = rows % kRowsOfX;
    return make_int2(full + (rest > 0),
                     full * kManyCost + (rest > few_rows(zeros) ? kManyCost : rest > 2 ? kFewCost : rest > 0 ? kTwoCost : 0));
}

// First unit (a tile of weights for a tile of x rows, in Run's order) of CTA `share`: the CTAs get equal costs.  The host sees
// to it that costs times tiles fit into 32 bits; a 64-bit division would take a microsecond here.
__device__ __forceinline__ unsigned unit_at_share(const Experts& ex, const MatvecArgs& a, unsigned share, unsigned tiles)
{
    const unsigned all = (unsigned)ex.cost[a.E] * tiles;
    if (share == gridDim.x || all == 0) return (unsigned)ex.first[a.E] * tiles;
    const unsigned at = __umulhi(all, share * a.share_step);
    const int e = last_at_or_below(ex.cost, a.E, at / tiles);
    const unsigned x_tiles = ex.first[e + 1] - ex.first[e], cost = ex.cost[e + 1] - ex.cost[e], rel = at - (unsigned)ex.cost[e] * tiles;
    const unsigned unit = x_tiles == 1 ? rel / cost : (unsigned)((unsigned long long)rel * x_tiles / cost);
    return (unsigned)ex.first[e] * tiles + unit;
}

// Work is laid out expert by expert.  An expert with more than eight rows meets its weights once per eight of them, in
// chunks of kChunkTiles tiles, so that the second read of a chunk finds it in L2 (148 CTAs x 8 tiles x 57 KB = 68 MB).
__device__ __forceinline__ Run run_at(const Experts& ex, const MatvecArgs& a, unsigned unit, unsigned end, int tiles)
{
    const int e = last_at_or_below(ex.first, a.E, unit / tiles);
    const int x_tiles = ex.first[e + 1] - ex.first[e], within = unit - ex.first[e] * tiles;
    if (x_tiles == 1) return {e, 0, within, (int)min((unsigned)(tiles - within), end - unit)};
    const int chunk = within / (kChunkTiles * x_tiles), rem = within - chunk * kChunkTiles * x_tiles;
    const int here = min(kChunkTiles, tiles - chunk * kChunkTiles), x_tile = rem / here;
    return {e, x_tile, chunk * kChunkTiles + rem - x_tile * here, (int)min((unsigned)(here - (rem - x_tile * here)), end - unit)};
}

// The rows of x and out that a run's tiles meet.
__device__ __forceinline__ int2 rows_of(const Experts& ex, const Run& r) {
    const int2 rows = ex.rows[r.expert];
    return make_int2(rows.x + r.x_tile * kRowsOfX, min(kRowsOfX, rows.y - r.x_tile * kRowsOfX));
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
// 2^e, -149 <= e <= 127
__device__ __forceinline__ float exp2_of(int e) {
    return e >= -126 ? __int_as_float((e + 127) << 23) : __int_as_float(1 << (e + 149));
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
    static constexpr int kMantissa = 7, kBias = 127;
    static constexpr uint32_t kInf = 0x7f80u;
    static __device__ __forceinline__ float value(uint16_t bits) { return __uint_as_float((uint32_t)bits << 16); }
    static __device__ __forceinline__ float scale(uint16_t bits) { return value(bits); }
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
    static constexpr int kMantissa = 10, kBias = 15;
    static constexpr uint32_t kInf = 0x7c00u;
    static __device__ __forceinline__ float value(uint16_t bits) { return __half2float(__ushort_as_half(bits)); }
    static __device__ __forceinline__ float scale(uint16_t bits) { return value(bits); }
    static __device__ __forceinline__ __half round(float v) { return __float2half_rn(v); }
};

__device__ __forceinline__ void mma_s8(int (&d)[4], const int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    asm("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "r"(c[0]), "r"(c[1]), "r"(c[2]), "r"(c[3]));
}
// The start of every sum by integers (see ByInteger).  With a scale per block there are so many that it is kept in four registers
// (16 tokens, groups of 32 with zero points: 63 us, 67 with four moves per sum); with one per pair the registers are worth
// more (one token, 256 experts: 39 us, 41 with Ones).
__host__ __device__ constexpr int one_of(bool zeros) { return 0x4b400000 - ((zeros ? 20 : 24) << 23); }
template <bool ZEROS>
struct Ones {
    int v[4];
    __device__ __forceinline__ Ones() {
#pragma unroll
        for (int i = 0; i < 4; ++i) asm volatile("mov.b32 %0, %1;" : "=r"(v[i]) : "n"(one_of(ZEROS)));
    }
};
// (a ^ b) & mask in one instruction
__device__ __forceinline__ uint32_t xor_and(uint32_t a, uint32_t b, uint32_t mask) {
    uint32_t d;
    asm("lop3.b32 %0, %1, %2, %3, 0x28;" : "=r"(d) : "r"(a), "r"(b), "r"(mask));
    return d;
}

// A thread's part of a tile in shared memory (bytes into the ring).  SPLIT warps share a tile, and each takes every SPLIT-th pair
// of 32-column blocks: its pairs lie SPLIT / 4 chunks apart.  With SPLIT a constant, so are the distances, and the loads need
// no arithmetic; registers are what this kernel has least of (a spilled one comes back out of L2, behind the weights).
struct TileView {
    const uint8_t* ring;
    int even;              // its word of the first pair's first block in weight row g (the second's: ^ 16); row g + 8 lies 1024 bytes further
    int scales, zeros;     // its row's scale and zero point of the first pair; row g + 8's lie 8 rows further
    int blocks;            // of the warp; a last pair's second block may not exist (its x is zero)
};

// The words of COUNT pairs of blocks from `pair` on, and the scales and zero points of one.
template <int SPLIT, int COUNT>
struct Words {
    uint32_t row0[2 * COUNT], row1[2 * COUNT];
    __device__ __forceinline__ Words(const TileView& v, int pair) {
#pragma unroll
        for (int p = 0; p < COUNT; ++p) {
            const uint8_t* at = v.ring + (pair + p) * (SPLIT * 512);
            const int odd = v.even ^ 16;
            row0[2 * p] = *reinterpret_cast<const uint32_t*>(at + v.even);
            row1[2 * p] = *reinterpret_cast<const uint32_t*>(at + v.even + 1024);
            row0[2 * p + 1] = *reinterpret_cast<const uint32_t*>(at + odd);
            row1[2 * p + 1] = *reinterpret_cast<const uint32_t*>(at + odd + 1024);
        }
    }
};
// `second`: the pair's second scale
template <typename H, bool ZEROS>
struct Scales {
    float s0, s1;
    uint32_t z0, z1;
    __device__ __forceinline__ Scales(const MatvecArgs& a, const TileView& v, int pair, bool second) {
        const int sa = v.scales + pair * (2 * a.scale_step) + (second ? 2 : 0), za = v.zeros + pair * a.scale_step + (second ? 1 : 0);
        s0 = H::scale(*reinterpret_cast<const uint16_t*>(v.ring + sa));
        s1 = H::scale(*reinterpret_cast<const uint16_t*>(v.ring + sa + 8 * a.scale_bytes));
        z0 = ZEROS ? v.ring[za] : 8u;
        z1 = ZEROS ? v.ring[za + 8 * a.zero_bytes] : 8u;
        if (second && 2 * pair + 1 >= v.blocks) s0 = s1 = 0.0f;   // what lies there is no scale
    }
};

// COUNT pairs of blocks from pair FIRST on, in one stretch without a branch, so that their loads, conversions and matrix
// instructions overlap.  The products of a pair are summed by the matrix
// instructions, one scale at a time (FINE: two scales in a pair).  Here in the type itself, for eight rows of x.
template <typename H, bool FINE, bool ZEROS, int SPLIT>
struct ByType {
    static constexpr int kAtOnce = 1;
    template <int FIRST, int COUNT>
    static __device__ __forceinline__ void multiply(float (&acc)[8], const uint32_t (&xr)[kMaxBlocks][4], const Ones<ZEROS>& ones, const MatvecArgs& a, const TileView& v) {
        constexpr int kScales = FINE ? 2 : 1, kBlocks = 2 / kScales;   // scales of a pair, blocks of a scale
        const Words<SPLIT, COUNT> w(v, FIRST);
#pragma unroll
        for (int p = 0; p < COUNT; ++p)
#pragma unroll
            for (int i = 0; i < kScales; ++i) {
                const Scales<H, ZEROS> s(a, v, FIRST + p, i != 0);
                const uint32_t off0 = H::offset(s.z0), off1 = H::offset(s.z1);
                float c[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 2 * p + i * kBlocks; j < 2 * p + (i + 1) * kBlocks; ++j) {
                    const uint32_t(&x)[4] = xr[2 * FIRST + j];
                    uint32_t q0[4], q1[4];
                    H::decode(w.row0[j], off0, q0);
                    H::decode(w.row1[j], off1, q1);
                    H::mma(c, c, q0[0], q1[0], q0[1], q1[1], x[0], x[1]);
                    H::mma(c, c, q0[2], q1[2], q0[3], q1[3], x[2], x[3]);
                }
                acc[0] = fmaf(s.s0, c[0], acc[0]);
                acc[1] = fmaf(s.s0, c[1], acc[1]);
                acc[2] = fmaf(s.s1, c[2], acc[2]);
                acc[3] = fmaf(s.s1, c[3], acc[3]);
            }
    }
};

// By integers, for 2 * MMAS rows of x: column 4 r + d of a product is byte d of row r.  At most 64 products of 2^7 by 2^7 meet in
// a sum (with zero points, of 15 by 2^7), so it stays below 2^22 and one_of + sum is a float's bit pattern whose value is
// (1.5 * 2^23 + sum) / 2^24 (/ 2^20).  That makes the sum at most 1/16 (0.12), and the eight scales of a warp (sixteen of half as
// many columns) add up to less than the largest of them: nothing leaves fp32 that the result does not leave.  At the other
// end a product with a scale is rounded to 2^-149, half of which is 2^(e - 136) in the result, e as in load_digits.
template <typename H, bool FINE, bool ZEROS, int SPLIT, int MMAS>
struct ByInteger {
    static constexpr int kAtOnce = MMAS == 1 ? 2 : 1;
    template <int FIRST, int COUNT>
    static __device__ __forceinline__ void multiply(float (&acc)[8], const uint32_t (&xr)[kMaxBlocks][4], const Ones<ZEROS>& ones, const MatvecArgs& a, const TileView& v) {
        constexpr int kScales = FINE ? 2 : 1, kBlocks = 2 / kScales;
        const Words<SPLIT, COUNT> w(v, FIRST);
#pragma unroll
        for (int p = 0; p < COUNT; ++p)
#pragma unroll
            for (int i = 0; i < kScales; ++i) {
                constexpr int kOne = one_of(ZEROS);
                const Scales<H, ZEROS> s(a, v, FIRST + p, i != 0);
                const uint32_t neg0 = __byte_perm(0u - s.z0, 0, 0), neg1 = __byte_perm(0u - s.z1, 0, 0);   // bytes -zero
                int c[MMAS][4];
                if (!FINE) {
#pragma unroll
                    for (int m = 0; m < MMAS; ++m) c[m][0] = c[m][1] = c[m][2] = c[m][3] = kOne;
                }
#pragma unroll
                for (int j = 2 * p + i * kBlocks; j < 2 * p + (i + 1) * kBlocks; ++j) {
                    const uint32_t(&x)[4] = xr[2 * FIRST + j];
                    uint32_t even0, odd0, even1, odd1;
                    if (ZEROS) {
                        even0 = w.row0[j] & 0x0f0f0f0fu, odd0 = (w.row0[j] >> 4) & 0x0f0f0f0fu;
                        even1 = w.row1[j] & 0x0f0f0f0fu, odd1 = (w.row1[j] >> 4) & 0x0f0f0f0fu;
                    } else {
                        even0 = xor_and(w.row0[j] << 4, 0x80808080u, 0xf0f0f0f0u), odd0 = xor_and(w.row0[j], 0x80808080u, 0xf0f0f0f0u);
                        even1 = xor_and(w.row1[j] << 4, 0x80808080u, 0xf0f0f0f0u), odd1 = xor_and(w.row1[j], 0x80808080u, 0xf0f0f0f0u);
                    }
#pragma unroll
                    for (int m = 0; m < MMAS; ++m) {
                        if (FINE) mma_s8(c[m], ones.v, even0, even1, odd0, odd1, x[2 * m], x[2 * m + 1]);
                        else mma_s8(c[m], c[m], even0, even1, odd0, odd1, x[2 * m], x[2 * m + 1]);
                        if (ZEROS) mma_s8(c[m], c[m], neg0, neg1, neg0, neg1, x[2 * m], x[2 * m + 1]);
                    }
                }
#pragma unroll
                for (int m = 0; m < MMAS; ++m)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        acc[4 * m + k] = fmaf(k < 2 ? s.s0 : s.s1, __int_as_float(c[m][k]) - __int_as_float(kOne), acc[4 * m + k]);
            }
    }
};

// All of a warp's pairs, two at a time where the registers allow it.
template <typename P, int FIRST = 0, typename O>
__device__ __forceinline__ void multiply_pairs(float (&acc)[8], const uint32_t (&xr)[kMaxBlocks][4], const O& ones, const MatvecArgs& a, const TileView& v)
{
    if constexpr (2 * FIRST < kMaxBlocks) {
        if (v.blocks > 2 * (FIRST + P::kAtOnce - 1)) {
            P::template multiply<FIRST, P::kAtOnce>(acc, xr, ones, a, v);
            multiply_pairs<P, FIRST + P::kAtOnce>(acc, xr, ones, a, v);
        } else if (v.blocks > 2 * FIRST) {
            P::template multiply<FIRST, 1>(acc, xr, ones, a, v);
        }
    }
}

// A tile's scales (or zero points) where they are no box: as they lie, in two halves if gated.
__device__ __forceinline__ void copy_side(const MatvecArgs& a, const uint8_t* src, int bytes, int expert, int row, uint32_t to,
                                          uint32_t bar) {
    const int rows = a.gated ? kTileRows / 2 : kTileRows;
    src += ((long long)expert * a.N + row) * bytes;
    bulk_load(to, src, rows * bytes, bar);
    if (a.gated) bulk_load(to + rows * bytes, src + (long long)(a.N / 2) * bytes, rows * bytes, bar);
}

// Row `i` of a run's x, from its member-th pair of blocks on.
__device__ __forceinline__ const uint8_t* x_row(const MatvecArgs& a, int row, int rows, int i, int member) {
    int src = row + min(i, rows - 1);
    if (a.by_token) src = a.row_pair[src] / a.top_k;
    src = min(max(src, 0), a.x_rows - 1);
    return a.x + src * a.x_stride + (member * 64 < a.K ? member * 128 : 0);
}

// Block j of a warp exists, and its place behind the warp's first one (one that does not exist: the first one's).
template <int SPLIT>
__device__ __forceinline__ bool block_exists(const MatvecArgs& a, int member, int j) {
    return (2 * (member + j / 2 * SPLIT) + j % 2) * 32 < a.K;
}
template <int SPLIT>
__device__ __forceinline__ int x_block(const MatvecArgs& a, int member, int j) {
    return block_exists<SPLIT>(a, member, j) ? j / 2 * SPLIT * 128 + j % 2 * 64 : 0;
}

// x for the products in its own type: thread (g, t) holds row g's columns 8t .. 8t+7 of each of its warp's blocks, as the pairs
// (0, 4) (1, 5) (2, 6) (3, 7); zeros behind the last column.  A row of bf16 values near the end of fp32's range is held 2^16
// times smaller, so that products with codes do not leave it; `unit` says so.  (Only values below 2^-110, 2^-222 of the largest one,
// lose bits by that.)
template <typename T, int SPLIT>
__device__ __forceinline__ void load_values(uint32_t (&xr)[kMaxBlocks][4], int* unit, const MatvecArgs& a, int row, int rows,
                                            int member, int lane)
{
    const int g = lane / 4, t = lane % 4;
    const uint8_t* xp = x_row(a, row, rows, g, member) + 16 * t;
    if (a.x_wide) {
        // without a branch, so that all are under way together
#pragma unroll
        for (int j = 0; j < kMaxBlocks; ++j) {
            const uint4 v = *reinterpret_cast<const uint4*>(xp + x_block<SPLIT>(a, member, j));
            xr[j][0] = v.x, xr[j][1] = v.y, xr[j][2] = v.z, xr[j][3] = v.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < kMaxBlocks; ++j) {
            const uint16_t* h = reinterpret_cast<const uint16_t*>(xp + x_block<SPLIT>(a, member, j));
#pragma unroll
            for (int i = 0; i < 4; ++i) xr[j][i] = (uint32_t)h[2 * i] | ((uint32_t)h[2 * i + 1] << 16);
        }
    }
#pragma unroll
    for (int j = 0; j < kMaxBlocks; ++j) {
        const bool there = block_exists<SPLIT>(a, member, j);
        const uint32_t v0 = there ? xr[j][0] : 0, v1 = there ? xr[j][1] : 0, v2 = there ? xr[j][2] : 0, v3 = there ? xr[j][3] : 0;
        xr[j][0] = __byte_perm(v0, v2, 0x5410);
        xr[j][1] = __byte_perm(v0, v2, 0x7632);
        xr[j][2] = __byte_perm(v1, v3, 0x5410);
        xr[j][3] = __byte_perm(v1, v3, 0x7632);
    }
    float by_row = 1.0f;
    if constexpr (Half2<T>::kMantissa == 7) {
        uint32_t most = 0;
#pragma unroll
        for (int j = 0; j < kMaxBlocks; ++j)
#pragma unroll
            for (int i = 0; i < 4; ++i) most = max(most, max(xr[j][i] & 0x7fffu, xr[j][i] >> 16 & 0x7fffu));
        most = max(most, __shfl_xor_sync(~0u, most, 1));
        most = max(most, __shfl_xor_sync(~0u, most, 2));
        const bool large = most >= (112u + 127u) << 7;
        if (__any_sync(~0u, large)) {
            const uint32_t by = large ? 0x37803780u : 0x3f803f80u;   // 2^-16 or 1, twice
#pragma unroll
            for (int j = 0; j < kMaxBlocks; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i) asm("mul.rn.bf16x2 %0, %0, %1;" : "+r"(xr[j][i]) : "r"(by));
            if (large) by_row = 65536.0f;
        }
    }
    if (t == 0) unit[g] = __float_as_int(by_row);
    __syncwarp();
}

// x for the products by integers: thread (g, t) holds byte g % 4 of rows g / 4 and 2 + g / 4, of the columns 8t, 8t+2, 8t+4,
// 8t+6 in one word and of the odd ones in the next.  A value is 31 bits below 2^e, the power of two above the largest of
// its row's values in this warp, split into signed bytes.  Each thread converts two columns of a block; four threads'
// words are then transposed byte by byte.  `unit` gets e of each row.  Returns the form that
// x is in (1 up to two rows, 2 up to four), or 0 if a value is not finite or has bits below 2^(e - 30).
template <typename T, int SPLIT>
__device__ __forceinline__ int load_digits(uint32_t (&xr)[kMaxBlocks][4], int* unit, const MatvecArgs& a, int row, int rows,
                                           int member, int lane)
{
    const int t = lane % 4, q = lane / 4 % 4, forms = rows <= 2 ? 1 : 2;
    const uint32_t swap2 = q < 2 ? 0x5410u : 0x3276u, swap1 = q & 1 ? 0x3715u : 0x6240u;
#pragma unroll
    for (int m = 0; m < 2; ++m) {
        if (m >= forms) break;
        const uint8_t* xp = x_row(a, row, rows, 2 * m + lane / 16, member) + 16 * t + 4 * q;
        uint32_t raw[kMaxBlocks], most = 0, least = ~0u;   // least: of the values but zero, minus one
        if (a.x_wide) {
#pragma unroll
            for (int j = 0; j < kMaxBlocks; ++j) raw[j] = *reinterpret_cast<const uint32_t*>(xp + x_block<SPLIT>(a, member, j));
        } else {
#pragma unroll
            for (int j = 0; j < kMaxBlocks; ++j) {
                const uint16_t* h = reinterpret_cast<const uint16_t*>(xp + x_block<SPLIT>(a, member, j));
                raw[j] = (uint32_t)h[0] | ((uint32_t)h[1] << 16);
            }
        }
#pragma unroll
        for (int j = 0; j < kMaxBlocks; ++j) {
            if (!block_exists<SPLIT>(a, member, j)) raw[j] = 0;
            const uint32_t lo = raw[j] & 0x7fffu, hi = raw[j] >> 16 & 0x7fffu;
            most = max(most, max(lo, hi));
            least = min(least, min(lo - 1, hi - 1));
        }
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) most = max(most, __shfl_xor_sync(~0u, most, d));
        // the last bit of a value lies kMantissa below its first one; a subnormal's where the smallest normal one's does
        const int lowest = (int)(most >> Half2<T>::kMantissa) - 29 + Half2<T>::kMantissa;
        const uint32_t exact = lowest > 1 ? ((uint32_t)lowest << Half2<T>::kMantissa) - 1 : 0;
        if (__any_sync(~0u, most >= Half2<T>::kInf || least < exact)) return 0;
        const int e = (int)(most >> Half2<T>::kMantissa) - Half2<T>::kBias + 1;   // all below 2^e
        const float scale = exp2_of(-e);
        if (lane % 16 == 0) unit[2 * m + lane / 16] = e;
#pragma unroll
        for (int j = 0; j < kMaxBlocks; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float x = Half2<T>::value((uint16_t)(raw[j] >> (16 * i)));
                uint32_t v = ((uint32_t)__float2int_rn(x * scale * 0x1p30f) + 0x80808080u) ^ 0x80808080u;   // bytes -128 .. 127
                v = __byte_perm(v, __shfl_xor_sync(~0u, v, 8), swap2);
                v = __byte_perm(v, __shfl_xor_sync(~0u, v, 4), swap1);
                xr[j][2 * m + i] = v;
            }
    }
    __syncwarp();
    return forms;
}

template <typename T, bool FINE, bool ZEROS, int SPLIT>
__global__ void __launch_bounds__(kThreads, 1) matvec4_kernel(const MatvecArgs a, const __grid_constant__ MatvecMaps maps)
{
    extern __shared__ uint8_t pool[];
    __shared__ Shared sh;
    typedef Half2<T> H;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint8_t* const ring = pool + (0u - smem_u32(pool)) % kSwizzleAtom;
    const uint32_t ring0 = smem_u32(ring);
    Experts ex;
    ex.rows = reinterpret_cast<int2*>(ring + a.stages * a.stage_bytes);
    ex.first = reinterpret_cast<int*>(ex.rows + a.E + 1);
    ex.cost = ex.first + a.E + 1;
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        sh.abort = 0;
        for (int i = 0; i < a.stages; ++i) {
            mbar_init(smem_u32(&sh.full_bar[i]), 1);
            mbar_init(smem_u32(&sh.empty_bar[i]), kWarps);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.done_bar[i]), kWarps);
            mbar_init(smem_u32(&sh.free_bar[i]), kSumWarps);
        }
        fence_mbar_init();
    }
    __syncthreads();
    pdl_wait();

    int2 mine = {0, 0};   // first row and rows of expert threadIdx.x
    if (a.expert_count && threadIdx.x < a.E) mine = make_int2(a.expert_offset[threadIdx.x], a.expert_count[threadIdx.x]);
    // x is asked into L2 while these come
    if (a.prefetch) {
        const int lines = (a.K * 2 + 127) / 128 + 1, all = a.x_rows * lines;
        for (int i = blockIdx.x * kThreads + threadIdx.x; i < all; i += gridDim.x * kThreads) {
            const int r = i / lines, at = min((i - r * lines) * 128, a.K * 2 - 1);
            prefetch_l2(a.x + r * a.x_stride + at);
        }
        if (a.by_token)
            for (int i = blockIdx.x * kThreads + threadIdx.x; i < (a.rows + 31) / 32; i += gridDim.x * kThreads) prefetch_l2(a.row_pair + i * 32);
    }

    // tiles of x rows per expert and their costs, summed up
    if (a.expert_count) {
        int2 before = {0, 0};
        for (int e0 = 0; e0 < a.E; e0 += kThreads) {
            const int e = e0 + threadIdx.x, sums = min(kThreads, a.E - e0 + 31) / 32;
            int2 own = {0, 0};
            if (e < a.E) {
                const int off = e0 ? a.expert_offset[e] : mine.x, count = e0 ? a.expert_count[e] : mine.y;
                const int2 rows = off >= 0 && count > 0 && off < a.rows ? make_int2(off, min(count, a.rows - off)) : make_int2(0, 0);
                own = x_tiles_of(rows.y, ZEROS);
                ex.rows[e] = rows;
            }
            int2 upto = own;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int x = __shfl_up_sync(~0u, upto.x, d), y = __shfl_up_sync(~0u, upto.y, d);
                if (lane >= d) upto.x += x, upto.y += y;
            }
            if (lane == 31) sh.warp_sum[warp] = upto;
            __syncthreads();
            int2 total = before;
            for (int w = 0; w < sums; ++w) {
                const int2 v = sh.warp_sum[w];
                if (w < warp) upto.x += v.x, upto.y += v.y;
                total.x += v.x, total.y += v.y;
            }
            if (e < a.E) {
                ex.first[e] = before.x + upto.x - own.x;
                ex.cost[e] = before.y + upto.y - own.y;
            }
            before = total;
            if (e == a.E - 1) {
                ex.first[a.E] = total.x;
                ex.cost[a.E] = total.y;
            }
            __syncthreads();
        }
    } else {
        if (threadIdx.x == 0) {
            const int2 v = x_tiles_of(a.rows, ZEROS);
            ex.first[0] = ex.cost[0] = 0;
            ex.first[1] = v.x;
            ex.cost[1] = v.y;
            ex.rows[0] = {0, a.rows};
        }
        __syncthreads();
    }

    const int tiles = a.N / kTileRows;
    constexpr int per_stage = kWarps / SPLIT;
    if (threadIdx.x == 0) {
        // a plan whose experts' rows overlap is none: nothing is done
        if (ex.first[a.E] > a.rows / kRowsOfX + a.E) ex.first[a.E] = ex.cost[a.E] = 0;
        const unsigned begin = unit_at_share(ex, a, blockIdx.x, tiles), end = unit_at_share(ex, a, blockIdx.x + 1, tiles);
        sh.begin = begin;
        sh.end = end;
        const int2 x = begin < end ? rows_of(ex, run_at(ex, a, begin, end, tiles)) : make_int2(-1, 0);
        sh.start = {x.x, x.y, 0, 1};
    }
    __syncthreads();
    bool ok = true;

    if (warp >= kWarps) {
        setmaxnreg_dec<kOtherRegisters>();
        if (warp == kLoadWarp) {
            // ---- the stages, one after the other, and the end.  Lane m requests tile m of a stage.
            if (lane == 0) prefetch_tmap(&maps.codes);
            const int rows = a.gated ? kTileRows / 2 : kTileRows;
            int it = 0, slot = 0, lap = 0;
            for (unsigned u = sh.begin; u < sh.end && ok;) {
                Run r = run_at(ex, a, u, sh.end, a.N / kTileRows);
                u += r.count;
                for (; r.count > 0; r.count -= per_stage, r.tile += per_stage) {
                    ok = it < a.stages || mbar_wait(smem_u32(&sh.empty_bar[slot]), lap ^ 1, &sh.abort);
                    if (!__all_sync(~0u, ok)) { ok = false; break; }
                    const int n = min(per_stage, r.count);
                    const uint32_t bar = smem_u32(&sh.full_bar[slot]);
                    if (lane == 0) {
                        const int2 x = rows_of(ex, r);
                        sh.info[it % kStageInfos] = {x.x, x.y, r.tile, n};
                        mbar_expect_tx(bar, (uint32_t)n * a.tile_bytes);
                    }
                    __syncwarp();
                    if (lane < n) {
                        const int row = (r.tile + lane) * rows;
                        uint32_t to = ring0 + slot * a.stage_bytes;
                        for (int c = 0; c < (a.whole ? 1 : a.chunks); ++c)
                            box_load_5d(to + (lane * a.chunks + c) * 2048, &maps.codes, bar, c * 128, row, 0, 0, r.expert);
                        if (a.scale_box) box_load_4d(to + a.scale_at + lane * kTileRows * a.scale_bytes, &maps.scales, bar, 0, row, 0, r.expert);
                        else copy_side(a, a.scales, a.scale_bytes, r.expert, row, to + a.scale_at + lane * kTileRows * a.scale_bytes, bar);
                        if (ZEROS) {
                            to += a.zero_at + lane * kTileRows * a.zero_bytes;
                            if (a.zero_box) box_load_4d(to, &maps.zeros, bar, 0, row, 0, r.expert);
                            else copy_side(a, a.zeros, a.zero_bytes, r.expert, row, to, bar);
                        }
                    }
                    ++it;
                    if (++slot == a.stages) {
                        slot = 0;
                        lap ^= 1;
                    }
                }
            }
            if (ok) ok = it < a.stages || mbar_wait(smem_u32(&sh.empty_bar[slot]), lap ^ 1, &sh.abort);
            if (ok && lane == 0) {
                sh.info[it % kStageInfos].tiles = 0;
                mbar_arrive(smem_u32(&sh.full_bar[slot]));
            }
            if (!ok) {
                // A wait of a second ran out (see mbar_wait): nothing of this CTA stays on its way.
                int waited = 0;
                for (int i = 0; i < a.stages; ++i) {
                    slot = slot == 0 ? a.stages - 1 : slot - 1;
                    if (slot == a.stages - 1) lap ^= 1;
                    if (it - 1 - i >= 0) mbar_wait(smem_u32(&sh.full_bar[slot]), lap, &waited);
                }
            }
        } else {
            // ---- results of a stage: 128 per tile, the sums of its `split` warps' partial sums.  Thread (i, lane) has weight row
            // g + 8 (i / 2) and x row 2t + i % 2.
            const int g = lane / 4, t = lane % 4;
            for (int it = 0;; ++it) {
                const int b = it & 1;
                ok = mbar_wait(smem_u32(&sh.done_bar[b]), (it >> 1) & 1, &sh.abort);
                if (!ok) break;
                const StageInfo s = sh.info[it % kStageInfos];
                if (s.tiles == 0) break;
                const float(*part)[128] = sh.part[b];
                for (int v = warp - kLoadWarp - 1; v < s.tiles * (a.gated ? 2 : 4); v += kSumWarps) {
                    const int m = a.gated ? v / 2 : v / 4, i = a.gated ? v % 2 : v % 4, x_row = 2 * t + (i & 1);
                    float y = 0.0f, gate = 0.0f;
#pragma unroll 4
                    for (int k = 0; k < SPLIT; ++k) {
                        y += part[m * SPLIT + k][i * 32 + lane];
                        if (a.gated) gate += part[m * SPLIT + k][(i + 2) * 32 + lane];
                    }
                    if (x_row < s.rows) {
                        if (a.gated) y = gate / (1.0f + __expf(-gate)) * y;
                        const int col = a.gated ? (s.tile + m) * 8 + g : (s.tile + m) * kTileRows + g + 8 * (i / 2);
                        reinterpret_cast<T*>(a.out + (s.row + x_row) * a.out_stride)[col] = H::round(y);
                    }
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.free_bar[b]));
            }
        }
        return;
    }

    // ---- `split` warps share a tile's K range, tile m of the stage belongs to warps [m * split, (m + 1) * split)
    setmaxnreg_inc<kMultiplyRegisters>();
    const int member = warp % SPLIT, of_stage = warp / SPLIT;
    const int g = lane / 4, t = lane % 4;
    TileView view;
    {
        const int unit = 2 * member % 8;   // 16-byte unit of the first pair's first block in its chunk
        const int row = of_stage * kTileRows + g, group = member * 64 / a.group;
        view.ring = ring;
        view.even = (of_stage * a.chunks + member / 4) * 2048 + g * 128 + 4 * t + ((unit ^ g) << 4);
        view.scales = a.scale_at + row * a.scale_bytes + 2 * group;
        view.zeros = a.zero_at + row * a.zero_bytes + group;
        const int pairs = ((a.K + 63) / 64 - member + SPLIT - 1) / SPLIT;
        view.blocks = pairs > 0 ? min(2 * pairs, a.K / 32 - 2 * (member + (pairs - 1) * SPLIT) + 2 * (pairs - 1)) : 0;
    }
    const Ones<ZEROS> ones;
    uint32_t xr[kMaxBlocks][4];
    int form = 0;                      // 0 in the type itself, 1 by integers for up to two rows, 2 for up to four
    int* const unit = sh.unit[warp];
    int slot = 0, lap = 0, row = -1;
    // round -1 only takes up the first x, while its weights are on their way
    for (int it = -1;; ++it) {
        if (it >= 0) {
            ok = mbar_wait(smem_u32(&sh.full_bar[slot]), lap, &sh.abort);
            if (!ok) break;
        }
        const StageInfo& s = it < 0 ? sh.start : sh.info[it % kStageInfos];
        const int b = it & 1;
        if (s.tiles == 0) {
            // the adding warps see the end, too; not before all have arrived for the stage two before it
            if (it >= 2) ok = mbar_wait(smem_u32(&sh.free_bar[b]), (it >> 1) - 1 & 1, &sh.abort);
            if (ok && lane == 0) mbar_arrive(smem_u32(&sh.done_bar[b]));
            break;
        }
        if (s.row != row) {
            row = s.row;
            form = 0;
            if (s.rows <= few_rows(ZEROS)) form = load_digits<T, SPLIT>(xr, unit, a, row, s.rows, member, lane);
            if (form == 0) load_values<T, SPLIT>(xr, unit, a, row, s.rows, member, lane);
        }
        if (it < 0) continue;
        float acc[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
        if (of_stage < s.tiles) {
            TileView v = view;
            const int at = slot * a.stage_bytes;
            v.ring += at;
            if (form == 1) multiply_pairs<ByInteger<H, FINE, ZEROS, SPLIT, 1>>(acc, xr, ones, a, v);
            else if (!ZEROS && form == 2) multiply_pairs<ByInteger<H, FINE, ZEROS, SPLIT, 2>>(acc, xr, ones, a, v);
            else multiply_pairs<ByType<H, FINE, ZEROS, SPLIT>>(acc, xr, ones, a, v);
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.empty_bar[slot]));
        if (it >= 2) ok = mbar_wait(smem_u32(&sh.free_bar[b]), (it >> 1) - 1 & 1, &sh.abort);
        if (!ok) break;
        float* part = sh.part[b][warp];
        if (form == 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) part[i * 32 + lane] = acc[i] * __int_as_float(unit[2 * t + (i & 1)]);
        } else {
            // this thread's columns 2t, 2t + 1 are bytes 0, 1 (t even) or 2, 3 of x row t / 2 (and 2 + t / 2).  With the larger one as
            // the unit they stand for 2^(e - 2) and 2^(e + 14), which is multiplied in as two halves: neither leaves the range alone.
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                if (m >= form) break;
                const int half = (unit[2 * m + (t >> 1)] >> 1) + 8 * (t & 1);
                const int rest = unit[2 * m + (t >> 1)] + 16 * (t & 1) - half;
                const float f0 = __int_as_float((half + 127) << 23), f1 = __int_as_float((rest + 125) << 23);
                float y0 = fmaf(0x1p-8f, acc[4 * m], acc[4 * m + 1]) * f0 * f1;
                float y1 = fmaf(0x1p-8f, acc[4 * m + 2], acc[4 * m + 3]) * f0 * f1;
                y0 += __shfl_xor_sync(~0u, y0, 1);
                y1 += __shfl_xor_sync(~0u, y1, 1);
                part[((t & 1) * 2 + (t >> 1)) * 32 + g * 4 + m] = t & 1 ? y1 : y0;
            }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&sh.done_bar[b]));
        if (++slot == a.stages) {
            slot = 0;
            lap ^= 1;
        }
    }
    if (!ok) {
        // a load that never came, or sums that nobody added: the results are NaN
        for (unsigned u = sh.begin + warp; u < sh.end; u += kWarps) {
            const Run r = run_at(ex, a, u, u + 1, a.N / kTileRows);
            const int2 x = rows_of(ex, r);
            const int cols = a.gated ? kTileRows / 2 : kTileRows;
            for (int i = lane; i < x.y * cols; i += 32)
                reinterpret_cast<T*>(a.out + (x.x + i / cols) * a.out_stride)[r.tile * cols + i % cols] = H::round(__int_as_float(0x7fc00000));
        }
    }
}

}  // namespace
}  // namespace moe

using namespace moe;

namespace {

template <typename T, bool FINE, bool ZEROS, int SPLIT>
cudaError_t launch_form(const MatvecArgs& a, const MatvecMaps& maps, int sms, cudaStream_t stream)
{
    const size_t smem = (size_t)a.stages * a.stage_bytes + experts_bytes(a.E) + kSwizzleAtom;
    const auto kernel = matvec4_kernel<T, FINE, ZEROS, SPLIT>;
    // the same value in every call: the attribute belongs to the kernel, and another thread's call may stand between this and the launch
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kDynamicLimit);
    if (e != cudaSuccess) return e;
    return launch_after(kernel, dim3(sms), dim3(kThreads), smem, 1, stream, a, maps);
}

template <typename T, bool FINE, bool ZEROS>
cudaError_t launch_split(const MatvecArgs& a, const MatvecMaps& maps, int split, int sms, cudaStream_t stream)
{
    return split == 4   ? launch_form<T, FINE, ZEROS, 4>(a, maps, sms, stream)
           : split == 8 ? launch_form<T, FINE, ZEROS, 8>(a, maps, sms, stream)
                        : launch_form<T, FINE, ZEROS, 16>(a, maps, sms, stream);
}

template <typename T>
cudaError_t launch_matvec(const MatvecArgs& a, const MatvecMaps& maps, int split, int sms, cudaStream_t stream)
{
    if (a.group == 32)
        return a.zeros ? launch_split<T, true, true>(a, maps, split, sms, stream) : launch_split<T, true, false>(a, maps, split, sms, stream);
    return a.zeros ? launch_split<T, false, true>(a, maps, split, sms, stream) : launch_split<T, false, false>(a, maps, split, sms, stream);
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
    if (rows > kMaxRows) return bad("%lld rows are more than %d", (long long)rows, kMaxRows);
    if ((rows / kRowsOfX + w->num_experts + 1) * kManyCost * (w->n / kTileRows) >= ((int64_t)1 << 31))
        return bad("%lld rows by n = %d are too many for a product of a small batch", (long long)rows, w->n);
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
                             {"zeros", w->zeros, 1, all * groups, 0},
                             {"expert_offset", plan ? plan->expert_offset : nullptr, 1, 4ll * (w->num_experts + 1), 0},
                             {"expert_count", plan ? plan->expert_count : nullptr, 1, 4ll * w->num_experts, 0},
                             // not read here (row_pair without by_token), but what combines the results reads them
                             {"pair_row", plan ? plan->pair_row : nullptr, 1, plan ? 4ll * plan->num_tokens * plan->top_k : 0, 0},
                             {"row_pair", plan ? plan->row_pair : nullptr, 1, 4ll * rows, 0}};
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
    a.group = w->group;
    a.gated = gated ? 1 : 0;
    a.rows = (int)rows;
    a.share_step = (unsigned)(((uint64_t)1 << 32) / (unsigned)sms);
    a.prefetch = x_rows * w->k * 2 <= ((int64_t)4 << 20);
    if (plan) {
        a.top_k = plan->top_k;
        a.expert_offset = plan->expert_offset;
        a.expert_count = plan->expert_count;
        a.row_pair = plan->row_pair;
    }
    // a warp holds at most kMaxBlocks blocks of x
    const int split = w->k <= 32 * kMaxBlocks * 4 ? 4 : w->k <= 32 * kMaxBlocks * 8 ? 8 : 16;
    a.chunks = (w->k / 2 + 127) / 128;
    a.whole = w->k % 256 == 0;
    // Scales and zero points come as boxes a little wider than their rows: eight rows start in different groups of four banks
    // if their pitch is an odd number of 16-byte units (a box has at most 256 values; K = 8192 with groups of 32 has that many)
    auto pitch = [](int bytes, int most) { return bytes % 32 || bytes >= most ? bytes : bytes + 16; };
    const int per_stage = kWarps / split;
    a.scale_step = 64 * split / w->group;
    a.scale_box = groups * 2 % 16 == 0;
    a.zero_box = groups % 16 == 0;
    a.scale_bytes = a.scale_box ? pitch(groups * 2, 512) : groups * 2;
    a.zero_bytes = a.zero_box ? pitch(groups, 256) : groups;
    a.scale_at = per_stage * a.chunks * 2048;
    a.zero_at = (a.scale_at + per_stage * kTileRows * a.scale_bytes + 127) / 128 * 128;
    a.stage_bytes = (a.zero_at + (w->zeros ? per_stage * kTileRows * a.zero_bytes : 0) + 1023) / 1024 * 1024;
    a.stages = (int)((kDynamicLimit - experts_bytes(a.E) - kSwizzleAtom) / a.stage_bytes);
    if (a.stages > kMaxStages) a.stages = kMaxStages;
    a.tile_bytes = kTileRows * (unsigned)(a.chunks * 128 + a.scale_bytes + (w->zeros ? a.zero_bytes : 0));
    MatvecMaps maps = {};
    int r = encode_weights(maps.codes, w->codes, a, gated != 0, w->k / 2, 128, true);
    if (r == 0 && a.scale_box) r = encode_weights(maps.scales, w->scales, a, gated != 0, groups * 2, a.scale_bytes, false);
    if (r == 0 && w->zeros && a.zero_box) r = encode_weights(maps.zeros, w->zeros, a, gated != 0, groups, a.zero_bytes, false);
    if (r != 0) return refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "cuTensorMapEncodeTiled(weights) failed: %d", r);
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    e = dtype == MOE_FP8_B200_BF16 ? launch_matvec<__nv_bfloat16>(a, maps, split, sms, s) : launch_matvec<__half>(a, maps, split, sms, s);
    return e == cudaSuccess ? MOE_FP8_B200_OK : refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
}
