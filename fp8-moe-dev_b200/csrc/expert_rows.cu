// Tokens sorted by expert and back (declared in include/moe_fp8_b200.h): the plan that gives every (token, expert) pair
// its packed row, the copy of the tokens to those rows, the weighted sum of a token's rows, and the gradients.
//
// The movement is bound by HBM: a row is read or written once, a token once.  There is no atomic anywhere, so results
// do not depend on the order in which CTAs run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstring>
#include <initializer_list>
#include <type_traits>

#include "call_checks.cuh"
#include "ptx.cuh"

namespace moe {
namespace {

constexpr int kMaxTopK = MOE_FP8_B200_PLAN_MAX_TOP_K;
constexpr int kMaxExperts = MOE_FP8_B200_PLAN_MAX_EXPERTS;
constexpr int kMaxAlign = 1024;

// The plan as the kernels take it.
struct PlanView {
    int T, K, E, align;
    int pairs, capacity;   // T * K, rows of the packed matrix
    int *pair_row, *row_pair, *expert_offset, *expert_count;
};

// The plan's arrays are the caller's: a row outside the matrix counts as none.
__device__ __forceinline__ int row_of_pair(const PlanView& p, long long pair) {
    const int r = p.pair_row[pair];
    return (unsigned)r < (unsigned)p.capacity ? r : -1;
}

// Rows of a strided matrix in bytes.
struct Rows {
    uint8_t* base;
    long long stride;
    __device__ uint8_t* operator[](long long r) const { return base + r * stride; }
};

// ---------------------------------------------------------------------------------------
// The sort: a counting sort by expert that keeps the order of the pairs.  One cluster of CTAs, one launch: every warp
// counts a contiguous range of pairs, a CTA's warps and then the cluster's CTAs are scanned per expert (the other CTAs'
// counts through distributed shared memory), and each warp walks its range again, where a pair's rank among the
// pairs of its expert in the same 32 comes from votes over the warp.
// ---------------------------------------------------------------------------------------
constexpr int kSortThreads = 1024;

__device__ __forceinline__ unsigned cluster_rank() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ unsigned cluster_size() {
    unsigned r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
__device__ __forceinline__ int load_cluster(const int* own, unsigned rank) {
    uint32_t addr;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(addr) : "r"(smem_u32(own)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

template <typename Id>
__device__ __forceinline__ int expert_of(const Id* ids, int pair, unsigned long long first, int E) {
    const unsigned long long d = (unsigned long long)(long long)ids[pair] - first;
    return d < (unsigned long long)E ? (int)d : -1;
}

size_t sort_smem_bytes(int threads, int E) { return sizeof(int) * (size_t)E * (threads / 32 + 4); }

// The lanes whose x agrees in its low bits.  A vote per bit: nine of them take less time than one match over the warp (98304
// pairs: 16.4 us, 18.5 with the match).
__device__ __forceinline__ unsigned lanes_with(int x, int bits) {
    unsigned same = ~0u;
    for (int b = 0; b < bits; ++b) {
        const bool one = x >> b & 1;
        const unsigned v = __ballot_sync(~0u, one);
        same &= one ? v : ~v;
    }
    return same;
}

// What a CTA knows after the sort (shared memory).
struct Sorted {
    int *seen, *mine, *first_row, *pad_begin, *pad_end;
    __device__ Sorted(int* smem, int E, int warps) {
        seen = smem;                // [warps][E] pairs of the expert in earlier warps, then in earlier rounds too
        mine = seen + warps * E;    // [E] pairs in this CTA
        first_row = mine + E;       // [E] row of this CTA's first pair
        pad_begin = first_row + E;  // [E] padding rows of the expert
        pad_end = pad_begin + E;
    }
};

// Sorts the pairs with the CTAs of the cluster (one, if the launch has none) and returns the end of the last expert.  The
// plan's arrays are written if `publish`; LOCAL: a CTA by itself, which also keeps the pairs' rows in `local_row`.
// The ids of eight rounds are requested together, since a warp's loads would otherwise wait for one another.
template <typename Id, bool LOCAL>
__device__ __forceinline__ int sort_pairs(const Id* ids, unsigned long long first, const PlanView& p, const Sorted& s, bool publish,
                                          int* local_row)
{
    constexpr int kBatch = 8;
    __shared__ int warp_sum[32];
    const int E = p.E, warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const unsigned rank = LOCAL ? 0 : cluster_rank(), ctas = LOCAL ? 1 : cluster_size();
    const int per_cta = (p.pairs + (int)ctas - 1) / (int)ctas;
    const int cta_end = min(p.pairs, ((int)rank + 1) * per_cta);
    const int per_warp = (per_cta + warps * 32 - 1) / (warps * 32) * 32;
    const int begin = min(cta_end, (int)rank * per_cta + warp * per_warp);
    const int end = min(cta_end, begin + per_warp);
    int* own = s.seen + warp * E;
    const int bits = 32 - __clz(E);   // -1 has a pattern of its own among them
    for (int i0 = begin + lane; i0 < end + lane; i0 += 32 * kBatch) {
        int x[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) x[b] = i0 + 32 * b < end ? expert_of(ids, i0 + 32 * b, first, E) : -1;
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
            if (x[b] >= 0) atomicAdd(own + x[b], 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int run = 0;
        for (int w0 = 0; w0 < warps; w0 += kBatch) {
            int c[kBatch];
#pragma unroll
            for (int b = 0; b < kBatch; ++b) c[b] = w0 + b < warps ? s.seen[(w0 + b) * E + e] : 0;
#pragma unroll
            for (int b = 0; b < kBatch; ++b) {
                if (w0 + b < warps) s.seen[(w0 + b) * E + e] = run;
                run += c[b];
            }
        }
        s.mine[e] = run;
    }
    if (!LOCAL) {
        cluster_arrive();
        cluster_wait();
    }
    // one thread per expert (the launch has at least E)
    const int e = threadIdx.x;
    int before = 0, all = 0, padded = 0;
    if (e < E) {
        if (LOCAL) {
            all = s.mine[e];
        } else {
            for (unsigned c = 0; c < ctas; ++c) {
                const int v = load_cluster(s.mine + e, c);
                if (c < rank) before += v;
                all += v;
            }
        }
        padded = (all + p.align - 1) / p.align * p.align;
    }
    if (!LOCAL) cluster_arrive();   // this CTA reads no other one's memory any more; the wait stands at the end
    int upto = padded;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < (E + 31) / 32; ++w) {
        if (w < warp) upto += warp_sum[w];
        total += warp_sum[w];
    }
    if (e < E) {
        const int offset = upto - padded;
        s.first_row[e] = offset + before;
        s.pad_begin[e] = offset + all;
        s.pad_end[e] = upto;
        if (publish && rank == 0) {
            p.expert_offset[e] = offset;
            p.expert_count[e] = all;
        }
    }
    if (publish && rank == 0 && threadIdx.x == 0) p.expert_offset[E] = total;
    __syncthreads();

    for (int i0 = begin; i0 < end; i0 += 32 * kBatch) {
        int batch[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) batch[b] = i0 + 32 * b + lane < end ? expert_of(ids, i0 + 32 * b + lane, first, E) : -1;
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
            if (i0 + 32 * b >= end) break;
            const int i = i0 + 32 * b + lane, x = batch[b];
            const unsigned same = lanes_with(x, bits);
            const int prior = x >= 0 ? own[x] : 0;
            __syncwarp();
            if (x >= 0 && lane == __ffs(same) - 1) own[x] = prior + __popc(same);
            __syncwarp();
            if (i < end) {
                const int row = x >= 0 ? s.first_row[x] + prior + __popc(same & ((1u << lane) - 1u)) : -1;
                if (LOCAL) local_row[i] = row;
                if (publish) {
                    p.pair_row[i] = row;
                    if (row >= 0) p.row_pair[row] = i;
                }
            }
        }
    }
    if (publish) {
        const int cluster_warp = (int)rank * warps + warp, cluster_warps = (int)ctas * warps;
        if (p.align > 1)
            for (int x = cluster_warp; x < E; x += cluster_warps)
                for (int r = s.pad_begin[x] + lane; r < s.pad_end[x]; r += 32) p.row_pair[r] = -1;
        for (int r = total + cluster_warp * 32 + lane; r < p.capacity; r += cluster_warps * 32) p.row_pair[r] = -1;
    }
    if (!LOCAL) cluster_wait();
    return total;
}

template <typename Id>
__global__ void __launch_bounds__(kSortThreads) sort_tokens_kernel(const Id* ids, unsigned long long first, PlanView p)
{
    extern __shared__ int sort_smem[];
    const Sorted s(sort_smem, p.E, blockDim.x / 32);
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < (int)blockDim.x / 32 * p.E; i += blockDim.x) s.seen[i] = 0;
    __syncthreads();
    pdl_wait();
    sort_pairs<Id, false>(ids, first, p, s, true, nullptr);
}

// ---------------------------------------------------------------------------------------
// Row types: a piece of N elements, 16 bytes where the rows allow it, else 8, 4 or 2.
// ---------------------------------------------------------------------------------------
// A piece stays in 32-bit words until its elements are used: as elements, eight bf16 values take eight registers (the
// combine kernel 100 instead of 64, at half the loads in flight).
template <typename T, int N>
struct Piece {
    typedef T Type;
    static constexpr int kBytes = sizeof(T) * N;
    static_assert(kBytes == 16 || kBytes == 8 || kBytes == 4 || kBytes == 2, "one load");
    typedef typename std::conditional<kBytes >= 8, typename std::conditional<kBytes == 16, uint4, uint2>::type,
                                      typename std::conditional<kBytes == 4, uint32_t, uint16_t>::type>::type Raw;
    Raw raw;
    __device__ __forceinline__ uint32_t& word(int i) { return reinterpret_cast<uint32_t*>(&raw)[i]; }
    __device__ __forceinline__ uint32_t word(int i) const { return reinterpret_cast<const uint32_t*>(&raw)[i]; }
};

__device__ __forceinline__ float low_half(uint32_t w, __nv_bfloat16) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_half(uint32_t w, __nv_bfloat16) { return __uint_as_float(w & 0xffff0000u); }
__device__ __forceinline__ float low_half(uint32_t w, __half) { return __half2float(__ushort_as_half((unsigned short)w)); }
__device__ __forceinline__ float high_half(uint32_t w, __half) { return __half2float(__ushort_as_half((unsigned short)(w >> 16))); }
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi, __nv_bfloat16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_halves(float lo, float hi, __half) {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, int N>
__device__ __forceinline__ void unpack(const Piece<T, N>& p, float (&f)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = __uint_as_float(p.word(i));
    } else if constexpr (N == 1) {
        f[0] = low_half(p.raw, T{});
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) {
            f[2 * i] = low_half(p.word(i), T{});
            f[2 * i + 1] = high_half(p.word(i), T{});
        }
    }
}
template <typename T, int N>
__device__ __forceinline__ void pack(const float (&f)[N], Piece<T, N>& p) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) p.word(i) = __float_as_uint(f[i]);
    } else if constexpr (N == 1) {
        p.raw = (uint16_t)pack_halves(f[0], 0.0f, T{});
    } else {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) p.word(i) = pack_halves(f[2 * i], f[2 * i + 1], T{});
    }
}

// Plain loads throughout: a kernel may start while the one that writes its inputs still runs (see pdl_wait), which the
// read-only path does not allow.
template <typename P>
__device__ __forceinline__ P load_piece(const uint8_t* row, int i) {
    P p;
    p.raw = reinterpret_cast<const typename P::Raw*>(row)[i];
    return p;
}
template <typename P>
__device__ __forceinline__ void store_piece(uint8_t* row, int i, const P& v) { reinterpret_cast<typename P::Raw*>(row)[i] = v.raw; }

// What the CTAs in front of the tokens' do: padding_split of them write zeros to the padding rows of an expert (align > 1), the
// others to the rows behind the last expert (zero_unused).  In front, since an expert's padding takes longer than a token.
constexpr int kUnusedCtas = 592;   // four per SM
struct Fill {
    int padding_split, padding_ctas, unused_ctas;
    __host__ __device__ int ctas() const { return padding_ctas + unused_ctas; }
};

// Zeros in rows begin, begin + step ... below end.
template <typename P>
__device__ __forceinline__ void zero_rows(const Rows& rows, int pieces, const PlanView& p, int begin, int end, int step)
{
    P zero;
    memset(&zero, 0, sizeof(P));
    const int threads = blockDim.x * blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
    end = min(p.capacity, end);
    for (int r = max(0, begin); r < end; r += step)
        for (int i = blockIdx.y * threads + tid; i < pieces; i += gridDim.y * threads) store_piece(rows[r], i, zero);
}

template <typename P>
__device__ void fill_rows(const Rows& rows, int pieces, const PlanView& p, const Fill& fill, int cta)
{
    if (cta < fill.padding_ctas) {
        const int e = cta / fill.padding_split;
        zero_rows<P>(rows, pieces, p, p.expert_offset[e] + p.expert_count[e] + cta % fill.padding_split, p.expert_offset[e + 1],
                     fill.padding_split);
    } else {
        zero_rows<P>(rows, pieces, p, p.expert_offset[p.E] + cta - fill.padding_ctas, p.capacity, fill.unused_ctas);
    }
}

// ---------------------------------------------------------------------------------------
// Dispatch: a token is read once and stored to each of its rows.  blockDim.y tokens per CTA, blockDim.x threads over
// the row's pieces.
// ---------------------------------------------------------------------------------------
template <typename P>
__device__ __forceinline__ void copy_token(const uint8_t* src, const Rows& rows, const int (&row)[kMaxTopK], int K, int pieces, int begin,
                                           int step)
{
    constexpr int kUnroll = P::kBytes == 16 ? 4 : 8;
    for (int i0 = begin; i0 < pieces; i0 += step * kUnroll) {
        P v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (i0 + u * step < pieces) v[u] = load_piece<P>(src, i0 + u * step);
#pragma unroll
        for (int k = 0; k < kMaxTopK; ++k) {
            if (k >= K) break;
            if (row[k] < 0) continue;
            uint8_t* dst = rows[row[k]];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (i0 + u * step < pieces) store_piece(dst, i0 + u * step, v[u]);
        }
    }
}

template <typename T, int N>
__global__ void __launch_bounds__(256) dispatch_rows_kernel(Rows x, Rows rows, int pieces, Fill fill, PlanView p)
{
    typedef Piece<T, N> P;
    pdl_launch_dependents();
    pdl_wait();
    const int cta = (int)blockIdx.x - fill.ctas();
    if (cta < 0) {
        fill_rows<P>(rows, pieces, p, fill, blockIdx.x);
        return;
    }
    const int t = cta * blockDim.y + threadIdx.y;
    if (t >= p.T) return;
    const long long pair0 = (long long)t * p.K;
    int row[kMaxTopK], any = -1;
#pragma unroll
    for (int k = 0; k < kMaxTopK; ++k) {
        row[k] = k < p.K ? row_of_pair(p, pair0 + k) : -1;
        any = max(any, row[k]);
    }
    if (any < 0) return;
    copy_token<P>(x[t], rows, row, p.K, pieces, blockIdx.y * blockDim.x + threadIdx.x, gridDim.y * blockDim.x);
}

// A small batch sorted and copied by one kernel: every CTA sorts all pairs for itself, one of them writes the plan.  Up to 2048
// pairs that costs less than a second launch and the wait between the two (top 8 of 256 experts, 7168 columns, align 1, given
// rows, us by one and by two kernels, call by call: 1 token 8.2 / 11.3, 128 tokens 13.2 / 17.4, 256 tokens 16.4 / 19.4, 512 tokens
// 28.7 / 25.6; replayed in a graph: 3.5 / 4.5, 7.9 / 9.1, 12.1 / 12.1; align 8 in a graph: 7.2 / 7.6, 12.5 / 14.0, 14.8 / 15.2).
// The rule looks at neither align nor new rows, where it costs more than it gives: the CTAs that write zeros sort as well, and
// there are thousands of them (in a graph, 1 token and 256 tokens: align 32 40 / 15 and 42 / 31, align 128 41 / 16 and 75 / 79;
// new rows at align 1 12.9 / 6.7 and 18.1 / 14.1).
constexpr int kSmallPairs = 2048, kSmallTokens = 256, kSmallThreads = 256;

template <typename Id, typename T, int N>
__global__ void __launch_bounds__(kSmallThreads) sort_and_dispatch_kernel(const Id* ids, unsigned long long first, Rows x, Rows rows,
                                                                          int pieces, Fill fill, PlanView p)
{
    typedef Piece<T, N> P;
    extern __shared__ int sort_smem[];
    const Sorted s(sort_smem, p.E, kSmallThreads / 32);
    int* const local_row = s.pad_end + p.E;
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < kSmallThreads / 32 * p.E; i += kSmallThreads) s.seen[i] = 0;
    __syncthreads();
    pdl_wait();
    const int total = sort_pairs<Id, true>(ids, first, p, s, blockIdx.x == 0 && blockIdx.y == 0, local_row);
    __syncthreads();
    const int cta = (int)blockIdx.x - fill.ctas();
    if (cta < 0) {
        if ((int)blockIdx.x < fill.padding_ctas) {
            const int e = blockIdx.x / fill.padding_split;
            zero_rows<P>(rows, pieces, p, s.pad_begin[e] + blockIdx.x % fill.padding_split, s.pad_end[e], fill.padding_split);
        } else {
            zero_rows<P>(rows, pieces, p, total + blockIdx.x - fill.padding_ctas, p.capacity, fill.unused_ctas);
        }
        return;
    }
    int row[kMaxTopK];
#pragma unroll
    for (int k = 0; k < kMaxTopK; ++k) row[k] = k < p.K ? local_row[cta * p.K + k] : -1;
    copy_token<P>(x[cta], rows, row, p.K, pieces, blockIdx.y * kSmallThreads + threadIdx.x, gridDim.y * kSmallThreads);
}

// ---------------------------------------------------------------------------------------
// Combine: eight rows' pieces of a column are requested together, then added in pair order.
// ---------------------------------------------------------------------------------------
constexpr int kRowsAtOnce = 8;

template <typename T, int N, bool WEIGHTED>
__global__ void __launch_bounds__(256, 4) combine_rows_kernel(Rows y, const float* weights, Rows out, int pieces,
                                                           PlanView p)
{
    typedef Piece<T, N> P;
    pdl_launch_dependents();
    pdl_wait();
    const int t = blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= p.T) return;
    const long long pair0 = (long long)t * p.K;
    for (int i = blockIdx.y * blockDim.x + threadIdx.x; i < pieces; i += gridDim.y * blockDim.x) {
        float acc[N];
#pragma unroll
        for (int j = 0; j < N; ++j) acc[j] = 0.0f;
        for (int k0 = 0; k0 < p.K; k0 += kRowsAtOnce) {
            int row[kRowsAtOnce];
            float w[kRowsAtOnce];
            P v[kRowsAtOnce];
#pragma unroll
            for (int k = 0; k < kRowsAtOnce; ++k) {
                row[k] = k0 + k < p.K ? row_of_pair(p, pair0 + k0 + k) : -1;
                w[k] = WEIGHTED && row[k] >= 0 ? weights[pair0 + k0 + k] : 1.0f;
            }
#pragma unroll
            for (int k = 0; k < kRowsAtOnce; ++k)
                if (row[k] >= 0) v[k] = load_piece<P>(y[row[k]], i);
#pragma unroll
            for (int k = 0; k < kRowsAtOnce; ++k)
                if (row[k] >= 0) {
                    float f[N];
                    unpack(v[k], f);
#pragma unroll
                    for (int j = 0; j < N; ++j) acc[j] = WEIGHTED ? fmaf(f[j], w[k], acc[j]) : acc[j] + f[j];
                }
        }
        P o;
        pack(acc, o);
        store_piece(out[t], i, o);
    }
}

// ---------------------------------------------------------------------------------------
// The combine's gradient: a CTA takes a token.  A thread reads a piece of the token's gradient once, and with it eight rows'
// pieces of y: it scales the gradient into those rows' gradients and adds up the products with them.  The sums meet over
// the warp and in shared memory, in a fixed order.
// ---------------------------------------------------------------------------------------
constexpr int kGradThreads = 256;

template <typename T, int N>
__global__ void __launch_bounds__(kGradThreads, 3) combine_grad_kernel(Rows grad_out, Rows y, const float* weights, Rows grad_y,
                                                                       float* grad_weights, int pieces, Fill fill, PlanView p)
{
    typedef Piece<T, N> P;
    __shared__ int live_row[kMaxTopK], live_k[kMaxTopK], live_count;
    __shared__ float part_sum[kRowsAtOnce][kGradThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int t = (int)blockIdx.x - fill.ctas();
    if (t < 0) {
        fill_rows<P>(grad_y, pieces, p, fill, blockIdx.x);
        return;
    }
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, warps = blockDim.x / 32;
    if (warp == 0) {
        const int row = lane < p.K ? row_of_pair(p, (long long)t * p.K + lane) : -1;
        const unsigned live = __ballot_sync(~0u, row >= 0);
        if (row >= 0) {
            const int at = __popc(live & ((1u << lane) - 1u));
            live_row[at] = row;
            live_k[at] = lane;
        } else if (lane < p.K && grad_weights) {
            grad_weights[(long long)t * p.K + lane] = 0.0f;
        }
        if (lane == 0) live_count = __popc(live);
    }
    __syncthreads();
    const int count = live_count;
    const uint8_t* src = grad_out[t];
    for (int base = 0; base < count; base += kRowsAtOnce) {
        const int rows = min(kRowsAtOnce, count - base);
        int row[kRowsAtOnce];
        float w[kRowsAtOnce], sum[kRowsAtOnce];
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) {
            row[k] = k < rows ? live_row[base + k] : 0;
            w[k] = k < rows && grad_y.base ? weights[(long long)t * p.K + live_k[base + k]] : 0.0f;
            sum[k] = 0.0f;
        }
        for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
            const P piece = load_piece<P>(src, i);
            P v[kRowsAtOnce];
            if (grad_weights) {
#pragma unroll
                for (int k = 0; k < kRowsAtOnce; ++k)
                    if (k < rows) v[k] = load_piece<P>(y[row[k]], i);
            }
#pragma unroll
            for (int k = 0; k < kRowsAtOnce; ++k) {
                if (k >= rows) break;
                float g[N], f[N];
                unpack(piece, g);
                if (grad_weights) {
                    unpack(v[k], f);
#pragma unroll
                    for (int n = 0; n < N; ++n) sum[k] = fmaf(g[n], f[n], sum[k]);
                }
                if (grad_y.base) {
                    P o;
#pragma unroll
                    for (int n = 0; n < N; ++n) f[n] = g[n] * w[k];
                    pack(f, o);
                    store_piece(grad_y[row[k]], i, o);
                }
            }
        }
        if (grad_weights) {
#pragma unroll
            for (int k = 0; k < kRowsAtOnce; ++k) {
                if (k >= rows) break;
                float s = sum[k];
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(~0u, s, d);
                if (lane == 0) part_sum[k][warp] = s;
            }
            __syncthreads();
            if ((int)threadIdx.x < rows) {
                float s = 0.0f;
                for (int q = 0; q < warps; ++q) s += part_sum[threadIdx.x][q];
                grad_weights[(long long)t * p.K + live_k[base + threadIdx.x]] = s;
            }
            __syncthreads();
        }
    }
}

// ---------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------
int64_t plan_rows(int64_t T, int64_t K, int64_t E, int64_t align)
{
    if (T < 0 || K < 1 || K > kMaxTopK || E < 1 || E > kMaxExperts || align < 1 || align > kMaxAlign) return -1;
    const int64_t pairs = T * K, most = pairs + (E < pairs ? E : pairs) * (align - 1);
    const int64_t rows = (most + align - 1) / align * align;
    return rows <= INT32_MAX - 2 * kSortThreads * 16 ? rows : -1;   // index arithmetic of the sort stays in 32 bits
}

struct Call {
    char* err;
    size_t err_len;
    int device = 0;
    const char* what = nullptr;

    template <typename... A>
    int bad(const char* fmt, A... a) const { return refuse(err, err_len, MOE_FP8_B200_ERR_INVALID_ARGUMENT, fmt, a...); }
    int cuda(cudaError_t e) const {
        return e == cudaSuccess ? MOE_FP8_B200_OK
                                : refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "launch failed: %s", cudaGetErrorString(e));
    }
    int begin() {
        if (cudaGetDevice(&device) != cudaSuccess) return refuse(err, err_len, MOE_FP8_B200_ERR_CUDA, "cudaGetDevice failed");
        return MOE_FP8_B200_OK;
    }
    int tensor(const char* name, const void* p, size_t align) const {
        if (!p) return bad("%s is NULL", name);
        if ((uintptr_t)p % align) return bad("%s is not aligned to its element size", name);
        if (!memory_of_device(p, device))
            return bad("%s does not live on the current CUDA device (make the tensors' GPU current before the call)", name);
        return MOE_FP8_B200_OK;
    }
};

int check_apart(const Call& call, const Extent& written, const Extent& other)
{
    return share_memory(written, other) ? call.bad("%s and %s share memory", written.name, other.name) : MOE_FP8_B200_OK;
}

struct PlanExtents {
    Extent a[4];
    explicit PlanExtents(const PlanView& p)
        : a{{"pair_row", p.pair_row, 1, 4ll * p.pairs, 0},
            {"row_pair", p.row_pair, 1, 4ll * p.capacity, 0},
            {"expert_offset", p.expert_offset, 1, 4ll * (p.E + 1), 0},
            {"expert_count", p.expert_count, 1, 4ll * p.E, 0}} {}
};

int check_apart_from_plan(const Call& call, const Extent& other, const PlanView& p)
{
    const PlanExtents plan(p);
    for (const Extent& e : plan.a)
        if (share_memory(other, e)) return call.bad("%s and the plan's %s share memory", other.name, e.name);
    return MOE_FP8_B200_OK;
}

int check_plan(Call& call, const moe_fp8_b200_plan* plan, PlanView& v)
{
    if (!plan) return call.bad("plan is NULL");
    const int64_t rows = plan_rows(plan->num_tokens, plan->top_k, plan->num_experts, plan->align);
    if (rows < 0)
        return call.bad("plan sizes out of range: num_tokens %d, top_k %d (1 .. %d), num_experts %d (1 .. %d), align %d (1 .. %d)",
                        plan->num_tokens, plan->top_k, kMaxTopK, plan->num_experts, kMaxExperts, plan->align, kMaxAlign);
    v = {plan->num_tokens, plan->top_k, plan->num_experts, plan->align, plan->num_tokens * plan->top_k, (int)rows,
         plan->pair_row, plan->row_pair, plan->expert_offset, plan->expert_count};
    const PlanExtents arrays(v);
    for (int i = 0; i < 4; ++i)
        for (int j = i + 1; j < 4; ++j) {
            const int rc = check_apart(call, arrays.a[i], arrays.a[j]);
            if (rc != MOE_FP8_B200_OK) return rc;
        }
    int rc = call.begin();
    if (rc == MOE_FP8_B200_OK && plan->num_tokens > 0) {
        rc = call.tensor("pair_row", plan->pair_row, 4);
        if (rc == MOE_FP8_B200_OK) rc = call.tensor("row_pair", plan->row_pair, 4);
    }
    if (rc == MOE_FP8_B200_OK) rc = call.tensor("expert_offset", plan->expert_offset, 4);
    if (rc == MOE_FP8_B200_OK) rc = call.tensor("expert_count", plan->expert_count, 4);
    return rc;
}

int element_size(int dtype)
{
    return dtype == MOE_FP8_B200_BF16 || dtype == MOE_FP8_B200_FP16 ? 2 : dtype == MOE_FP8_B200_FP32 ? 4 : 0;
}

int check_rows(const Call& call, const char* name, const void* p, int64_t stride, int64_t rows, int dtype, int hidden, bool written,
               Extent& out)
{
    const int size = element_size(dtype);
    if (!size) return call.bad("unknown row type %d", dtype);
    if (hidden < 1 || hidden > (1 << 24)) return call.bad("hidden %d is not in 1 .. 2^24", hidden);
    if (stride < 0 || stride > ((int64_t)1 << 40)) return call.bad("%s: row stride out of range", name);
    if (written && rows > 1 && stride < hidden) return call.bad("%s: rows of %d elements overlap at a stride of %lld", name, hidden, (long long)stride);
    const int rc = call.tensor(name, p, size);
    out = {name, p, rows, (int64_t)hidden * size, stride * size};
    return rc;
}

// The widest piece, up to 16 bytes, that the rows of both matrices consist of.
int piece_bytes(const Extent& a, const Extent& b, const Extent& c = {})
{
    uintptr_t all = 16;
    for (const Extent* e : {&a, &b, &c})
        if (e->base) all |= (uintptr_t)e->base | (uintptr_t)e->row_bytes | (e->rows > 1 ? (uintptr_t)e->stride_bytes : 0);
    return (int)(all & (~all + 1));
}

// f(type, elements of a piece)
template <typename F>
cudaError_t with_pieces(int dtype, int bytes, F f)
{
    auto of = [&](auto type) {
        typedef decltype(type) T;
        if constexpr (sizeof(T) == 2)
            if (bytes == 2) return f(type, std::integral_constant<int, 1>{});
        return bytes == 16  ? f(type, std::integral_constant<int, 16 / sizeof(T)>{})
               : bytes == 8 ? f(type, std::integral_constant<int, 8 / sizeof(T)>{})
                            : f(type, std::integral_constant<int, 4 / sizeof(T)>{});
    };
    return dtype == MOE_FP8_B200_BF16 ? of(__nv_bfloat16{}) : dtype == MOE_FP8_B200_FP16 ? of(__half{}) : of(float{});
}

Rows as_rows(const Extent& e) { return {static_cast<uint8_t*>(const_cast<void*>(e.base)), e.stride_bytes}; }

// Threads and CTAs of a kernel that walks rows of `pieces` pieces: as few passes over a row as 256 threads allow, spread
// evenly; several short rows per CTA; where tokens are few, a row's passes become CTAs of their own so that every SM has
// work.
struct Shape {
    dim3 block;
    int token_ctas, splits;
};
Shape shape_for(int T, int pieces)
{
    constexpr int kThreads = 256, kManyCtas = 148 * 8;
    const int passes = (pieces + kThreads - 1) / kThreads;
    const int threads = ((pieces + passes - 1) / passes + 31) / 32 * 32;
    const int tokens = kThreads / threads;
    const int ctas = (T + tokens - 1) / tokens;
    int splits = (kManyCtas + ctas - 1) / ctas;
    if (splits > passes) splits = passes;
    return {dim3(threads, tokens), ctas, splits};
}

template <typename Id>
cudaError_t launch_sort(const void* ids, int64_t first, const PlanView& p, cudaStream_t stream)
{
    // The cluster grows with the batch: a CTA takes 32 pairs per warp at least.  Sixteen CTAs (98304 pairs: 16.4 us, 22.5 with
    // eight) have to be allowed for, and lie within one GPC.
    unsigned ctas = 1;
    while (ctas < 16 && p.pairs > (int)ctas * kSortThreads) ctas *= 2;
    if (ctas == 16) {
        const cudaError_t e = cudaFuncSetAttribute(sort_tokens_kernel<Id>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
    }
    const int need = p.E > p.pairs ? p.E : p.pairs;
    const int threads = need >= kSortThreads ? kSortThreads : need <= 128 ? 128 : (need + 31) / 32 * 32;
    const size_t smem = sort_smem_bytes(threads, p.E);
    if (smem > 48 * 1024) {
        // the same value in every call: the attribute belongs to the kernel, and another thread's call may stand between this and the launch
        const cudaError_t e = cudaFuncSetAttribute(sort_tokens_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)sort_smem_bytes(kSortThreads, kMaxExperts));
        if (e != cudaSuccess) return e;
    }
    return launch_after(sort_tokens_kernel<Id>, dim3(ctas), dim3(threads), smem, ctas, stream, static_cast<const Id*>(ids),
                        (unsigned long long)first, p);
}

cudaError_t enqueue_sort(const void* ids, int id_bits, int64_t first, const PlanView& p, cudaStream_t stream)
{
    return id_bits == 32 ? launch_sort<int32_t>(ids, first, p, stream) : launch_sort<int64_t>(ids, first, p, stream);
}

template <typename T, int N>
cudaError_t launch_dispatch(const Extent& x, const Extent& rows, const PlanView& p, const Fill& fill, cudaStream_t stream)
{
    const int pieces = (int)(x.row_bytes / (int64_t)(sizeof(T) * N));
    const Shape s = shape_for(p.T, pieces);
    return launch_after(dispatch_rows_kernel<T, N>, dim3(fill.ctas() + s.token_ctas, s.splits), s.block, 0, 1, stream, as_rows(x),
                        as_rows(rows), pieces, fill, p);
}

Fill fill_for(const PlanView& p, int zero_unused)
{
    const int split = p.align >= 32 ? 8 : 1;   // an expert's padding is align / 2 rows on average
    return {split, p.align > 1 ? p.E * split : 0, zero_unused ? kUnusedCtas : 0};
}

template <typename Id, typename T, int N>
cudaError_t launch_small(const void* ids, int64_t first, const Extent& x, const Extent& rows, const PlanView& p, const Fill& fill,
                         cudaStream_t stream)
{
    const int pieces = (int)(x.row_bytes / (int64_t)(sizeof(T) * N));
    const int passes = (pieces + kSmallThreads - 1) / kSmallThreads;
    int splits = (148 + p.T - 1) / p.T;
    if (splits > passes) splits = passes;
    const size_t smem = sort_smem_bytes(kSmallThreads, p.E) + sizeof(int) * (size_t)p.pairs;
    return launch_after(sort_and_dispatch_kernel<Id, T, N>, dim3(fill.ctas() + p.T, splits), dim3(kSmallThreads), smem, 1, stream,
                        static_cast<const Id*>(ids), (unsigned long long)first, as_rows(x), as_rows(rows), pieces, fill, p);
}

// The copy needs no arithmetic: one form per element size.  `ids`: sorted here first, if the batch is small in the same kernel.
cudaError_t enqueue_dispatch(const void* ids, int id_bits, int64_t first, const Extent& x, const Extent& rows, int dtype,
                             const PlanView& p, int zero_unused, cudaStream_t stream)
{
    const Fill fill = fill_for(p, zero_unused);
    return with_pieces(element_size(dtype) == 2 ? MOE_FP8_B200_FP16 : dtype, piece_bytes(x, rows), [&](auto type, auto n) {
        typedef decltype(type) T;
        constexpr int N = decltype(n)::value;
        if (ids && p.pairs <= kSmallPairs && p.T <= kSmallTokens && p.E <= kSmallThreads)
            return id_bits == 32 ? launch_small<int32_t, T, N>(ids, first, x, rows, p, fill, stream)
                                 : launch_small<int64_t, T, N>(ids, first, x, rows, p, fill, stream);
        const cudaError_t e = ids ? enqueue_sort(ids, id_bits, first, p, stream) : cudaSuccess;
        return e == cudaSuccess ? launch_dispatch<T, N>(x, rows, p, fill, stream) : e;
    });
}

template <typename T, int N>
cudaError_t launch_combine_rows(const Extent& y, const float* weights, const Extent& out, const PlanView& p, cudaStream_t stream)
{
    const int pieces = (int)(y.row_bytes / (int64_t)(sizeof(T) * N));
    const Shape s = shape_for(p.T, pieces);
    return launch_after(weights ? combine_rows_kernel<T, N, true> : combine_rows_kernel<T, N, false>, dim3(s.token_ctas, s.splits),
                        s.block, 0, 1, stream, as_rows(y), weights, as_rows(out), pieces, p);
}

template <typename T, int N>
cudaError_t launch_combine_grad(const Extent& grad_out, const Extent& y, const float* weights, const Extent& grad_y,
                                float* grad_weights, const PlanView& p, int zero_unused, cudaStream_t stream)
{
    const int pieces = (int)(grad_out.row_bytes / (int64_t)(sizeof(T) * N));
    const Fill fill = grad_y.base ? fill_for(p, zero_unused) : Fill{1, 0, 0};
    const int passes = (pieces + kGradThreads - 1) / kGradThreads, threads = ((pieces + passes - 1) / passes + 31) / 32 * 32;
    return launch_after(combine_grad_kernel<T, N>, dim3(fill.ctas() + p.T), dim3(threads), 0, 1, stream, as_rows(grad_out), as_rows(y),
                        weights, as_rows(grad_y), grad_weights, pieces, fill, p);
}

// The ids are read twice, by every CTA of the small kernel: the plan written over them would be read as ids.
int check_ids(const Call& call, const void* ids, int id_bits, int64_t first, const PlanView& p)
{
    if (id_bits != 32 && id_bits != 64) return call.bad("id_bits must be 32 or 64, got %d", id_bits);
    if (first > INT64_MAX - (p.E - 1)) return call.bad("first_expert %lld: %d experts from it on are not 64-bit ids", (long long)first, p.E);
    const int rc = call.tensor("topk_idx", ids, id_bits / 8);
    return rc == MOE_FP8_B200_OK ? check_apart_from_plan(call, {"topk_idx", ids, 1, (int64_t)p.pairs * (id_bits / 8), 0}, p) : rc;
}

}  // namespace
}  // namespace moe

using namespace moe;

extern "C" {

int64_t moe_fp8_b200_plan_rows(int num_tokens, int top_k, int num_experts, int align)
{
    return plan_rows(num_tokens, top_k, num_experts, align);
}

int moe_fp8_b200_sort_tokens(const void* topk_idx, int id_bits, int64_t first_expert, const moe_fp8_b200_plan* plan,
                             void* stream, char* err, size_t err_len)
{
    Call call{err, err_len};
    PlanView p;
    int rc = check_plan(call, plan, p);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_ids(call, topk_idx, id_bits, first_expert, p);
    if (rc != MOE_FP8_B200_OK) return rc;
    return call.cuda(enqueue_sort(topk_idx, id_bits, first_expert, p, static_cast<cudaStream_t>(stream)));
}

int moe_fp8_b200_dispatch_rows(const void* x, int64_t x_stride, void* rows, int64_t rows_stride, int dtype, int hidden,
                               const moe_fp8_b200_plan* plan, int zero_unused, void* stream, char* err, size_t err_len)
{
    Call call{err, err_len};
    PlanView p;
    Extent ex, er;
    int rc = check_plan(call, plan, p);
    if (rc != MOE_FP8_B200_OK || p.T == 0) return rc;
    rc = check_rows(call, "x", x, x_stride, p.T, dtype, hidden, false, ex);
    if (rc == MOE_FP8_B200_OK) rc = check_rows(call, "rows", rows, rows_stride, p.capacity, dtype, hidden, true, er);
    if (rc == MOE_FP8_B200_OK) rc = check_apart(call, er, ex);
    if (rc == MOE_FP8_B200_OK) rc = check_apart_from_plan(call, er, p);
    if (rc != MOE_FP8_B200_OK) return rc;
    return call.cuda(enqueue_dispatch(nullptr, 0, 0, ex, er, dtype, p, zero_unused, static_cast<cudaStream_t>(stream)));
}

int moe_fp8_b200_sort_and_dispatch(const void* topk_idx, int id_bits, int64_t first_expert, const void* x, int64_t x_stride,
                                   void* rows, int64_t rows_stride, int dtype, int hidden, const moe_fp8_b200_plan* plan,
                                   int zero_unused, void* stream, char* err, size_t err_len)
{
    Call call{err, err_len};
    PlanView p;
    Extent ex, er;
    int rc = check_plan(call, plan, p);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_ids(call, topk_idx, id_bits, first_expert, p);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_rows(call, "x", x, x_stride, p.T, dtype, hidden, false, ex);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_rows(call, "rows", rows, rows_stride, p.capacity, dtype, hidden, true, er);
    if (rc == MOE_FP8_B200_OK && p.T > 0) {
        Extent ei = {"topk_idx", topk_idx, 1, (int64_t)p.pairs * (id_bits / 8), 0};
        for (const Extent* other : {&ex, &ei})
            if (rc == MOE_FP8_B200_OK) rc = check_apart(call, er, *other);
        for (const Extent* other : {&er, &ex})
            if (rc == MOE_FP8_B200_OK) rc = check_apart_from_plan(call, *other, p);
    }
    if (rc != MOE_FP8_B200_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return call.cuda(p.T > 0 ? enqueue_dispatch(topk_idx, id_bits, first_expert, ex, er, dtype, p, zero_unused, s)
                             : enqueue_sort(topk_idx, id_bits, first_expert, p, s));
}

int moe_fp8_b200_combine_rows(const void* y, int64_t y_stride, const float* weights, void* out, int64_t out_stride, int dtype,
                              int hidden, const moe_fp8_b200_plan* plan, void* stream, char* err, size_t err_len)
{
    Call call{err, err_len};
    PlanView p;
    Extent ey, eo;
    int rc = check_plan(call, plan, p);
    if (rc != MOE_FP8_B200_OK || p.T == 0) return rc;
    rc = check_rows(call, "y", y, y_stride, p.capacity, dtype, hidden, false, ey);
    if (rc == MOE_FP8_B200_OK) rc = check_rows(call, "out", out, out_stride, p.T, dtype, hidden, true, eo);
    if (rc == MOE_FP8_B200_OK && weights) rc = call.tensor("weights", weights, 4);
    if (rc == MOE_FP8_B200_OK) rc = check_apart(call, eo, ey);
    if (rc == MOE_FP8_B200_OK) rc = check_apart_from_plan(call, eo, p);
    if (rc == MOE_FP8_B200_OK && weights) rc = check_apart(call, eo, {"weights", weights, 1, 4ll * p.pairs, 0});
    if (rc != MOE_FP8_B200_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return call.cuda(with_pieces(dtype, piece_bytes(ey, eo), [&](auto type, auto n) {
        return launch_combine_rows<decltype(type), decltype(n)::value>(ey, weights, eo, p, s);
    }));
}

int moe_fp8_b200_combine_rows_backward(const void* grad_out, int64_t grad_out_stride, const void* y, int64_t y_stride,
                                       const float* weights, void* grad_y, int64_t grad_y_stride, float* grad_weights, int dtype,
                                       int hidden, const moe_fp8_b200_plan* plan, int zero_unused, void* stream, char* err,
                                       size_t err_len)
{
    Call call{err, err_len};
    PlanView p;
    Extent eg, ey = {}, ed = {};
    int rc = check_plan(call, plan, p);
    if (rc != MOE_FP8_B200_OK || p.T == 0 || (!grad_y && !grad_weights)) return rc;
    rc = check_rows(call, "grad_out", grad_out, grad_out_stride, p.T, dtype, hidden, false, eg);
    if (rc == MOE_FP8_B200_OK && (grad_y || weights)) rc = call.tensor("weights", weights, 4);
    if (rc == MOE_FP8_B200_OK && grad_y) {
        rc = check_rows(call, "grad_y", grad_y, grad_y_stride, p.capacity, dtype, hidden, true, ed);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, ed, eg);
        if (rc == MOE_FP8_B200_OK) rc = check_apart_from_plan(call, ed, p);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, ed, {"weights", weights, 1, 4ll * p.pairs, 0});
    }
    if (rc == MOE_FP8_B200_OK && grad_weights) {
        rc = check_rows(call, "y", y, y_stride, p.capacity, dtype, hidden, false, ey);
        if (rc == MOE_FP8_B200_OK) rc = call.tensor("grad_weights", grad_weights, 4);
        const Extent dw = {"grad_weights", grad_weights, 1, 4ll * p.pairs, 0};
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, ed, ey);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, eg);
        if (rc == MOE_FP8_B200_OK) rc = check_apart_from_plan(call, dw, p);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, ey);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, ed);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, {"weights", weights, 1, 4ll * p.pairs, 0});
    }
    if (rc != MOE_FP8_B200_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    return call.cuda(with_pieces(dtype, piece_bytes(eg, ey, ed), [&](auto type, auto n) {
        return launch_combine_grad<decltype(type), decltype(n)::value>(eg, ey, weights, ed, grad_weights, p, zero_unused, s);
    }));
}

}  // extern "C"
