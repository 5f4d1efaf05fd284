// Tokens sorted by expert and back (declared in include/moe_fp8_b200.h): the plan that gives every (token, expert) pair
// its packed row, the copy of the tokens to those rows, the weighted sum of a token's rows, and the gradients.
//
// The movement is bound by HBM: a row is read or written once, a token once.  There is no atomic anywhere, so results
// do not depend on the order in which CTAs run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstring>

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
// pairs of its expert in the same 32 comes from a match over the warp.
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

template <typename Id>
__global__ void __launch_bounds__(kSortThreads) sort_tokens_kernel(const Id* ids, unsigned long long first,
                                                                   PlanView p)
{
    extern __shared__ int sort_smem[];
    __shared__ int warp_sum[32];
    const int E = p.E, warps = blockDim.x / 32, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    int* seen = sort_smem;              // [warps][E] pairs of the expert in earlier warps, then in earlier rounds too
    int* mine = seen + warps * E;       // [E] pairs in this CTA
    int* first_row = mine + E;          // [E] row of this CTA's first pair
    int* pad_begin = first_row + E;     // [E] padding rows of the expert
    int* pad_end = pad_begin + E;
    const unsigned rank = cluster_rank(), ctas = cluster_size();
    pdl_launch_dependents();
    for (int i = threadIdx.x; i < warps * E; i += blockDim.x) seen[i] = 0;
    __syncthreads();
    pdl_wait();

    const int per_cta = (p.pairs + (int)ctas - 1) / (int)ctas;
    const int cta_end = min(p.pairs, ((int)rank + 1) * per_cta);
    const int per_warp = (per_cta + warps * 32 - 1) / (warps * 32) * 32;
    const int begin = min(cta_end, (int)rank * per_cta + warp * per_warp);
    const int end = min(cta_end, begin + per_warp);
    int* own = seen + warp * E;
    for (int i = begin + lane; i < end; i += 32) {
        const int e = expert_of(ids, i, first, E);
        if (e >= 0) atomicAdd(own + e, 1);
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int run = 0;
        for (int w = 0; w < warps; ++w) {
            const int c = seen[w * E + e];
            seen[w * E + e] = run;
            run += c;
        }
        mine[e] = run;
    }
    cluster_arrive();
    cluster_wait();
    // one thread per expert (the launch has at least E)
    const int e = threadIdx.x;
    int before = 0, all = 0, padded = 0;
    if (e < E) {
        for (unsigned c = 0; c < ctas; ++c) {
            const int v = load_cluster(mine + e, c);
            if (c < rank) before += v;
            all += v;
        }
        padded = (all + p.align - 1) / p.align * p.align;
    }
    cluster_arrive();   // this CTA reads no other one's memory any more; the wait stands at the end
    int upto = padded;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int v = __shfl_up_sync(~0u, upto, d);
        if (lane >= d) upto += v;
    }
    if (lane == 31) warp_sum[warp] = upto;
    __syncthreads();
    int total = 0;
    for (int w = 0; w < warps; ++w) {
        if (w < warp) upto += warp_sum[w];
        total += warp_sum[w];
    }
    if (e < E) {
        const int offset = upto - padded;
        first_row[e] = offset + before;
        pad_begin[e] = offset + all;
        pad_end[e] = upto;
        if (rank == 0) {
            p.expert_offset[e] = offset;
            p.expert_count[e] = all;
        }
    }
    if (rank == 0 && threadIdx.x == 0) p.expert_offset[E] = total;
    __syncthreads();

    for (int i0 = begin; i0 < end; i0 += 32) {
        const int i = i0 + lane;
        const int x = i < end ? expert_of(ids, i, first, E) : -1;
        const unsigned same = __match_any_sync(~0u, x);
        const int prior = x >= 0 ? own[x] : 0;
        __syncwarp();
        if (x >= 0 && lane == __ffs(same) - 1) own[x] = prior + __popc(same);
        __syncwarp();
        if (i < end) {
            const int row = x >= 0 ? first_row[x] + prior + __popc(same & ((1u << lane) - 1u)) : -1;
            p.pair_row[i] = row;
            if (row >= 0) p.row_pair[row] = i;
        }
    }
    const int cluster_warp = (int)rank * warps + warp, cluster_warps = (int)ctas * warps;
    if (p.align > 1)
        for (int x = cluster_warp; x < E; x += cluster_warps)
            for (int r = pad_begin[x] + lane; r < pad_end[x]; r += 32) p.row_pair[r] = -1;
    for (int r = total + cluster_warp * 32 + lane; r < p.capacity; r += cluster_warps * 32) p.row_pair[r] = -1;
    cluster_wait();
}

// ---------------------------------------------------------------------------------------
// Row types: a piece of N elements, 16 bytes where the rows allow it, else one element.
// ---------------------------------------------------------------------------------------
template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ float from_float(float v) { return v; }

template <typename T, int N>
struct alignas(sizeof(T) * N) Piece {
    T v[N];
};

// Plain loads throughout: a kernel may start while the one that writes its inputs still runs (see pdl_wait), which the
// read-only path does not allow.
template <typename P>
__device__ __forceinline__ P load_piece(const uint8_t* row, int i) { return reinterpret_cast<const P*>(row)[i]; }
template <typename P>
__device__ __forceinline__ void store_piece(uint8_t* row, int i, const P& v) { reinterpret_cast<P*>(row)[i] = v; }

// What the CTAs behind the tokens' do: CTA i < E writes zeros to the padding rows of expert i (align > 1), the others to the
// rows behind the last expert (zero_unused).
constexpr int kUnusedCtas = 592;   // four per SM
struct Fill {
    int padding_ctas, unused_ctas;
    int ctas() const { return padding_ctas + unused_ctas; }
};

template <typename P>
__device__ void fill_rows(const Rows& rows, int pieces, const PlanView& p, const Fill& fill, int cta)
{
    int begin, end, step = 1;
    if (cta < fill.padding_ctas) {
        begin = p.expert_offset[cta] + p.expert_count[cta];
        end = p.expert_offset[cta + 1];
    } else {
        begin = p.expert_offset[p.E];
        end = p.capacity;
        step = fill.unused_ctas;
    }
    begin = max(0, begin) + (step > 1 ? cta - fill.padding_ctas : 0);
    end = min(p.capacity, end);
    P zero;
    memset(&zero, 0, sizeof(P));
    const int threads = blockDim.x * blockDim.y, tid = threadIdx.y * blockDim.x + threadIdx.x;
    for (int r = begin; r < end; r += step)
        for (int i = blockIdx.y * threads + tid; i < pieces; i += gridDim.y * threads) store_piece(rows[r], i, zero);
}

// ---------------------------------------------------------------------------------------
// Dispatch: a token is read once and stored to each of its rows.  blockDim.y tokens per CTA, blockDim.x threads over
// the row's pieces; the CTAs behind the tokens' write the padding.
// ---------------------------------------------------------------------------------------
constexpr int kUnroll = 4;

template <typename T, int N>
__global__ void __launch_bounds__(256) dispatch_rows_kernel(Rows x, Rows rows, int pieces, int token_ctas, Fill fill,
                                                            PlanView p)
{
    typedef Piece<T, N> P;
    pdl_launch_dependents();
    pdl_wait();
    if ((int)blockIdx.x >= token_ctas) {
        fill_rows<P>(rows, pieces, p, fill, (int)blockIdx.x - token_ctas);
        return;
    }
    const int t = blockIdx.x * blockDim.y + threadIdx.y;
    if (t >= p.T) return;
    const long long pair0 = (long long)t * p.K;
    int row[kMaxTopK], any = -1;
#pragma unroll
    for (int k = 0; k < kMaxTopK; ++k) {
        row[k] = k < p.K ? row_of_pair(p, pair0 + k) : -1;
        any = max(any, row[k]);
    }
    if (any < 0) return;
    const uint8_t* src = x[t];
    const int step = gridDim.y * blockDim.x;
    for (int i0 = blockIdx.y * blockDim.x + threadIdx.x; i0 < pieces; i0 += step * kUnroll) {
        P v[kUnroll];
#pragma unroll
        for (int u = 0; u < kUnroll; ++u)
            if (i0 + u * step < pieces) v[u] = load_piece<P>(src, i0 + u * step);
#pragma unroll
        for (int k = 0; k < kMaxTopK; ++k) {
            if (k >= p.K) break;
            if (row[k] < 0) continue;
            uint8_t* dst = rows[row[k]];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u)
                if (i0 + u * step < pieces) store_piece(dst, i0 + u * step, v[u]);
        }
    }
}

// ---------------------------------------------------------------------------------------
// Combine: eight rows' pieces of a column are requested together, then added in pair order.
// ---------------------------------------------------------------------------------------
constexpr int kRowsAtOnce = 8;

template <typename T, int N, bool WEIGHTED>
__global__ void __launch_bounds__(256) combine_rows_kernel(Rows y, const float* weights, Rows out, int pieces,
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
                if (row[k] >= 0)
#pragma unroll
                    for (int j = 0; j < N; ++j)
                        acc[j] = WEIGHTED ? fmaf(to_float(v[k].v[j]), w[k], acc[j]) : acc[j] + to_float(v[k].v[j]);
        }
        P o;
#pragma unroll
        for (int j = 0; j < N; ++j) o.v[j] = from_float<T>(acc[j]);
        store_piece(out[t], i, o);
    }
}

// ---------------------------------------------------------------------------------------
// The combine's gradient: a CTA takes a token, its warps share the token's rows.  A row's warps walk its pieces, scale
// the token's gradient into the row's gradient and sum the products with the row; the sums meet in shared memory in a
// fixed order.  The token's gradient is read by every row's warps, out of L1 after the first.
// ---------------------------------------------------------------------------------------
constexpr int kGradWarps = 8;

template <typename T, int N>
__global__ void __launch_bounds__(kGradWarps * 32) combine_grad_kernel(Rows grad_out, Rows y, const float* weights,
                                                                       Rows grad_y, float* grad_weights,
                                                                       int pieces, Fill fill, PlanView p)
{
    typedef Piece<T, N> P;
    __shared__ int live_row[kMaxTopK], live_k[kMaxTopK], live_count;
    __shared__ float part_sum[kGradWarps];
    pdl_launch_dependents();
    pdl_wait();
    if ((int)blockIdx.x >= p.T) {
        fill_rows<P>(grad_y, pieces, p, fill, (int)blockIdx.x - p.T);
        return;
    }
    const int t = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
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
    for (int base = 0; base < count; base += kGradWarps) {
        // rows base .. base + rows - 1; warps with the same remainder share one
        const int rows = min(kGradWarps, count - base);
        const int j = base + warp % rows, part = warp / rows, parts = (kGradWarps - warp % rows + rows - 1) / rows;
        const float w = weights[(long long)t * p.K + live_k[j]];
        float sum = 0.0f;
        for (int i0 = part * 32 + lane; i0 < pieces; i0 += parts * 32 * kUnroll) {
            P g[kUnroll], v[kUnroll];
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = i0 + u * parts * 32;
                if (i < pieces) {
                    if (grad_weights) v[u] = load_piece<P>(y[live_row[j]], i);
                    g[u] = load_piece<P>(src, i);
                }
            }
#pragma unroll
            for (int u = 0; u < kUnroll; ++u) {
                const int i = i0 + u * parts * 32;
                if (i < pieces) {
                    P o;
#pragma unroll
                    for (int n = 0; n < N; ++n) {
                        const float f = to_float(g[u].v[n]);
                        o.v[n] = from_float<T>(f * w);
                        if (grad_weights) sum = fmaf(f, to_float(v[u].v[n]), sum);
                    }
                    if (grad_y.base) store_piece(grad_y[live_row[j]], i, o);
                }
            }
        }
        if (grad_weights) {
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) sum += __shfl_xor_sync(~0u, sum, d);
            if (lane == 0) part_sum[warp] = sum;
            __syncthreads();
            if ((int)threadIdx.x < rows) {
                float s = 0.0f;
                for (int q = threadIdx.x; q < kGradWarps; q += rows) s += part_sum[q];
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
    return rows <= INT32_MAX - 2 * kSortThreads * 8 ? rows : -1;   // index arithmetic of the sort stays in 32 bits
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

int check_plan(Call& call, const moe_fp8_b200_plan* plan, PlanView& v)
{
    if (!plan) return call.bad("plan is NULL");
    const int64_t rows = plan_rows(plan->num_tokens, plan->top_k, plan->num_experts, plan->align);
    if (rows < 0)
        return call.bad("plan sizes out of range: num_tokens %d, top_k %d (1 .. %d), num_experts %d (1 .. %d), align %d (1 .. %d)",
                        plan->num_tokens, plan->top_k, kMaxTopK, plan->num_experts, kMaxExperts, plan->align, kMaxAlign);
    int rc = call.begin();
    if (rc == MOE_FP8_B200_OK && plan->num_tokens > 0) {
        rc = call.tensor("pair_row", plan->pair_row, 4);
        if (rc == MOE_FP8_B200_OK) rc = call.tensor("row_pair", plan->row_pair, 4);
    }
    if (rc == MOE_FP8_B200_OK) rc = call.tensor("expert_offset", plan->expert_offset, 4);
    if (rc == MOE_FP8_B200_OK) rc = call.tensor("expert_count", plan->expert_count, 4);
    if (rc != MOE_FP8_B200_OK) return rc;
    v = {plan->num_tokens, plan->top_k, plan->num_experts, plan->align, plan->num_tokens * plan->top_k, (int)rows,
         plan->pair_row, plan->row_pair, plan->expert_offset, plan->expert_count};
    return MOE_FP8_B200_OK;
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

int check_apart(const Call& call, const Extent& written, const Extent& other)
{
    return share_memory(written, other) ? call.bad("%s and %s share memory", written.name, other.name) : MOE_FP8_B200_OK;
}

bool on_16_bytes(const Extent& e)
{
    return !e.base || (((uintptr_t)e.base | (uintptr_t)e.row_bytes | (e.rows > 1 ? (uintptr_t)e.stride_bytes : 0)) & 15u) == 0;
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
    // the cluster grows with the batch: a CTA takes 32 pairs per warp at least
    const unsigned ctas = p.pairs <= kSortThreads ? 1 : p.pairs <= 2 * kSortThreads ? 2 : p.pairs <= 4 * kSortThreads ? 4 : 8;
    const int need = p.E > p.pairs ? p.E : p.pairs;
    const int threads = need >= kSortThreads ? kSortThreads : need <= 128 ? 128 : (need + 31) / 32 * 32;
    const size_t smem = sort_smem_bytes(threads, p.E);
    if (smem > 48 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(sort_tokens_kernel<Id>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
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
    return launch_after(dispatch_rows_kernel<T, N>, dim3(s.token_ctas + fill.ctas(), s.splits), s.block, 0, 1, stream,
                        as_rows(x), as_rows(rows), pieces, s.token_ctas, fill, p);
}

Fill fill_for(const PlanView& p, int zero_unused) { return {p.align > 1 ? p.E : 0, zero_unused ? kUnusedCtas : 0}; }

cudaError_t enqueue_dispatch(const Extent& x, const Extent& rows, int dtype, const PlanView& p, int zero_unused,
                             cudaStream_t stream)
{
    const Fill fill = fill_for(p, zero_unused);
    // the copy needs no arithmetic: one form per element size
    const bool wide = on_16_bytes(x) && on_16_bytes(rows);
    if (element_size(dtype) == 4)
        return wide ? launch_dispatch<float, 4>(x, rows, p, fill, stream) : launch_dispatch<float, 1>(x, rows, p, fill, stream);
    return wide ? launch_dispatch<__half, 8>(x, rows, p, fill, stream) : launch_dispatch<__half, 1>(x, rows, p, fill, stream);
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
    const Fill fill = grad_y.base ? fill_for(p, zero_unused) : Fill{0, 0};
    return launch_after(combine_grad_kernel<T, N>, dim3(p.T + fill.ctas()), dim3(kGradWarps * 32), 0, 1, stream, as_rows(grad_out),
                        as_rows(y), weights, as_rows(grad_y), grad_weights, pieces, fill, p);
}

int check_ids(const Call& call, const void* ids, int id_bits)
{
    if (id_bits != 32 && id_bits != 64) return call.bad("id_bits must be 32 or 64, got %d", id_bits);
    return call.tensor("topk_idx", ids, id_bits / 8);
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
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_ids(call, topk_idx, id_bits);
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
    if (rc != MOE_FP8_B200_OK) return rc;
    return call.cuda(enqueue_dispatch(ex, er, dtype, p, zero_unused, static_cast<cudaStream_t>(stream)));
}

int moe_fp8_b200_sort_and_dispatch(const void* topk_idx, int id_bits, int64_t first_expert, const void* x, int64_t x_stride,
                                   void* rows, int64_t rows_stride, int dtype, int hidden, const moe_fp8_b200_plan* plan,
                                   int zero_unused, void* stream, char* err, size_t err_len)
{
    Call call{err, err_len};
    PlanView p;
    Extent ex, er;
    int rc = check_plan(call, plan, p);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_ids(call, topk_idx, id_bits);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_rows(call, "x", x, x_stride, p.T, dtype, hidden, false, ex);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_rows(call, "rows", rows, rows_stride, p.capacity, dtype, hidden, true, er);
    if (rc == MOE_FP8_B200_OK && p.T > 0) rc = check_apart(call, er, ex);
    if (rc != MOE_FP8_B200_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = enqueue_sort(topk_idx, id_bits, first_expert, p, s);
    if (e == cudaSuccess && p.T > 0) e = enqueue_dispatch(ex, er, dtype, p, zero_unused, s);
    return call.cuda(e);
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
    if (rc == MOE_FP8_B200_OK && weights) rc = check_apart(call, eo, {"weights", weights, 1, 4ll * p.pairs, 0});
    if (rc != MOE_FP8_B200_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = on_16_bytes(ey) && on_16_bytes(eo);
    switch (dtype) {
        case MOE_FP8_B200_BF16:
            return call.cuda(wide ? launch_combine_rows<__nv_bfloat16, 8>(ey, weights, eo, p, s)
                                  : launch_combine_rows<__nv_bfloat16, 1>(ey, weights, eo, p, s));
        case MOE_FP8_B200_FP16:
            return call.cuda(wide ? launch_combine_rows<__half, 8>(ey, weights, eo, p, s)
                                  : launch_combine_rows<__half, 1>(ey, weights, eo, p, s));
        default:
            return call.cuda(wide ? launch_combine_rows<float, 4>(ey, weights, eo, p, s)
                                  : launch_combine_rows<float, 1>(ey, weights, eo, p, s));
    }
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
    if (rc == MOE_FP8_B200_OK) rc = call.tensor("weights", weights, 4);
    if (rc == MOE_FP8_B200_OK && grad_y) {
        rc = check_rows(call, "grad_y", grad_y, grad_y_stride, p.capacity, dtype, hidden, true, ed);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, ed, eg);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, ed, {"weights", weights, 1, 4ll * p.pairs, 0});
    }
    if (rc == MOE_FP8_B200_OK && grad_weights) {
        rc = check_rows(call, "y", y, y_stride, p.capacity, dtype, hidden, false, ey);
        if (rc == MOE_FP8_B200_OK) rc = call.tensor("grad_weights", grad_weights, 4);
        const Extent dw = {"grad_weights", grad_weights, 1, 4ll * p.pairs, 0};
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, ed, ey);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, eg);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, ey);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, ed);
        if (rc == MOE_FP8_B200_OK) rc = check_apart(call, dw, {"weights", weights, 1, 4ll * p.pairs, 0});
    }
    if (rc != MOE_FP8_B200_OK) return rc;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const bool wide = on_16_bytes(eg) && on_16_bytes(ey) && on_16_bytes(ed);
    switch (dtype) {
        case MOE_FP8_B200_BF16:
            return call.cuda(wide ? launch_combine_grad<__nv_bfloat16, 8>(eg, ey, weights, ed, grad_weights, p, zero_unused, s)
                                  : launch_combine_grad<__nv_bfloat16, 1>(eg, ey, weights, ed, grad_weights, p, zero_unused, s));
        case MOE_FP8_B200_FP16:
            return call.cuda(wide ? launch_combine_grad<__half, 8>(eg, ey, weights, ed, grad_weights, p, zero_unused, s)
                                  : launch_combine_grad<__half, 1>(eg, ey, weights, ed, grad_weights, p, zero_unused, s));
        default:
            return call.cuda(wide ? launch_combine_grad<float, 4>(eg, ey, weights, ed, grad_weights, p, zero_unused, s)
                                  : launch_combine_grad<float, 1>(eg, ey, weights, ed, grad_weights, p, zero_unused, s));
    }
}

}  // extern "C"
