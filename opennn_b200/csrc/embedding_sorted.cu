// Gradient of the embedding table, summed by token in a fixed order:
//   dW[v, :] (+)= sqrt(E) * sum over the positions n with id v of (dY + dY2)[n, :],   0 < v < V.
// No atomics on floating-point values: the same inputs give the same bits.
//
// Bound by HBM: every gradient row is read once and every table row written once.  Three launches:
//   1  one cluster sorts the positions by id (stable radix sort, its passes joined by cluster barriers), while the other
//      clusters mark the ids that occur in their part of the table and write the zeros of the rows that do not;
//   2  the sorted positions are cut into equal chunks, whatever their ids, so that a frequent token is spread over many
//      CTAs; a group of threads adds the rows of a chunk, and writes the table row of each run of equal ids that lies inside it.
//      Runs that cross the edge of a chunk leave a partial sum;
//   3  the partial sums of each such run are added in order.
// Few positions take one launch instead: every CTA owns some rows of the table and looks for their ids itself.
#include <cooperative_groups.h>

#include "common.cuh"
#include "launch_counter.h"

namespace onn
{

namespace
{

namespace cg = cooperative_groups;

// ---------------------------------------------------------------------------------------
// Few positions
// ---------------------------------------------------------------------------------------

constexpr int kOwnerThreads = 256;
constexpr int kOwnerWarps = kOwnerThreads / 32;
constexpr int kTile = 1024;                       // ids looked at together
constexpr int kOwnerColumns = 256;                // one per thread
constexpr int kMaxOwned = 32;                     // rows of a CTA, summed in shared memory

// CTA (x, y) owns `owned` consecutive rows of the table, 256 columns of them.  It walks over all ids in order, keeps those that
// are its own (in order: prefix sums) and adds their gradient rows; a thread always has the same column.
__global__ void __launch_bounds__(kOwnerThreads)
embedding_owner_kernel(const float* __restrict__ ids, const float* __restrict__ dY, const float* __restrict__ dY2,
                       float* __restrict__ dW, int tokens, int E, int V, float scale, int owned, int accumulate)
{
    __shared__ float sums[kMaxOwned][kOwnerColumns];
    __shared__ unsigned char present[kMaxOwned];
    __shared__ int list_row[kTile];
    __shared__ int list_token[kTile];
    __shared__ int warp_count[kOwnerWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int v0 = blockIdx.x * owned, v1 = min(v0 + owned, V);
    const int column = blockIdx.y * kOwnerColumns + tid;
    for(int r = 0; r < owned; r++) sums[r][tid] = 0.f;
    if(tid < kMaxOwned) present[tid] = 0;
    for(int first = 0; first < tokens; first += kTile)
    {
        constexpr int kEach = kTile / kOwnerThreads;
        int found[kEach];
        int mine = 0;
#pragma unroll
        for(int k = 0; k < kEach; k++)
        {
            const int n = first + tid * kEach + k;
            const long long v = n < tokens ? token_index(__ldg(ids + n)) : 0;
            found[k] = v > 0 && v >= v0 && v < v1 ? (int)v - v0 : -1;
            mine += found[k] >= 0;
        }
        int before = mine;
#pragma unroll
        for(int offset = 1; offset < 32; offset <<= 1)
        {
            const int other = __shfl_up_sync(0xffffffffu, before, offset);
            if(lane >= offset) before += other;
        }
        __syncthreads();                               // the lists of the tile before have been read
        if(lane == 31) warp_count[warp] = before;
        __syncthreads();
        before -= mine;
        int total = 0;
#pragma unroll
        for(int w = 0; w < kOwnerWarps; w++)
        {
            if(w < warp) before += warp_count[w];
            total += warp_count[w];
        }
#pragma unroll
        for(int k = 0; k < kEach; k++)
        {
            if(found[k] < 0) continue;
            list_row[before] = found[k];
            list_token[before] = first + tid * kEach + k;
            present[found[k]] = 1;
            before++;
        }
        __syncthreads();
        if(column < E)
        {
            for(int i = 0; i < total; i += 4)
            {
                float g[4];
#pragma unroll
                for(int k = 0; k < 4; k++)
                {
                    const long long at = i + k < total ? (long long)list_token[i + k] * E + column : -1;
                    g[k] = at >= 0 ? __ldg(dY + at) : 0.f;
                    if(dY2 && at >= 0) g[k] += __ldg(dY2 + at);
                }
#pragma unroll
                for(int k = 0; k < 4; k++)
                    if(i + k < total) sums[list_row[i + k]][tid] += g[k];
            }
        }
    }
    __syncthreads();
    if(column >= E) return;
    for(int v = v0; v < v1; v++)
    {
        float* to = dW + (long long)v * E + column;
        const float sum = sums[v - v0][tid] * scale;
        if(!accumulate) *to = sum;
        else if(present[v - v0]) *to += sum;
    }
}

// ---------------------------------------------------------------------------------------
// 1: sort, and the zeros
// ---------------------------------------------------------------------------------------

constexpr int kSortCtas = 8;
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;
constexpr int kZeroClusters = 17;                 // 18 clusters of 8: 144 of the 148 SMs

struct SortShared
{
    unsigned int count[kSortWarps][kMaxBins];     // of each warp's positions: digits seen; then where its next one goes
    unsigned int total[kSortCtas][kMaxBins];      // written by every CTA of the cluster
    unsigned int base[kMaxBins];
    unsigned int warp_sum[kMaxBins / 32];
};

__device__ __forceinline__ unsigned int sort_key(const float* __restrict__ ids, long long n, unsigned int V)
{
    const long long v = token_index(__ldg(ids + n));
    return v > 0 && v < (long long)V ? (unsigned int)v : V;         // V: padding, sorted behind everything
}

__device__ void sort_by_id(SortShared& shared, const float* __restrict__ ids, uint2* buffer0, uint2* buffer1, int tokens, unsigned int V,
                           int passes, int digit_bits, cg::cluster_group& cluster)
{
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank();
    const int bins = 1 << digit_bits;
    // warp w of CTA r has positions [from, to): in order of warp, so the sort is stable
    const int warps = kSortCtas * kSortWarps;
    const int each = ((tokens + warps - 1) / warps + 31) & ~31;
    const long long begin = (long long)(rank * kSortWarps + warp) * each;
    const int from = (int)(begin < tokens ? begin : tokens), to = (int)(begin + each < tokens ? begin + each : tokens);
    cluster.sync();                                                  // every CTA is running: its shared memory may be written
    for(int pass = 0; pass < passes; pass++)
    {
        const int shift = pass * digit_bits;
        const uint2* source = (pass & 1) ? buffer0 : buffer1;        // of passes after the first
        uint2* destination = (pass & 1) ? buffer1 : buffer0;
        unsigned int* count = shared.count[warp];
        for(int b = lane; b < bins; b += 32) count[b] = 0;
        __syncwarp();
        auto item = [&](int n)
        {
            if(n >= to) return make_uint2(0xffffffffu, 0u);
            return pass == 0 ? make_uint2(sort_key(ids, n, V), (unsigned int)n) : __ldcg(source + n);
        };
        for(int n = from; n < to; n += 32)
        {
            const uint2 it = item(n + lane);
            const bool there = n + lane < to;
            const unsigned int digit = there ? (it.x >> shift) & (unsigned int)(bins - 1) : 0xffffu;
            const unsigned int same = __match_any_sync(0xffffffffu, digit);
            if(there && lane == __ffs(same) - 1) count[digit] += __popc(same);
            __syncwarp();
        }
        __syncthreads();
        if(tid < bins)
        {
            // where each warp's share of a digit starts inside the CTA's
            unsigned int run = 0;
            for(int w = 0; w < kSortWarps; w++)
            {
                const unsigned int c = shared.count[w][tid];
                shared.count[w][tid] = run;
                run += c;
            }
            for(int r = 0; r < kSortCtas; r++) cluster.map_shared_rank(&shared, r)->total[rank][tid] = run;
        }
        cluster.sync();
        unsigned int all = 0, before = 0;
        if(tid < bins)
        {
#pragma unroll
            for(int r = 0; r < kSortCtas; r++)
            {
                if(r < rank) before += shared.total[r][tid];
                all += shared.total[r][tid];
            }
        }
        unsigned int upto = all;
        if(tid < kMaxBins)
        {
#pragma unroll
            for(int offset = 1; offset < 32; offset <<= 1)
            {
                const unsigned int other = __shfl_up_sync(0xffffffffu, upto, offset);
                if(lane >= offset) upto += other;
            }
            if(lane == 31) shared.warp_sum[warp] = upto;
        }
        __syncthreads();
        if(tid < bins)
        {
            unsigned int lower = 0;
            for(int w = 0; w < warp; w++) lower += shared.warp_sum[w];
            shared.base[tid] = lower + upto - all + before;
        }
        __syncthreads();
        for(int n = from; n < to; n += 32)
        {
            const uint2 it = item(n + lane);
            const bool there = n + lane < to;
            const unsigned int digit = there ? (it.x >> shift) & (unsigned int)(bins - 1) : 0xffffu;
            const unsigned int same = __match_any_sync(0xffffffffu, digit);
            const unsigned int at = there ? shared.base[digit] + count[digit] + __popc(same & ((1u << lane) - 1u)) : 0u;
            __syncwarp();
            if(there)
            {
                destination[at] = it;
                if(lane == __ffs(same) - 1) count[digit] += __popc(same);
            }
            __syncwarp();
        }
        cluster.sync();                                              // what this pass wrote is there for the next one
    }
}

// The rows [v0, v1) of the table that no position has become zero.
__device__ void zero_absent_rows(unsigned int* present, const float* __restrict__ ids, float* __restrict__ dW, int tokens, int E,
                                 int v0, int v1)
{
    const int tid = threadIdx.x;
    for(int i = tid; i < (v1 - v0 + 31) / 32; i += kSortThreads) present[i] = 0;
    __syncthreads();
#pragma unroll 8
    for(int n = tid; n < tokens; n += kSortThreads)
    {
        const long long v = token_index(__ldg(ids + n));
        if(v > 0 && v >= v0 && v < v1) atomicOr(present + (int)(v - v0) / 32, 1u << ((int)(v - v0) & 31));
    }
    __syncthreads();
    const bool vec = (E & 3) == 0 && aligned16(dW);
    if(E >= 64)
    {
        for(int v = v0 + (tid >> 5); v < v1; v += kSortWarps)
        {
            if((present[(v - v0) / 32] >> ((v - v0) & 31)) & 1u) continue;
            float* row = dW + (long long)v * E;
            if(vec) for(int e = (tid & 31) * 4; e < E; e += 128) st4_stream(row + e, make_float4(0.f, 0.f, 0.f, 0.f));
            else for(int e = tid & 31; e < E; e += 32) row[e] = 0.f;
        }
    }
    else
    {
        for(long long i = tid; i < (long long)(v1 - v0) * E; i += kSortThreads)
        {
            const int r = (int)(i / E);
            if(!((present[r / 32] >> (r & 31)) & 1u)) dW[(long long)v0 * E + i] = 0.f;
        }
    }
}

__global__ void __cluster_dims__(kSortCtas, 1, 1) __launch_bounds__(kSortThreads, 1)
embedding_sort_kernel(const float* __restrict__ ids, float* __restrict__ dW, uint2* buffer0, uint2* buffer1, int* owner_count,
                      int tokens, int E, int V, int passes, int digit_bits)
{
    extern __shared__ __align__(16) unsigned char bytes[];
    pdl_launch_dependents();
    cg::cluster_group cluster = cg::this_cluster();
    if(blockIdx.x < kSortCtas)
    {
        if(blockIdx.x == 0 && threadIdx.x == 0) *owner_count = 0;
        sort_by_id(*reinterpret_cast<SortShared*>(bytes), ids, buffer0, buffer1, tokens, (unsigned int)V, passes, digit_bits, cluster);
        return;
    }
    const int ctas = gridDim.x - kSortCtas, z = blockIdx.x - kSortCtas;
    const int rows = (V + ctas - 1) / ctas;
    const long long v0 = (long long)z * rows;
    if(v0 < V) zero_absent_rows(reinterpret_cast<unsigned int*>(bytes), ids, dW, tokens, E, (int)v0, (int)(v0 + rows < V ? v0 + rows : V));
}

// ---------------------------------------------------------------------------------------
// 2: chunks, and 3: runs that cross their edges
// ---------------------------------------------------------------------------------------

constexpr int kReduceThreads = 256;
constexpr int kInFlight = 8;                      // gradient rows a thread has under way

template <int VEC> struct Piece;
template <> struct Piece<4>
{
    using type = float4;
    static __device__ __forceinline__ float4 zero() { return make_float4(0.f, 0.f, 0.f, 0.f); }
    static __device__ __forceinline__ float4 load(const float* p) { return ld4_stream(p); }
    static __device__ __forceinline__ void store(float* p, float4 v) { st4(p, v); }
    static __device__ __forceinline__ float4 add(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
    static __device__ __forceinline__ float4 scaled(float4 a, float s) { return make_float4(a.x * s, a.y * s, a.z * s, a.w * s); }
};
template <> struct Piece<1>
{
    using type = float;
    static __device__ __forceinline__ float zero() { return 0.f; }
    static __device__ __forceinline__ float load(const float* p) { return __ldcs(p); }
    static __device__ __forceinline__ void store(float* p, float v) { *p = v; }
    static __device__ __forceinline__ float add(float a, float b) { return a + b; }
    static __device__ __forceinline__ float scaled(float a, float s) { return a * s; }
};

template <int VEC>
__device__ __forceinline__ void put_row(float* to, typename Piece<VEC>::type sum, float scale, int accumulate)
{
    using P = Piece<VEC>;
    sum = P::scaled(sum, scale);
    if(accumulate) sum = P::add(sum, P::load(to));
    P::store(to, sum);
}

// A group of `group` threads adds one chunk, group * VEC columns of it.
template <int VEC, bool TWO>
__global__ void __launch_bounds__(kReduceThreads)
embedding_chunk_kernel(const uint2* sorted, const float* __restrict__ dY, const float* __restrict__ dY2, float* __restrict__ dW,
                       float* __restrict__ partial, int* __restrict__ owners, int* owner_count,
                       int tokens, int E, int V, int chunk, int group, float scale, int accumulate)
{
    using P = Piece<VEC>;
    using T = typename P::type;
    pdl_launch_dependents();
    pdl_wait();
    const int which = threadIdx.x / group;
    const int index = blockIdx.x * (kReduceThreads / group) + which;
    const int column = (blockIdx.y * group + threadIdx.x % group) * VEC;
    const long long start = (long long)index * chunk;
    if(start >= tokens || column >= E) return;
    const int end = (int)(start + chunk < tokens ? start + chunk : tokens);
    const unsigned int before = start > 0 ? sorted[start - 1].x : 0xffffffffu, behind = end < tokens ? sorted[end].x : 0xffffffffu;

    unsigned int current = sorted[start].x;
    bool starts_here = before != current;
    T sum = P::zero();
    auto finish = [&](bool ends_here)
    {
        if(current >= (unsigned int)V) return;         // padding
        if(starts_here && ends_here) put_row<VEC>(dW + (long long)current * E + column, sum, scale, accumulate);
        else
        {
            P::store(partial + ((long long)index * 2 + (starts_here ? 1 : 0)) * E + column, sum);
            if(starts_here && column == 0) owners[atomicAdd(owner_count, 1)] = index;
        }
    };
    for(int i = (int)start; i < end && current < (unsigned int)V; i += kInFlight)
    {
        uint2 item[kInFlight];
        T row[kInFlight];
#pragma unroll
        for(int u = 0; u < kInFlight; u++) item[u] = i + u < end ? sorted[i + u] : make_uint2(0xffffffffu, 0u);
#pragma unroll
        for(int u = 0; u < kInFlight; u++)
        {
            row[u] = P::zero();
            if(item[u].x >= (unsigned int)V) continue;
            const long long at = (long long)item[u].y * E + column;
            row[u] = P::load(dY + at);
            if(TWO) row[u] = P::add(row[u], P::load(dY2 + at));
        }
#pragma unroll
        for(int u = 0; u < kInFlight; u++)
        {
            if(i + u >= end) break;
            if(item[u].x != current)
            {
                finish(true);
                current = item[u].x;
                starts_here = true;
                sum = P::zero();
            }
            sum = P::add(sum, row[u]);
        }
    }
    finish(behind != current);
}

// A run that starts in one chunk and goes on in the next ones: its last partial of the first chunk, then the first of each
// following chunk.  Eight warps take every eighth, 32 * VEC columns; their sums are added in order.
template <int VEC>
__global__ void __launch_bounds__(kReduceThreads)
embedding_join_kernel(const uint2* sorted, const float* partial, const int* owners, const int* owner_count, float* __restrict__ dW,
                      int tokens, int E, int chunk, float scale, int accumulate)
{
    using P = Piece<VEC>;
    using T = typename P::type;
    __shared__ T warp_sums[kReduceThreads / 32][32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int blocks = (E + 32 * VEC - 1) / (32 * VEC);
    const long long items = (long long)*owner_count * blocks;
    for(long long i = blockIdx.x; i < items; i += gridDim.x)
    {
        const int index = owners[i / blocks];
        const int column = ((int)(i % blocks) * 32 + lane) * VEC;
        const long long last = (long long)(index + 1) * chunk - 1;       // the chunk is whole: its run goes on behind it
        const unsigned int v = sorted[last].x;
        // chunks behind it that begin with the same id
        int more = 0;
        while(true)
        {
            const long long at = (long long)(index + 1 + more + tid) * chunk;
            const int here = __syncthreads_count(at < tokens && sorted[at].x == v);
            more += here;
            if(here < kReduceThreads) break;
        }
        T sum = P::zero();
        if(column < E)
        {
            // part 0 is the first chunk's, part j that of the j-th behind it
            auto part = [&](int j) { return P::load(partial + ((long long)(index + j) * 2 + (j == 0 ? 1 : 0)) * E + column); };
            for(int j = warp; j <= more; j += 4 * (kReduceThreads / 32))
            {
                T four[4];
#pragma unroll
                for(int k = 0; k < 4; k++) four[k] = j + k * (kReduceThreads / 32) <= more ? part(j + k * (kReduceThreads / 32)) : P::zero();
#pragma unroll
                for(int k = 0; k < 4; k++) sum = P::add(sum, four[k]);
            }
        }
        warp_sums[warp][lane] = sum;
        __syncthreads();
        if(warp == 0 && column < E)
        {
            sum = warp_sums[0][lane];
#pragma unroll
            for(int w = 1; w < kReduceThreads / 32; w++) sum = P::add(sum, warp_sums[w][lane]);
            put_row<VEC>(dW + (long long)v * E + column, sum, scale, accumulate);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------

constexpr int64_t kFewTokens = 2048;

// Positions of a chunk: enough chunks to fill the GPU, few enough that partial sums stay a small share of the traffic.
int chunk_of(int64_t tokens) { return tokens <= 65536 ? 16 : tokens <= 1048576 ? 32 : 64; }

struct Layout { int64_t buffer0, buffer1, partial, owners, count, words; int chunks; };

Layout layout_of(int64_t tokens, int64_t E)
{
    auto up = [](int64_t words) { return (words + 3) / 4 * 4; };
    Layout l;
    l.chunks = (int)((tokens + chunk_of(tokens) - 1) / chunk_of(tokens));
    l.buffer0 = 0;
    l.buffer1 = l.buffer0 + up(2 * tokens);
    l.partial = l.buffer1 + up(2 * tokens);
    l.owners = l.partial + up(2 * (int64_t)l.chunks * E);
    l.count = l.owners + up(l.chunks);
    l.words = l.count + 4;
    return l;
}

}  // namespace

}  // namespace onn

using namespace onn;

static bool sorted_sizes_ok(int64_t B, int64_t S, int64_t E, int64_t V)
{
    return B > 0 && S > 0 && E > 0 && V > 0 && E < (1LL << 23) && V < (1LL << 24) && B < (1LL << 31) && S < (1LL << 31) && B * S < (1LL << 31) - 65536;
}

extern "C" size_t onn_embedding_bwd_sorted_workspace_floats(int64_t B, int64_t S, int64_t E, int64_t V)
{
    if(!sorted_sizes_ok(B, S, E, V) || B * S <= kFewTokens) return 0;
    return (size_t)layout_of(B * S, E).words;
}

extern "C" int onn_embedding_bwd_sorted(const float* ids, const float* dY, const float* dY2, float* dW,
                                        int64_t B, int64_t S, int64_t E, int64_t V, int scale,
                                        float* workspace, uint32_t flags, void* stream)
{
    ONN_CHECK_ARG(ids && dY && dW && sorted_sizes_ok(B, S, E, V));
    ONN_CHECK_ARG((flags & ~ONN_ACCUMULATE) == 0);
    const int64_t tokens = B * S;
    const float scale_value = scale ? sqrtf((float)E) : 1.f;
    const int accumulate = (flags & ONN_ACCUMULATE) ? 1 : 0;
    cudaStream_t s = (cudaStream_t)stream;
    if(tokens <= kFewTokens)
    {
        // a CTA for each SM if the table is that tall, but no more rows than fit in shared memory
        const int columns = (int)((E + kOwnerColumns - 1) / kOwnerColumns);
        int64_t owned = (V * columns + 2 * kSmCount - 1) / (2 * kSmCount);
        owned = owned < 1 ? 1 : owned > kMaxOwned ? kMaxOwned : owned;
        embedding_owner_kernel<<<dim3((unsigned)((V + owned - 1) / owned), columns), kOwnerThreads, 0, s>>>(
            ids, dY, dY2, dW, (int)tokens, (int)E, (int)V, scale_value, (int)owned, accumulate);
        count_launch();
        return launch_status();
    }
    if(!workspace) return ONN_ERR_WORKSPACE;
    ONN_CHECK_ARG(host_aligned16(workspace));
    const Layout l = layout_of(tokens, E);
    uint2* buffer0 = reinterpret_cast<uint2*>(workspace + l.buffer0);
    uint2* buffer1 = reinterpret_cast<uint2*>(workspace + l.buffer1);
    float* partial = workspace + l.partial;
    int* owners = reinterpret_cast<int*>(workspace + l.owners);
    int* owner_count = reinterpret_cast<int*>(workspace + l.count);

    int bits = 1;
    while((V >> bits) != 0) bits++;                    // the largest key is V, for padding
    const int passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits, digit_bits = (bits + passes - 1) / passes;
    static PerDeviceBytes configured;
    const int rows_of_zero_cta = (int)((V + kZeroClusters * kSortCtas - 1) / (kZeroClusters * kSortCtas));
    const size_t bitmap = ((size_t)rows_of_zero_cta + 31) / 32 * 4;
    const size_t shared = sizeof(SortShared) > bitmap ? sizeof(SortShared) : bitmap;
    if(!ensure_dynamic_smem(embedding_sort_kernel, configured, shared)) return ONN_ERR_CUDA;
    embedding_sort_kernel<<<kSortCtas * (accumulate ? 1 : 1 + kZeroClusters), kSortThreads, shared, s>>>(
        ids, dW, buffer0, buffer1, owner_count, (int)tokens, (int)E, (int)V, passes, digit_bits);
    count_launch();
    if(launch_status() != ONN_OK) return ONN_ERR_CUDA;

    const uint2* sorted = (passes & 1) ? buffer0 : buffer1;
    const bool vec = (E & 3) == 0 && host_aligned16(dY) && host_aligned16(dY2) && host_aligned16(dW);
    const int pieces = (int)(vec ? E / 4 : E);
    int group = 32;
    while(group < kReduceThreads && group < pieces) group *= 2;
    const int chunk = chunk_of(tokens), groups = kReduceThreads / group;
    const dim3 grid((unsigned)((l.chunks + groups - 1) / groups), (unsigned)((pieces + group - 1) / group));
    auto add = [&](auto kernel)
    {
        return launch_overlapped(kernel, grid, dim3(kReduceThreads), 0, s, sorted, dY, dY2, dW, partial, owners, owner_count, (int)tokens,
                                 (int)E, (int)V, chunk, group, scale_value, accumulate);
    };
    cudaError_t error = vec ? (dY2 ? add(embedding_chunk_kernel<4, true>) : add(embedding_chunk_kernel<4, false>))
                            : (dY2 ? add(embedding_chunk_kernel<1, true>) : add(embedding_chunk_kernel<1, false>));
    count_launch();
    if(error != cudaSuccess) return ONN_ERR_CUDA;
    auto join = [&](auto kernel)
    {
        return launch_overlapped(kernel, dim3(2 * kSmCount), dim3(kReduceThreads), 0, s, sorted, (const float*)partial, (const int*)owners,
                                 (const int*)owner_count, dW, (int)tokens, (int)E, chunk, scale_value, accumulate);
    };
    error = vec ? join(embedding_join_kernel<4>) : join(embedding_join_kernel<1>);
    count_launch();
    if(error != cudaSuccess) return ONN_ERR_CUDA;
    return launch_status();
}
