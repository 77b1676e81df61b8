// Gradient of the embedding table, summed by token in a fixed order:
//   dW[v, :] (+)= sqrt(E) * sum over the positions n with id v, in order of position, of (dY + dY2)[n, :],   0 < v < V.
// No atomics on floating-point values: the same inputs give the same bits.
#include "common.cuh"
#include "launch_counter.h"

namespace onn
{

namespace
{

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kTile = 1024;                       // ids looked at together

// A CTA owns `owned` consecutive rows of the table.  It walks over all ids in order, keeps those that are its own (in
// order: ballots and prefix sums) and adds their gradient rows to its rows; a thread always has the same columns, so
// its additions to a row follow one another.
__global__ void __launch_bounds__(kThreads)
embedding_owner_kernel(const float* __restrict__ ids, const float* __restrict__ dY, const float* __restrict__ dY2,
                       float* __restrict__ dW, long long tokens, int E, int V, float scale, int owned, int accumulate)
{
    __shared__ int list_row[kTile];
    __shared__ int list_token[kTile];
    __shared__ int warp_count[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int v0 = blockIdx.x * owned, v1 = min(v0 + owned, V);
    if(!accumulate)
    {
        for(int v = v0; v < v1; v++)
            for(int e = tid; e < E; e += kThreads) dW[(long long)v * E + e] = 0.f;
    }
    for(long long first = 0; first < tokens; first += kTile)
    {
        int found[kTile / kThreads];
        int mine = 0;
#pragma unroll
        for(int k = 0; k < kTile / kThreads; k++)
        {
            const long long n = first + tid * (kTile / kThreads) + k;
            long long v = n < tokens ? token_index(__ldg(ids + n)) : 0;
            found[k] = v > 0 && v >= v0 && v < v1 ? (int)v : -1;
            mine += found[k] >= 0;
        }
        int before = mine;
#pragma unroll
        for(int offset = 1; offset < 32; offset <<= 1)
        {
            const int other = __shfl_up_sync(0xffffffffu, before, offset);
            if(lane >= offset) before += other;
        }
        __syncthreads();
        if(lane == 31) warp_count[warp] = before;
        __syncthreads();
        before -= mine;
        int total = 0;
        for(int w = 0; w < kWarps; w++)
        {
            if(w < warp) before += warp_count[w];
            total += warp_count[w];
        }
#pragma unroll
        for(int k = 0; k < kTile / kThreads; k++)
        {
            if(found[k] < 0) continue;
            list_row[before] = found[k];
            list_token[before] = tid * (kTile / kThreads) + k;
            before++;
        }
        __syncthreads();
        for(int i = 0; i < total; i++)
        {
            float* row = dW + (long long)list_row[i] * E;
            const long long n = first + list_token[i];
            for(int e = tid; e < E; e += kThreads)
            {
                float g = __ldg(dY + n * E + e);
                if(dY2) g += __ldg(dY2 + n * E + e);
                row[e] += g * scale;
            }
        }
    }
}

}  // namespace

}  // namespace onn

using namespace onn;

extern "C" size_t onn_embedding_bwd_sorted_workspace_floats(int64_t B, int64_t S, int64_t E, int64_t V)
{
    (void)B; (void)S; (void)E; (void)V;
    return 0;
}

extern "C" int onn_embedding_bwd_sorted(const float* ids, const float* dY, const float* dY2, float* dW,
                                        int64_t B, int64_t S, int64_t E, int64_t V, int scale,
                                        float* workspace, uint32_t flags, void* stream)
{
    (void)workspace;
    ONN_CHECK_ARG(ids && dY && dW && B > 0 && S > 0 && E > 0 && V > 0);
    ONN_CHECK_ARG(E < (1LL << 24) && V < (1LL << 24) && B < (1LL << 31) && S < (1LL << 31) && B * S < (1LL << 31));
    ONN_CHECK_ARG((flags & ~ONN_ACCUMULATE) == 0);
    const float scale_value = scale ? sqrtf((float)E) : 1.f;
    const int owned = 32;
    embedding_owner_kernel<<<(unsigned)((V + owned - 1) / owned), kThreads, 0, (cudaStream_t)stream>>>(
        ids, dY, dY2, dW, B * S, (int)E, (int)V, scale_value, owned, (flags & ONN_ACCUMULATE) ? 1 : 0);
    count_launch();
    return launch_status();
}
