// Log probabilities of given tokens with entropy and the top alternatives, and their gradient.
//
//   z = x / T,  lse = log sum_i exp z_i,  p = exp(z - lse)
//   forward   logprob = z_t - lse,  entropy = -sum_i p_i log p_i,  the K largest x with z - lse
//   backward  dx_i = [ g (1[i = t] - p_i) - h p_i (log p_i + entropy) ] / T
//
// Both are bound by HBM: the forward pass reads each logit once, the backward pass reads and writes each once.
#include <cooperative_groups.h>

#include "logit_rows.cuh"

namespace onn
{

namespace
{

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 8;                        // 16-byte vectors a thread has in flight

// Running statistics of a set of logits, in base 2 and relative to the largest logit m seen: with c = log2(e) / T and
// d = c (x - m),  s = sum 2^d  and  w = sum 2^d d.  The difference is taken before the scale, so logits of any finite
// size (a mask of the type's lowest value) leave it finite or at -inf; -inf adds nothing to either sum; NaN and +inf
// make both NaN.
struct Running { float m, s, w; };

constexpr float kNothing = -1e4f;                 // 2^-10000 = 0: the bound that keeps 0 * -inf out of w

__device__ __forceinline__ float finite_anchor(float m) { return m > -INFINITY ? m : 0.f; }

// The sums of r relative to another, larger m.
__device__ __forceinline__ void rebase(Running& r, float m, float c)
{
    const float d = fmaxf((r.m - finite_anchor(m)) * c, kNothing);
    const float f = exp2_approx(d);
    r.w = fmaf(d, r.s, r.w) * f;
    r.s *= f;
    r.m = m;
}

__device__ __forceinline__ Running merge(Running a, Running b, float c)
{
    const float m = fmaxf(a.m, b.m);
    rebase(a, m, c);
    rebase(b, m, c);
    a.s += b.s;
    a.w += b.w;
    return a;
}

// Adds the logits of kUnroll vectors, of which the largest is `m`: one rescaling for all of them, then two logits per
// instruction (packed fp32).
template <int DTYPE>
__device__ __forceinline__ void add_vectors(Running& r, const uint4 (&v)[kUnroll], float m, float c)
{
    using L = Logit<DTYPE>;
    if(m > r.m) rebase(r, m, c);
    const float base = finite_anchor(r.m);
    const float2 minus_base = make_float2(-base, -base), c2 = make_float2(c, c);
    float2 s2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);
#pragma unroll
    for(int u = 0; u < kUnroll; u++)
    {
        float x[L::VE];
        L::unpack(v[u], x);
#pragma unroll
        for(int e = 0; e < L::VE; e += 2)
        {
            const float2 d = mul2(add2(make_float2(x[e], x[e + 1]), minus_base), c2);
            const float2 p = make_float2(exp2_approx(d.x), exp2_approx(d.y));
            s2 = add2(s2, p);
            w2 = fma2(p, make_float2(fmaxf(d.x, kNothing), fmaxf(d.y, kNothing)), w2);
        }
    }
    r.s += s2.x + s2.y;
    r.w += w2.x + w2.y;
}

// Order of the alternatives as one number: the larger logit first, then the lower index.  0 = not in the list at all
// (-inf and NaN).
__device__ __forceinline__ unsigned long long key_of(float x, int index)
{
    if(!(x > -INFINITY)) return 0ull;
    const unsigned int bits = __float_as_uint(x + 0.f);             // -0 and +0 are the same logit
    const unsigned int order = bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
    return ((unsigned long long)order << 32) | (0xffffffffu - (unsigned int)index);
}
__device__ __forceinline__ int key_index(unsigned long long key) { return (int)(0xffffffffu - (unsigned int)key); }
__device__ __forceinline__ float key_logit(unsigned long long key)
{
    const unsigned int order = (unsigned int)(key >> 32);
    return __uint_as_float(order ^ ((order >> 31) ? 0x80000000u : 0xffffffffu));
}

// k-th largest of the lanes' values (k from 1 to 32): a bitonic sort across the warp.
__device__ __forceinline__ float warp_kth_largest(float v, int k)
{
    const int lane = threadIdx.x & 31;
#pragma unroll
    for(int size = 2; size <= 32; size <<= 1)
    {
#pragma unroll
        for(int stride = size >> 1; stride > 0; stride >>= 1)
        {
            const float other = __shfl_xor_sync(0xffffffffu, v, stride);
            const bool falling = (lane & size) == 0 || size == 32, first = (lane & stride) == 0;
            v = falling == first ? fmaxf(v, other) : fminf(v, other);
        }
    }
    return __shfl_sync(0xffffffffu, v, k - 1);
}

constexpr int kMaxCluster = 8;
constexpr int kList = 2048;                       // candidates a CTA can hold

// What a warp knows of its part of the row.
struct alignas(16) Part { float m, s, w, top; };

// Shared memory of a CTA.  `parts` and, in the first CTA of a cluster, `candidates` are written by the whole cluster.
template <bool TOP>
struct Shared
{
    Part parts[kMaxCluster * kWarps];
    float m, log_s;
};
template <>
struct Shared<true>
{
    Part parts[kMaxCluster * kWarps];
    float m, log_s;
    volatile float warp_top[kWarps];
    int listed, candidate_count;
    unsigned long long best[kWarps];
    unsigned long long list[kList];
    unsigned long long candidates[kList];
};

// One cluster of CTAs (often of one) per row; each CTA streams its part of the row once.
//
// The alternatives come out of the same pass.  If every warp knows k logits that are at least t, with k = ceil(top /
// warps), no logit below t can stand in the list.  So after its first batch every warp sorts its lanes' maxima and takes
// the k-th as its bound; the smallest bound of all warps is the CTA's, and logits that reach it are put on a list in shared
// memory (a compare per vector; for logits in no particular order a few hundred of them).  The bounds rise after 2, 4, 8 ... batches.  At
// the end the bound of all maxima thins the lists out to little more than `top` candidates in the first CTA, which ranks
// them.  A list that overflows (thousands of equal logits, a rising row) is done without: the first CTA then scans
// the row once for each place.
template <int DTYPE, bool TOP>
__global__ void __launch_bounds__(kThreads, TOP ? 3 : 4)
token_logprobs_kernel(const typename Logit<DTYPE>::type* __restrict__ logits, long long pitch, const float* __restrict__ tokens,
                      float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ lse,
                      int* __restrict__ top_ids, float* __restrict__ top_logprobs, int top, int V, float c, float inverse_temperature)
{
    using L = Logit<DTYPE>;
    constexpr int VE = L::VE;
    __shared__ Shared<TOP> shared;
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    bool active;
    const long long token = row_token(tokens, row, V, &active);
    if(!active)                                        // the same for the whole cluster
    {
        if(rank != 0) return;
        if(tid == 0)
        {
            if(logprobs) logprobs[row] = 0.f;
            if(entropy) entropy[row] = 0.f;
            if(lse) lse[row] = 0.f;
        }
        for(int k = tid; k < top; k += kThreads) { top_ids[row * top + k] = -1; top_logprobs[row * top + k] = -INFINITY; }
        return;
    }

    const typename L::type* x = logits + row * pitch;
    const RowCut cut = cut_row<DTYPE>(x, V);
    const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
    const int after = cut.head + cut.vectors * VE;
    // the element of the row's ends that this thread looks after, if any
    int end_index = tid < cut.head ? tid : tid < cut.head + cut.tail ? after + tid - cut.head : -1;
    if(rank != 0) end_index = -1;
    const int share = (cut.vectors + ctas - 1) / ctas;
    const int begin = min(rank * share, cut.vectors), end = min(begin + share, cut.vectors);

    if constexpr(TOP)
    {
        if(tid == 0) { shared.listed = 0; shared.candidate_count = 0; }
    }
    // all CTAs of a cluster must be running before one writes into another
    if(ctas > 1) cluster.sync();
    else if constexpr(TOP) __syncthreads();

    [[maybe_unused]] auto list_one = [&](float value, int index)
    {
        if constexpr(TOP)
        {
            const unsigned long long key = key_of(value, index);
            if(key == 0) return;
            const int at = atomicAdd(&shared.listed, 1);
            if(at < kList) shared.list[at] = key;
        }
    };

    Running r = {-INFINITY, 0.f, 0.f};
    float end_value = -INFINITY;
    if(end_index >= 0)
    {
        end_value = L::get(x + end_index);
        // as a batch of its own; NaN is never larger, and reaches the sum
        r.m = end_value > -INFINITY ? end_value : -INFINITY;
        r.s = exp2_approx((end_value - finite_anchor(r.m)) * c);
    }
    const int wanted = TOP ? (top + kWarps - 1) / kWarps : 1;
    float bound = -INFINITY;
    for(int first = begin, batch = 0; first < end || batch == 0; first += kThreads * kUnroll, batch++)
    {
        uint4 v[kUnroll];
#pragma unroll
        for(int u = 0; u < kUnroll; u++)
        {
            const int i = first + u * kThreads + tid;
            v[u] = i < end ? __ldg(body + i) : L::lowest();
        }
        float vector_max[kUnroll];
        float m = r.m;
#pragma unroll
        for(int u = 0; u < kUnroll; u++)
        {
            vector_max[u] = L::max(v[u]);
            m = fmaxf(m, vector_max[u]);
        }
        add_vectors<DTYPE>(r, v, m, c);
        if constexpr(TOP)
        {
            if((batch & (batch - 1)) == 0)             // after 1, 2, 3, 5, 9 ... batches
            {
                const float mine = warp_kth_largest(r.m, wanted);
                if(lane == 0) shared.warp_top[warp] = mine;
                // the first bound needs every warp's; later ones take what is there, since bounds only rise
                if(batch == 0) __syncthreads();
                bound = shared.warp_top[0];
#pragma unroll
                for(int w = 1; w < kWarps; w++) bound = fminf(bound, shared.warp_top[w]);
                if(batch == 0 && end_value >= bound) list_one(end_value, end_index);
            }
#pragma unroll
            for(int u = 0; u < kUnroll; u++)
            {
                if(vector_max[u] < bound || vector_max[u] == -INFINITY) continue;
                float part[VE];
                L::unpack(v[u], part);
                const int index = cut.head + (first + u * kThreads + tid) * VE;
#pragma unroll
                for(int e = 0; e < VE; e++)
                    if(part[e] >= bound) list_one(part[e], index + e);
            }
        }
    }

    // every warp's part to every CTA of the cluster
    const float own_max = r.m;
    const float warp_m = warp_max(r.m);
    rebase(r, warp_m, c);
    Part part;
    part.m = warp_m;
    part.s = warp_sum(r.s);
    part.w = warp_sum(r.w);
    const int parts = ctas * kWarps;
    const int wanted_all = TOP ? (top + parts - 1) / parts : 1;
    part.top = TOP ? warp_kth_largest(own_max, wanted_all) : 0.f;
    if(ctas == 1)
    {
        if(lane == 0) shared.parts[warp] = part;
        __syncthreads();
    }
    else
    {
        if(lane < ctas) cluster.map_shared_rank(&shared, lane)->parts[rank * kWarps + warp] = part;
        cluster.sync();
    }

    if(rank == 0 && warp == 0)
    {
        Running all = {-INFINITY, 0.f, 0.f};
        for(int i = lane; i < parts; i += 32) all = merge(all, Running{shared.parts[i].m, shared.parts[i].s, shared.parts[i].w}, c);
        rebase(all, warp_max(all.m), c);
        all.s = warp_sum(all.s);
        all.w = warp_sum(all.w);
        if(lane == 0)
        {
            const bool none = all.s == 0.f;            // a row without a finite logit has no distribution
            const float log_s = none ? INFINITY : logf(all.s);
            shared.m = finite_anchor(all.m);
            shared.log_s = log_s;
            if(logprobs) logprobs[row] = none ? -INFINITY : (L::get(x + token) - all.m) * inverse_temperature - log_s;
            if(entropy)
            {
                const float value = log_s - all.w / all.s * kLn2;
                entropy[row] = none || value < 0.f ? 0.f : value;
            }
            if(lse) lse[row] = none ? -INFINITY : fmaf(all.m, inverse_temperature, log_s);
        }
    }

    if constexpr(TOP)
    {
        // the bound of all maxima
        if(wanted_all == 1 && parts >= 2 * top)
        {
            // more warps than places: the bound is the top-th largest of their maxima
            float found = -INFINITY;
            for(int i = lane; i < parts; i += 32)
            {
                const float mine = shared.parts[i].m;
                int larger = 0;
                for(int j = 0; j < parts; j++) larger += shared.parts[j].m > mine || (shared.parts[j].m == mine && j < i);
                if(larger == top - 1) found = mine;
            }
            bound = warp_max(found);
        }
        else
        {
            float lowest = INFINITY;
            for(int i = lane; i < parts; i += 32) lowest = fminf(lowest, shared.parts[i].top);
            bound = -warp_max(-lowest);
        }
        const int listed = shared.listed;
        Shared<TOP>* leader = ctas == 1 ? &shared : cluster.map_shared_rank(&shared, 0);
        if(listed > kList)
        {
            if(tid == 0) atomicAdd(&leader->candidate_count, kList + 1);
        }
        else
        {
            for(int i = tid; i < listed; i += kThreads)
            {
                const unsigned long long key = shared.list[i];
                if(key_logit(key) < bound) continue;
                const int at = atomicAdd(&leader->candidate_count, 1);
                if(at < kList) leader->candidates[at] = key;
            }
        }
        if(ctas == 1) __syncthreads();
        else cluster.sync();
        if(rank != 0) return;

        auto place = [&](int k, unsigned long long key)
        {
            top_ids[row * top + k] = key ? key_index(key) : -1;
            top_logprobs[row * top + k] = key ? (key_logit(key) - shared.m) * inverse_temperature - shared.log_s : -INFINITY;
        };
        int n = shared.candidate_count;
        if(n < 0 || n > kList)
        {
            // one place after the other: the largest key below the last one
            unsigned long long last = ~0ull;
            for(int k = 0; k < top; k++)
            {
                unsigned long long best = 0;
                auto look = [&](float value, int index)
                {
                    const unsigned long long key = key_of(value, index);
                    if(key < last && key > best) best = key;
                };
                if(last != 0)
                {
                    if(end_index >= 0) look(end_value, end_index);
                    for(int i = tid; i < cut.vectors; i += kThreads)
                    {
                        float values[VE];
                        L::unpack(__ldg(body + i), values);
#pragma unroll
                        for(int e = 0; e < VE; e++) look(values[e], cut.head + i * VE + e);
                    }
                }
#pragma unroll
                for(int offset = 16; offset > 0; offset >>= 1)
                {
                    const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, offset);
                    best = other > best ? other : best;
                }
                __syncthreads();
                if(lane == 0) shared.best[warp] = best;
                __syncthreads();
                best = shared.best[0];
#pragma unroll
                for(int w = 1; w < kWarps; w++) best = shared.best[w] > best ? shared.best[w] : best;
                last = best;
                if(tid == 0) place(k, best);
            }
            return;
        }
        for(int k = n + tid; k < top; k += kThreads) place(k, 0);
        if(n <= kThreads)
        {
            // few: a candidate's place is the number of larger ones
            if(tid < n)
            {
                const unsigned long long key = shared.candidates[tid];
                int larger = 0;
                for(int j = 0; j < n; j++) larger += shared.candidates[j] > key;
                if(larger < top) place(larger, key);
            }
            return;
        }
        int padded = 2 * kThreads;
        while(padded < n) padded *= 2;
        for(int i = n + tid; i < padded; i += kThreads) shared.candidates[i] = 0;
        for(int size = 2; size <= padded; size <<= 1)
        {
            for(int stride = size >> 1; stride > 0; stride >>= 1)
            {
                __syncthreads();
                for(int pair = tid; pair < padded / 2; pair += kThreads)
                {
                    const int i = 2 * pair - (pair & (stride - 1)), j = i + stride;
                    const unsigned long long a = shared.candidates[i], b = shared.candidates[j];
                    if(((i & size) == 0) != (a > b)) { shared.candidates[i] = b; shared.candidates[j] = a; }
                }
            }
        }
        __syncthreads();
        for(int k = tid; k < min(top, n); k += kThreads) place(k, shared.candidates[k]);
    }
}

// One CTA per piece of a row: the row's scalars, then load, compute, store.
template <int DTYPE>
__global__ void __launch_bounds__(kThreads)
token_logprobs_bwd_kernel(const typename Logit<DTYPE>::type* logits, long long pitch, const float* __restrict__ tokens,
                          const float* __restrict__ lse, const float* __restrict__ entropy,
                          const float* __restrict__ d_logprobs, const float* __restrict__ d_entropy,
                          typename Logit<DTYPE>::type* dlogits, long long d_pitch, int V, float inverse_temperature)
{
    using L = Logit<DTYPE>;
    constexpr int VE = L::VE;
    const long long row = blockIdx.y;
    const int tid = threadIdx.x;
    bool active;
    const long long token = row_token(tokens, row, V, &active);
    const typename L::type* x = logits + row * pitch;
    typename L::type* dx = dlogits + row * d_pitch;
    const RowCut cut = cut_row<DTYPE>(dx, V);
    const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;

    const float g = active ? d_logprobs[row] * inverse_temperature : 0.f;
    const float h = active && d_entropy ? d_entropy[row] * inverse_temperature : 0.f;
    const float H = h != 0.f ? entropy[row] : 0.f;
    float row_lse = active ? lse[row] : 0.f;
    if(row_lse == -INFINITY) row_lse = 0.f;            // a row without a finite logit: every p is 0

    auto one = [&](float value, long long index)
    {
        if(!active) return 0.f;
        const float log_p = fmaf(value, inverse_temperature, -row_lse);
        const float p = exp2_approx(log_p * kLog2E);
        float r = -g * p;
        if(h != 0.f) r = fmaf(-h * p, fmaxf(log_p, kNothing) + H, r);
        if(index == token) r += g;
        return r;
    };

    const int after = cut.head + cut.vectors * VE;
    if(blockIdx.x == 0 && tid < cut.head + cut.tail)
    {
        const int i = tid < cut.head ? tid : after + tid - cut.head;
        L::put(dx + i, one(active ? L::get(x + i) : 0.f, i));
    }
    for(int i = blockIdx.x * kThreads + tid; i < cut.vectors; i += gridDim.x * kThreads)
    {
        const int index = cut.head + i * VE;
        float f[VE];
        if(!active)
        {
#pragma unroll
            for(int e = 0; e < VE; e++) f[e] = 0.f;
        }
        else if(together) L::unpack(*reinterpret_cast<const uint4*>(x + index), f);
        else
        {
#pragma unroll
            for(int e = 0; e < VE; e++) f[e] = L::get(x + index + e);
        }
#pragma unroll
        for(int e = 0; e < VE; e++) f[e] = one(f[e], index + e);
        *reinterpret_cast<uint4*>(dx + index) = L::pack(f);
    }
}

template <int DTYPE, bool TOP>
int launch_fwd_as(const void* logits, int64_t pitch, const float* tokens, float* logprobs, float* entropy, float* lse,
                  int32_t* top_ids, float* top_logprobs, int64_t top, int64_t rows, int64_t V, float c, float inverse_temperature,
                  cudaStream_t stream)
{
    using L = Logit<DTYPE>;
    // few rows: a row is shared by the CTAs of a cluster, as long as each has two vectors per thread to read
    int ctas = 1;
    while(ctas < kMaxCluster && rows * ctas * 2 <= 4 * kSmCount && V / L::VE >= (int64_t)ctas * 2 * kThreads * 2) ctas *= 2;
    if(launch_clusters(token_logprobs_kernel<DTYPE, TOP>, (unsigned)(rows * ctas), kThreads, ctas, stream,
                       static_cast<const typename L::type*>(logits), (long long)pitch, tokens, logprobs, entropy, lse, top_ids,
                       top_logprobs, (int)top, (int)V, c, inverse_temperature) != cudaSuccess) return ONN_ERR_CUDA;
    count_launch();
    return launch_status();
}

template <int DTYPE>
int launch_fwd(const void* logits, int64_t pitch, const float* tokens, float* logprobs, float* entropy, float* lse,
               int32_t* top_ids, float* top_logprobs, int64_t top, int64_t rows, int64_t V, float c, float inverse_temperature,
               cudaStream_t stream)
{
    const auto launch = top > 0 ? launch_fwd_as<DTYPE, true> : launch_fwd_as<DTYPE, false>;
    return launch(logits, pitch, tokens, logprobs, entropy, lse, top_ids, top_logprobs, top, rows, V, c, inverse_temperature, stream);
}

template <int DTYPE>
int launch_bwd(const void* logits, int64_t pitch, const float* tokens, const float* lse, const float* entropy,
               const float* d_logprobs, const float* d_entropy, void* dlogits, int64_t d_pitch, int64_t rows, int64_t V,
               float inverse_temperature, cudaStream_t stream)
{
    using L = Logit<DTYPE>;
    const int pieces = (int)((V / L::VE + kThreads * kUnroll - 1) / (kThreads * kUnroll));
    // the second grid dimension holds at most 65535 rows
    for(int64_t first = 0; first < rows; first += 65535)
    {
        const int64_t n = rows - first < 65535 ? rows - first : 65535;
        token_logprobs_bwd_kernel<DTYPE><<<dim3(pieces > 0 ? pieces : 1, (unsigned)n), kThreads, 0, stream>>>(
            static_cast<const typename L::type*>(logits) + first * pitch, pitch, tokens ? tokens + first : nullptr, lse + first,
            entropy ? entropy + first : nullptr, d_logprobs + first, d_entropy ? d_entropy + first : nullptr,
            static_cast<typename L::type*>(dlogits) + first * d_pitch, d_pitch, (int)V, inverse_temperature);
        count_launch();
        if(launch_status() != ONN_OK) return ONN_ERR_CUDA;
    }
    return ONN_OK;
}

}  // namespace

}  // namespace onn

using namespace onn;

extern "C" int onn_token_logprobs(const void* logits, int dtype, int64_t pitch, const float* tokens,
                                  float* logprobs, float* entropy, float* lse, int32_t* top_ids, float* top_logprobs, int64_t top,
                                  int64_t rows, int64_t V, float temperature, void* stream)
{
    ONN_CHECK_ARG(logit_arguments_ok(logits, dtype, pitch, rows, V) && temperature_ok(temperature));
    ONN_CHECK_ARG(top >= 0 && (top == 0 || (top_ids && top_logprobs)));
    ONN_CHECK_ARG((tokens || !logprobs) && (logprobs || entropy || lse || top > 0));
    if(top > ONN_TOP_MAX) return ONN_ERR_LIMIT;
    const float c = kLog2E / temperature, inverse = 1.0f / temperature;
    cudaStream_t s = (cudaStream_t)stream;
    switch(dtype)
    {
        case ONN_F32: return launch_fwd<ONN_F32>(logits, pitch, tokens, logprobs, entropy, lse, top_ids, top_logprobs, top, rows, V, c, inverse, s);
        case ONN_BF16: return launch_fwd<ONN_BF16>(logits, pitch, tokens, logprobs, entropy, lse, top_ids, top_logprobs, top, rows, V, c, inverse, s);
        default: return launch_fwd<ONN_F16>(logits, pitch, tokens, logprobs, entropy, lse, top_ids, top_logprobs, top, rows, V, c, inverse, s);
    }
}

extern "C" int onn_token_logprobs_bwd(const void* logits, int dtype, int64_t pitch, const float* tokens, const float* lse,
                                      const float* entropy, const float* d_logprobs, const float* d_entropy,
                                      void* dlogits, int64_t d_pitch, int64_t rows, int64_t V, float temperature, void* stream)
{
    ONN_CHECK_ARG(logit_arguments_ok(logits, dtype, pitch, rows, V) && temperature_ok(temperature));
    ONN_CHECK_ARG(tokens && lse && d_logprobs && (entropy || !d_entropy));
    ONN_CHECK_ARG(logit_arguments_ok(dlogits, dtype, d_pitch, rows, V));
    const float inverse = 1.0f / temperature;
    cudaStream_t s = (cudaStream_t)stream;
    switch(dtype)
    {
        case ONN_F32: return launch_bwd<ONN_F32>(logits, pitch, tokens, lse, entropy, d_logprobs, d_entropy, dlogits, d_pitch, rows, V, inverse, s);
        case ONN_BF16: return launch_bwd<ONN_BF16>(logits, pitch, tokens, lse, entropy, d_logprobs, d_entropy, dlogits, d_pitch, rows, V, inverse, s);
        default: return launch_bwd<ONN_F16>(logits, pitch, tokens, lse, entropy, d_logprobs, d_entropy, dlogits, d_pitch, rows, V, inverse, s);
    }
}
