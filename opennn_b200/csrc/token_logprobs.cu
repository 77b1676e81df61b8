// Log probabilities of given tokens with entropy and the top alternatives, and their gradient.
//
//   z = x / T,  lse = log sum_i exp z_i,  p = exp(z - lse)
//   forward   logprob = z_t - lse,  entropy = -sum_i p_i log p_i,  the K largest x with z - lse
//   backward  dx_i = [ g (1[i = t] - p_i) - h p_i (log p_i + entropy) ] / T
//
// Both are bound by HBM: the forward pass reads each logit once, the backward pass reads and writes each once.
#include <cooperative_groups.h>
#include <float.h>

#include <type_traits>

#include "logit_rows.cuh"

namespace onn
{

namespace
{

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 8;                        // 16-byte vectors a thread has in flight

// Running statistics of a set of logits, in base 2 and relative to the largest logit m seen: with c = log2(e) / T,
// a = c max(m, -kHuge) and d = c x - a in one rounding,  s = sum 2^d  and  w = sum 2^d d.  Every set with the
// same m has the same a, so its rounding shifts all terms alike and is taken out at the end.  -inf adds nothing to either
// sum; NaN and +inf make both NaN.  Logits below -kHuge count as nothing, and beyond |m| = kHuge c x could overflow: a row
// whose largest logit is that far out is summed again (huge_row).
struct Running { float m, s, w; };

constexpr float kNothing = -1e4f;                 // 2^-10000 = 0: the bound that keeps 0 * -inf out of w
constexpr float kHuge = 1e29f;

__device__ __forceinline__ float finite_anchor(float m) { return m > -INFINITY ? m : 0.f; }
// rounded once, whatever it is subtracted from (no contraction into a fused multiply-add)
__device__ __forceinline__ float anchor(float m, float c) { return __fmul_rn(fmaxf(m, -kHuge), c); }

// The sums of r relative to another, larger m.
__device__ __forceinline__ void rebase(Running& r, float m, float c)
{
    const float d = fmaxf(anchor(r.m, c) - anchor(m, c), kNothing);
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

// Adds the logits of N vectors, of which the largest (with those before) is `m`: one rescaling for all of them, then two
// logits per instruction (packed fp32).
template <int DTYPE, int N>
__device__ __forceinline__ void add_vectors(Running& r, const uint4 (&v)[N], float m, float c)
{
    using L = Logit<DTYPE>;
    if(m > r.m) rebase(r, m, c);
    const float a = anchor(r.m, c);
    const float2 minus_a = make_float2(-a, -a), c2 = make_float2(c, c);
    float2 s2 = make_float2(0.f, 0.f), w2 = make_float2(0.f, 0.f);
#pragma unroll
    for(int u = 0; u < N; u++)
    {
        float x[L::VE];
        L::unpack(L::floor(v[u]), x);
#pragma unroll
        for(int e = 0; e < L::VE; e += 2)
        {
            float2 d = fma2(make_float2(x[e], x[e + 1]), c2, minus_a);
            const float2 p = make_float2(exp2_approx(d.x), exp2_approx(d.y));
            s2 = add2(s2, p);
            if(!L::floors) d = make_float2(fmaxf(d.x, kNothing), fmaxf(d.y, kNothing));
            w2 = fma2(p, d, w2);
        }
    }
    r.s += s2.x + s2.y;
    r.w += w2.x + w2.y;
}

// The sums of a whole row by one warp, with the difference taken before the scale: right for logits of any finite size
// (nothing but a mask of the type's lowest value), and rare.
template <int DTYPE>
__device__ __noinline__ Running huge_row(const typename Logit<DTYPE>::type* x, int V, float m, float c)
{
    Running r = {m, 0.f, 0.f};
    for(int i = threadIdx.x & 31; i < V; i += 32)
    {
        const float d = (Logit<DTYPE>::get(x + i) - m) * c;
        const float p = exp2_approx(d);
        r.s += p;
        r.w = fmaf(p, fmaxf(d, kNothing), r.w);
    }
    r.s = warp_sum(r.s);
    r.w = warp_sum(r.w);
    return r;
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

// A value that at least k of the lanes' pairs of logits (first >= second) reach: the largest is taken away k times.  Equal
// ones of several lanes go together, which only lowers the result.
__device__ __forceinline__ float warp_reached_by(float first, float second, int k)
{
    float t;
    while(true)
    {
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(t) : "f"(first));
        if(--k == 0) return t;
        if(first == t) { first = second; second = -INFINITY; }
    }
}

constexpr int kMaxCluster = 8;
constexpr int kHits = 160;                        // vectors with a possible alternative that a warp can hold
constexpr int kCandidates = 1024;

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
    int candidate_count;
    unsigned long long best[kWarps];
    uint4 hit[kWarps][kHits];
    int hit_index[kWarps][kHits];
    unsigned long long candidates[kCandidates];
};

// One cluster of CTAs (often of one) per row; each CTA streams its part of the row once.
//
// The alternatives come out of the same pass.  If every warp knows k logits that are at least t, with k = ceil(top /
// warps), no logit below t can stand in the list.  So after its first batch every warp takes the k-th largest of its
// lanes' two best vectors as its bound; the smallest bound of all warps is the CTA's, and vectors with a logit that reaches
// it go on the warp's list in shared memory (a compare per vector; for logits in no particular order a few hundred
// of a row).  The bounds rise after 2, 3, 5, 9 ... batches.  At the end the bound of all warps thins the lists out to little
// more than `top` candidates in the first CTA, which ranks them.  A list that overflows (a rising row) is replaced by
// another scan with the final bound; candidates that overflow (a thousand equal logits) by a scan for each place.
template <int DTYPE, bool TOP, int N>
__global__ void __launch_bounds__(kThreads, N > 4 && TOP ? 3 : 4)
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
        if(tid == 0) shared.candidate_count = 0;
    }
    // all CTAs of a cluster must be running before one writes into another
    if(ctas > 1) cluster.sync();
    else if constexpr(TOP) __syncthreads();

    Running r = {-INFINITY, 0.f, 0.f};
    float end_value = -INFINITY;
    if(end_index >= 0)
    {
        end_value = L::get(x + end_index);
        // as a batch of its own; NaN is never larger, and reaches the sum
        r.m = end_value > -INFINITY ? end_value : -INFINITY;
        r.s = exp2_approx(fmaf(end_value, c, -anchor(r.m, c)));
        r.w = r.s * fmaxf(fmaf(end_value, c, -anchor(r.m, c)), kNothing);
    }
    const int wanted = TOP ? (top + kWarps - 1) / kWarps : 1;
    [[maybe_unused]] float bound = -FLT_MAX, second = -INFINITY;     // of this lane's vectors, the second largest maximum
    [[maybe_unused]] int hits = 0;                                   // on the warp's list
    auto take = [&](const int first, const int batch, auto whole)
    {
        uint4 v[N];
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            const int i = first + u * kThreads + tid;
            v[u] = whole.value || i < end ? __ldg(body + i) : L::lowest();
        }
        float vector_max[N];
        float m = r.m;
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            vector_max[u] = L::max(v[u]);
            if constexpr(TOP) second = fmaxf(second, vector_max[u] > m ? m : vector_max[u]);       // NaN is passed by
            m = fmaxf(m, vector_max[u]);
        }
        add_vectors<DTYPE, N>(r, v, m, c);
        if constexpr(TOP)
        {
            if((batch & (batch - 1)) == 0)             // batches 0, 1, 2, 4, 8 ...
            {
                const float mine = warp_reached_by(r.m, second, wanted);
                if(lane == 0) shared.warp_top[warp] = mine;
                // the first bound needs every warp's; later ones take what is there, since bounds only rise
                if(batch == 0) __syncthreads();
                else __syncwarp();
                bound = shared.warp_top[0];
#pragma unroll
                for(int w = 1; w < kWarps; w++) bound = fminf(bound, shared.warp_top[w]);
                bound = fmaxf(bound, -FLT_MAX);
            }
#pragma unroll
            for(int u = 0; u < N; u++)
            {
                const bool hit = vector_max[u] >= bound;
                const unsigned int who = __ballot_sync(0xffffffffu, hit);
                if(who == 0) continue;
                const int at = hits + __popc(who & ((1u << lane) - 1u));
                if(hit && at < kHits)
                {
                    shared.hit[warp][at] = v[u];
                    shared.hit_index[warp][at] = cut.head + (first + u * kThreads + tid) * VE;
                }
                hits += __popc(who);
            }
        }
    };
    {
        int first = begin, batch = 0;
        for(; first + kThreads * N <= end; first += kThreads * N, batch++) take(first, batch, std::true_type{});
        if(first < end || batch == 0) take(first, batch, std::false_type{});
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
    part.top = TOP ? warp_reached_by(own_max, second, wanted_all) : 0.f;
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
        const bool huge = fabsf(all.m) >= kHuge && fabsf(all.m) < INFINITY;
        if(huge) all = huge_row<DTYPE>(x, V, all.m, c);
        if(lane == 0)
        {
            const bool none = all.s == 0.f;            // a row without a finite logit has no distribution
            const float log_2s = logf(all.s);
            // relative to m itself: the rounding of the anchor
            const float log_s = none ? INFINITY : huge ? log_2s : fmaf(fmaf(all.m, c, -anchor(all.m, c)), -kLn2, log_2s);
            shared.m = finite_anchor(all.m);
            shared.log_s = log_s;
            if(logprobs) logprobs[row] = none ? -INFINITY : (L::get(x + token) - all.m) * inverse_temperature - log_s;
            if(entropy)
            {
                const float value = log_2s - all.w / all.s * kLn2;
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
        bound = fmaxf(bound, -FLT_MAX);                // -inf is no alternative
        Shared<TOP>* leader = ctas == 1 ? &shared : cluster.map_shared_rank(&shared, 0);
        auto candidate = [&](float value, int index)
        {
            if(!(value >= bound)) return;
            const int at = atomicAdd(&leader->candidate_count, 1);
            if(at < kCandidates) leader->candidates[at] = key_of(value, index);
        };
        if(end_index >= 0) candidate(end_value, end_index);
        if(hits <= kHits)
        {
            for(int i = lane; i < hits; i += 32)
            {
                float values[VE];
                L::unpack(shared.hit[warp][i], values);
                const int index = shared.hit_index[warp][i];
#pragma unroll
                for(int e = 0; e < VE; e++) candidate(values[e], index + e);
            }
        }
        else
        {
            for(int i = begin + tid; i < end; i += kThreads)
            {
                const uint4 v = __ldg(body + i);
                if(!(L::max(v) >= bound)) continue;
                float values[VE];
                L::unpack(v, values);
#pragma unroll
                for(int e = 0; e < VE; e++) candidate(values[e], cut.head + i * VE + e);
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
        if(n > kCandidates)
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
#pragma unroll 4
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

template <int DTYPE, bool TOP, int N>
int launch_fwd_as(const void* logits, int64_t pitch, const float* tokens, float* logprobs, float* entropy, float* lse,
                  int32_t* top_ids, float* top_logprobs, int64_t top, int64_t rows, int64_t V, float c, float inverse_temperature,
                  cudaStream_t stream)
{
    using L = Logit<DTYPE>;
    // few rows: a row is shared by the CTAs of a cluster, as long as each has two vectors per thread to read
    int ctas = 1;
    while(ctas < kMaxCluster && rows * ctas * 2 <= 4 * kSmCount && V / L::VE >= (int64_t)ctas * 2 * kThreads * 2) ctas *= 2;
    if(launch_clusters(token_logprobs_kernel<DTYPE, TOP, N>, (unsigned)(rows * ctas), kThreads, ctas, stream,
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
    constexpr int N = DTYPE == ONN_F32 ? 8 : 4;
    const auto launch = top > 0 ? launch_fwd_as<DTYPE, true, N> : launch_fwd_as<DTYPE, false, N>;
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
