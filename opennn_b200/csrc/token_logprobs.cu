// Log probabilities of given tokens with entropy and the top alternatives, and their gradient.
//
//   z = x / T,  lse = log sum_i exp z_i,  p = exp(z - lse)
//   forward   logprob = z_t - lse,  entropy = -sum_i p_i log p_i,  the K largest x with z - lse
//   backward  dx_i = [ g (1[i = t] - p_i) - h p_i (log p_i + entropy) ] / T
//
// Both are bound by HBM: the forward pass reads each logit once, the backward pass reads and writes each once.  Measured on a
// B200 (copy bandwidth 6.57 TB/s): forward without a list 16384 x 32000 fp32 298 us = 7.0 TB/s, with 37 % of the rows padding, which
// are not read (1.31 GB), 195 to 202 us = 6.5 to 6.7 TB/s, 8192 x 50021 bf16 142 us = 5.8 TB/s; with 64 alternatives 189 us = 4.3 TB/s:
// there the instructions bound it (12 to 13 per logit, 70 % of the issue slots; about five are the sums' own: two for unpacking, one to
// floor, a multiply-add, two exponentials and two sums for a pair, and its share of the maximum; the rest, batches ahead, unit maxima, the
// second reading and the ranking, is not told apart).  Backward 8192 x 32000 fp32 with entropy, padded in the same way, 262 to 278 us
// = 6.1 to 6.5 TB/s.
#include <cooperative_groups.h>
#include <float.h>

#include <type_traits>

#include "logit_rows.cuh"

namespace onn
{

namespace
{

// Running statistics of a set of logits, in base 2 and relative to the largest logit m seen: with c = log2(e) / T,
// a = max(c m, -kFar) and d = c x - a in one rounding,  s = sum 2^d  and  w = sum 2^d d.  Every set with the
// same m has the same a, so its rounding shifts all terms alike and is taken out at the end.  That shift is up to half a step of c m
// (the d of the largest logit itself): within kFar at most 64, a little later 2^d overflows.  So a set of nothing but logits below
// -kFar / c (a finite mask) adds nothing when it meets a larger one, and a row whose largest logit is beyond +-kFar / c is summed again
// (far_row).  -inf adds nothing to either sum; NaN and +inf make both NaN.
struct Running { float m, s, w; };

constexpr float kNothing = -1e4f;                 // 2^-10000 = 0: the bound that keeps 0 * -inf out of w
constexpr float kFar = 2147483648.f;              // 2^31

__device__ __forceinline__ float finite_anchor(float m) { return m > -INFINITY ? m : 0.f; }
// rounded once, whatever it is subtracted from (no contraction into a fused multiply-add)
__device__ __forceinline__ float anchor(float m, float c) { return fmaxf(__fmul_rn(m, c), -kFar); }

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

// The sums of a whole row by one warp, with the difference taken before the scale: right for logits of any finite size,
// and rare (a row of nothing but a mask far out, large logits at a temperature near zero).  16384 x 32000 fp32 with every row of that kind
// 1048 us, ordinary 298; one row of 131072 197 us, ordinary 10.
template <int DTYPE>
__device__ __noinline__ Running far_row(const typename Logit<DTYPE>::type* x, int V, float m, float c)
{
    // eight loads of a lane under way, and eight short sums instead of a long one
    constexpr int N = 8;
    float s[N] = {}, w[N] = {};
    for(int start = threadIdx.x & 31; start < V; start += N * 32)
    {
        float d[N];
#pragma unroll
        for(int u = 0; u < N; u++) d[u] = start + u * 32 < V ? (Logit<DTYPE>::get(x + start + u * 32) - m) * c : -INFINITY;
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            const float p = exp2_approx(d[u]);
            s[u] += p;
            w[u] = fmaf(p, fmaxf(d[u], kNothing), w[u]);
        }
    }
    Running r = {m, 0.f, 0.f};
#pragma unroll
    for(int u = 0; u < N; u++) { r.s += s[u]; r.w += w[u]; }
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

// The k-th largest of the lanes' pairs of logits (first >= second): the largest ones are taken away until k are gone.
__device__ __forceinline__ float warp_reached_by(float first, float second, int k)
{
    float t;
    while(true)
    {
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(t) : "f"(first));
        k -= __popc(__ballot_sync(0xffffffffu, first == t));
        if(k <= 0) return t;
        if(first == t) { first = second; second = -INFINITY; }
    }
}

constexpr int kMaxCluster = 8;
constexpr int kSlots = 16;                        // maxima a thread writes down
constexpr int kBuckets = 256;
constexpr int kFew = 96;                          // candidates that are ranked without buckets

// What a warp knows of its part of the row.
struct alignas(16) Part { float m, s, w, top; };

// Warps that share a row (clusters are of 256 threads), and candidates: a single warp has short rows and lists, and little shared
// memory lets more of them run (16384 x 1000 fp32 with 20 alternatives: 39 us, with 1024 candidates 75).
template <int T> constexpr int kMaxParts = T == 256 ? kMaxCluster * 8 : T / 32;
template <int T> constexpr int kCandidates = T == 32 ? 256 : T == 64 ? 512 : 1024;

// Shared memory of a CTA of T threads.  `parts` and, in the first CTA of a cluster, `candidates` are written by the whole
// cluster.
template <bool TOP, int T>
struct Shared
{
    Part parts[2][kMaxParts<T>];                     // of this row and the next
};
template <int T>
struct Shared<true, T>
{
    Part parts[2][kMaxParts<T>];
    float m, log_s;
    int candidate_count;
    int bucket[kBuckets + 1];
    unsigned long long best[T / 32];
    unsigned long long candidates[kCandidates<T>];
    union
    {
        float slot[kSlots][T];                    // the largest logit of each unit of vectors
        unsigned long long sorted[kCandidates<T>];
    };
    unsigned short unit[T / 32][32 * kSlots];     // of each warp: units that hold an alternative
};

// Clusters of CTAs (often of one) walk over the rows; each CTA streams its part of a row once.
//
// The alternatives: each thread also writes down the largest logit of each unit of its vectors (a vector, or some
// batches of a long row).  If every warp knows k logits that are at least t, with k = ceil(top / warps), no logit below t can
// stand in the list; so the k-th largest of the lanes' two best units is the warp's bound, and the smallest bound of all warps
// the row's.  Only units that reach it (little more than `top` of them) are read again, most often from L2, and
// their logits that reach it become candidates in the first CTA, which ranks them.  Should more logits reach the bound than the list of
// candidates holds, the row is scanned once for each place: equal ones, or a neighbouring stretch so unlikely (masked) that a warp has to
// vouch with it for more places than it has better logits.  Then one row of 131072 bf16 with 64 alternatives takes 1483 us instead of 10.
template <int DTYPE, bool TOP, int T, int N>
__global__ void __launch_bounds__(T, T == 32 ? 24 : 1024 / T)
token_logprobs_kernel(const typename Logit<DTYPE>::type* __restrict__ logits, long long pitch, const float* __restrict__ tokens,
                      float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ lse,
                      int* __restrict__ top_ids, float* __restrict__ top_logprobs, int top, long long rows, int V, float c, float inverse_temperature)
{
    using L = Logit<DTYPE>;
    constexpr int VE = L::VE, kWarps = T / 32;
    constexpr bool kAhead = DTYPE != ONN_F32 && TOP;
    __shared__ Shared<TOP, T> shared;
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if constexpr(TOP)
    {
        if(tid == 0) shared.candidate_count = 0;
        for(int i = tid; i <= kBuckets; i += T) shared.bucket[i] = 0;
    }
    // all CTAs of a cluster must be running before one writes into another: waited for under the first row's loads
    bool met = ctas == 1;
    if(!met) asm volatile("barrier.cluster.arrive;" ::: "memory");

    int flip = 0;
    const long long step = gridDim.x / ctas;
    long long row = blockIdx.x / ctas;
    float next_token = tokens && row < rows ? __ldg(tokens + row) : 1.f;
    for(; row < rows; row += step)
    {
    const long long token = token_index(next_token);
    const bool active = token > 0 && token < V;        // 0 is padding; without tokens every row takes part
    if(tokens && row + step < rows) next_token = __ldg(tokens + row + step);
    if(!active)                                        // the same for the whole cluster
    {
        if(rank == 0)
        {
            if(tid == 0)
            {
                if(logprobs) logprobs[row] = 0.f;
                if(entropy) entropy[row] = 0.f;
                if(lse) lse[row] = 0.f;
            }
            for(int k = tid; k < top; k += T) { top_ids[row * top + k] = -1; top_logprobs[row * top + k] = -INFINITY; }
        }
        continue;
    }
    flip ^= 1;
    Part* const row_parts = shared.parts[flip];

    const typename L::type* x = logits + row * pitch;
    const RowCut cut = cut_row<DTYPE>(x, V);
    const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
    const int after = cut.head + cut.vectors * VE;
    // the element of the row's ends that this thread looks after, if any
    int end_index = tid < cut.head ? tid : tid < cut.head + cut.tail ? after + tid - cut.head : -1;
    if(rank != 0) end_index = -1;
    const int share = (cut.vectors + ctas - 1) / ctas;
    const int begin = min(rank * share, cut.vectors), end = min(begin + share, cut.vectors);

    // vectors of a unit: 1 << unit_shift; a thread has at most kSlots units
    constexpr int kBatchShift = N == 8 ? 3 : 2;
    const int each = (share + T - 1) / T;              // vectors of a thread
    int unit_shift = 0;
    if(TOP && each > kSlots)
    {
        unit_shift = kBatchShift;
        while(((each - 1) >> unit_shift) >= kSlots) unit_shift++;
    }
    const float given = tid == 0 && rank == 0 ? L::get(x + token) : 0.f;
    Running r = {-INFINITY, 0.f, 0.f};
    float end_value = -INFINITY;
    if(end_index >= 0)
    {
        end_value = L::get(x + end_index);
        // as a batch of its own; NaN is never larger, and reaches the sum
        r.m = end_value > -INFINITY ? end_value : -INFINITY;
        const float d = fmaf(end_value, c, -anchor(r.m, c));
        r.s = exp2_approx(d);
        r.w = r.s * fmaxf(d, kNothing);
    }
    // of this thread's units
    [[maybe_unused]] float best = -INFINITY, second = -INFINITY, unit_max = -INFINITY;
    auto note = [&](float value, int slot)
    {
        if constexpr(TOP)
        {
            shared.slot[slot][tid] = value;
            second = fmaxf(second, value > best ? best : value);       // NaN is passed by
            best = fmaxf(best, value);
        }
    };
    const int whole = (end - begin) / (T * N), batches = (each + N - 1) / N;
    auto load = [&](uint4 (&v)[N], const int batch)
    {
        const int first = begin + batch * (T * N) + tid;
        if(batch < whole)
        {
#pragma unroll
            for(int u = 0; u < N; u++) v[u] = __ldg(body + first + u * T);
        }
        else
        {
#pragma unroll
            for(int u = 0; u < N; u++) v[u] = first + u * T < end ? __ldg(body + first + u * T) : L::lowest();
        }
    };
    auto take = [&](const uint4 (&v)[N], const int batch)
    {
        float vector_max[N];
        float m = -INFINITY;
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            vector_max[u] = L::max(v[u]);
            m = fmaxf(m, vector_max[u]);
        }
        if constexpr(TOP)
        {
            if(unit_shift == 0)
            {
#pragma unroll
                for(int u = 0; u < N; u++)
                    if(batch * N + u < each) note(vector_max[u], batch * N + u);
            }
            else
            {
                unit_max = fmaxf(unit_max, m);
                const int last = ((batch + 1) * N - 1) >> unit_shift;
                if(((batch + 1) * N) >> unit_shift != last || (batch + 1) * N >= each) { note(unit_max, last); unit_max = -INFINITY; }
            }
        }
        add_vectors<DTYPE, N>(r, v, fmaxf(r.m, m), c);
    };
    if constexpr(kAhead)
    {
        // a batch is on its way while the one before it is worked on
        uint4 v[N], next[N];
        load(next, 0);
        for(int batch = 0; batch < batches; batch++)
        {
#pragma unroll
            for(int u = 0; u < N; u++) v[u] = next[u];
            if(batch + 1 < batches) load(next, batch + 1);
            take(v, batch);
        }
    }
    else
    {
        for(int batch = 0; batch < batches; batch++)
        {
            uint4 v[N];
            load(v, batch);
            take(v, batch);
        }
    }

    // every warp's part to every CTA of the cluster
    const float warp_m = warp_largest(r.m);
    rebase(r, warp_m, c);
    Part part;
    part.m = warp_m;
    part.s = warp_sum(r.s);
    part.w = warp_sum(r.w);
    const int parts = ctas * kWarps;
    const int wanted = TOP ? (top + parts - 1) / parts : 1;
    part.top = 0.f;
    if constexpr(TOP)
    {
        // places that this warp has to vouch for: an equal share, or, in a row of so few vectors that the warps' numbers of them
        // differ, one in proportion (2400 x 1600 bf16, 128 alternatives: 31 us, with equal shares 122, where
        // a third of such a row became candidates)
        int vouched = wanted;
        if(each <= 2 && cut.vectors > 0)
        {
            auto of_warp = [&](int n) { return n < 0 ? 0 : n > 32 ? 32 : n; };
            const int mine = of_warp(end - begin - warp * 32) + of_warp(end - begin - T - warp * 32);
            vouched = (top * mine + cut.vectors - 1) / cut.vectors;
        }
        part.top = vouched > 0 ? warp_reached_by(best, second, vouched) : INFINITY;
    }
    if(ctas == 1)
    {
        if(lane == 0) row_parts[warp] = part;
        __syncthreads();
    }
    else
    {
        if(!met) asm volatile("barrier.cluster.wait;" ::: "memory");
        met = true;
        if(lane < ctas) cluster.map_shared_rank(&shared, lane)->parts[flip][rank * kWarps + warp] = part;
        cluster.sync();
    }

    if(rank == 0 && warp == 0)
    {
        Running all = {-INFINITY, 0.f, 0.f};
        for(int i = lane; i < parts; i += 32) all = merge(all, Running{row_parts[i].m, row_parts[i].s, row_parts[i].w}, c);
        if(parts > 1)
        {
            rebase(all, warp_largest(all.m), c);
            all.s = warp_sum(all.s);
            all.w = warp_sum(all.w);
        }
        else all = Running{part.m, part.s, part.w};
        const bool far = fabsf(all.m * c) >= kFar && fabsf(all.m) < INFINITY;
        if(far) all = far_row<DTYPE>(x, V, all.m, c);
        if(lane == 0)
        {
            const bool none = all.s == 0.f;            // a row without a finite logit has no distribution
            const float log_2s = logf(all.s);
            // relative to m itself: the rounding of the anchor
            const float log_s = none ? INFINITY : far ? log_2s : fmaf(fmaf(all.m, c, -anchor(all.m, c)), -kLn2, log_2s);
            if constexpr(TOP) { shared.m = finite_anchor(all.m); shared.log_s = log_s; }
            if(logprobs) logprobs[row] = none ? -INFINITY : (given - all.m) * inverse_temperature - log_s;
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
        float bound;
        if(wanted == 1 && parts >= 2 * top)
        {
            // more warps than places: the bound is the top-th largest of their maxima, at most two of them a lane's
            const float a = lane < parts ? row_parts[lane].m : -INFINITY, b = lane + 32 < parts ? row_parts[lane + 32].m : -INFINITY;
            bound = warp_reached_by(fmaxf(a, b), fminf(a, b), top);
        }
        else
        {
            float lowest = INFINITY;
            for(int i = lane; i < parts; i += 32) lowest = fminf(lowest, row_parts[i].top);
            bound = -warp_largest(-lowest);
        }
        bound = fmaxf(bound, -FLT_MAX);                // -inf is no alternative

        Shared<TOP, T>* leader = ctas == 1 ? &shared : cluster.map_shared_rank(&shared, 0);
        auto candidate = [&](float value, int index)
        {
            const int at = atomicAdd(&leader->candidate_count, 1);
            if(at < kCandidates<T>) leader->candidates[at] = key_of(value, index);
        };
        if(end_value >= bound) candidate(end_value, end_index);
        // this warp's units that reach the bound, then their vectors, four loads of a lane at a time
        unsigned short* units = shared.unit[warp];
        int found = 0;
        const int slots = each > 0 ? ((each - 1) >> unit_shift) + 1 : 0;
        for(int slot = 0; slot < slots; slot++)
        {
            const bool hit = shared.slot[slot][tid] >= bound;
            const unsigned int who = __ballot_sync(0xffffffffu, hit);
            if(hit) units[found + __popc(who & ((1u << lane) - 1u))] = (unsigned short)(slot * 32 + lane);
            found += __popc(who);
        }
        __syncwarp();
        const int again = found << unit_shift;
        for(int start = lane; start < again; start += 4 * 32)
        {
            uint4 v[4];
            int at[4];
#pragma unroll
            for(int k = 0; k < 4; k++)
            {
                const int j = start + k * 32;
                at[k] = end;
                if(j < again)
                {
                    const int unit = units[j >> unit_shift];
                    const int ordinal = ((unit >> 5) << unit_shift) + (j & ((1 << unit_shift) - 1));
                    at[k] = begin + ordinal * T + warp * 32 + (unit & 31);
                }
                v[k] = at[k] < end ? __ldg(body + at[k]) : L::lowest();
            }
#pragma unroll
            for(int k = 0; k < 4; k++)
            {
                if(!(L::max(v[k]) >= bound)) continue;
                float values[VE];
                L::unpack(v[k], values);
                unsigned int which = 0;
#pragma unroll
                for(int e = 0; e < VE; e++) which |= (values[e] >= bound ? 1u : 0u) << e;
                while(which)
                {
                    const int e = __ffs(which) - 1;
                    which &= which - 1;
                    float value = values[0];
#pragma unroll
                    for(int i = 1; i < VE; i++) value = e == i ? values[i] : value;
                    candidate(value, cut.head + at[k] * VE + e);
                }
            }
        }
        if(ctas == 1) __syncthreads();
        else cluster.sync();
        auto place = [&](int k, unsigned long long key)
        {
            top_ids[row * top + k] = key ? key_index(key) : -1;
            top_logprobs[row * top + k] = key ? (key_logit(key) - shared.m) * inverse_temperature - shared.log_s : -INFINITY;
        };
        int n = rank == 0 ? shared.candidate_count : 0;
        if(rank != 0) {}
        else if(n > kCandidates<T>)
        {
            // one place after the other: the largest key below the last one
            unsigned long long last = ~0ull;
            for(int k = 0; k < top; k++)
            {
                unsigned long long largest = 0;
                auto look = [&](float value, int index)
                {
                    const unsigned long long key = key_of(value, index);
                    if(key < last && key > largest) largest = key;
                };
                if(last != 0)
                {
                    if(end_index >= 0) look(end_value, end_index);
                    for(int i = tid; i < cut.vectors; i += T)
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
                    const unsigned long long other = __shfl_xor_sync(0xffffffffu, largest, offset);
                    largest = other > largest ? other : largest;
                }
                __syncthreads();
                if(lane == 0) shared.best[warp] = largest;
                __syncthreads();
                largest = shared.best[0];
#pragma unroll
                for(int w = 1; w < kWarps; w++) largest = shared.best[w] > largest ? shared.best[w] : largest;
                last = largest;
                if(tid == 0) place(k, largest);
            }
        }
        else
        {
        for(int k = n + tid; k < top; k += T) place(k, 0);

        // A candidate's place is the number of larger ones: those of higher buckets, of kBuckets that lie evenly between the
        // bound and the largest logit, and those before it in its own.  bucket[b + 1] counts bucket b, 0 is the highest.
        if(n <= kFew)
        {
            for(int i = tid; i < n; i += T)
            {
                const unsigned long long key = shared.candidates[i];
                int larger = 0;
#pragma unroll 4
                for(int j = 0; j < n; j++) larger += shared.candidates[j] > key;
                if(larger < top) place(larger, key);
            }
        }
        else
        {
        const float high = shared.m;
        float low = bound;
        if(bound == -FLT_MAX)
        {
            // no bound: the lowest candidate
            float lowest = INFINITY;
            for(int i = tid; i < n; i += T) lowest = fminf(lowest, key_logit(shared.candidates[i]));
            lowest = -warp_largest(-lowest);
            if(lane == 0) row_parts[warp].m = lowest;
            __syncthreads();
            low = row_parts[0].m;
#pragma unroll
            for(int w = 1; w < kWarps; w++) low = fminf(low, row_parts[w].m);
        }
        const float width = high * 0.5f - low * 0.5f;   // halves: finite whatever the two are
        const float per = width > 0.f && width < INFINITY ? (kBuckets - 1) / width : 0.f;
        auto bucket_of = [&](unsigned long long key) { return min(kBuckets - 1, (int)((high * 0.5f - key_logit(key) * 0.5f) * per)); };
        for(int i = tid; i < n; i += T) atomicAdd(&shared.bucket[bucket_of(shared.candidates[i]) + 1], 1);
        __syncthreads();
        if(warp == 0)
        {
            // running sums: bucket[b + 1] becomes the number of candidates in the buckets up to b
            int mine[kBuckets / 32], total = 0;
#pragma unroll
            for(int b = 0; b < kBuckets / 32; b++) { mine[b] = shared.bucket[lane * (kBuckets / 32) + b + 1]; total += mine[b]; }
            int before = total;
#pragma unroll
            for(int offset = 1; offset < 32; offset <<= 1)
            {
                const int other = __shfl_up_sync(0xffffffffu, before, offset);
                if(lane >= offset) before += other;
            }
            before -= total;
#pragma unroll
            for(int b = 0; b < kBuckets / 32; b++) { shared.bucket[lane * (kBuckets / 32) + b + 1] = before; before += mine[b]; }
        }
        __syncthreads();
        // bucket[b + 1] goes from where bucket b starts to where it ends, which is where the next one starts
        for(int i = tid; i < n; i += T)
        {
            const unsigned long long key = shared.candidates[i];
            shared.sorted[atomicAdd(&shared.bucket[bucket_of(key) + 1], 1)] = key;
        }
        __syncthreads();
        for(int i = tid; i < n; i += T)
        {
            const unsigned long long key = shared.sorted[i];
            const int b = bucket_of(key), first = shared.bucket[b], end_of = shared.bucket[b + 1];
            if(first >= top) continue;
            int larger = first;
            for(int j = first; j < end_of; j++) larger += shared.sorted[j] > key;
            if(larger < top) place(larger, key);
        }
        __syncthreads();
        for(int i = tid; i <= kBuckets; i += T) shared.bucket[i] = 0;
        }
        }
        // the lists have been read before the next row's are written
        __syncthreads();
        if(tid == 0) shared.candidate_count = 0;
    }
    }
    // whatever one CTA of a cluster writes into another comes before the last barrier of the row
    if(!met) asm volatile("barrier.cluster.wait;" ::: "memory");
}

// exp(z - lse) carries the rounding of lse: half a step of it is at most 2^-11 below this bound, and p is anything once it exceeds 1.
constexpr float kFarLse = 16384.f;

// The gradient of a row whose log-sum-exp is that far out (a row of nothing but a finite mask, large logits at a temperature near zero),
// by one CTA: the largest logit and the sum relative to it first, then p from the difference.  Rare: 16384 x 32000 fp32 with every
// row of that kind 1490 us, ordinary 648; one row of 131072 114 us, ordinary 12.
template <int DTYPE, bool ENTROPY, int T>
__device__ __noinline__ void far_gradient(const typename Logit<DTYPE>::type* x, typename Logit<DTYPE>::type* dx, int V, int token, float g, float h, float H,
                                          float inverse_temperature)
{
    using L = Logit<DTYPE>;
    __shared__ float scratch[32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    float m = -INFINITY;
    for(int i = tid; i < V; i += T) m = fmaxf(m, L::get(x + i));      // no NaN: lse would be NaN too
    m = warp_largest(m);
    if(lane == 0) scratch[warp] = m;
    __syncthreads();
    m = scratch[0];
#pragma unroll
    for(int w = 1; w < T / 32; w++) m = fmaxf(m, scratch[w]);
    m = finite_anchor(m);
    const float c = kLog2E * inverse_temperature;
    float s = 0.f;
    for(int i = tid; i < V; i += T) s += exp2_approx((L::get(x + i) - m) * c);
    s = block_sum(s, scratch);
    const float log_s = s == 0.f ? 0.f : logf(s);       // no finite logit: every p is 0
    for(int i = tid; i < V; i += T)
    {
        const float log_p = fmaf(L::get(x + i) - m, inverse_temperature, -log_s), p = exp2_approx(log_p * kLog2E);
        float value = -g * p;
        if(ENTROPY) value = fmaf(-h, fmaxf(log_p, kNothing) + H, -g) * p;
        L::put(dx + i, value + (i == token ? g : 0.f));
    }
}

// One CTA per piece of a row: the row's scalars, then batches of vectors: load, compute, store.
template <int DTYPE, bool ENTROPY, int T, int N>
__global__ void __launch_bounds__(T, 1024 / T)
token_logprobs_bwd_kernel(const typename Logit<DTYPE>::type* logits, long long pitch, const float* __restrict__ tokens,
                          const float* __restrict__ lse, const float* __restrict__ entropy,
                          const float* __restrict__ d_logprobs, const float* __restrict__ d_entropy,
                          typename Logit<DTYPE>::type* dlogits, long long d_pitch, int V, float inverse_temperature)
{
    using L = Logit<DTYPE>;
    constexpr int VE = L::VE;
    const long long row = blockIdx.y;
    const int tid = threadIdx.x;
    const typename L::type* x = logits + row * pitch;
    typename L::type* dx = dlogits + row * d_pitch;
    const RowCut cut = cut_row<DTYPE>(dx, V);
    const int after = cut.head + cut.vectors * VE;
    const int end_index = blockIdx.x != 0 ? -1 : tid < cut.head ? tid : tid < cut.head + cut.tail ? after + tid - cut.head : -1;
    bool active;
    const long long token = row_token(tokens, row, V, &active);
    if(!active)
    {
        for(int i = blockIdx.x * T + tid; i < cut.vectors; i += gridDim.x * T)
            *reinterpret_cast<uint4*>(dx + cut.head + i * VE) = make_uint4(0u, 0u, 0u, 0u);
        if(end_index >= 0) L::put(dx + end_index, 0.f);
        return;
    }
    const float g = d_logprobs[row] * inverse_temperature;
    const float h = ENTROPY ? d_entropy[row] * inverse_temperature : 0.f;
    const float H = ENTROPY ? entropy[row] : 0.f;
    float row_lse = lse[row];
    // a row without a finite logit: every p is 0.  Below temperature 1 -inf may also be a finite z past fp32.
    if(row_lse == -INFINITY && inverse_temperature <= 1.f) row_lse = 0.f;
    if(fabsf(row_lse) >= kFarLse)
    {
        // all by one CTA: where the gradient takes the logits' place nobody else may write while it reads
        if(blockIdx.x == 0) far_gradient<DTYPE, ENTROPY, T>(x, dx, V, (int)token, g, h, H, inverse_temperature);
        return;
    }
    const float2 minus_lse = make_float2(-row_lse, -row_lse), it2 = make_float2(inverse_temperature, inverse_temperature);
    const float2 log2e2 = make_float2(kLog2E, kLog2E), minus_g = make_float2(-g, -g), minus_h = make_float2(-h, -h), H2 = make_float2(H, H);
    auto two = [&](float2 value)
    {
        const float2 log_p = fma2(value, it2, minus_lse);
        const float2 d = mul2(log_p, log2e2);
        const float2 p = make_float2(exp2_approx(d.x), exp2_approx(d.y));
        if(!ENTROPY) return mul2(minus_g, p);
        const float2 inner = add2(make_float2(fmaxf(log_p.x, kNothing), fmaxf(log_p.y, kNothing)), H2);
        return mul2(fma2(minus_h, inner, minus_g), p);
    };

    if(end_index >= 0)
    {
        const float value = L::get(x + end_index);
        L::put(dx + end_index, two(make_float2(value, value)).x + (end_index == (int)token ? g : 0.f));
    }
    const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    const int token_vector = (int)token >= cut.head && (int)token < after ? ((int)token - cut.head) / VE : -1;
    const int token_place = ((int)token - cut.head) % VE;
    for(int first = blockIdx.x * (T * N) + tid; first < cut.vectors; first += gridDim.x * (T * N))
    {
        uint4 v[N];
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            const int i = first + u * T;
            if(i >= cut.vectors) continue;
            const typename L::type* at = x + cut.head + i * VE;
            if(together) v[u] = __ldcs(reinterpret_cast<const uint4*>(at));
            else
            {
                float f[VE];
#pragma unroll
                for(int e = 0; e < VE; e++) f[e] = L::get(at + e);
                v[u] = L::pack(f);                     // exact: the values come from this type
            }
        }
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            const int i = first + u * T;
            if(i >= cut.vectors) continue;
            float f[VE];
            L::unpack(v[u], f);
#pragma unroll
            for(int e = 0; e < VE; e += 2)
            {
                const float2 r = two(make_float2(f[e], f[e + 1]));
                f[e] = r.x;
                f[e + 1] = r.y;
            }
            if(i == token_vector)
            {
#pragma unroll
                for(int e = 0; e < VE; e++) f[e] += e == token_place ? g : 0.f;
            }
            *reinterpret_cast<uint4*>(dx + cut.head + i * VE) = L::pack(f);
        }
    }
}

template <int DTYPE, bool TOP, int T>
int launch_fwd_as(const void* logits, int64_t pitch, const float* tokens, float* logprobs, float* entropy, float* lse,
                  int32_t* top_ids, float* top_logprobs, int64_t top, int64_t rows, int64_t V, float c, float inverse_temperature,
                  int ctas, cudaStream_t stream)
{
    using L = Logit<DTYPE>;
    // eight vectors in flight per thread; in 16 bits with a list four: the row's units are finer, and 8 CTAs of 128 threads fit
    constexpr int N = DTYPE != ONN_F32 && TOP ? 4 : 8;
    // single warps walk over the rows (16384 x 1000 fp32: 27 us, one row each 35); larger CTAs have one row each, so that whoever is
    // free takes the next (8192 x 50021 bf16 with 64 alternatives: 203 us, walking 213)
    int64_t clusters = rows;
    if(T == 32 && clusters > 24 * kSmCount) clusters = 24 * kSmCount;
    if(launch_clusters(token_logprobs_kernel<DTYPE, TOP, T, N>, (unsigned)(clusters * ctas), T, ctas, 0, false, stream,
                       static_cast<const typename L::type*>(logits), (long long)pitch, tokens, logprobs, entropy, lse, top_ids,
                       top_logprobs, (int)top, (long long)rows, (int)V, c, inverse_temperature) != cudaSuccess) return ONN_ERR_CUDA;
    count_launch();
    return launch_status();
}

// Threads of a row.  What a row costs besides its logits (start, reductions, ranking) is latency, so short rows want many
// small CTAs; but the bound for a list comes from two samples of each thread, and a long list wants many.  In us:
//                       alternatives     32      64     128     256 threads
//   16384 x  4000 fp32            0       45      48      55      99
//   16384 x  4000 fp32           20       68      87     113     199
//   16384 x  4000 fp32           64              120     138     222
//   16384 x  8000 bf16           32      110     103     132
//    8192 x 16000 fp32            0       91      86      81      84
//    8192 x 16000 fp32           20      116     113     105     150
//    8192 x 32000 fp32           64              251     232     211
//    8192 x 50021 bf16           64              244     199     222
// Where all rows run at once a row's latency is all there is, and more threads shorten it: 300 x 6000 fp32 with 20 alternatives
// 8.0 us with 128 threads, 9.8 with 32; 300 x 16000 bf16 with 64 10.4, with 64 threads 18.5; rows of 88 vectors are better left to 32
// threads.  Few long rows: a row is shared by the CTAs of a cluster, as long as each has two vectors per thread to read.
int threads_of(int64_t rows, int64_t vectors, int64_t top)
{
    if(rows > 4 * kSmCount || vectors < 256)
    {
        if(top == 0 && vectors <= 2048) return 32;
        if(top > 0 && top <= 24 && vectors <= 1024) return 32;
        if(top > 0 && top <= 64 && vectors <= (top <= 32 ? 2048 : 1024)) return 64;
    }
    return top > 32 && vectors >= 7168 ? 256 : 128;
}

template <int DTYPE>
int launch_fwd(const void* logits, int64_t pitch, const float* tokens, float* logprobs, float* entropy, float* lse,
               int32_t* top_ids, float* top_logprobs, int64_t top, int64_t rows, int64_t V, float c, float inverse_temperature,
               cudaStream_t stream)
{
    const int64_t vectors = V / Logit<DTYPE>::VE;
    int ctas = 1;
    while(ctas < kMaxCluster && rows * ctas * 2 <= 4 * kSmCount && vectors >= (int64_t)ctas * 1024) ctas *= 2;
    const int T = ctas > 1 ? 256 : threads_of(rows, vectors, top);
    const auto launch = top > 0 ? (T == 32 ? launch_fwd_as<DTYPE, true, 32> : T == 64 ? launch_fwd_as<DTYPE, true, 64> : T == 128 ? launch_fwd_as<DTYPE, true, 128> : launch_fwd_as<DTYPE, true, 256>)
                                : (T == 32 ? launch_fwd_as<DTYPE, false, 32> : T == 128 ? launch_fwd_as<DTYPE, false, 128> : launch_fwd_as<DTYPE, false, 256>);
    return launch(logits, pitch, tokens, logprobs, entropy, lse, top_ids, top_logprobs, top, rows, V, c, inverse_temperature, ctas, stream);
}

template <int DTYPE>
int launch_bwd(const void* logits, int64_t pitch, const float* tokens, const float* lse, const float* entropy,
               const float* d_logprobs, const float* d_entropy, void* dlogits, int64_t d_pitch, int64_t rows, int64_t V,
               float inverse_temperature, cudaStream_t stream)
{
    using L = Logit<DTYPE>;
    // small CTAs for short rows (16384 x 1000 bf16: 14.7 us, with 256 threads 35), pieces of eight vectors per thread
    const int64_t vectors = V / L::VE;
    const int T = vectors <= 256 ? 64 : vectors <= 2048 ? 128 : 256;
    const int pieces = (int)((vectors + T * 8 - 1) / (T * 8));
    const auto kernel = T == 64 ? (d_entropy ? token_logprobs_bwd_kernel<DTYPE, true, 64, 4> : token_logprobs_bwd_kernel<DTYPE, false, 64, 4>)
                      : T == 128 ? (d_entropy ? token_logprobs_bwd_kernel<DTYPE, true, 128, 4> : token_logprobs_bwd_kernel<DTYPE, false, 128, 4>)
                                 : (d_entropy ? token_logprobs_bwd_kernel<DTYPE, true, 256, 4> : token_logprobs_bwd_kernel<DTYPE, false, 256, 4>);
    // the second grid dimension holds at most 65535 rows
    for(int64_t first = 0; first < rows; first += 65535)
    {
        const int64_t n = rows - first < 65535 ? rows - first : 65535;
        kernel<<<dim3(pieces > 0 ? pieces : 1, (unsigned)n), T, 0, stream>>>(
            static_cast<const typename L::type*>(logits) + first * pitch, pitch, tokens + first, lse + first,
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
    ONN_CHECK_ARG(logit_arguments_ok(dlogits, dtype, d_pitch, rows, V) && gradient_place_ok(logits, pitch, dlogits, d_pitch));
    const float inverse = 1.0f / temperature;
    cudaStream_t s = (cudaStream_t)stream;
    switch(dtype)
    {
        case ONN_F32: return launch_bwd<ONN_F32>(logits, pitch, tokens, lse, entropy, d_logprobs, d_entropy, dlogits, d_pitch, rows, V, inverse, s);
        case ONN_BF16: return launch_bwd<ONN_BF16>(logits, pitch, tokens, lse, entropy, d_logprobs, d_entropy, dlogits, d_pitch, rows, V, inverse, s);
        default: return launch_bwd<ONN_F16>(logits, pitch, tokens, lse, entropy, d_logprobs, d_entropy, dlogits, d_pitch, rows, V, inverse, s);
    }
}
