// Distillation from a teacher's top logits, mixed with the hard-label cross entropy: loss and gradient in one call.
//
// For an active row (target in (0, V)) with student logits x, temperature T, a teacher's list (id_k, u_k), and
//   q = softmax over the valid places of u / T     p = softmax(x / T)     p1 = softmax(x)
//   soft = T^2 sum_k q_k (log q_k - log p_{id_k})   hard = -log(p1_target + FLT_EPSILON)
//   dx_i = [ soft_weight T (p_i - sum over k with id_k = i of q_k) + hard_weight (p1_i - 1[i = target]) ] / #active
#include <cooperative_groups.h>
#include <float.h>

#include "logit_rows.cuh"

namespace onn
{

namespace
{

constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ float finite_anchor(float m) { return m > -INFINITY ? m : 0.f; }

// What a row's softmaxes come to: p_i = 2^((x_i - m) c) * inv and p1_i = 2^((x_i - m) log2 e) * inv1.
struct Softmaxes
{
    float m, c, inverse_temperature, s, s1;
    __device__ __forceinline__ float p(float x) const { return s > 0.f || s != s ? exp2_approx((x - m) * c) / s : 0.f; }
    __device__ __forceinline__ float p1(float x) const { return s1 > 0.f || s1 != s1 ? exp2_approx((x - m) * kLog2E) / s1 : 0.f; }
    __device__ __forceinline__ float log_p(float x) const { return s == 0.f ? -INFINITY : (x - m) * inverse_temperature - logf(s); }
};

// The teacher's distribution over the places of its list, in shared memory: q[k] (0 for a place that is not valid) and
// the first place k' <= k with the same id.  Called by the whole CTA; returns whether there is any.
struct Teacher
{
    float q[ONN_TOP_MAX];
    int id[ONN_TOP_MAX];
    float reduce[kWarps];
};

__device__ __forceinline__ float cta_max(float v, float* scratch)
{
    v = warp_max(v);
    __syncthreads();
    if((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for(int w = 1; w < kWarps; w++) v = fmaxf(v, scratch[w]);
    return v;
}

__device__ __forceinline__ float cta_sum(float v, float* scratch)
{
    v = warp_sum(v);
    __syncthreads();
    if((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for(int w = 0; w < kWarps; w++) v += scratch[w];
    return v;
}

// Rows longer than a cluster can hold: one CTA per row, which sweeps it three times.
template <int DTYPE>
__global__ void __launch_bounds__(kThreads)
distill3d_sweeps_kernel(const typename Logit<DTYPE>::type* logits, long long pitch, const float* __restrict__ targets,
                 const float* __restrict__ active_count, const int* __restrict__ teacher_ids, const float* __restrict__ teacher_logits,
                 int top, float inverse_temperature, float temperature, float soft_weight, float hard_weight,
                 typename Logit<DTYPE>::type* dlogits, long long d_pitch, float* __restrict__ row_losses, long long rows, int V)
{
    using L = Logit<DTYPE>;
    __shared__ Teacher teacher;
    const long long row = blockIdx.x;
    const int tid = threadIdx.x;
    const typename L::type* x = logits + row * pitch;
    typename L::type* dx = dlogits ? dlogits + row * d_pitch : nullptr;
    bool active;
    const long long target = row_token(targets, row, V, &active);
    if(!active)
    {
        if(dx) for(int i = tid; i < V; i += kThreads) L::put(dx + i, 0.f);
        if(tid == 0) { row_losses[row] = 0.f; row_losses[rows + row] = 0.f; }
        return;
    }

    // the teacher
    float u = -INFINITY;
    int id = -1;
    if(tid < top)
    {
        id = teacher_ids[row * top + tid];
        if(id < 0 || id >= V) id = -1;
        else u = teacher_logits[row * top + tid];
    }
    const float u_max = cta_max(u, teacher.reduce);
    // NaN passes the maximum by: it comes in through the sum
    const float e = id < 0 ? 0.f : exp2_approx((u - finite_anchor(u_max)) * (kLog2E * inverse_temperature));
    const float e_sum = cta_sum(e, teacher.reduce);
    const bool taught = e_sum != 0.f;                    // some place is valid and not -inf
    const float q = taught && id >= 0 ? e / e_sum : 0.f;
    if(tid < ONN_TOP_MAX) { teacher.q[tid] = q; teacher.id[tid] = id; }
    __syncthreads();

    // the student's softmaxes
    float m = -INFINITY;
    for(int i = tid; i < V; i += kThreads) m = fmaxf(m, L::get(x + i));
    Softmaxes f;
    f.m = finite_anchor(cta_max(m, teacher.reduce));
    f.inverse_temperature = inverse_temperature;
    f.c = kLog2E * inverse_temperature;
    float s = 0.f, s1 = 0.f;
    for(int i = tid; i < V; i += kThreads)
    {
        const float d = L::get(x + i) - f.m;
        s += exp2_approx(d * f.c);
        s1 += exp2_approx(d * kLog2E);
    }
    f.s = cta_sum(s, teacher.reduce);
    f.s1 = cta_sum(s1, teacher.reduce);

    float term = 0.f;
    if(taught && id >= 0 && q != 0.f)
        term = q * ((u - finite_anchor(u_max)) * inverse_temperature - logf(e_sum) - f.log_p(L::get(x + id)));
    term = cta_sum(term, teacher.reduce);
    if(tid == 0)
    {
        row_losses[row] = term * temperature * temperature;
        row_losses[rows + row] = hard_weight != 0.f ? -logf(f.p1(L::get(x + target)) + FLT_EPSILON) : 0.f;
    }
    if(!dx) return;

    const float count = active_count[0];
    const float scale = count > 0.f ? 1.f / count : 0.f;
    const float soft = taught ? soft_weight * temperature * scale : 0.f, hard = hard_weight * scale;
    // the elements that the list or the target singles out: their student logits, before the gradient takes their place
    float special = 0.f;
    int special_index = -1;
    if(tid <= top)
    {
        // one thread for each place of the list, the one after the last place for the target; an index that stands in
        // several places is done by the first of them
        special_index = tid < top ? id : (int)target;
        float q_there = 0.f;
        for(int k = 0; k < top; k++)
        {
            if(teacher.id[k] != special_index || special_index < 0) continue;
            if(k < tid) { special_index = -1; break; }
            q_there += teacher.q[k];
        }
        if(special_index >= 0)
        {
            const float there = L::get(x + special_index);
            special = soft * (f.p(there) - q_there) + (hard != 0.f ? hard * (f.p1(there) - (special_index == target ? 1.f : 0.f)) : 0.f);
        }
    }
    __syncthreads();
    for(int i = tid; i < V; i += kThreads)
    {
        const float value = L::get(x + i);
        L::put(dx + i, soft * f.p(value) + (hard != 0.f ? hard * f.p1(value) : 0.f));
    }
    __syncthreads();
    if(special_index >= 0) L::put(dx + special_index, special);
}

constexpr int kMaxCluster = 8;
constexpr int kCountInside = 2048;                // up to so many rows a CTA counts the active ones itself

struct alignas(16) Part { float m, s, s1, unused; };

struct Held
{
    Part parts[kMaxCluster * 32];
    float q[ONN_TOP_MAX];
    float log_q[ONN_TOP_MAX];
    alignas(16) int id[ONN_TOP_MAX];
    float term[ONN_TOP_MAX / 32];
    int taught;
    float count[32];
};

// One cluster of CTAs (often of one) per row, which holds the row in its registers: each logit is read from global memory
// once, and its gradient written once.  N vectors of 16 bytes per thread.
//   1  the loads, with the teacher's list under way beside them (one warp does its softmax in each CTA);
//   2  sums relative to each thread's largest logit, joined over the warp, and put into every CTA's shared memory;
//   3  the row's maximum and sums, then the gradient from the registers: with one softmax in fp32 (SETS = 1: the
//      temperature is 1 or there is no hard-label part) the exponentials are kept, else they are formed again;
//   4  the elements that the list or the target singles out are written again by one thread each.
template <int DTYPE, int SETS, int T, int N>
__global__ void __launch_bounds__(T, 1024 / T)
distill3d_kernel(const typename Logit<DTYPE>::type* logits, long long pitch, const float* __restrict__ targets,
                 const float* active_count, const int* __restrict__ teacher_ids, const float* __restrict__ teacher_logits,
                 int top, float inverse_temperature, float temperature, float soft_weight, float hard_weight,
                 typename Logit<DTYPE>::type* dlogits, long long d_pitch, float* __restrict__ row_losses, long long rows, int V)
{
    using L = Logit<DTYPE>;
    constexpr int VE = L::VE, kWarpsHere = T / 32;
    constexpr bool kKeep = DTYPE == ONN_F32 && SETS == 1;
    __shared__ Held held;
    pdl_launch_dependents();
    pdl_wait();
    cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
    const int ctas = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const long long row = blockIdx.x / ctas;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const typename L::type* x = logits + row * pitch;
    typename L::type* dx = dlogits ? dlogits + row * d_pitch : nullptr;
    bool active;
    const long long target = row_token(targets, row, V, &active);

    const RowCut cut = cut_row<DTYPE>(x, V);
    const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
    const int after = cut.head + cut.vectors * VE;
    const int end_index = rank != 0 ? -1 : tid < cut.head ? tid : tid < cut.head + cut.tail ? after + tid - cut.head : -1;
    const int share = (cut.vectors + ctas - 1) / ctas;
    const int begin = min(rank * share, cut.vectors), end = min(begin + share, cut.vectors);
    const bool together = ((reinterpret_cast<uintptr_t>(x) ^ reinterpret_cast<uintptr_t>(dx)) & 15) == 0;
    auto store = [&](int vector, const float (&f)[VE])
    {
        typename L::type* to = dx + cut.head + vector * VE;
        if(together) __stcs(reinterpret_cast<uint4*>(to), L::pack(f));
        else
        {
#pragma unroll
            for(int e = 0; e < VE; e++) L::put(to + e, f[e]);
        }
    };

    if(!active)                                        // the same for the whole cluster
    {
        if(dx)
        {
            const float zeros[VE] = {};
            for(int i = begin + tid; i < end; i += T) store(i, zeros);
            if(end_index >= 0) L::put(dx + end_index, 0.f);
        }
        if(rank == 0 && tid == 0) { row_losses[row] = 0.f; row_losses[rows + row] = 0.f; }
        return;
    }
    // all CTAs of the cluster must be running before one writes into another: waited for below, under the loads
    if(ctas > 1) asm volatile("barrier.cluster.arrive;" ::: "memory");

    // ---- 1
    uint4 v[N];
#pragma unroll
    for(int u = 0; u < N; u++)
    {
        const int i = begin + u * T + tid;
        v[u] = i < end ? __ldcs(body + i) : L::lowest();
    }
    const float end_value = end_index >= 0 ? L::get(x + end_index) : -INFINITY;
    // thread k < top looks after place k of the list, thread `top` after the target: the logit there, if this CTA needs it
    int index = -1;
    if(tid < top) index = __ldg(teacher_ids + row * top + tid);
    else if(tid == top) index = (int)target;
    if(index < 0 || index >= V) index = -1;
    bool mine = false;                                 // the element is one of this CTA's
    if(index >= 0)
    {
        const int vector = index < cut.head || index >= after ? -1 : (index - cut.head) / VE;
        mine = vector < 0 ? rank == 0 : vector >= begin && vector < end;
    }
    const float special_logit = mine || (rank == 0 && index >= 0) ? L::get(x + index) : -INFINITY;

    if(warp == 0)
    {
        // the teacher's softmax over the valid places
        constexpr int kPlaces = ONN_TOP_MAX / 32;
        float u[kPlaces], largest = -INFINITY;
        int id[kPlaces];
#pragma unroll
        for(int k = 0; k < kPlaces; k++)
        {
            const int at = k * 32 + lane;
            id[k] = at < top ? __ldg(teacher_ids + row * top + at) : -1;
            if(id[k] < 0 || id[k] >= V) id[k] = -1;
            u[k] = id[k] >= 0 ? __ldg(teacher_logits + row * top + at) : -INFINITY;
            largest = fmaxf(largest, u[k]);
        }
        largest = finite_anchor(warp_max(largest));
        float e[kPlaces], sum = 0.f;
#pragma unroll
        for(int k = 0; k < kPlaces; k++)
        {
            // NaN passes the maximum by: it comes in through the sum
            e[k] = id[k] < 0 ? 0.f : exp2_approx((u[k] - largest) * (kLog2E * inverse_temperature));
            sum += e[k];
        }
        sum = warp_sum(sum);
        const float inverse = 1.f / sum, log_sum = logf(sum);
#pragma unroll
        for(int k = 0; k < kPlaces; k++)
        {
            const int at = k * 32 + lane;
            held.id[at] = id[k];
            held.q[at] = sum != 0.f && id[k] >= 0 ? e[k] * inverse : 0.f;
            held.log_q[at] = (u[k] - largest) * inverse_temperature - log_sum;
        }
        if(lane == 0) held.taught = sum != 0.f;
    }
    float counted = 0.f;
    if(!active_count)
    {
        for(long long i = tid; i < rows; i += T)
        {
            const long long t = token_index(__ldg(targets + i));
            counted += t > 0 && t < V ? 1.f : 0.f;
        }
        counted = warp_sum(counted);
        if(lane == 0) held.count[warp] = counted;
    }

    // ---- 2
    const float c = kLog2E * inverse_temperature;
    float m = end_value > -INFINITY ? end_value : -INFINITY;
#pragma unroll
    for(int u = 0; u < N; u++) m = fmaxf(m, L::max(v[u]));
    const float base = finite_anchor(m);
    float s, s1 = 0.f;
    {
        const float2 minus = make_float2(-base, -base), c2 = make_float2(c, c), c1 = make_float2(kLog2E, kLog2E);
        float2 s2 = make_float2(0.f, 0.f), s12 = make_float2(0.f, 0.f);
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            float f[VE];
            L::unpack(v[u], f);
#pragma unroll
            for(int e = 0; e < VE; e += 2)
            {
                const float2 d = add2(make_float2(f[e], f[e + 1]), minus), d2 = mul2(d, c2);
                const float2 p = make_float2(exp2_approx(d2.x), exp2_approx(d2.y));
                s2 = add2(s2, p);
                if(kKeep) { f[e] = p.x; f[e + 1] = p.y; }
                if(SETS == 2)
                {
                    const float2 d1 = mul2(d, c1);
                    s12 = add2(s12, make_float2(exp2_approx(d1.x), exp2_approx(d1.y)));
                }
            }
            if(kKeep) v[u] = L::pack(f);
        }
        s = s2.x + s2.y;
        s1 = s12.x + s12.y;
        if(end_index >= 0)
        {
            s += exp2_approx((end_value - base) * c);
            if(SETS == 2) s1 += exp2_approx((end_value - base) * kLog2E);
        }
    }
    const float warp_m = warp_max(m);
    {
        const float down = m > -INFINITY ? m - finite_anchor(warp_m) : -INFINITY;
        s = warp_sum(s * exp2_approx(down * c));
        if(SETS == 2) s1 = warp_sum(s1 * exp2_approx(down * kLog2E));
    }
    const Part part = {warp_m, s, s1, 0.f};
    const int parts = ctas * kWarpsHere;
    if(ctas == 1)
    {
        if(lane == 0) held.parts[warp] = part;
        __syncthreads();
    }
    else
    {
        asm volatile("barrier.cluster.wait;" ::: "memory");
        if(lane < ctas) cluster.map_shared_rank(&held, lane)->parts[rank * kWarpsHere + warp] = part;
        cluster.sync();
    }

    // ---- 3
    float row_m = -INFINITY;
    for(int i = lane; i < parts; i += 32) row_m = fmaxf(row_m, held.parts[i].m);
    row_m = warp_max(row_m);
    const float M = finite_anchor(row_m);
    s = 0.f;
    s1 = 0.f;
    for(int i = lane; i < parts; i += 32)
    {
        const Part other = held.parts[i];
        const float down = other.m > -INFINITY ? other.m - M : -INFINITY;
        s = fmaf(other.s, exp2_approx(down * c), s);
        if(SETS == 2) s1 = fmaf(other.s1, exp2_approx(down * kLog2E), s1);
    }
    s = warp_sum(s);
    s1 = SETS == 2 ? warp_sum(s1) : s;
    // a student without a finite logit has no distribution: p = 0
    const float inverse = s == 0.f ? 0.f : 1.f / s, inverse1 = s1 == 0.f ? 0.f : 1.f / s1;
    float count = 0.f;
    if(active_count) count = *active_count;
    else
    {
#pragma unroll
        for(int w = 0; w < kWarpsHere; w++) count += held.count[w];
    }
    const float scale = count > 0.f ? 1.f / count : 0.f;
    const bool taught = held.taught != 0;
    const float soft = taught ? soft_weight * temperature * scale : 0.f, hard = hard_weight * scale;
    // one softmax serves both parts at temperature 1
    const float weight = SETS == 2 ? soft * inverse : (soft + hard) * inverse, weight1 = hard * inverse1;
    auto p_of = [&](float logit) { return exp2_approx((logit - M) * c) * inverse; };
    auto p1_of = [&](float logit) { return exp2_approx((logit - M) * kLog2E) * inverse1; };
    auto gradient = [&](float logit)
    {
        const float g = weight * exp2_approx((logit - M) * c);
        return SETS == 2 ? fmaf(weight1, exp2_approx((logit - M) * kLog2E), g) : g;
    };
    if(dx)
    {
        const float again = (m > -INFINITY ? exp2_approx((m - M) * c) : 0.f) * weight;
        const float2 minus = make_float2(-M, -M), c2 = make_float2(c, c), c1 = make_float2(kLog2E, kLog2E);
        const float2 again2 = make_float2(again, again), w2 = make_float2(weight, weight), w12 = make_float2(weight1, weight1);
#pragma unroll
        for(int u = 0; u < N; u++)
        {
            const int i = begin + u * T + tid;
            if(i >= end) continue;
            float f[VE];
            L::unpack(v[u], f);
#pragma unroll
            for(int e = 0; e < VE; e += 2)
            {
                float2 g = make_float2(f[e], f[e + 1]);
                if(kKeep) g = mul2(g, again2);
                else
                {
                    const float2 d = add2(g, minus), d2 = mul2(d, c2);
                    g = mul2(make_float2(exp2_approx(d2.x), exp2_approx(d2.y)), w2);
                    if(SETS == 2)
                    {
                        const float2 d1 = mul2(d, c1);
                        g = fma2(make_float2(exp2_approx(d1.x), exp2_approx(d1.y)), w12, g);
                    }
                }
                f[e] = g.x;
                f[e + 1] = g.y;
            }
            store(i, f);
        }
        if(end_index >= 0) L::put(dx + end_index, gradient(end_value));
    }

    // ---- 4
    float special = 0.f;
    if(mine)
    {
        // an index that stands in several places is done by the first of them, the target by its place in the list if it has one
        int equal = 0;
        for(int k = 0; k < top; k += 4)
        {
            const int4 four = *reinterpret_cast<const int4*>(held.id + k);     // places past the list hold -1
            equal += (four.x == index) + (four.y == index) + (four.z == index) + (four.w == index);
        }
        float q = tid < top ? held.q[tid] : 0.f;
        if(equal > (tid < top ? 1 : 0))
        {
            q = 0.f;
            for(int k = 0; k < top; k++)
            {
                if(held.id[k] != index) continue;
                if(k < tid) { mine = false; break; }
                q += held.q[k];
            }
        }
        special = soft * (p_of(special_logit) - q);
        if(hard != 0.f) special += hard * ((SETS == 2 ? p1_of(special_logit) : p_of(special_logit)) - (index == (int)target ? 1.f : 0.f));
    }
    if(rank == 0)
    {
        if(warp < ONN_TOP_MAX / 32)
        {
            float term = 0.f;
            if(tid < top && index >= 0 && held.q[tid] != 0.f)
            {
                const float log_p = s == 0.f ? -INFINITY : (special_logit - M) * inverse_temperature - logf(s);
                term = held.q[tid] * (held.log_q[tid] - log_p);
            }
            term = warp_sum(term);
            if(lane == 0) held.term[warp] = term;
        }
        if(tid == top) row_losses[rows + row] = hard_weight != 0.f ? -logf((SETS == 2 ? p1_of(special_logit) : p_of(special_logit)) + FLT_EPSILON) : 0.f;
    }
    __syncthreads();                                   // the stores of 3 come before those that replace them
    if(dx && mine) L::put(dx + index, special);
    if(rank == 0 && tid == 0)
    {
        float term = 0.f;
#pragma unroll
        for(int w = 0; w < (kWarpsHere < ONN_TOP_MAX / 32 ? kWarpsHere : ONN_TOP_MAX / 32); w++) term += held.term[w];
        row_losses[row] = term * temperature * temperature;
    }
}

// stats = {sum of the soft losses, sum of the hard losses, #active}: one CTA, fixed order.
__global__ void __launch_bounds__(1024)
distill3d_finish_kernel(const float* __restrict__ row_losses, const float* __restrict__ targets, long long rows, long long V,
                        float* __restrict__ stats)
{
    __shared__ float scratch[32];
    pdl_wait();
    float soft = 0.f, hard = 0.f, active = 0.f;
    for(long long i = threadIdx.x; i < rows; i += blockDim.x)
    {
        soft += row_losses[i];
        hard += row_losses[rows + i];
        const long long t = token_index(targets[i]);
        active += t > 0 && t < V ? 1.f : 0.f;
    }
    soft = block_sum(soft, scratch);
    hard = block_sum(hard, scratch);
    active = block_sum(active, scratch);
    if(threadIdx.x == 0) { stats[0] = soft; stats[1] = hard; stats[2] = active; }
}

__global__ void __launch_bounds__(1024)
distill3d_count_kernel(const float* __restrict__ targets, long long rows, long long V, float* __restrict__ stats)
{
    __shared__ float scratch[32];
    pdl_launch_dependents();
    float active = 0.f;
#pragma unroll 8
    for(long long i = threadIdx.x; i < rows; i += blockDim.x)
    {
        const long long t = token_index(__ldg(targets + i));
        active += t > 0 && t < V ? 1.f : 0.f;
    }
    active = block_sum(active, scratch);
    if(threadIdx.x == 0) stats[2] = active;
}

template <int DTYPE>
int launch(const void* logits, int64_t pitch, const float* targets, const float* active_count, const int32_t* teacher_ids,
           const float* teacher_logits, int64_t top, float temperature, float soft_weight, float hard_weight, void* dlogits,
           int64_t d_pitch, float* row_losses, float* stats, int64_t rows, int64_t V, cudaStream_t stream)
{
    using E = typename Logit<DTYPE>::type;
    // CTAs of a row: as many as hold it at 8 vectors per thread of 256 threads, 512 or 1024 for the longest; more while the GPU
    // is not full and each has two vectors per thread
    const int64_t vectors = V / Logit<DTYPE>::VE + 1;
    int T = 256;
    while(T < 1024 && vectors > (int64_t)kMaxCluster * T * 8) T *= 2;
    const bool fits = vectors <= (int64_t)kMaxCluster * T * 8;
    int ctas = (int)((vectors + T * 8 - 1) / (T * 8));
    while(ctas < kMaxCluster && rows * ctas < 2 * kSmCount && vectors > (int64_t)ctas * T * 2) ctas++;
    const int64_t each = (vectors + ctas * T - 1) / (ctas * T);

    bool counted = false;
    if(!active_count && (rows > kCountInside || !fits))
    {
        distill3d_count_kernel<<<1, 1024, 0, stream>>>(targets, rows, V, stats);
        count_launch();
        if(launch_status() != ONN_OK) return ONN_ERR_CUDA;
        active_count = stats + 2;
        counted = true;
    }
    const E* x = static_cast<const E*>(logits);
    E* dx = static_cast<E*>(dlogits);
    const float inverse_temperature = 1.f / temperature;
    cudaError_t error;
    if(!fits)
    {
        distill3d_sweeps_kernel<DTYPE><<<(unsigned)rows, kThreads, 0, stream>>>(
            x, pitch, targets, active_count, teacher_ids, teacher_logits, (int)top, inverse_temperature, temperature, soft_weight,
            hard_weight, dx, d_pitch, row_losses, rows, (int)V);
        error = cudaGetLastError();
    }
    else
    {
        const bool two = hard_weight != 0.f && temperature != 1.f;
        auto held = [&](auto kernel)
        {
            return launch_clusters(kernel, (unsigned)(rows * ctas), T, ctas, counted, stream, x, (long long)pitch, targets, active_count,
                                   teacher_ids, teacher_logits, (int)top, inverse_temperature, temperature, soft_weight, hard_weight, dx,
                                   (long long)d_pitch, row_losses, (long long)rows, (int)V);
        };
#define ONN_HELD(SETS) (T == 1024 ? held(distill3d_kernel<DTYPE, SETS, 1024, 8>) : T == 512 ? held(distill3d_kernel<DTYPE, SETS, 512, 8>) : \
                        each > 4 ? held(distill3d_kernel<DTYPE, SETS, 256, 8>) : each > 2 ? held(distill3d_kernel<DTYPE, SETS, 256, 4>) : \
                        each > 1 ? held(distill3d_kernel<DTYPE, SETS, 256, 2>) : held(distill3d_kernel<DTYPE, SETS, 256, 1>))
        error = two ? ONN_HELD(2) : ONN_HELD(1);
#undef ONN_HELD
    }
    count_launch();
    if(error != cudaSuccess) return ONN_ERR_CUDA;
    return launch_status();
}

}  // namespace

}  // namespace onn

using namespace onn;

extern "C" int onn_distill3d_fwd_bwd(const void* logits, int dtype, int64_t pitch, const float* targets, const float* active_count,
                                     const int32_t* teacher_ids, const float* teacher_logits, int64_t top, float temperature,
                                     float soft_weight, float hard_weight, void* dlogits, int64_t d_pitch, float* stats,
                                     float* row_losses, int64_t rows, int64_t V, void* stream)
{
    ONN_CHECK_ARG(logit_arguments_ok(logits, dtype, pitch, rows, V) && temperature_ok(temperature));
    ONN_CHECK_ARG(targets && teacher_ids && teacher_logits && stats && row_losses && top >= 1);
    ONN_CHECK_ARG(isfinite(soft_weight) && isfinite(hard_weight));
    ONN_CHECK_ARG(!dlogits || logit_arguments_ok(dlogits, dtype, d_pitch, rows, V));
    if(top > ONN_TOP_MAX) return ONN_ERR_LIMIT;
    cudaStream_t s = (cudaStream_t)stream;
    int status;
    switch(dtype)
    {
        case ONN_F32: status = launch<ONN_F32>(logits, pitch, targets, active_count, teacher_ids, teacher_logits, top, temperature, soft_weight, hard_weight, dlogits, d_pitch, row_losses, stats, rows, V, s); break;
        case ONN_BF16: status = launch<ONN_BF16>(logits, pitch, targets, active_count, teacher_ids, teacher_logits, top, temperature, soft_weight, hard_weight, dlogits, d_pitch, row_losses, stats, rows, V, s); break;
        default: status = launch<ONN_F16>(logits, pitch, targets, active_count, teacher_ids, teacher_logits, top, temperature, soft_weight, hard_weight, dlogits, d_pitch, row_losses, stats, rows, V, s); break;
    }
    if(status != ONN_OK) return status;
    if(launch_overlapped(distill3d_finish_kernel, dim3(1), dim3(1024), 0, s, (const float*)row_losses, targets, (long long)rows, (long long)V, stats) != cudaSuccess)
        return ONN_ERR_CUDA;
    count_launch();
    return launch_status();
}
