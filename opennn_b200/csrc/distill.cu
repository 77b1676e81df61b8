// Distillation from a teacher's top logits, mixed with the hard-label cross entropy: loss and gradient in one call.
//
// For an active row (target in (0, V)) with student logits x, temperature T, a teacher's list (id_k, u_k), and
//   q = softmax over the valid places of u / T     p = softmax(x / T)     p1 = softmax(x)
//   soft = T^2 sum_k q_k (log q_k - log p_{id_k})   hard = -log(p1_target + FLT_EPSILON)
//   dx_i = [ soft_weight T (p_i - sum over k with id_k = i of q_k) + hard_weight (p1_i - 1[i = target]) ] / #active
//
// Bound by HBM at one read and one write of each logit: DRAM traffic is that (0.30 GB read for 0.30 GB of logits), the second
// sweep comes from L1 (45 % of all loads) and L2.  Measured on a B200 (copy bandwidth 6.57 TB/s): 16384 x 32000 fp32 with both
// parts at temperature 2, 37 % of the rows padding, 577 us = 5.9 TB/s, 8192 x 32000 fp32 at temperature 1 341 us = 6.1 TB/s;
// 4096 x 131072 bf16 with the soft part 388 us = 5.5 TB/s, where the exponentials (two per logit, 16 per clock and SM) take 238 us by
// themselves (times of the kernel alone).  Holding the row on chip instead was
// slower: in the registers of a cluster of CTAs 789 and 776 us, in a persistent cluster with the next row's copies under way
// 1163 and 1220 us (a cluster barrier and some 500 instructions per thread and row had nothing to hide behind).
#include <float.h>

#include <type_traits>

#include "logit_rows.cuh"

namespace onn
{

namespace
{

__device__ __forceinline__ float finite_anchor(float m) { return m > -INFINITY ? m : 0.f; }

constexpr int kCountInside = 2048;                // up to so many rows a CTA counts the active ones itself

struct Part { float m, s, s1; };

struct Shared
{
    Part parts[32];
    float q[ONN_TOP_MAX];
    float log_q[ONN_TOP_MAX];
    alignas(16) int id[ONN_TOP_MAX];
    float term[ONN_TOP_MAX / 32];
    int taught;
    float count[32];
};

// SETS: 1 where one softmax serves both parts (temperature 1, or no hard-label part), 2 where there are two, 3 where the second one
// is the square of the first (temperature 2, the usual choice: half the exponentials, which bound 16-bit logits: 2048 x 131072
// bf16 285 us with two softmaxes, 213 with squares, 207 with one).
// One CTA per row, two sweeps: sums relative to the largest logit on the way up, the gradient on the way down, so that what was
// read last, and is still in L1, is read again first; the rest comes from L2, which holds the rows that the GPU works on.
template <int DTYPE, int SETS, int T, int N>
__global__ void __launch_bounds__(T, 1024 / T)
distill3d_kernel(const typename Logit<DTYPE>::type* logits, long long pitch, const float* __restrict__ targets,
                     const float* active_count, const int* __restrict__ teacher_ids, const float* __restrict__ teacher_logits,
                     int top, float inverse_temperature, float temperature, float soft_weight, float hard_weight,
                     typename Logit<DTYPE>::type* dlogits, long long d_pitch, float* __restrict__ row_losses, long long rows, int V)
{
    using L = Logit<DTYPE>;
    constexpr int VE = L::VE, kWarpsHere = T / 32;
    __shared__ Shared shared;
    pdl_launch_dependents();
    pdl_wait();
    const long long row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const typename L::type* x = logits + row * pitch;
    typename L::type* dx = dlogits ? dlogits + row * d_pitch : nullptr;
    // the target and the teacher's list (all of it in the first warp) are asked for together
    constexpr int kPlaces = ONN_TOP_MAX / 32;
    int index = tid < top ? __ldg(teacher_ids + row * top + tid) : -1;
    int id[kPlaces];
    float u[kPlaces];
#pragma unroll
    for(int k = 0; k < kPlaces; k++)
    {
        const int at = k * 32 + lane;
        const bool there = warp == 0 && at < top;
        id[k] = there ? __ldg(teacher_ids + row * top + at) : -1;
        u[k] = there ? __ldg(teacher_logits + row * top + at) : -INFINITY;
    }
    bool active;
    const long long target = row_token(targets, row, V, &active);

    const RowCut cut = cut_row<DTYPE>(x, V);
    const uint4* body = reinterpret_cast<const uint4*>(x + cut.head);
    const int after = cut.head + cut.vectors * VE;
    const int end_index = tid < cut.head ? tid : tid < cut.head + cut.tail ? after + tid - cut.head : -1;
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
    if(!active)
    {
        if(dx)
        {
            const float zeros[VE] = {};
            for(int i = tid; i < cut.vectors; i += T) store(i, zeros);
            if(end_index >= 0) L::put(dx + end_index, 0.f);
        }
        if(tid == 0) { row_losses[row] = 0.f; row_losses[rows + row] = 0.f; }
        return;
    }
    // thread k < top looks after place k of the list, thread `top` after the target
    if(tid == top) index = (int)target;
    if(index < 0 || index >= V) index = -1;
    const float special_logit = index >= 0 ? L::get(x + index) : -INFINITY;
    const float end_value = end_index >= 0 ? L::get(x + end_index) : -INFINITY;

    float counted = 0.f;
    if(!active_count)
    {
        for(long long i = tid; i < rows; i += T)
        {
            const long long t = token_index(__ldg(targets + i));
            counted += t > 0 && t < V ? 1.f : 0.f;
        }
        counted = warp_sum(counted);
        if(lane == 0) shared.count[warp] = counted;
    }

    // ---- up
    const float c = kLog2E * inverse_temperature;
    float m = end_value > -INFINITY ? end_value : -INFINITY;
    float s = 0.f, s1 = 0.f;
    if(end_index >= 0) { s = exp2_approx((end_value - finite_anchor(m)) * c); s1 = exp2_approx((end_value - finite_anchor(m)) * kLog2E); }
    // whole batches need no look at the row's end, and their addresses differ by constants
    const int batches = (cut.vectors + T * N - 1) / (T * N), whole = cut.vectors / (T * N);
    const uint4* const mine_body = body + tid;
    for(int batch = 0; batch < batches; batch++)
    {
        uint4 v[N];
        float larger = m;
        const uint4* const at = mine_body + (size_t)batch * (T * N);
        if(batch < whole)
        {
#pragma unroll
            for(int u = 0; u < N; u++) v[u] = at[u * T];
        }
        else
        {
#pragma unroll
            for(int u = 0; u < N; u++) v[u] = (batch * N + u) * T + tid < cut.vectors ? at[u * T] : L::lowest();
        }
#pragma unroll
        for(int u = 0; u < N; u++) larger = fmaxf(larger, L::max(v[u]));
        if(larger > m)
        {
            const float down = m > -INFINITY ? m - larger : -INFINITY;
            s *= exp2_approx(down * c);
            if(SETS >= 2) s1 *= exp2_approx(down * kLog2E);
            m = larger;
        }
        const float base = finite_anchor(m);
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
                if(SETS == 2)
                {
                    const float2 d1 = mul2(d, c1);
                    s12 = add2(s12, make_float2(exp2_approx(d1.x), exp2_approx(d1.y)));
                }
                if(SETS == 3) s12 = fma2(p, p, s12);
            }
        }
        s += s2.x + s2.y;
        s1 += s12.x + s12.y;
    }
    if(warp == 0)
    {
        // the teacher's softmax over the valid places
        float largest = -INFINITY;
#pragma unroll
        for(int k = 0; k < kPlaces; k++)
        {
            if(id[k] < 0 || id[k] >= V) { id[k] = -1; u[k] = -INFINITY; }
            largest = fmaxf(largest, u[k]);
        }
        largest = finite_anchor(warp_largest(largest));
        float e[kPlaces], sum = 0.f;
#pragma unroll
        for(int k = 0; k < kPlaces; k++)
        {
            // NaN passes the maximum by: it comes in through the sum
            e[k] = id[k] < 0 ? 0.f : exp2_approx((u[k] - largest) * c);
            sum += e[k];
        }
        sum = warp_sum(sum);
        const float inverse = 1.f / sum, log_sum = logf(sum);
#pragma unroll
        for(int k = 0; k < kPlaces; k++)
        {
            const int at = k * 32 + lane;
            shared.id[at] = id[k];
            if(k * 32 >= top) continue;
            shared.q[at] = sum != 0.f && id[k] >= 0 ? e[k] * inverse : 0.f;
            shared.log_q[at] = (u[k] - largest) * inverse_temperature - log_sum;
        }
        if(lane == 0) shared.taught = sum != 0.f;
    }
    const float warp_m = warp_largest(m);
    {
        const float down = m > -INFINITY ? m - finite_anchor(warp_m) : -INFINITY;
        s = warp_sum(s * exp2_approx(down * c));
        if(SETS >= 2) s1 = warp_sum(s1 * exp2_approx(down * kLog2E));
    }
    if(lane == 0) shared.parts[warp] = Part{warp_m, s, s1};
    __syncthreads();
    const Part other = lane < kWarpsHere ? shared.parts[lane] : Part{-INFINITY, 0.f, 0.f};
    const float M = finite_anchor(warp_largest(other.m));
    {
        const float down = other.m > -INFINITY ? other.m - M : -INFINITY;
        s = warp_sum(other.s * exp2_approx(down * c));
        s1 = SETS >= 2 ? warp_sum(other.s1 * exp2_approx(down * kLog2E)) : s;
    }
    // a student without a finite logit has no distribution: p = 0
    const float inverse = s == 0.f ? 0.f : 1.f / s, inverse1 = s1 == 0.f ? 0.f : 1.f / s1;
    float count = 0.f;
    if(active_count) count = *active_count;
    else
    {
#pragma unroll
        for(int w = 0; w < kWarpsHere; w++) count += shared.count[w];
    }
    const float scale = count > 0.f ? 1.f / count : 0.f;
    const bool taught = shared.taught != 0;
    const float soft = taught ? soft_weight * temperature * scale : 0.f, hard = hard_weight * scale;
    // one softmax serves both parts at temperature 1
    const float weight = SETS >= 2 ? soft * inverse : (soft + hard) * inverse, weight1 = hard * inverse1;
    auto p_of = [&](float logit) { return exp2_approx((logit - M) * c) * inverse; };
    auto p1_of = [&](float logit) { return exp2_approx((logit - M) * kLog2E) * inverse1; };
    auto gradient = [&](float logit)
    {
        const float g = weight * exp2_approx((logit - M) * c);
        return SETS >= 2 ? fmaf(weight1, exp2_approx((logit - M) * kLog2E), g) : g;
    };

    // ---- down
    if(dx)
    {
        const float2 minus = make_float2(-M, -M), c2 = make_float2(c, c), c1 = make_float2(kLog2E, kLog2E);
        const float2 w2 = make_float2(weight, weight), w12 = make_float2(weight1, weight1);
        auto gradients = [&](const uint4& v, float (&f)[VE])
        {
            L::unpack(v, f);
#pragma unroll
            for(int e = 0; e < VE; e += 2)
            {
                const float2 d = add2(make_float2(f[e], f[e + 1]), minus), d2 = mul2(d, c2);
                const float2 p = make_float2(exp2_approx(d2.x), exp2_approx(d2.y));
                float2 g = mul2(p, w2);
                if(SETS == 2)
                {
                    const float2 d1 = mul2(d, c1);
                    g = fma2(make_float2(exp2_approx(d1.x), exp2_approx(d1.y)), w12, g);
                }
                if(SETS == 3) g = mul2(p, fma2(p, w12, w2));
                f[e] = g.x;
                f[e + 1] = g.y;
            }
        };
        uint4* const mine_out = reinterpret_cast<uint4*>(dx + cut.head) + tid;
        for(int batch = batches - 1; batch >= 0; batch--)
        {
            uint4 v[N];
            const uint4* const at = mine_body + (size_t)batch * (T * N);
            if(batch < whole && together)
            {
                uint4* const to = mine_out + (size_t)batch * (T * N);
#pragma unroll
                for(int u = 0; u < N; u++) v[u] = __ldcs(at + u * T);
#pragma unroll
                for(int u = 0; u < N; u++)
                {
                    float f[VE];
                    gradients(v[u], f);
                    __stcs(to + u * T, L::pack(f));
                }
            }
            else
            {
#pragma unroll
                for(int u = 0; u < N; u++)
                {
                    const int i = (batch * N + u) * T + tid;
                    if(i < cut.vectors) v[u] = __ldcs(at + u * T);
                }
#pragma unroll
                for(int u = 0; u < N; u++)
                {
                    const int i = (batch * N + u) * T + tid;
                    if(i >= cut.vectors) continue;
                    float f[VE];
                    gradients(v[u], f);
                    store(i, f);
                }
            }
        }
        if(end_index >= 0) L::put(dx + end_index, gradient(end_value));
    }

    // ---- the elements that the list or the target singles out
    float special = 0.f;
    bool mine = index >= 0;
    if(mine)
    {
        // an index that stands in several places is done by the first of them, the target by its place in the list if it has one
        int equal = 0;
        for(int k = 0; k < top; k += 4)
        {
            const int4 four = *reinterpret_cast<const int4*>(shared.id + k);     // places past the list hold -1
            equal += (four.x == index) + (four.y == index) + (four.z == index) + (four.w == index);
        }
        float q = tid < top ? shared.q[tid] : 0.f;
        if(equal > (tid < top ? 1 : 0))
        {
            q = 0.f;
            for(int k = 0; k < top; k++)
            {
                if(shared.id[k] != index) continue;
                if(k < tid) { mine = false; break; }
                q += shared.q[k];
            }
        }
        special = soft * (p_of(special_logit) - q);
        if(hard != 0.f) special += hard * ((SETS >= 2 ? p1_of(special_logit) : p_of(special_logit)) - (index == (int)target ? 1.f : 0.f));
    }
    if(warp < ONN_TOP_MAX / 32)
    {
        float term = 0.f;
        if(tid < top && index >= 0 && shared.q[tid] != 0.f)
        {
            const float log_p = s == 0.f ? -INFINITY : (special_logit - M) * inverse_temperature - logf(s);
            term = shared.q[tid] * (shared.log_q[tid] - log_p);
        }
        term = warp_sum(term);
        if(lane == 0) shared.term[warp] = term;
    }
    if(tid == top) row_losses[rows + row] = hard_weight != 0.f ? -logf((SETS >= 2 ? p1_of(special_logit) : p_of(special_logit)) + FLT_EPSILON) : 0.f;
    __syncthreads();                                   // the stores of the sweep come before those that replace them
    if(dx && mine) L::put(dx + index, special);
    if(tid == 0)
    {
        float term = 0.f;
#pragma unroll
        for(int w = 0; w < (kWarpsHere < ONN_TOP_MAX / 32 ? kWarpsHere : ONN_TOP_MAX / 32); w++) term += shared.term[w];
        row_losses[row] = term * temperature * temperature;
    }
}

// Sums over a CTA of 1024 threads, for thread 0, in a fixed order.
template <typename T>
__device__ __forceinline__ T cta_total(T v, T* scratch)
{
#pragma unroll
    for(int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
    if((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    if(threadIdx.x < 32)
    {
        v = scratch[threadIdx.x];
#pragma unroll
        for(int offset = 16; offset > 0; offset >>= 1) v += __shfl_xor_sync(0xffffffffu, v, offset);
    }
    return v;
}

// stats = {sum of the soft losses, sum of the hard losses, #active}: one CTA, fixed order.  The sums are held in 64 bits (a thread adds
// rows / 1024 losses one after the other: 4 M equal ones were off by 650 units of 2^-24 in fp32) and the rows counted in whole
// numbers; each is rounded once.
__global__ void __launch_bounds__(1024)
distill3d_finish_kernel(const float* __restrict__ row_losses, const float* __restrict__ targets, long long rows, long long V,
                        float* __restrict__ stats)
{
    __shared__ double soft_parts[32], hard_parts[32];
    __shared__ int active_parts[32];
    pdl_wait();
    double soft = 0.0, hard = 0.0;
    int active = 0;
#pragma unroll 8
    for(long long i = threadIdx.x; i < rows; i += blockDim.x)
    {
        soft += row_losses[i];
        hard += row_losses[rows + i];
        const long long t = token_index(targets[i]);
        active += t > 0 && t < V;
    }
    soft = cta_total(soft, soft_parts);
    hard = cta_total(hard, hard_parts);
    active = cta_total(active, active_parts);
    if(threadIdx.x == 0) { stats[0] = (float)soft; stats[1] = (float)hard; stats[2] = (float)active; }
}

__global__ void __launch_bounds__(1024)
distill3d_count_kernel(const float* __restrict__ targets, long long rows, long long V, float* __restrict__ stats)
{
    __shared__ int parts[32];
    pdl_launch_dependents();
    int active = 0;
#pragma unroll 8
    for(long long i = threadIdx.x; i < rows; i += blockDim.x)
    {
        const long long t = token_index(__ldg(targets + i));
        active += t > 0 && t < V;
    }
    active = cta_total(active, parts);
    if(threadIdx.x == 0) stats[2] = (float)active;
}

template <int DTYPE>
int launch(const void* logits, int64_t pitch, const float* targets, const float* active_count, const int32_t* teacher_ids,
           const float* teacher_logits, int64_t top, float temperature, float soft_weight, float hard_weight, void* dlogits,
           int64_t d_pitch, float* row_losses, float* stats, int64_t rows, int64_t V, cudaStream_t stream)
{
    using E = typename Logit<DTYPE>::type;
    bool counted = false;
    if(!active_count && rows > kCountInside)
    {
        distill3d_count_kernel<<<1, 1024, 0, stream>>>(targets, rows, V, stats);
        count_launch();
        if(launch_status() != ONN_OK) return ONN_ERR_CUDA;
        active_count = stats + 2;
        counted = true;
    }
    // Threads of a row.  The rows that the GPU works on should stay in L2 (and in part in L1) between the two sweeps, so long rows
    // want few large CTAs; what a row costs besides its logits is latency, so short ones want many small CTAs.  In us:
    //                          128     256     512    1024
    //   16384 x   8000 fp32    210     239     322     591
    //    8192 x  32000 fp32    454     393     385     531
    //    8192 x  50021 fp32    771     679     631     752
    //    2048 x 131072 fp32            490     454     435
    //    8192 x  32000 bf16    212     217     266     459
    //    8192 x  50021 bf16    362     335     384     539
    //    2048 x 131072 bf16            241     218     256
    // With less than two rows for each SM nothing is gained by small CTAs.
    const int64_t vectors = V / Logit<DTYPE>::VE;
    const bool wide = DTYPE == ONN_F32;
    int T = vectors >= (wide ? 24576 : 49152) ? 1024 : vectors >= (wide ? 6144 : 10240) ? 512 : vectors >= 4000 || top >= 128 ? 256 : 128;
    while(T < 1024 && rows * T <= 512 * kSmCount && vectors >= 4 * T) T *= 2;

    const E* x = static_cast<const E*>(logits);
    E* dx = static_cast<E*>(dlogits);
    const int sets = hard_weight == 0.f || temperature == 1.f ? 1 : temperature == 2.f ? 3 : 2;
    auto run = [&](auto kernel)
    {
        return launch_clusters(kernel, (unsigned)rows, T, 1, 0, counted, stream, x, (long long)pitch, targets, active_count, teacher_ids,
                               teacher_logits, (int)top, 1.f / temperature, temperature, soft_weight, hard_weight, dx, (long long)d_pitch,
                               row_losses, (long long)rows, (int)V);
    };
    auto with = [&](auto sets_of)
    {
        constexpr int SETS = sets_of.value;
        return T == 1024 ? run(distill3d_kernel<DTYPE, SETS, 1024, 8>) : T == 512 ? run(distill3d_kernel<DTYPE, SETS, 512, 8>)
             : T == 256 ? run(distill3d_kernel<DTYPE, SETS, 256, 8>) : run(distill3d_kernel<DTYPE, SETS, 128, 4>);
    };
    const cudaError_t error = sets == 1 ? with(std::integral_constant<int, 1>{}) : sets == 2 ? with(std::integral_constant<int, 2>{})
                                                                                            : with(std::integral_constant<int, 3>{});
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
    ONN_CHECK_ARG(!dlogits || (logit_arguments_ok(dlogits, dtype, d_pitch, rows, V) && gradient_place_ok(logits, pitch, dlogits, d_pitch)));
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
