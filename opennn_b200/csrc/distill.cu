// Distillation from a teacher's top logits, mixed with the hard-label cross entropy: loss and gradient in one call.
//
// For an active row (target in (0, V)) with student logits x, temperature T, a teacher's list (id_k, u_k), and
//   q = softmax over the valid places of u / T     p = softmax(x / T)     p1 = softmax(x)
//   soft = T^2 sum_k q_k (log q_k - log p_{id_k})   hard = -log(p1_target + FLT_EPSILON)
//   dx_i = [ soft_weight T (p_i - sum over k with id_k = i of q_k) + hard_weight (p1_i - 1[i = target]) ] / #active
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

template <int DTYPE>
__global__ void __launch_bounds__(kThreads)
distill3d_kernel(const typename Logit<DTYPE>::type* logits, long long pitch, const float* __restrict__ targets,
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

// stats = {sum of the soft losses, sum of the hard losses, #active}: one CTA, fixed order.
__global__ void __launch_bounds__(1024)
distill3d_finish_kernel(const float* __restrict__ row_losses, const float* __restrict__ targets, long long rows, long long V,
                        float* __restrict__ stats)
{
    __shared__ float scratch[32];
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
    float active = 0.f;
    for(long long i = threadIdx.x; i < rows; i += blockDim.x)
    {
        const long long t = token_index(targets[i]);
        active += t > 0 && t < V ? 1.f : 0.f;
    }
    active = block_sum(active, scratch);
    if(threadIdx.x == 0) stats[2] = active;
}

template <int DTYPE>
int launch(const void* logits, int64_t pitch, const float* targets, const float* active_count, const int32_t* teacher_ids,
           const float* teacher_logits, int64_t top, float temperature, float soft_weight, float hard_weight, void* dlogits,
           int64_t d_pitch, float* row_losses, int64_t rows, int64_t V, cudaStream_t stream)
{
    using T = typename Logit<DTYPE>::type;
    distill3d_kernel<DTYPE><<<(unsigned)rows, kThreads, 0, stream>>>(
        static_cast<const T*>(logits), pitch, targets, active_count, teacher_ids, teacher_logits, (int)top, 1.f / temperature,
        temperature, soft_weight, hard_weight, static_cast<T*>(dlogits), d_pitch, row_losses, rows, (int)V);
    count_launch();
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
    if(!active_count)
    {
        distill3d_count_kernel<<<1, 1024, 0, s>>>(targets, rows, V, stats);
        count_launch();
        if(launch_status() != ONN_OK) return ONN_ERR_CUDA;
        active_count = stats + 2;
    }
    int status;
    switch(dtype)
    {
        case ONN_F32: status = launch<ONN_F32>(logits, pitch, targets, active_count, teacher_ids, teacher_logits, top, temperature, soft_weight, hard_weight, dlogits, d_pitch, row_losses, rows, V, s); break;
        case ONN_BF16: status = launch<ONN_BF16>(logits, pitch, targets, active_count, teacher_ids, teacher_logits, top, temperature, soft_weight, hard_weight, dlogits, d_pitch, row_losses, rows, V, s); break;
        default: status = launch<ONN_F16>(logits, pitch, targets, active_count, teacher_ids, teacher_logits, top, temperature, soft_weight, hard_weight, dlogits, d_pitch, row_losses, rows, V, s); break;
    }
    if(status != ONN_OK) return status;
    distill3d_finish_kernel<<<1, 1024, 0, s>>>(row_losses, targets, rows, V, stats);
    count_launch();
    return launch_status();
}
