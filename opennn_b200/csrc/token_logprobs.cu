// Log probabilities of given tokens with entropy and the top alternatives, and their gradient.
//
//   z = x / T,  lse = log sum_i exp z_i,  p = exp(z - lse)
//   forward   logprob = z_t - lse,  entropy = -sum_i p_i log p_i,  the K largest x with z - lse
//   backward  dx_i = [ g (1[i = t] - p_i) - h p_i (log p_i + entropy) ] / T
//
// Both are bound by HBM: the forward pass reads each logit once, the backward pass reads and writes each once.
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

// Adds N logits at once.  One rescaling for all of them.
template <int N>
__device__ __forceinline__ void add_logits(Running& r, const float (&x)[N], float c)
{
    float m = r.m;
#pragma unroll
    for(int i = 0; i < N; i++) m = fmaxf(m, x[i]);
    if(m > r.m) rebase(r, m, c);
    const float base = finite_anchor(m);
#pragma unroll
    for(int i = 0; i < N; i++)
    {
        const float d = (x[i] - base) * c;
        const float e = exp2_approx(d);
        r.s += e;
        r.w = fmaf(e, fmaxf(d, kNothing), r.w);
    }
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

template <int DTYPE>
__global__ void __launch_bounds__(kThreads)
token_logprobs_kernel(const typename Logit<DTYPE>::type* __restrict__ logits, long long pitch, const float* __restrict__ tokens,
                      float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ lse,
                      int* __restrict__ top_ids, float* __restrict__ top_logprobs, int top, int V, float c, float inverse_temperature)
{
    using L = Logit<DTYPE>;
    constexpr int VE = L::VE;
    __shared__ Running parts[kWarps];
    __shared__ unsigned long long best_keys[kWarps];
    const long long row = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

    bool active;
    const long long token = row_token(tokens, row, V, &active);
    if(!active)
    {
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
    const int end_index = tid < cut.head ? tid : tid < cut.head + cut.tail ? after + tid - cut.head : -1;

    Running r = {-INFINITY, 0.f, 0.f};
    if(end_index >= 0)
    {
        const float one[1] = {L::get(x + end_index)};
        add_logits<1>(r, one, c);
    }
    for(int first = 0; first < cut.vectors; first += kThreads * kUnroll)
    {
        uint4 v[kUnroll];
#pragma unroll
        for(int u = 0; u < kUnroll; u++)
        {
            const int i = first + u * kThreads + tid;
            v[u] = i < cut.vectors ? __ldg(body + i) : L::lowest();
        }
        float f[kUnroll * VE];
#pragma unroll
        for(int u = 0; u < kUnroll; u++)
        {
            float part[VE];
            L::unpack(v[u], part);
#pragma unroll
            for(int e = 0; e < VE; e++) f[u * VE + e] = part[e];
        }
        add_logits<kUnroll * VE>(r, f, c);
    }
#pragma unroll
    for(int offset = 16; offset > 0; offset >>= 1)
    {
        Running o;
        o.m = __shfl_xor_sync(0xffffffffu, r.m, offset);
        o.s = __shfl_xor_sync(0xffffffffu, r.s, offset);
        o.w = __shfl_xor_sync(0xffffffffu, r.w, offset);
        r = merge(r, o, c);
    }
    if(lane == 0) parts[warp] = r;
    __syncthreads();
    r = parts[0];
#pragma unroll
    for(int w = 1; w < kWarps; w++) r = merge(r, parts[w], c);

    const bool none = r.s == 0.f;                      // a row without a finite logit has no distribution
    const float log_s = logf(r.s);
    auto log_probability = [&](float value) { return none ? -INFINITY : (value - r.m) * inverse_temperature - log_s; };
    if(tid == 0)
    {
        if(logprobs) logprobs[row] = log_probability(L::get(x + token));
        if(entropy)
        {
            const float value = log_s - r.w / r.s * kLn2;
            entropy[row] = none || value < 0.f ? 0.f : value;
        }
        if(lse) lse[row] = none ? -INFINITY : fmaf(r.m, inverse_temperature, log_s);
    }

    // the alternatives, one after the other: the largest key below the last one
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
            if(end_index >= 0) look(L::get(x + end_index), end_index);
            for(int i = tid; i < cut.vectors; i += kThreads)
            {
                float part[VE];
                L::unpack(__ldg(body + i), part);
#pragma unroll
                for(int e = 0; e < VE; e++) look(part[e], cut.head + i * VE + e);
            }
        }
#pragma unroll
        for(int offset = 16; offset > 0; offset >>= 1)
        {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, offset);
            best = other > best ? other : best;
        }
        __syncthreads();
        if(lane == 0) best_keys[warp] = best;
        __syncthreads();
        best = best_keys[0];
#pragma unroll
        for(int w = 1; w < kWarps; w++) best = best_keys[w] > best ? best_keys[w] : best;
        last = best;
        if(tid == 0)
        {
            top_ids[row * top + k] = best ? key_index(best) : -1;
            top_logprobs[row * top + k] = best ? log_probability(key_logit(best)) : -INFINITY;
        }
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

template <int DTYPE>
int launch_fwd(const void* logits, int64_t pitch, const float* tokens, float* logprobs, float* entropy, float* lse,
               int32_t* top_ids, float* top_logprobs, int64_t top, int64_t rows, int64_t V, float c, float inverse_temperature, cudaStream_t stream)
{
    token_logprobs_kernel<DTYPE><<<(unsigned)rows, kThreads, 0, stream>>>(
        static_cast<const typename Logit<DTYPE>::type*>(logits), pitch, tokens, logprobs, entropy, lse, top_ids, top_logprobs,
        (int)top, (int)V, c, inverse_temperature);
    count_launch();
    return launch_status();
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
