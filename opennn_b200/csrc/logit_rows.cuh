// Rows of logits in fp32, bf16 or fp16: 16-byte vectors of a row and the elements around them, shared by the kernels
// that read logits (token_logprobs.cu, distill.cu).
//
// A row starts wherever `pitch` puts it, so it is cut into up to VE - 1 leading elements, a body of 16-byte vectors that
// starts on a 16-byte boundary, and up to VE - 1 trailing elements.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <math.h>

#include "common.cuh"
#include "launch_counter.h"

namespace onn
{

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

template <int DTYPE> struct Logit;

template <> struct Logit<ONN_F32>
{
    using type = float;
    static constexpr int VE = 4;                     // elements of a 16-byte vector
    static __device__ __forceinline__ float get(const type* p) { return *p; }
    static __device__ __forceinline__ void put(type* p, float v) { *p = v; }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[VE])
    {
        x[0] = __uint_as_float(v.x); x[1] = __uint_as_float(v.y); x[2] = __uint_as_float(v.z); x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[VE])
    {
        return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
    }
    // the largest element; NaN is passed by (NaN for nothing but NaN)
    static __device__ __forceinline__ float max(const uint4& v)
    {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    }
    static constexpr bool floors = false;                // -inf stays: a sum that multiplies by it has to look
    static __device__ __forceinline__ uint4 floor(const uint4& v) { return v; }
    static __device__ __forceinline__ uint4 lowest() { const unsigned int v = 0xff800000u; return make_uint4(v, v, v, v); }
};

template <> struct Logit<ONN_BF16>
{
    using type = __nv_bfloat16;
    static constexpr int VE = 8;
    static __device__ __forceinline__ float get(const type* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ void put(type* p, float v) { *p = __float2bfloat16_rn(v); }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[VE])
    {
        const unsigned int w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for(int i = 0; i < 4; i++) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[VE])
    {
        unsigned int w[4];
#pragma unroll
        for(int i = 0; i < 4; i++)
        {
            const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned int*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float max(const uint4& v)
    {
        auto h = [](unsigned int w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
        const float2 f = __bfloat1622float2(__hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w))));
        return fmaxf(f.x, f.y);
    }
    // -inf (and anything below -1e30) as -1e30, NaN as it is: finite, and as far below any other logit as makes no difference
    static constexpr bool floors = true;
    static __device__ __forceinline__ uint4 floor(const uint4& v)
    {
        const unsigned int bound = 0xf14af14au;              // -1.0e30 twice
        auto at_least = [&](unsigned int w)
        {
            const __nv_bfloat162 h = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&w), *reinterpret_cast<const __nv_bfloat162*>(&bound));
            return *reinterpret_cast<const unsigned int*>(&h);
        };
        return make_uint4(at_least(v.x), at_least(v.y), at_least(v.z), at_least(v.w));
    }
    static __device__ __forceinline__ uint4 lowest() { const unsigned int v = 0xff80ff80u; return make_uint4(v, v, v, v); }
};

template <> struct Logit<ONN_F16>
{
    using type = __half;
    static constexpr int VE = 8;
    static __device__ __forceinline__ float get(const type* p) { return __half2float(*p); }
    static __device__ __forceinline__ void put(type* p, float v) { *p = __float2half_rn(v); }
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[VE])
    {
        const unsigned int w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for(int i = 0; i < 4; i++)
        {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            x[2 * i] = f.x; x[2 * i + 1] = f.y;
        }
    }
    static __device__ __forceinline__ uint4 pack(const float (&x)[VE])
    {
        unsigned int w[4];
#pragma unroll
        for(int i = 0; i < 4; i++)
        {
            const __half2 h = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const unsigned int*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    static __device__ __forceinline__ float max(const uint4& v)
    {
        auto h = [](unsigned int w) { return *reinterpret_cast<const __half2*>(&w); };
        const float2 f = __half22float2(__hmax2(__hmax2(h(v.x), h(v.y)), __hmax2(h(v.z), h(v.w))));
        return fmaxf(f.x, f.y);
    }
    static constexpr bool floors = false;                // -inf stays: a sum that multiplies by it has to look
    static __device__ __forceinline__ uint4 floor(const uint4& v) { return v; }
    static __device__ __forceinline__ uint4 lowest() { const unsigned int v = 0xfc00fc00u; return make_uint4(v, v, v, v); }
};

// head + VE * vectors + tail = V; the body starts 16-byte aligned.
struct RowCut { int head, vectors, tail; };

template <int DTYPE>
__device__ __forceinline__ RowCut cut_row(const void* row, int V)
{
    constexpr int VE = Logit<DTYPE>::VE;
    RowCut c;
    c.head = (int)((-reinterpret_cast<intptr_t>(row)) & 15) / (16 / VE);
    if(c.head > V) c.head = V;
    c.vectors = (V - c.head) / VE;
    c.tail = V - c.head - c.vectors * VE;
    return c;
}

__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The largest of the lanes' values in one instruction; NaN is passed by.
__device__ __forceinline__ float warp_largest(float value)
{
    float t;
    asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(t) : "f"(value));
    return t;
}

// Two fp32 operations per instruction.
__device__ __forceinline__ unsigned long long pair_bits(float2 v)
{
    unsigned long long r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(v.x), "f"(v.y));
    return r;
}
__device__ __forceinline__ float2 pair_of(unsigned long long r)
{
    float2 v;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(v.x), "=f"(v.y) : "l"(r));
    return v;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    unsigned long long r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return pair_of(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    unsigned long long r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
    return pair_of(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    unsigned long long r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
    return pair_of(r);
}

// A row takes part when its token is in (0, V): 0 is padding, as in the loss.  Without tokens every row does.
__device__ __forceinline__ long long row_token(const float* tokens, long long row, int V, bool* active)
{
    if(!tokens) { *active = true; return -1; }
    const long long t = token_index(__ldg(tokens + row));
    *active = t > 0 && t < V;
    return t;
}

// A launch in clusters of `ctas` CTAs.  overlapped: as launch_overlapped (the kernel calls pdl_wait first).
template <typename... KernelArgs, typename... Args>
inline cudaError_t launch_clusters(void (*kernel)(KernelArgs...), unsigned int grid, int threads, int ctas, size_t dynamic_bytes, bool overlapped, cudaStream_t stream, Args&&... args)
{
    if(ctas == 1 && !overlapped)
    {
        kernel<<<grid, threads, dynamic_bytes, stream>>>(std::forward<Args>(args)...);      // half the host's time of the launch below
        return cudaGetLastError();
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = dynamic_bytes;
    config.stream = stream;
    cudaLaunchAttribute attribute[2];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim.x = ctas;
    attribute[0].val.clusterDim.y = 1;
    attribute[0].val.clusterDim.z = 1;
    attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[1].val.programmaticStreamSerializationAllowed = overlapped && pdl_enabled() ? 1 : 0;
    config.attrs = attribute;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
}

inline int logit_bytes(int dtype) { return dtype == ONN_F32 ? 4 : 2; }
inline bool logit_arguments_ok(const void* logits, int dtype, int64_t pitch, int64_t rows, int64_t V)
{
    return logits && dtype >= ONN_F32 && dtype <= ONN_F16 && V > 1 && V < (1LL << 31) - 4096 && pitch >= V &&
           rows > 0 && rows < (1LL << 27) && reinterpret_cast<uintptr_t>(logits) % logit_bytes(dtype) == 0;
}
// Gradients in the logits' place keep their rows' places.
inline bool gradient_place_ok(const void* logits, int64_t pitch, const void* dlogits, int64_t d_pitch) { return logits != dlogits || pitch == d_pitch; }
inline bool temperature_ok(float t) { return t > 0.f && t <= 1e6f && t >= 1e-6f; }

}  // namespace onn
