// What the kernels over 16- and 32-bit activations share: the element types of the
// ABI, vector loads and stores that convert to and from fp32, and the guard that
// makes a context's device the current one for the length of a call.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace sb200 {

using bf16 = __nv_bfloat16;
using f16 = __half;

inline bool known_type(int t) { return t == SB200_F32 || t == SB200_BF16 || t == SB200_F16; }
inline int type_bytes(int t) { return t == SB200_F32 ? 4 : 2; }

// Makes ctx->device current and puts the caller's device back: the torch side of a
// program keeps its own idea of the current device.
struct DeviceGuard {
    int before = -1;
    bool ok;
    explicit DeviceGuard(int device)
    {
        ok = cudaGetDevice(&before) == cudaSuccess &&
             (before == device || cudaSetDevice(device) == cudaSuccess);
        if (before == device) before = -1;
    }
    ~DeviceGuard() { if (before >= 0) cudaSetDevice(before); }
    DeviceGuard(const DeviceGuard&) = delete;
    DeviceGuard& operator=(const DeviceGuard&) = delete;
};

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// A launch that may overlap the tail of the kernel before; the kernel itself waits for that
// one (ptx::griddep_wait) before it touches global memory.
template <typename... A, typename... B>
inline int launch_after(sb200_ctx* ctx, void (*kern)(A...), dim3 grid, int block, size_t smem, cudaStream_t stream, B... args)
{
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(static_cast<unsigned>(block));
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    ctx->launches += 1;
    return cudaLaunchKernelEx(&cfg, kern, static_cast<A>(args)...) == cudaSuccess ? SB200_OK : SB200_ERR_CUDA;
}

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f(f16 x) { return __half2float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ f16 from_f<f16>(float x) { return __float2half_rn(x); }

// Two fp32 operations an instruction (each element rounded as by the scalar one).
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 d;
    asm("add.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 d;
    asm("mul.rn.f32x2 %0, %1, %2;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)));
    return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;"
        : "=l"(reinterpret_cast<unsigned long long&>(d))
        : "l"(reinterpret_cast<const unsigned long long&>(a)), "l"(reinterpret_cast<const unsigned long long&>(b)),
          "l"(reinterpret_cast<const unsigned long long&>(c)));
    return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// Two neighbouring elements of an array, as fp32.
__device__ __forceinline__ float2 pair_f(const float* p) { return make_float2(p[0], p[1]); }
__device__ __forceinline__ float2 pair_f(const bf16* p) { return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p)); }
__device__ __forceinline__ float2 pair_f(const f16* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }
__device__ __forceinline__ void set_pair(float* p, float2 v) { p[0] = v.x; p[1] = v.y; }
__device__ __forceinline__ void set_pair(bf16* p, float2 v) { *reinterpret_cast<__nv_bfloat162*>(p) = __float22bfloat162_rn(v); }
__device__ __forceinline__ void set_pair(f16* p, float2 v) { *reinterpret_cast<__half2*>(p) = __float22half2_rn(v); }

// VEC consecutive elements as raw words; the pointer is aligned to min(16, VEC * sizeof(T)).
template <typename T, int VEC>
struct Raw {
    static constexpr int BYTES = VEC * static_cast<int>(sizeof(T));
    static_assert(BYTES == 2 || BYTES == 4 || BYTES == 8 || BYTES == 16 || BYTES == 32, "vector width");
    alignas(BYTES < 16 ? BYTES : 16) T e[VEC];
};

// STREAM: data that is read or written once, which need not stay in the caches.
template <bool STREAM, typename T, int VEC>
__device__ __forceinline__ void load_raw(Raw<T, VEC>& r, const T* p)
{
    constexpr int B = Raw<T, VEC>::BYTES;
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) {
            const uint4* q = reinterpret_cast<const uint4*>(p) + i;
            reinterpret_cast<uint4*>(r.e)[i] = STREAM ? __ldcs(q) : *q;
        }
    } else if constexpr (B == 8) {
        *reinterpret_cast<uint2*>(r.e) = STREAM ? __ldcs(reinterpret_cast<const uint2*>(p)) : *reinterpret_cast<const uint2*>(p);
    } else if constexpr (B == 4) {
        *reinterpret_cast<uint32_t*>(r.e) =
            STREAM ? __ldcs(reinterpret_cast<const uint32_t*>(p)) : *reinterpret_cast<const uint32_t*>(p);
    } else {
        *reinterpret_cast<unsigned short*>(r.e) = STREAM ? __ldcs(reinterpret_cast<const unsigned short*>(p))
                                                         : *reinterpret_cast<const unsigned short*>(p);
    }
}

template <bool STREAM, typename T, int VEC>
__device__ __forceinline__ void store_raw(T* p, const Raw<T, VEC>& r)
{
    constexpr int B = Raw<T, VEC>::BYTES;
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) {
            uint4* q = reinterpret_cast<uint4*>(p) + i;
            const uint4 v = reinterpret_cast<const uint4*>(r.e)[i];
            if (STREAM) __stcs(q, v); else *q = v;
        }
    } else if constexpr (B == 8) {
        const uint2 v = *reinterpret_cast<const uint2*>(r.e);
        if (STREAM) __stcs(reinterpret_cast<uint2*>(p), v); else *reinterpret_cast<uint2*>(p) = v;
    } else if constexpr (B == 4) {
        const uint32_t v = *reinterpret_cast<const uint32_t*>(r.e);
        if (STREAM) __stcs(reinterpret_cast<uint32_t*>(p), v); else *reinterpret_cast<uint32_t*>(p) = v;
    } else {
        const unsigned short v = *reinterpret_cast<const unsigned short*>(r.e);
        if (STREAM) __stcs(reinterpret_cast<unsigned short*>(p), v); else *reinterpret_cast<unsigned short*>(p) = v;
    }
}

template <bool STREAM, typename T, int VEC>
__device__ __forceinline__ void load_f(float (&f)[VEC], const T* p)
{
    Raw<T, VEC> r;
    load_raw<STREAM>(r, p);
#pragma unroll
    for (int i = 0; i < VEC; ++i) f[i] = to_f(r.e[i]);
}

template <bool STREAM, typename T, int VEC>
__device__ __forceinline__ void store_f(T* p, const float (&f)[VEC])
{
    Raw<T, VEC> r;
#pragma unroll
    for (int i = 0; i < VEC; ++i) r.e[i] = from_f<T>(f[i]);
    store_raw<STREAM>(p, r);
}

}  // namespace sb200
