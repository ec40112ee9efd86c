// What the two ways of sb200_orthogonalize share.
#pragma once
#include "typed.cuh"

namespace sb200 {

constexpr float ORTH_SCALE = 8192.0f;            // 2^13: matrices are kept as fp16 parts of 2^13 times their values
constexpr float ORTH_INV_SCALE = 1.0f / 8192.0f;

struct OrthCall {
    void* out; int64_t ldo, stride_out;
    const void* g; int64_t ldg, stride_g;
    int64_t rows, cols, batch;
    int steps;
    float a, b, c, eps;
    int type;
};

// x -> 2^13 x / (norm + eps), from the sum of squares.  The factor leaves the fp32 range for
// norms below about 1e-35: then in fp64.
struct OrthInverse {
    double exact;
    float quick;
    bool beyond;
    __device__ OrthInverse(double squares, float eps)
        : exact(static_cast<double>(ORTH_SCALE) / (sqrt(squares) + static_cast<double>(eps))), quick(static_cast<float>(exact)),
          beyond(exact > 1e38) {}
    __device__ float operator()(float x) const { return beyond ? static_cast<float>(static_cast<double>(x) * exact) : x * quick; }
};

// hi = fp16(v), lo = fp16(v - hi)
template <int N>
__device__ __forceinline__ void split_f16(const float* v, Raw<f16, N>& hi, Raw<f16, N>& lo)
{
#pragma unroll
    for (int e = 0; e < N; e += 2) {
        const __half2 h = __floats2half2_rn(v[e], v[e + 1]);
        const float2 f = __half22float2(h);
        *reinterpret_cast<__half2*>(&hi.e[e]) = h;
        *reinterpret_cast<__half2*>(&lo.e[e]) = __floats2half2_rn(v[e] - f.x, v[e + 1] - f.y);
    }
}

// v += hi (or lo) of eight elements
__device__ __forceinline__ void join_f16(float (&v)[8], const Raw<f16, 8>& part)
{
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&part.e[e]));
        v[e] += f.x;
        v[e + 1] += f.y;
    }
}

// orthogonalize_small.cu: matrices whose shorter side is at most 128, whole in one cluster.
// always: as large as a portable cluster holds, so that no other way is taken on any device;
// fits: as large as the cluster that the context's device grants.
bool orthogonalize_small_always(int64_t rows, int64_t cols);
bool orthogonalize_small_fits(const sb200_ctx* ctx, const OrthCall& q);
int launch_orthogonalize_small(sb200_ctx* ctx, const OrthCall& q, cudaStream_t stream);

}  // namespace sb200
