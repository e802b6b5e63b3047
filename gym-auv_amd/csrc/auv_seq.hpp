// Shared pieces of the sequence operators (auv_conv.hpp, auv_scan.hpp, auv_norm.hpp): the three activation types, the
// scalar functions they apply per element, lane exchanges, and the fixed-order sum over slices.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace auv {
namespace seq {

using bf16 = __bf16;
using f16 = _Float16;

template <class T, int V>
struct __attribute__((aligned(sizeof(T) * V))) Vec {
    T v[V];
};

// V elements of T as floats; the address must be a multiple of V * sizeof(T).
template <class T, int V>
__device__ __forceinline__ void load(const T* p, float (&out)[V]) {
    const Vec<T, V> t = *reinterpret_cast<const Vec<T, V>*>(p);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = (float)t.v[i];
}
// The one rounding an output gets: to the nearest value of its type, ties to even.
template <class T, int V>
__device__ __forceinline__ void store(T* p, const float (&in)[V]) {
    Vec<T, V> t;
#pragma unroll
    for (int i = 0; i < V; ++i) t.v[i] = (T)in[i];
    *reinterpret_cast<Vec<T, V>*>(p) = t;
}

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLow = (float)(1.44269504088896340736 - (double)kLog2e);
constexpr float kLn2 = 0.69314718055994530942f;

// 2^x by the hardware's instruction (one unit in the last place; results below 2^-126 are 0).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }

// e^x with the product x log2(e) carried to twice the width: e^x = 2^(hi + lo), 2^lo = 1 + lo ln 2.  Without the low
// part the rounding of the product alone costs |x| 2^-24 of relative error.
__device__ __forceinline__ float exp_f(float x) {
    const float hi = x * kLog2e;
    const float lo = fmaf(x, kLog2e, -hi) + x * kLog2eLow;
    const float e = exp2_hw(hi);
    // e = 0 and e = inf stand as they are (lo is NaN where hi is infinite)
    return (e > 0.0f && e < __builtin_inff()) ? fmaf(e, lo * kLn2, e) : e;
}

__device__ __forceinline__ float sigmoid_f(float x) { return rcp_hw(1.0f + exp_f(-x)); }

// log(1 + e) for 0 <= e <= 1: 2 artanh(s), s = e / (2 + e) <= 1/3, by its series; the first term left out is
// s^17 / 17 <= 5e-10, below the last place of s.  No cancellation for small e, unlike log(1 + e) itself.
__device__ __forceinline__ float log1p_unit(float e) {
    const float s = e * rcp_hw(2.0f + e);
    const float q = s * s;
    float p = 1.0f / 15.0f;
    p = fmaf(p, q, 1.0f / 13.0f);
    p = fmaf(p, q, 1.0f / 11.0f);
    p = fmaf(p, q, 1.0f / 9.0f);
    p = fmaf(p, q, 1.0f / 7.0f);
    p = fmaf(p, q, 1.0f / 5.0f);
    p = fmaf(p, q, 1.0f / 3.0f);
    return 2.0f * fmaf(s * q, p, s);
}
// softplus(x) = log(1 + e^x) = max(x, 0) + log(1 + e^-|x|); its derivative is the sigmoid, from the same exponential.
// Both select with comparisons that are false for NaN, so NaN comes out as NaN.
__device__ __forceinline__ float softplus_f(float x) {
    const float e = exp_f(-__builtin_fabsf(x));
    return (x < 0.0f ? 0.0f : x) + log1p_unit(e);
}

// One value passed within the wave to the lane whose number differs in bit `BIT`.
template <int BIT>
__device__ __forceinline__ float lane_xor(float x) {
    return __shfl_xor(x, 1 << BIT, 64);
}
// Sum over the lanes that differ in bits LO .. HI-1, left in all of them.
template <int LO, int HI>
__device__ __forceinline__ float lane_sum(float x) {
    if constexpr (LO < HI) {
        x += lane_xor<LO>(x);
        x = lane_sum<LO + 1, HI>(x);
    }
    return x;
}

// dst[m] = sum over s of src[s * stride + m], in a fixed order: 32 partial sums of every 32nd slice, then those in
// ascending order.  One workgroup per 32 outputs; 1024 threads = 32 outputs x 32 partial sums, so that a few thousand
// slices cost tens of loads per thread and not a chain of thousands.
constexpr int kSumOutputs = 32, kSumLanes = 32;
struct SumArgs {
    const float* src;
    int64_t slices, stride, count;
    // output m goes to dst[part][...]: a slice holds `inner` numbers per channel, the first n[0] of them belong to
    // dst[0], the next n[1] to dst[1], ...; a null dst takes nothing
    int32_t inner;
    int32_t n[3];
    float* dst[3];
};
static __global__ __launch_bounds__(kSumOutputs * kSumLanes) void k_seq_sum(SumArgs a) {
    __shared__ float part[kSumLanes][kSumOutputs + 1];
    const int o = threadIdx.x % kSumOutputs, s0 = threadIdx.x / kSumOutputs;
    const int64_t m = (int64_t)blockIdx.x * kSumOutputs + o;
    float acc = 0.0f;
    if (m < a.count) {
#pragma unroll 8
        for (int64_t s = s0; s < a.slices; s += kSumLanes) acc += a.src[s * a.stride + m];
    }
    part[s0][o] = acc;
    __syncthreads();
    if (s0 == 0 && m < a.count) {
        float t = 0.0f;
        for (int i = 0; i < kSumLanes; ++i) t += part[i][o];
        const int64_t chan = m / a.inner;
        int k = (int)(m - chan * a.inner);
        for (int p = 0; p < 3; ++p) {
            if (k < a.n[p]) {
                if (a.dst[p]) a.dst[p][chan * a.n[p] + k] = t;
                break;
            }
            k -= a.n[p];
        }
    }
}

}  // namespace seq
}  // namespace auv
