// Shared pieces of the sequence operators (auv_conv.hpp, auv_scan.hpp, auv_norm.hpp): the three activation types, the
// scalar functions they apply per element, lane exchanges, and the fixed-order sum over slices.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>
#include <utility>

namespace auv {
namespace seq {

using bf16 = __bf16;
using f16 = _Float16;

// V adjacent elements.  The hardware takes wide accesses at any address, so the type asks for no more alignment than an
// element's: rows of an odd number of channels are read as wide as others.
template <class T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
    T v[V];
};

// V elements of T as floats.
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

// V adjacent elements as they lie in memory, in 32-bit words.  Taking the elements out, or merging them with the zeros of
// a load left out, would wait for the load there and then; words wait until they are used.
template <class T, int V>
struct Raw {
    static_assert(V == 1 || sizeof(T) * V % 4 == 0, "whole words, or one element");
    static constexpr int kWords = ((int)sizeof(T) * V + 3) / 4;
    unsigned w[kWords];
    __device__ __forceinline__ float at(int i) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[i]);
        else return (float)__builtin_bit_cast(T, (unsigned short)(w[i / 2] >> (16 * (i % 2))));
    }
};
// The first `count` (0 to V) of V elements at p; the others come out as 0.
template <class T, int V>
__device__ __forceinline__ void fetch(Raw<T, V>& out, const T* p, int count) {
    struct __attribute__((packed, aligned(sizeof(T)))) Words {
        unsigned w[Raw<T, V>::kWords];
    };
#pragma unroll
    for (int i = 0; i < Raw<T, V>::kWords; ++i) out.w[i] = 0;
    if constexpr (sizeof(T) * V == 2) {
        if (count) out.w[0] = *reinterpret_cast<const unsigned short*>(p);
    } else if (count == V) {
        const Words t = *reinterpret_cast<const Words*>(p);
#pragma unroll
        for (int i = 0; i < Raw<T, V>::kWords; ++i) out.w[i] = t.w[i];
    } else if (count > 0) {
#pragma unroll
        for (int i = 0; i < V - 1; ++i)
            if (i < count) {
                if constexpr (sizeof(T) == 4) out.w[i] = reinterpret_cast<const unsigned*>(p)[i];
                else out.w[i / 2] |= (unsigned)reinterpret_cast<const unsigned short*>(p)[i] << (16 * (i % 2));
            }
    }
}
// The first `count` of V elements to p.
template <class T, int V>
__device__ __forceinline__ void put(T* p, int count, const float (&in)[V]) {
    if (count == V) {
        store<T, V>(p, in);
        asm volatile("");   // else the compiler shares this store's last element with the other branch, and splits it
    } else {
#pragma unroll
        for (int i = 0; i < V - 1; ++i)
            if (i < count) p[i] = (T)in[i];
    }
}
__device__ __forceinline__ int clamp_count(int64_t left, int most) { return left >= most ? most : left > 0 ? (int)left : 0; }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLog2eLow = (float)(1.44269504088896340736 - (double)kLog2e);
constexpr float kLn2 = 0.69314718055994530942f;

// 2^x by the hardware's instruction (one unit in the last place; results below 2^-126 are 0).
__device__ __forceinline__ float exp2_hw(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float rcp_hw(float x) { return __builtin_amdgcn_rcpf(x); }

// e^x for activations of type T.  The rounding of the product x log2(e) moves the result by |x| 2^-24 of itself: nothing
// beside what a 16-bit x was rounded by itself (by up to half a step, which moves e^x by |x| 2^-8 or 2^-11 of itself; so it is for
// the scan's step width, whose x has a 32-bit bias added), but for 32-bit ones the product is carried to twice the width,
// e^x = 2^(hi + lo), 2^lo = 1 + lo ln 2.
template <class T>
__device__ __forceinline__ float exp_f(float x) {
    const float hi = x * kLog2e;
    if constexpr (sizeof(T) == 2) return exp2_hw(hi);
    // (infinite x: the low part is NaN, which the median of three turns into a finite number; e is then 0, infinite or NaN)
    const float lo = __builtin_amdgcn_fmed3f(fmaf(x, kLog2eLow, fmaf(x, kLog2e, -hi)), -1.0f, 1.0f);
    return exp2_hw(hi) * fmaf(lo, kLn2, 1.0f);
}

template <class T>
__device__ __forceinline__ float sigmoid_f(float x) { return rcp_hw(1.0f + exp_f<T>(-x)); }

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
template <class T>
__device__ __forceinline__ float softplus_f(float x) {
    const float e = exp_f<T>(-__builtin_fabsf(x));
    return (x < 0.0f ? 0.0f : x) + log1p_unit(e);
}

// A value that is the same in every lane, as a scalar: what is computed from it needs no vector instructions.
__device__ __forceinline__ int uniform(int x) { return __builtin_amdgcn_readfirstlane(x); }

// Lane exchanges.  Within 16 lanes by data-parallel operands, which cost the instruction that uses them nothing; across
// by the two instructions that swap halves of two registers.  No LDS traffic, unlike a general permutation.
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
constexpr int kQuadXor1 = 0xb1, kQuadXor2 = 0x4e, kQuadXor3 = 0x1b, kHalfMirror = 0x141, kMirror = 0x140, kRotate8 = 0x128;

// f(0), f(1), ... f(N - 1) with the number as a compile-time constant.
template <class F, int... I>
__device__ __forceinline__ void static_for_(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, class F>
__device__ __forceinline__ void static_for(F&& f) {
    static_for_(f, std::make_integer_sequence<int, N>{});
}

// What lane FROM of every group of S adjacent lanes holds, in all of the group.
template <int S, int FROM>
__device__ __forceinline__ float lane_spread(float x) {
    static_assert(FROM < S, "a lane of the group");
    if constexpr (S == 1) return x;
    else if constexpr (S == 2) return dpp<FROM ? 0xf5 : 0xa0>(x);
    else if constexpr (S == 4) return dpp<FROM * 0x55>(x);
    else if constexpr (S == 16) return dpp<0x150 + FROM>(x);
    else {
        const float low = dpp<0x150 + FROM>(x), high = dpp<0x158 + FROM>(x);
        return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)) & 8 ? high : low;
    }
}

// After this, a holds both registers' low (BIT clear) parts side by side and b both high parts.
template <int BIT>
__device__ __forceinline__ void swap_halves(float& a, float& b) {
    static_assert(BIT == 4 || BIT == 5, "rows of 16 or halves of 32 lanes");
    const unsigned x = __builtin_bit_cast(unsigned, a), y = __builtin_bit_cast(unsigned, b);
    if constexpr (BIT == 5) {
        const auto r = __builtin_amdgcn_permlane32_swap(x, y, false, false);
        a = __builtin_bit_cast(float, (unsigned)r[0]), b = __builtin_bit_cast(float, (unsigned)r[1]);
    } else {
        const auto r = __builtin_amdgcn_permlane16_swap(x, y, false, false);
        a = __builtin_bit_cast(float, (unsigned)r[0]), b = __builtin_bit_cast(float, (unsigned)r[1]);
    }
}

// Sum over the lanes that differ in bits 0 .. HI-1, left in all of them.  (Mirrors do for single bits: the lanes of the
// lower bits already agree.)
template <int HI>
__device__ __forceinline__ float lane_sum(float x) {
    if constexpr (HI > 0) x += dpp<kQuadXor1>(x);
    if constexpr (HI > 1) x += dpp<kQuadXor2>(x);
    if constexpr (HI > 2) x += dpp<kHalfMirror>(x);
    if constexpr (HI > 3) x += dpp<kMirror>(x);
    if constexpr (HI > 4) {
        float y = x;
        swap_halves<4>(x, y);
        x += y;
    }
    if constexpr (HI > 5) {
        float y = x;
        swap_halves<5>(x, y);
        x += y;
    }
    return x;
}

// r = a + a of the lane 8 (4) away in lanes 0-7 (0-3, 8-11) of each 16, and b + b of that lane in the others: an add that
// writes only some banks of four lanes, so that a pair takes two instructions and no selects.  Four pairs at a time, which
// keeps the two wait states between a register's write and its use as a shifted operand to one s_nop on either side.
__device__ __forceinline__ void pair_sum8(float* v, int h) {
    float r0, r1, r2, r3;
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %4, %4 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %1, %5, %5 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %2, %6, %6 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %3, %7, %7 row_ror:8 row_mask:0xf bank_mask:0x3\n\t"
        "v_add_f32_dpp %0, %8, %8 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %1, %9, %9 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %2, %10, %10 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "v_add_f32_dpp %3, %11, %11 row_ror:8 row_mask:0xf bank_mask:0xc\n\t"
        "s_nop 1"
        : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[h]), "v"(v[h + 1]), "v"(v[h + 2]), "v"(v[h + 3]));
    v[0] = r0, v[1] = r1, v[2] = r2, v[3] = r3;
}
__device__ __forceinline__ void pair_sum4(float* v, int h) {
    float r0, r1, r2, r3;
    asm("s_nop 1\n\t"
        "v_add_f32_dpp %0, %4, %4 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %1, %5, %5 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %2, %6, %6 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %3, %7, %7 row_shl:4 row_mask:0xf bank_mask:0x5\n\t"
        "v_add_f32_dpp %0, %8, %8 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %1, %9, %9 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %2, %10, %10 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "v_add_f32_dpp %3, %11, %11 row_shr:4 row_mask:0xf bank_mask:0xa\n\t"
        "s_nop 1"
        : "=&v"(r0), "=&v"(r1), "=&v"(r2), "=&v"(r3)
        : "v"(v[0]), "v"(v[1]), "v"(v[2]), "v"(v[3]), "v"(v[h]), "v"(v[h + 1]), "v"(v[h + 2]), "v"(v[h + 3]));
    v[0] = r0, v[1] = r1, v[2] = r2, v[3] = r3;
}

// One halving step of the sums below: v[0 .. H) become the sums over the lanes that differ in bit BIT, of v[0 .. H) where
// that bit is clear and of v[H .. 2H) where it is set.
template <int BIT, int H>
__device__ __forceinline__ void halve(float* v) {
    if constexpr ((BIT == 3 || BIT == 2) && H % 4 == 0) {
#pragma unroll
        for (int i = 0; i < H; i += 4) {
            if constexpr (BIT == 3) pair_sum8(v + i, H);
            else pair_sum4(v + i, H);
        }
    } else if constexpr (BIT >= 4) {
#pragma unroll
        for (int i = 0; i < H; ++i) {
            swap_halves<BIT>(v[i], v[i + H]);
            v[i] += v[i + H];
        }
    } else {
        const bool high = __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)) >> BIT & 1;
#pragma unroll
        for (int i = 0; i < H; ++i) {
            const float keep = high ? v[i + H] : v[i], give = high ? v[i] : v[i + H];
            if constexpr (BIT == 3) v[i] = keep + dpp<kRotate8>(give);
            else if constexpr (BIT == 2) v[i] = keep + dpp<kQuadXor3>(dpp<kHalfMirror>(give));   // 7-i, then 3-i: i xor 4
            else if constexpr (BIT == 1) v[i] = keep + dpp<kQuadXor2>(give);
            else v[i] = keep + dpp<kQuadXor1>(give);
        }
    }
}

// Sums of N values at once over the lanes that differ in some bits, each left in one lane only: with every bit the number
// of values halves, so that they cost some 2 N instructions in place of N times the bits.  v[0 .. R) hold the sums, R = N
// over the number of lanes (at least 1), and lane_place says which values' they are.  The bits whose steps are cheapest, 3
// and 2, go first, while the values are many.
template <int HI, int LO, int N>
__device__ __forceinline__ void lane_scatter_sum(float* v) {
    constexpr int order[6] = {3, 2, 5, 4, 1, 0};
    constexpr auto count = [](int upto) {   // values left before step `upto`
        int n = N;
        for (int k = 0; k < upto; ++k)
            if (order[k] < HI && order[k] >= LO && n > 1) n /= 2;
        return n;
    };
    if constexpr (3 < HI && 3 >= LO && count(0) > 1) halve<3, count(0) / 2>(v);
    if constexpr (2 < HI && 2 >= LO && count(1) > 1) halve<2, count(1) / 2>(v);
    if constexpr (5 < HI && 5 >= LO && count(2) > 1) halve<5, count(2) / 2>(v);
    if constexpr (4 < HI && 4 >= LO && count(3) > 1) halve<4, count(3) / 2>(v);
    if constexpr (1 < HI && 1 >= LO && count(4) > 1) halve<1, count(4) / 2>(v);
    if constexpr (0 < HI && 0 >= LO && count(5) > 1) halve<0, count(5) / 2>(v);
}
// The number of the first of the values whose sums lane_scatter_sum leaves in this lane.
template <int HI, int LO, int N>
__device__ __forceinline__ int lane_place(int lane) {
    constexpr int order[6] = {3, 2, 5, 4, 1, 0};
    int n = N, at = 0;
    for (int k = 0; k < 6; ++k)
        if (order[k] < HI && order[k] >= LO && n > 1) {
            n /= 2;
            if (lane >> order[k] & 1) at += n;
        }
    return at;
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
    int64_t first;          // workgroup of this launch
};
static __global__ __launch_bounds__(kSumOutputs * kSumLanes) void k_seq_sum(SumArgs a) {
    __shared__ float part[kSumLanes][kSumOutputs + 1];
    const int o = threadIdx.x % kSumOutputs, s0 = threadIdx.x / kSumOutputs;
    const int64_t m = (a.first + blockIdx.x) * kSumOutputs + o;
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
