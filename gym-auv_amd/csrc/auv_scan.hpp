// The selective state space scan: per channel d of a row, N states h[n] with decays that depend on the token,
//
//   dt = softplus(delta + delta_bias)          h[n] <- exp(dt A[d,n]) h[n] + dt u B[g,n]
//   y  = sum_n C[g,n] h[n] + D[d] u            out = y silu(z)
//
// g is the channel's group (channels / groups adjacent channels share B and C).  A token marked in `start` opens an
// episode: the states are cleared before it.  Tokens at and behind lengths[b] are not read and give zeros; the states
// handed on are those after the row's last token.  Everything between the loads and the one rounding of each output is
// in 32 bits.
//
// Two bounds lie close together: 4 elements of traffic per (token, channel), and per state one exponential (two issue
// slots), two multiplications and two fused multiply-adds on the vector unit.  4,096 rows x 128 tokens x 128 channels, bf16,
// 16 states: the traffic (638 MB) asks for 124 us, 96 slots for the states and some 45 for widths, gates, sums and their
// loads and stores for 290 us.  It takes 297 us with the vector unit at work in 92 % of the busy cycles: bound by arithmetic.
// The product x B as a rank-1 matrix instruction (4 x 4 x 1, in 32 bits) took 444 us, C h by them as well 506 us.
#pragma once

#include <type_traits>

#include "auv_seq.hpp"
#include "auv_conv.hpp"   // row_length

namespace auv {
namespace seq {

constexpr int kSegment = 16;         // tokens between the states kept for the backward pass
constexpr int kScanWaves = 4;        // waves per workgroup of the forward kernels

struct ScanArgs {
    int64_t B, L, D, G;
    int32_t N, softplus;
    const void *u, *delta, *z;
    int64_t u_row, u_token, delta_row, delta_token, z_row, z_token;
    const void *Bm, *Cm;
    int64_t B_row, B_token, B_group, C_row, C_token, C_group;
    const float *A, *Dv, *bias;
    const uint8_t* start;
    int64_t start_row, start_token;
    const int32_t* lengths;
    const float* state;      // [B,D,N]
    float* new_state;        // [B,D,N]
    void* y;
    int64_t y_row, y_token;
    float* segments;         // [B, ceil(L/16), D, NP]: the states before every 16th token
    int64_t chunk, chunks;   // tokens per chunk (a multiple of 16), chunks per row
    float *chunk_state, *chunk_decay;   // [chunks, B, D, NP]; decays as chunk_log gives them
    // backward
    const void* dy;
    int64_t dy_row, dy_token;
    const float* dnew_state; // [B,D,N]
    void *du, *ddelta, *dz;
    int64_t du_row, du_token, ddelta_row, ddelta_token, dz_row, dz_token;
    void *dB, *dC;
    int64_t dB_row, dB_token, dB_group, dC_row, dC_token, dC_group;
    float* dstate;           // [B,D,N]
    float* partial;          // [gridDim.x * units per workgroup, D, N + 2]: dA, dD, ddelta_bias
    int32_t lanes;           // threads side by side on a row's channels in a step
    int32_t whole;           // rows of activations and of their gradients may be read and written in fours
    float* bc_partial;       // [tile blocks, B, L, G, 2, NP] when a group's channels fill more than one workgroup
    int64_t first;           // forwards and in k_scan_sum_bc: workgroup of this launch
};

__device__ __forceinline__ void wave_sync() {
    // LDS traffic of one wave is in order; this keeps the compiler from moving it across
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// delta -> step width, and the width's derivative with respect to delta
template <class T>
__device__ __forceinline__ float step_width(float raw, int softplus) { return softplus ? softplus_f<T>(raw) : raw; }
template <class T>
__device__ __forceinline__ float step_slope(float raw, int softplus) { return softplus ? sigmoid_f<T>(raw) : 1.0f; }

// ----------------------------------------------------------------------------------------------------------------
// Forward.  S lanes per channel, NPL states per lane: 64 / S channels per wave, a wave per (channel tile, group, row,
// chunk of time).  With S > 1 the lanes of a channel share the element-wise work of its tokens.  B and C of the next tokens
// go through LDS once per wave as floats, zero-padded to NP states, which takes care of odd counts and strides; every lane
// of a channel reads them from there at the same address.
//
// MODE 0 computes outputs (from `state`, or from the chunk's entry state when the row is split into chunks).
// MODE 1 starts each chunk from zero and leaves only its end state and its decay, exp(A sum dt), as its logarithm.
// ----------------------------------------------------------------------------------------------------------------
// A chunk's decay is handed on as its logarithm (to base 2): the decay itself leaves the 32 bits' range long before what it
// is a factor of does, 16 tokens that each take e^-6, or give it, suffice.  Kept finite, so that logarithms can be added
// up; negative infinity stands for a start within the chunk and for nothing else.  (A step width that is no number makes
// the chunk's own end state one that is none, whatever stands here.)
constexpr float kCut = -__builtin_inff();
__device__ __forceinline__ float chunk_log(bool cut, float log) { return cut ? kCut : __builtin_amdgcn_fmed3f(log, -1e30f, 1e30f); }

template <int S>
constexpr int lane_bits() { return S >= 16 ? 4 : S >= 8 ? 3 : S >= 4 ? 2 : S >= 2 ? 1 : 0; }
// Tokens at a time: at least one for every lane of a channel.  Four where a lane has whole channels: eight take 233
// registers (two waves per SIMD, 324 us for 4,096 x 128 x 128 in bf16 with 16 states), four 165 (three, 297 us).
template <int S>
constexpr int scan_tile() { return S > 8 ? S : S == 1 ? 4 : 8; }

template <class T, int NPL, int S, int MODE>
__global__ __launch_bounds__(kScanWaves * 64) void k_scan_forward(ScanArgs a) {
    constexpr int NP = NPL * S, CW = 64 / S, TQ = scan_tile<S>(), KT = TQ / S, SB = lane_bits<S>();
    constexpr int BE = (TQ * NP + 63) / 64;   // elements of B (and of C) a lane carries into LDS per tile
    __shared__ __align__(16) float tile[kScanWaves][TQ][2][NP];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int q = lane % S, c = lane / S;
    const int Dg = (int)(a.D / a.G), tiles = (Dg + CW - 1) / CW;
    unsigned id = ((unsigned)a.first + blockIdx.x) * kScanWaves + wave;             // the host sees to it that there are fewer than 2^31
    const int ct = id % tiles;
    id /= tiles;
    const int g = id % (unsigned)a.G;
    id /= (unsigned)a.G;
    const unsigned chunk = id / (unsigned)a.B, b32 = id - chunk * (unsigned)a.B;
    if (chunk >= a.chunks) return;
    const int64_t b = b32;
    const int d_first = g * Dg + ct * CW, d_left = Dg - ct * CW;
    const bool live = c < d_left;
    const int dl = live ? c : d_left - 1;      // channel within the wave's tile
    const int64_t d = d_first + dl;
    const int64_t n = row_length(a.lengths, b, a.L);
    const int64_t t_begin = chunk * a.chunk, t_end = t_begin + a.chunk < a.L ? t_begin + a.chunk : a.L;
    const int64_t stop = t_end < n ? t_end : n;

    float h[NPL], A2[NPL];
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
        const int s = q * NPL + j;
        A2[j] = s < a.N ? a.A[d * a.N + s] * kLog2e : 0.0f;
        h[j] = 0.0f;
        if (MODE == 0) {
            if (a.chunks > 1) h[j] = a.chunk_state[((chunk * a.B + b) * a.D + d) * NP + s];
            else if (a.state && s < a.N) h[j] = a.state[(b * a.D + d) * a.N + s];
        }
    }
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dv ? a.Dv[d] : 0.0f;
    // the wave's place in each array is a scalar; a lane adds its channel and its first token
    const T* const u = (const T*)a.u + b * a.u_row + d_first;
    const T* const delta = (const T*)a.delta + b * a.delta_row + d_first;
    const T* const z = (const T*)a.z + b * a.z_row + d_first;
    const T* const Bm = (const T*)a.Bm + b * a.B_row + g * a.B_group;
    const T* const Cm = (const T*)a.Cm + b * a.C_row + g * a.C_group;
    T* const y = (T*)a.y + b * a.y_row + d_first;
    const int64_t u_lane = q * a.u_token + dl, delta_lane = q * a.delta_token + dl, z_lane = q * a.z_token + dl, y_lane = q * a.y_token + dl;
    float sum_dt = 0.0f;
    bool cut = false;

    // What a tile needs from memory, fetched one tile ahead.  The lanes of a channel take a token each, form its width and
    // its gate, and hand them round.
    T ru[KT], rd[KT], rz[KT], rB[BE], rC[BE];
    uint8_t mark = 0;
    auto ask = [&](int64_t t0) {
        if (t0 >= stop) return;
        const int left = stop - t0 < TQ ? (int)(stop - t0) : TQ;
#pragma unroll
        for (int k = 0; k < KT; ++k)
            if (k * S + q < left) {
                const int64_t t = t0 + k * S;
                ru[k] = (u + t * a.u_token)[u_lane];
                rd[k] = (delta + t * a.delta_token)[delta_lane];
                if (MODE == 0 && a.z) rz[k] = (z + t * a.z_token)[z_lane];
            }
#pragma unroll
        for (int k = 0; k < BE; ++k) {
            const int e = k * 64 + lane, i = e / NP, s = e % NP;
            const bool in = i < left && s < a.N;
            rB[k] = in ? (Bm + t0 * a.B_token)[i * a.B_token + s] : (T)0.0f;
            if (MODE == 0) rC[k] = in ? (Cm + t0 * a.C_token)[i * a.C_token + s] : (T)0.0f;
        }
        mark = 0;
        if (a.start && lane < left) mark = a.start[b * a.start_row + (t0 + lane) * a.start_token];
    };
#pragma unroll
    for (int k = 0; k < KT; ++k) ru[k] = rd[k] = rz[k] = (T)0.0f;
    ask(t_begin);
    for (int64_t t0 = t_begin; t0 < stop; t0 += TQ) {
        const int left = stop - t0 < TQ ? (int)(stop - t0) : TQ;
        if (MODE == 0 && a.segments && t0 % kSegment == 0 && live) {
            float* const seg = a.segments + ((b * ((a.L + kSegment - 1) / kSegment) + t0 / kSegment) * a.D + d) * NP + q * NPL;
#pragma unroll
            for (int j = 0; j < NPL; j += 4) *reinterpret_cast<float4*>(seg + j) = make_float4(h[j], h[j + 1], h[j + 2], h[j + 3]);
        }
        const unsigned long long marks = __ballot(mark != 0);
        float uu[KT], dt[KT], du[KT], sz[KT];
#pragma unroll
        for (int k = 0; k < KT; ++k) {
            uu[k] = (float)ru[k];
            dt[k] = step_width<T>((float)rd[k] + bias, a.softplus);
            du[k] = dt[k] * uu[k];
            sz[k] = 1.0f;
            if (MODE == 0 && a.z) {
                const float zz = (float)rz[k];
                sz[k] = zz * sigmoid_f<T>(zz);
            }
            if (MODE == 1 && k * S + q < left) sum_dt += dt[k];
        }
        wave_sync();
#pragma unroll
        for (int k = 0; k < BE; ++k) {
            const int e = k * 64 + lane, i = e / NP, s = e % NP;
            if (TQ * NP >= 64 || e < TQ * NP) {
                tile[wave][i][0][s] = (float)rB[k];
                if (MODE == 0) tile[wave][i][1][s] = (float)rC[k];
            }
        }
        wave_sync();
        ask(t0 + TQ);
        auto tokens = [&](auto plain) {
            constexpr bool PLAIN = decltype(plain)::value;      // a whole tile without a start in it
            static_for<KT>([&](auto kk) {
                constexpr int k = decltype(kk)::value;
                float part[S];
                static_for<S>([&](auto oo) {
                    constexpr int o = decltype(oo)::value, i = k * S + o;
                    part[o] = 0.0f;
                    if (PLAIN || i < left) {
                        if (!PLAIN && (marks >> i & 1)) {
                            cut = true;
#pragma unroll
                            for (int j = 0; j < NPL; ++j) h[j] = 0.0f;
                        }
                        const float w = lane_spread<S, o>(dt[k]), x = lane_spread<S, o>(du[k]);
                        float e[NPL], acc0, acc1;
#pragma unroll
                        for (int j = 0; j < NPL; ++j) e[j] = exp2_hw(w * A2[j]);
#pragma unroll
                        for (int j = 0; j < NPL; ++j) h[j] = fmaf(e[j], h[j], x * tile[wave][i][0][q * NPL + j]);
                        if (MODE == 0) {
                            acc0 = h[0] * tile[wave][i][1][q * NPL];
                            acc1 = h[1] * tile[wave][i][1][q * NPL + 1];
#pragma unroll
                            for (int j = 2; j < NPL; j += 2) {
                                acc0 = fmaf(h[j], tile[wave][i][1][q * NPL + j], acc0);
                                acc1 = fmaf(h[j + 1], tile[wave][i][1][q * NPL + j + 1], acc1);
                            }
                            part[o] = acc0 + acc1;
                        }
                        // sixteen states a token are enough to schedule among; more tokens at once cost registers, that is waves
                        if (NPL >= 16) __builtin_amdgcn_sched_barrier(0);
                    }
                });
                if (MODE == 0) {
                    lane_scatter_sum<SB, 0, S>(part);      // lane q gets the sum of token k S + q
                    if (live && (PLAIN || k * S + q < left))
                        (y + (t0 + k * S) * a.y_token)[y_lane] = (T)(fmaf(skip, uu[k], part[0]) * sz[k]);
                }
            });
        };
        if (left == TQ && marks == 0) tokens(std::true_type{});
        else tokens(std::false_type{});
    }
    if (MODE == 1) {
        sum_dt = lane_sum<SB>(sum_dt);     // over the tokens that a channel's lanes had
        if (live) {
            const int64_t o = ((chunk * a.B + b) * a.D + d) * NP + q * NPL;
#pragma unroll
            for (int j = 0; j < NPL; ++j) {
                a.chunk_state[o + j] = h[j];
                a.chunk_decay[o + j] = chunk_log(cut, sum_dt * A2[j]);
            }
        }
        return;
    }
    if (a.new_state && live && stop == n && (t_begin < n || (n == 0 && chunk == 0))) {
#pragma unroll
        for (int j = 0; j < NPL; ++j)
            if (q * NPL + j < a.N) a.new_state[(b * a.D + d) * a.N + q * NPL + j] = h[j];
    }
    if (live && q == 0)
        for (int64_t t = t_begin > n ? t_begin : n; t < t_end; ++t) (y + t * a.y_token)[dl] = (T)0.0f;
}

// Joins the chunks of a row: chunk_state[c] becomes the state the chunk starts from (forwards from `state`) or, going
// backwards, the gradient that reaches the chunk's last state from behind (from the gradient of the states handed on,
// which lands in dstate at the front).  A workgroup takes LANES numbers and splits the chunks over 1,024 / LANES rows of
// threads.  Bound by the latency of its loads: few numbers want many rows.
constexpr int kJoinThreads = 1024;
struct JoinArgs {
    float *chunk_state, *chunk_decay;
    const float* first;     // [B,D,N] or null
    float* last;            // [B,D,N] or null
    int64_t chunks, count;  // count = B D NP
    int32_t N, NP, reverse;
};
template <int LANES>
__global__ __launch_bounds__(kJoinThreads) void k_scan_join(JoinArgs a) {
    constexpr int ROWS = kJoinThreads / LANES;
    __shared__ float hs[ROWS][LANES], ps[ROWS][LANES];
    const int lane = threadIdx.x % LANES, row = threadIdx.x / LANES;
    const int64_t i = (int64_t)blockIdx.x * LANES + lane;
    const bool live = i < a.count;
    const int64_t per = (a.chunks + ROWS - 1) / ROWS;
    const int64_t c0 = row * per < a.chunks ? row * per : a.chunks, c1 = c0 + per < a.chunks ? c0 + per : a.chunks;
    auto at = [&](int64_t c) { return (a.reverse ? a.chunks - 1 - c : c) * a.count + i; };
    // s + 2^p x.  Behind a start whatever came before (also an infinity or NaN) has no part in what follows.  Everywhere else
    // it has one: 2^p is multiplied in by halves within [2^-126, 2^127], so that an infinity or NaN stays one however small the
    // decay, a 0 stays 0 however large, and what is cut off at either end is off by less than 2^-124, or beyond 2^128 too.  No
    // half is 0, which therefore stands for a start.
    auto half = [](float p) { return p == kCut ? 0.0f : exp2_hw(__builtin_amdgcn_fmed3f(0.5f * p, -126.0f, 127.0f)); };
    auto join = [](float half, float x, float s) { return half == 0.0f ? s : fmaf(x * half, half, s); };
    float h = 0.0f, p = 0.0f;
    if (live) {
#pragma unroll 4
        for (int64_t c = c0; c < c1; ++c) {
            const float s = a.chunk_state[at(c)], q = a.chunk_decay[at(c)];
            h = join(half(q), h, s);
            p += q;
        }
    }
    hs[row][lane] = h;
    ps[row][lane] = half(p);
    __syncthreads();
    if (!live) return;
    const int64_t bd = i / a.NP;
    const int s = (int)(i - bd * a.NP);
    float x = a.first && s < a.N ? a.first[bd * a.N + s] : 0.0f;
#pragma unroll 8
    for (int r = 0; r < row; ++r) x = join(ps[r][lane], x, hs[r][lane]);
    for (int64_t c = c0; c < c1; c += 4) {      // four at a time: no load waits behind the stores before it
        float e[4], q[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k < c1) e[k] = a.chunk_state[at(c + k)], q[k] = a.chunk_decay[at(c + k)];
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (c + k < c1) {
                a.chunk_state[at(c + k)] = x;
                x = join(half(q[k]), x, e[k]);
            }
    }
    if (a.last && s < a.N && row == ROWS - 1) a.last[bd * a.N + s] = x;
}

// ----------------------------------------------------------------------------------------------------------------
// Backward.  With g = dout silu(z) the gradient of y, and dh[n] the gradient of the state after a token,
//
//   dh = carry + g C       dC += g h      dB += dh dt u     s1 = sum_n dh B     carry = exp(dt A) dh
//   through = carry h_before     dA += through dt     du = s1 dt + g D     ddelta = (s1 u + sum_n through A) softplus'
//   dz = dout y silu'(z)         dD += g u            carry = through = 0 at a start
//
// The states are formed again from the ones kept before every 16th token: a lane holds 4 states of one channel over 16
// tokens in registers, S = NP / 4 lanes make a channel, a wave 64 / S channels.  dB and dC are sums over a group's
// channels: over the lanes of a wave, then over the waves of the workgroup through LDS, in a fixed order.  dA, dD and
// ddelta_bias are sums over rows and tokens: each wave keeps them in registers over all rows it works on.
// ----------------------------------------------------------------------------------------------------------------
// The element-wise parts (widths, gates and their derivatives; the stores of du, ddelta, dz) belong to the workgroup: a
// thread takes four adjacent channels of a token, so that loads and stores are 8 or 16 bytes wide and a token's channels
// go in one piece.  Two-byte accesses by the lanes of the sweeps, 32 bytes of a token at a time, took longer than the
// arithmetic.  4,096 rows x 64 tokens x 128 channels, bf16, 16 states: 669 us (1,878 us in the first form, with lanes that
// loaded for themselves and sums through shuffles) at 2,425 vector instructions per 16 tokens of 16 channels, the vector unit
// at work in 94 % of the busy cycles: bound by instructions issued.  Not all of them are arithmetic: 128 registers, which two
// workgroups per CU leave, do not hold a tile, so that 116 scalars lie in vector lanes and are moved there and back, and 21
// vector registers (25 of 32-bit activations) in scratch memory, a good half of the 21 memory instructions per tile.
template <int S>
constexpr int scan_back_waves() { return S <= 4 ? 8 : 4; }
// tokens whose states a lane holds at a time: half a segment, so that two waves more fit on a SIMD (with S = 16 the sums
// over a channel's lanes want all sixteen together)
template <int S>
constexpr int scan_back_hold() { return S <= 8 ? 8 : 16; }
template <int S>
constexpr size_t scan_back_lds(int units) {
    constexpr int NP = 4 * S, W = scan_back_waves<S>(), CH = 64 / S * W;
    // per token and channel four numbers; delta_bias and D per channel; sums of dD and ddelta_bias per thread; sums of dB
    // and dC per wave; row lengths; B and C per row
    return (size_t)4 * (4 * 16 * CH + 2 * CH + 2 * 4 * W * 64 + W * 16 * 2 * NP + 2 * W + units * 16 * 2 * NP);
}

// The kernel's arguments, read where they are used: some sixty addresses and strides held in scalar registers through
// the tile loop would push its own scalars out to vector lanes.
__device__ __forceinline__ ScanArgs scan_args() {
    const __attribute__((address_space(4))) ScanArgs* p = (const __attribute__((address_space(4))) ScanArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    ScanArgs r;
    __builtin_memcpy(&r, (const ScanArgs*)p, sizeof(ScanArgs));
    return r;
}

// Four adjacent channels of one token as they lie in memory, in 32-bit words: taking the elements out, or merging them
// with the zeros of a load left out, would wait for the load there and then.
template <class T>
struct Quad {
    unsigned w[sizeof(T)];
    __device__ __forceinline__ float at(int j) const {
        if constexpr (sizeof(T) == 4) return __builtin_bit_cast(float, w[j]);
        else return (float)__builtin_bit_cast(T, (unsigned short)(w[j / 2] >> (16 * (j % 2))));
    }
};
// `count` of the four are real (the others come out as 0); `whole`: the address allows one access.
template <class T>
__device__ __forceinline__ void load4(Quad<T>& out, const T* p, int count, bool whole) {
    using Words = Vec<unsigned, sizeof(T)>;
#pragma unroll
    for (int j = 0; j < (int)sizeof(T); ++j) out.w[j] = 0;
    if (whole) {
        if (count == 4) {
            const Words t = *reinterpret_cast<const Words*>(p);
#pragma unroll
            for (int j = 0; j < (int)sizeof(T); ++j) out.w[j] = t.v[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) {
                if constexpr (sizeof(T) == 4) out.w[j] = reinterpret_cast<const unsigned*>(p)[j];
                else out.w[j / 2] |= (unsigned)reinterpret_cast<const unsigned short*>(p)[j] << (16 * (j % 2));
            }
    }
}
template <class T>
__device__ __forceinline__ void store4(T* p, int count, bool whole, const float (&in)[4]) {
    if (whole) {
        if (count == 4) store<T, 4>(p, in);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < count) p[j] = (T)in[j];
    }
}

// The thread's number, in a form whose derivatives the compiler does not carry from one use to the next.
__device__ __forceinline__ int thread_anew() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// i times a stride, of two instructions
__device__ __forceinline__ int64_t times(int i, int64_t stride) { return (int64_t)((uint64_t)(unsigned)i * (uint64_t)stride); }

// MODE 0: gradients.  MODE 1: from zero at the end of each chunk, only the carry at its front and its decay.
// TAIL: rows may end within a tile.  The tokens behind have a width of 0, which hands states and carry on as they are; but
// where these are infinite, 0 times them is not 0, and dA, dB and dC leave such tokens out.
template <class T, int S, int MODE, bool TAIL>
__global__ __launch_bounds__(scan_back_waves<S>() * 64, S == 4 ? 4 : S == 8 ? 3 : 2) void k_scan_backward(ScanArgs a) {
    constexpr int NP = 4 * S, CW = 64 / S, W = scan_back_waves<S>(), Q = kSegment, HQ = scan_back_hold<S>(), KT = HQ / S, SB = lane_bits<S>();
    constexpr int TH = W * 64, CH = W * CW;
    constexpr int QUADS = CH / 4, STEP = TH / QUADS, IT = Q > STEP ? Q / STEP : 1;   // a thread's tokens: first, first + STEP, ...
    constexpr int BE = Q * 2 * NP / 64;                                             // its share of B and C at the most
    // dB and dC of GT tokens are summed over the wave's channels together: as many values as lanes to sum over
    // A second form of the sweeps, without the selects for starts and row ends, pays where the registers of both fit: forwards
    // and backwards, 128 channels x 64 tokens, 8 states 650 us with it and 661 without, 32 states 991 and 1,013, 64 states 1,294
    // and 1,342; but 16 states (128 registers) 849 and 822, 4 states (256) 596 and 481.
    constexpr bool kPlainToo = S == 2 || S > 4;
    constexpr int GT = CW >= 8 ? CW / 8 : 1, GV = GT * 8, GR = GV / CW > 1 ? GV / CW : 1;
    static_assert(S <= HQ && GT <= HQ && CW >= 4, "the sums over lanes are formed for whole groups of tokens");
    extern __shared__ __align__(16) float lds[];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int q = lane % S, c = lane / S;
    // [token][channel]: the step's width; width u, then the sweeps' s1; g, then the sum of through A2; the sum of C h
    float(*const width)[CH] = reinterpret_cast<float(*)[CH]>(lds);
    float(*const wu)[CH] = width + Q, (*const gate)[CH] = wu + Q, (*const sum_y)[CH] = gate + Q;
    float(*const param)[CH] = sum_y + Q;                                                    // delta_bias, D
    float(*const sums)[4] = reinterpret_cast<float(*)[4]>(param + 2);                       // a thread's dD, ddelta_bias
    float* const red = lds + 4 * Q * CH + 2 * CH + 2 * 4 * TH;                              // [wave][token][2][NP]
    int64_t* const len = reinterpret_cast<int64_t*>(red + W * Q * 2 * NP);                  // tokens of each row at work
    float(*const bc_all)[Q][2][NP] = reinterpret_cast<float(*)[Q][2][NP]>(len + W);         // [row at work]

    const int Dg = (int)(a.D / a.G);
    const int tiles = (Dg + CW - 1) / CW;                    // waves a group's channels take
    const int per = tiles < W ? tiles : W, units = W / per;  // ... of them in this workgroup; rows side by side in it
    const int blocks = (tiles + per - 1) / per;
    const int tb = blockIdx.y % blocks;
    const int g = blockIdx.y / blocks;
    const int N = a.N, softplus = a.softplus;
    const bool gated = a.z != nullptr, whole = a.whole != 0;

    // the sweeps' view: a lane has states 4 q .. 4 q + 3 of channel c of its wave
    const int unit = wave / per, ct = tb * per + wave % per;
    const bool working = unit < units && ct * CW < Dg;
    const bool live = working && c < Dg - ct * CW;
    const int64_t d = working ? g * Dg + ct * CW + (live ? c : Dg - ct * CW - 1) : 0;
    float(*const bc)[2][NP] = bc_all[unit < units ? unit : 0];
    float A2[4], dA[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int s = q * 4 + j;
        A2[j] = s < N ? a.A[d * N + s] * kLog2e : 0.0f;
        dA[j] = 0.0f;
    }
    // the element-wise view: a thread has channels quad_d .. quad_d + quad_n - 1 of tokens quad_t, quad_t + STEP, ...
    const int slot = threadIdx.x % QUADS * 4, quad_t = threadIdx.x / QUADS;
    const int wave_t = uniform(wave * 64 / QUADS), lane_t = QUADS < 64 ? lane / QUADS : 0;    // quad_t = wave_t + lane_t
    const int quad_unit = slot / CW / per, quad_c = (tb * per + slot / CW % per) * CW + slot % CW;
    const int quad_n = quad_unit >= units || quad_t >= Q ? 0 : Dg - quad_c < 4 ? (Dg - quad_c > 0 ? Dg - quad_c : 0) : 4;
    const int64_t quad_d = (int64_t)g * Dg + quad_c;
    // where a thread's first token lies, from its workgroup's first row and its wave's first token: formed anew for each
    // tile, the registers are worth more than the arithmetic
    auto away = [&](int64_t row, int64_t token) {
        int64_t at = quad_c;
        if constexpr (QUADS == 32) at += lane_t ? token : 0;
        else if constexpr (QUADS < 32) at += (int64_t)lane_t * token;
        if (units > 1) at += (int64_t)quad_unit * row;
        return at;
    };
#pragma unroll
    for (int j = 0; j < 4; ++j) sums[threadIdx.x][j] = sums[TH + threadIdx.x][j] = 0.0f;
    if (quad_t == 0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            param[0][slot + j] = a.bias && j < quad_n ? a.bias[quad_d + j] : 0.0f;
            param[1][slot + j] = a.Dv && j < quad_n ? a.Dv[quad_d + j] : 0.0f;
        }
    }

    const int64_t groups = (a.B + units - 1) / units, items = groups * a.chunks;
    for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const int64_t chunk = item / groups;
        const int64_t row0 = (item - chunk * groups) * units;
        int64_t b, n, t_begin, t_end;
        bool on;
        float carry[4];
        {
            const ScanArgs r = scan_args();
            __syncthreads();
            if ((int)threadIdx.x < units) len[threadIdx.x] = row0 + threadIdx.x < r.B ? row_length(r.lengths, row0 + threadIdx.x, r.L) : 0;
            __syncthreads();
            on = working && row0 + unit < r.B;                  // the same for all lanes of a wave
            b = on ? row0 + unit : r.B - 1;
            n = on ? row_length(r.lengths, b, r.L) : 0;
            t_begin = chunk * r.chunk, t_end = t_begin + r.chunk < r.L ? t_begin + r.chunk : r.L;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int s = q * 4 + j;
                carry[j] = 0.0f;
                if (MODE == 0 && on) {
                    if (r.chunks > 1) carry[j] = r.chunk_state[((chunk * r.B + b) * r.D + d) * NP + s];
                    else if (r.dnew_state && s < N) carry[j] = r.dnew_state[(b * r.D + d) * N + s];
                }
            }
        }
        float sum_dt = 0.0f;
        bool cut = false;

        // what a tile needs from memory; the next tile's is asked for before this one's results are written
        Quad<T> fu[IT] = {}, fd[IT] = {}, fz[IT] = {}, fy[IT] = {};
        T fbc[BE] = {};
        float4 fh = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        uint8_t mark = 0;
        auto fetch = [&](int64_t t0) {
            const ScanArgs r = scan_args();
            const int64_t quad_len = quad_n > 0 ? len[quad_unit] : 0, quad_0 = t0 + wave_t;
            auto from = [&](Quad<T>(&to)[IT], const void* base, int64_t row, int64_t token) {
                const T* const p = (const T*)base + row0 * row + quad_0 * token + (int64_t)g * Dg;
                const int64_t off = away(row, token);
#pragma unroll
                for (int k = 0; k < IT; ++k)
                    load4(to[k], p + k * STEP * token + off, quad_0 + k * STEP + lane_t < quad_len ? quad_n : 0, whole);
            };
            from(fd, r.delta, r.delta_row, r.delta_token);
            from(fy, r.dy, r.dy_row, r.dy_token);
            if (gated) from(fz, r.z, r.z_row, r.z_token);
            if (MODE == 0) from(fu, r.u, r.u_row, r.u_token);
            const int tid = thread_anew();
#pragma unroll
            for (int k = 0; k < BE; ++k) {
                const int e = tid + k * TH;
                if (k * TH < units * Q * 2 * NP) {
                    // (rows of a workgroup's worth of numbers or more: the row is the same for all threads)
                    const int un = TH <= Q * 2 * NP ? k * TH / (Q * 2 * NP) : e / (Q * 2 * NP);
                    const int i = e / (2 * NP) % Q, which = e / NP % 2, s = e % NP;
                    fbc[k] = (T)0.0f;
                    if (un < units && s < N && t0 + i < len[un]) {
                        if (which == 1)
                            fbc[k] = ((const T*)r.Cm + (row0 + un) * r.C_row + g * r.C_group + t0 * r.C_token)[times(i, r.C_token) + s];
                        else if (MODE == 0)
                            fbc[k] = ((const T*)r.Bm + (row0 + un) * r.B_row + g * r.B_group + t0 * r.B_token)[times(i, r.B_token) + s];
                    }
                }
            }
            mark = 0;
            if (r.start && lane < Q && t0 + lane < n) mark = r.start[b * r.start_row + (t0 + lane) * r.start_token];
            if (MODE == 0 && t0 < n)
                fh = *reinterpret_cast<const float4*>(r.segments + ((b * ((r.L + Q - 1) / Q) + t0 / Q) * r.D + d) * NP + q * 4);
        };
        const int64_t t_last = (t_end - 1) / Q * Q;
        fetch(t_last);
        for (int64_t t0 = t_last; t0 >= t_begin; t0 -= Q) {
            const int here = t0 >= n ? 0 : n - t0 < Q ? (int)(n - t0) : Q;   // tokens of this wave's row in the tile
            const unsigned marks = (unsigned)__ballot(mark != 0);
            const float h0[4] = {fh.x, fh.y, fh.z, fh.w};
            Quad<T> gu[IT], gd[IT], gz[IT], gy[IT];      // this tile's elements
            const int64_t quad_len = quad_n > 0 ? len[quad_unit] : 0;
            // param and, from the tile before, the elements, bc and red: everything is read by now
            __syncthreads();
            const int tid = thread_anew();
#pragma unroll
            for (int k = 0; k < BE; ++k) {
                const int e = tid + k * TH;
                if (e < units * Q * 2 * NP) (&bc_all[0][0][0][0])[e] = (float)fbc[k];
            }
#pragma unroll
            for (int k = 0; k < IT; ++k) {
                const int i = quad_t + k * STEP;
                const int count = t0 + i < quad_len ? quad_n : 0;
                gu[k] = fu[k], gd[k] = fd[k], gz[k] = fz[k], gy[k] = fy[k];
                float w[4], x[4], o[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    // tokens behind the row's last and lanes without a channel: width 0 (decay 1), and they add nothing
                    w[j] = j < count ? step_width<T>(gd[k].at(j) + param[0][slot + j], softplus) : 0.0f;
                    x[j] = w[j] * gu[k].at(j);
                    const float zz = gz[k].at(j);
                    o[j] = gated ? gy[k].at(j) * (zz * sigmoid_f<T>(zz)) : gy[k].at(j);
                }
                if (i < Q) {
                    store<float, 4>(&width[i][slot], w);
                    if (MODE == 0) store<float, 4>(&wu[i][slot], x);
                    store<float, 4>(&gate[i][slot], o);
                }
            }
            __syncthreads();
            const int me = wave * CW + c, mine = lane_place<SB, 0, S>(lane);
            if (MODE == 1) {
                if (t0 > t_begin) fetch(t0 - Q);
#pragma unroll
                for (int i = Q - 1; i >= 0; --i) {
                    const float w = width[i][me], o = gate[i][me];
                    sum_dt += w;
#pragma unroll
                    for (int j = 0; j < 4; ++j) carry[j] = fmaf(o, bc[i][1][q * 4 + j], carry[j]) * exp2_hw(w * A2[j]);
                    if (marks >> i & 1) {
                        cut = true;
#pragma unroll
                        for (int j = 0; j < 4; ++j) carry[j] = 0.0f;
                    }
                }
                continue;
            }
            // HQ tokens from `first` on, forwards and backwards.  PLAIN: no token of the tile opens an episode or lies behind
            // the row's last.
            auto sweep = [&](auto plain, int first) {
                constexpr bool PLAIN = decltype(plain)::value;
                float hist[HQ + 1][4];
#pragma unroll
                for (int j = 0; j < 4; ++j) hist[0][j] = h0[j];
                for (int i = 0; i < first; ++i) {       // up to the first of them, from the state kept before the tile
                    const float w = width[i][me], x = wu[i][me];
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        float before = hist[0][j];
                        if (!PLAIN && (marks >> i & 1)) before = 0.0f;
                        hist[0][j] = fmaf(exp2_hw(w * A2[j]), before, x * bc[i][0][q * 4 + j]);
                    }
                }
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    float part[S];
#pragma unroll
                    for (int o = 0; o < S; ++o) {
                        const int m = k * S + o, i = first + m;
                        const float w = width[i][me], x = wu[i][me];
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            float before = hist[m][j];
                            if (!PLAIN && (marks >> i & 1)) before = 0.0f;
                            hist[m + 1][j] = fmaf(exp2_hw(w * A2[j]), before, x * bc[i][0][q * 4 + j]);
                            const float C = bc[i][1][q * 4 + j];
                            part[o] = j == 0 ? hist[m + 1][j] * C : fmaf(hist[m + 1][j], C, part[o]);
                        }
                    }
                    lane_scatter_sum<SB, 0, S>(part);      // a channel's lanes get the sums of S tokens, one each
                    sum_y[first + k * S + mine][me] = part[0];
                    __builtin_amdgcn_sched_barrier(0);
                }
                float p1[S], p2[S], bcsum[GV], s1[KT], s2[KT];
#pragma unroll
                for (int m = HQ - 1; m >= 0; --m) {
                    const int i = first + m;
                    const float w = width[i][me], x = wu[i][me], o = gate[i][me];
                    float x1, x2;
                    float* const to = bcsum + (m % GT) * 8;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float dh = fmaf(o, bc[i][1][q * 4 + j], carry[j]);
                        to[j] = dh * x;
                        to[4 + j] = o * hist[m + 1][j];
                        const float B = bc[i][0][q * 4 + j];
                        x1 = j == 0 ? dh * B : fmaf(dh, B, x1);
                        carry[j] = dh * exp2_hw(w * A2[j]);
                        float through = carry[j] * hist[m][j];
                        if (!PLAIN && (marks >> i & 1)) carry[j] = through = 0.0f;   // (hist may be anything here)
                        if (!PLAIN && TAIL && i >= here) through = 0.0f;
                        x2 = j == 0 ? through * A2[j] : fmaf(through, A2[j], x2);
                        dA[j] = fmaf(through, w, dA[j]);
                    }
                    p1[m % S] = x1, p2[m % S] = x2;
                    if (m % S == 0) {
                        lane_scatter_sum<SB, 0, S>(p1);
                        lane_scatter_sum<SB, 0, S>(p2);
                        s1[m / S] = p1[0], s2[m / S] = p2[0];
                    }
                    if (m % GT == 0) {
                        lane_scatter_sum<6, SB, GV>(bcsum);
                        // value v of GV is token i + v / 8, dB (0) or dC (1), state 4 q + v % 4
                        const int v = lane_place<6, SB, GV>(lane);
                        float* const at = red + ((wave * Q + i + v / 8) * 2 + v / 4 % 2) * NP + q * 4 + v % 4;
#pragma unroll
                        for (int r = 0; r < GR; ++r) at[r] = bcsum[r];
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                // these tokens' width u and g have been read for the last time, and by this wave alone
#pragma unroll
                for (int k = 0; k < KT; ++k) wu[first + k * S + mine][me] = s1[k], gate[first + k * S + mine][me] = s2[k];
            };
            if (here == 0) {
                for (int e = lane; e < Q * 2 * NP; e += 64) red[wave * Q * 2 * NP + e] = 0.0f;
            } else {
#pragma unroll 1
                for (int first = Q - HQ; first >= 0; first -= HQ) {
                    if (TAIL && HQ < Q && here <= first) {
                        for (int e = lane; e < HQ * 2 * NP; e += 64) red[(wave * Q + first) * 2 * NP + e] = 0.0f;
                        continue;
                    }
                    if (kPlainToo && marks == 0 && (!TAIL || here == Q)) sweep(std::true_type{}, first);
                    else sweep(std::false_type{}, first);
                }
            }
            __syncthreads();
            if (t0 > t_begin) fetch(t0 - Q);
            const ScanArgs r = scan_args();
            if (quad_n > 0 && row0 + quad_unit < r.B) {
                const int64_t quad_len = len[quad_unit], quad_0 = t0 + wave_t;
                float dD[4], dbias[4];
                load<float, 4>(sums[threadIdx.x], dD);
                load<float, 4>(sums[TH + threadIdx.x], dbias);
#pragma unroll
                for (int k = 0; k < IT; ++k) {
                    const int i = quad_t + k * STEP;
                    const int64_t t = t0 + i;
                    if (t < t_end) {
                        const bool in = t < quad_len;
                        float w[4], s1[4], s2[4], sy[4], ou[4], od[4], oz[4];
                        load<float, 4>(&width[i][slot], w);
                        load<float, 4>(&wu[i][slot], s1);
                        load<float, 4>(&gate[i][slot], s2);
                        load<float, 4>(&sum_y[i][slot], sy);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const float skip = param[1][slot + j], uu = gu[k].at(j), out = gy[k].at(j), zz = gz[k].at(j);
                            const float sg = sigmoid_f<T>(zz), gg = gated ? out * (zz * sg) : out;
                            ou[j] = in ? fmaf(s1[j], w[j], gg * skip) : 0.0f;
                            // sum of through A = sum of through A2, times ln 2
                            od[j] = in ? fmaf(s1[j], uu, s2[j] * kLn2) * step_slope<T>(gd[k].at(j) + param[0][slot + j], softplus) : 0.0f;
                            oz[j] = in ? out * fmaf(skip, uu, sy[j]) * (sg * fmaf(zz, 1.0f - sg, 1.0f)) : 0.0f;
                            dbias[j] += od[j];
                            if (in) dD[j] = fmaf(gg, uu, dD[j]);
                        }
                        auto to = [&](void* base, int64_t row, int64_t token, const float(&v)[4]) {
                            store4((T*)base + row0 * row + (quad_0 + k * STEP) * token + (int64_t)g * Dg + away(row, token), quad_n, whole, v);
                        };
                        to(r.du, r.du_row, r.du_token, ou);
                        to(r.ddelta, r.ddelta_row, r.ddelta_token, od);
                        if (gated) to(r.dz, r.dz_row, r.dz_token, oz);
                    }
                }
                store<float, 4>(sums[threadIdx.x], dD);
                store<float, 4>(sums[TH + threadIdx.x], dbias);
            }
            const int me_again = thread_anew();
            for (int k = 0; k * TH < units * Q * 2 * NP; ++k) {
                const int e = me_again + k * TH;
                const int un = TH <= Q * 2 * NP ? k * TH / (Q * 2 * NP) : e / (Q * 2 * NP);
                const int i = e / (2 * NP) % Q, which = e / NP % 2, s = e % NP;
                if (un < units && row0 + un < r.B && t0 + i < t_end && s < N) {
                    const int64_t br = row0 + un;
                    float sum = 0.0f;
                    for (int w = 0; w < per; ++w) sum += red[((un * per + w) * Q + i) * 2 * NP + which * NP + s];
                    if (TAIL && t0 + i >= len[un]) sum = 0.0f;
                    if (r.bc_partial)
                        (r.bc_partial + (((int64_t)tb * r.B + br) * r.L + t0) * r.G * 2 * NP)[times(i, r.G * 2 * NP) + (g * 2 + which) * NP + s] = sum;
                    else if (which == 0)
                        ((T*)r.dB + br * r.dB_row + t0 * r.dB_token + g * r.dB_group)[times(i, r.dB_token) + s] = (T)sum;
                    else
                        ((T*)r.dC + br * r.dC_row + t0 * r.dC_token + g * r.dC_group)[times(i, r.dC_token) + s] = (T)sum;
                }
            }
        }
        const ScanArgs r = scan_args();
        if (MODE == 1) {
            if (live && on) {
                const int64_t o = ((chunk * r.B + b) * r.D + d) * NP + q * 4;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    r.chunk_state[o + j] = carry[j];
                    r.chunk_decay[o + j] = chunk_log(cut, sum_dt * A2[j]);
                }
            }
        } else if (r.dstate && r.chunks == 1 && live && on) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (q * 4 + j < N) r.dstate[(b * r.D + d) * N + q * 4 + j] = carry[j];
        }
    }
    if (MODE == 1) return;
    // this workgroup's record: dA from the sweeps' lanes; dD and ddelta_bias of the threads that share channels, in order
    const int K = N + 2;
    float* const rec = a.partial + (int64_t)blockIdx.x * units * a.D * K;
    if (live) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (q * 4 + j < N) rec[((int64_t)unit * a.D + d) * K + q * 4 + j] = dA[j];
    }
    __syncthreads();
    if (quad_t == 0 && quad_n > 0) {
        for (int j = 0; j < quad_n; ++j) {
            float x = 0.0f, y = 0.0f;
            for (int i = 0; i < STEP; ++i) x += sums[i * QUADS + threadIdx.x][j], y += sums[TH + i * QUADS + threadIdx.x][j];
            rec[((int64_t)quad_unit * a.D + quad_d + j) * K + N] = x;
            rec[((int64_t)quad_unit * a.D + quad_d + j) * K + N + 1] = y;
        }
    }
}

// dB and dC of groups wider than one workgroup: the workgroups' sums in ascending order, rounded once.
template <class T>
__global__ __launch_bounds__(256) void k_scan_sum_bc(ScanArgs a, int NP, int blocks) {
    const int64_t count = a.B * a.L * a.G * 2 * NP;
    const int64_t i = (a.first + blockIdx.x) * 256 + threadIdx.x;
    if (i >= count) return;
    const int s = (int)(i % NP), which = (int)(i / NP % 2);
    const int64_t g = i / (2 * NP) % a.G, t = i / (2 * NP * a.G) % a.L, b = i / (2 * NP * a.G * a.L);
    if (s >= a.N) return;
    float sum = 0.0f;
    for (int k = 0; k < blocks; ++k) sum += a.bc_partial[k * count + i];
    if (which == 0) ((T*)a.dB + b * a.dB_row + t * a.dB_token + g * a.dB_group)[s] = (T)sum;
    else ((T*)a.dC + b * a.dC_row + t * a.dC_token + g * a.dC_group)[s] = (T)sum;
}

// ----------------------------------------------------------------------------------------------------------------
// One token per row: the states once in, once out, 8 N bytes per channel against some 50 bytes of everything else.  A
// lane holds 4 states, S lanes a channel, so that a wave reads 1 KiB of adjacent states per load; it keeps its channel's
// parameters for all the rows it takes and asks for the next row's states while it works on one.  state and new_state may
// be the same memory: a lane writes only what it alone has read.  65,536 rows x 64 channels x 16 states: 117 to 126 us (575
// MB, 4.6 to 4.9 TB/s); 146 us with parameters fetched for every row and nothing asked for ahead.
// ----------------------------------------------------------------------------------------------------------------
constexpr int kStepThreads = 256;
template <class T, int S>
__global__ __launch_bounds__(kStepThreads) void k_scan_step(ScanArgs a) {
    constexpr int SB = lane_bits<S>();
    // a.lanes threads (a multiple of S) take a row's channels, as many of them as there are or as a workgroup holds
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes, slots = kStepThreads / a.lanes;
    const int64_t d = (int64_t)blockIdx.y * (a.lanes / S) + lane / S;
    const int q = lane % S;
    if (slot >= slots || d >= a.D) return;      // all lanes of a channel or none
    const int g = (int)(d / (a.D / a.G)), count = clamp_count(a.N - q * 4, 4);
    float A2[4];
    Raw<float, 4> rA;
    fetch(rA, a.A + d * a.N + q * 4, count);
#pragma unroll
    for (int j = 0; j < 4; ++j) A2[j] = rA.at(j) * kLog2e;
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dv ? a.Dv[d] : 0.0f;
    Raw<float, 4> rh = {};
    Raw<T, 4> rB = {}, rC = {};
    T ru = (T)0.0f, rd = (T)0.0f, rz = (T)0.0f;
    uint8_t mark = 0;
    auto ask = [&](int64_t b) {
        if (b >= a.B) return;
        fetch(rh, a.state + (b * a.D + d) * a.N + q * 4, count);
        fetch(rB, (const T*)a.Bm + b * a.B_row + g * a.B_group + q * 4, count);
        fetch(rC, (const T*)a.Cm + b * a.C_row + g * a.C_group + q * 4, count);
        ru = ((const T*)a.u)[b * a.u_row + d];
        rd = ((const T*)a.delta)[b * a.delta_row + d];
        if (a.z) rz = ((const T*)a.z)[b * a.z_row + d];
        if (a.start) mark = a.start[b * a.start_row];
    };
    const int64_t step = (int64_t)gridDim.x * slots;
    int64_t b = (int64_t)blockIdx.x * slots + slot;
    ask(b);
    for (; b < a.B; b += step) {
        float h[4], x[4], C[4];
        const float u = (float)ru, z = (float)rz;
        const float dt = step_width<T>((float)rd + bias, a.softplus);
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = mark ? 0.0f : rh.at(j), x[j] = dt * u * rB.at(j), C[j] = rC.at(j);
        ask(b + step);
        float acc = 0.0f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = fmaf(exp2_hw(dt * A2[j]), h[j], x[j]);
            acc = fmaf(h[j], C[j], acc);
        }
        acc = lane_sum<SB>(acc);
        put(a.new_state + (b * a.D + d) * a.N + q * 4, count, h);
        if (q == 0) {
            acc = fmaf(skip, u, acc);
            if (a.z) acc *= z * sigmoid_f<T>(z);
            ((T*)a.y)[b * a.y_row + d] = (T)acc;
        }
    }
}

}  // namespace seq
}  // namespace auv
