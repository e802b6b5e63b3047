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
// Two bounds lie close together: 4 elements of traffic per (token, channel), and per state one exponential, two
// multiplications and two fused multiply-adds on the vector unit.
#pragma once

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
    float *chunk_state, *chunk_decay;   // [chunks, B, D, NP]
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
    float* bc_partial;       // [tile blocks, B, L, G, 2, NP] when a group's channels fill more than one workgroup
};

__device__ __forceinline__ void wave_sync() {
    // LDS traffic of one wave is in order; this keeps the compiler from moving it across
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// delta -> step width, and the width's derivative with respect to delta
__device__ __forceinline__ float step_width(float raw, int softplus) { return softplus ? softplus_f(raw) : raw; }
__device__ __forceinline__ float step_slope(float raw, int softplus) { return softplus ? sigmoid_f(raw) : 1.0f; }

// ----------------------------------------------------------------------------------------------------------------
// Forward.  S lanes per channel, NPL states per lane: 64 / S channels per wave, a wave per (channel tile, group, row,
// chunk of time).  B and C of the next tokens go through LDS once per wave as floats, zero-padded to NP states, which
// takes care of odd counts and strides; every lane of a channel reads them from there at the same address.
//
// MODE 0 computes outputs (from `state`, or from the chunk's entry state when the row is split into chunks).
// MODE 1 starts each chunk from zero and leaves only its end state and its decay, exp(A sum dt) (0 behind a start).
// ----------------------------------------------------------------------------------------------------------------
constexpr int kScanTile = 8;

template <class T, int NPL, int S, int MODE>
__global__ __launch_bounds__(kScanWaves * 64) void k_scan_forward(ScanArgs a) {
    constexpr int NP = NPL * S, CW = 64 / S, TQ = kScanTile;
    __shared__ __align__(16) float tile[kScanWaves][TQ][2][NP];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int q = lane % S, c = lane / S;
    const int64_t Dg = a.D / a.G, tiles = (Dg + CW - 1) / CW;
    int64_t id = (int64_t)blockIdx.x * kScanWaves + wave;
    const int64_t ct = id % tiles;
    id /= tiles;
    const int64_t g = id % a.G;
    id /= a.G;
    const int64_t b = id % a.B, chunk = id / a.B;
    if (chunk >= a.chunks) return;
    const bool live = ct * CW + c < Dg;
    const int64_t d = g * Dg + (live ? ct * CW + c : Dg - 1);
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
    const T* const u = (const T*)a.u + b * a.u_row + d;
    const T* const delta = (const T*)a.delta + b * a.delta_row + d;
    const T* const z = (const T*)a.z + b * a.z_row + d;
    const T* const Bm = (const T*)a.Bm + b * a.B_row + g * a.B_group;
    const T* const Cm = (const T*)a.Cm + b * a.C_row + g * a.C_group;
    T* const y = (T*)a.y + b * a.y_row + d;
    float sum_dt = 0.0f;
    bool cut = false;

    for (int64_t t0 = t_begin; t0 < stop; t0 += TQ) {
        if (MODE == 0 && a.segments && t0 % kSegment == 0 && live) {
            float* const seg = a.segments + ((b * ((a.L + kSegment - 1) / kSegment) + t0 / kSegment) * a.D + d) * NP + q * NPL;
#pragma unroll
            for (int j = 0; j < NPL; j += 4) *reinterpret_cast<float4*>(seg + j) = make_float4(h[j], h[j + 1], h[j + 2], h[j + 3]);
        }
        float uu[TQ], dd[TQ], zz[TQ];
#pragma unroll
        for (int i = 0; i < TQ; ++i) {
            const int64_t t = t0 + i < stop ? t0 + i : stop - 1;
            uu[i] = (float)u[t * a.u_token];
            dd[i] = (float)delta[t * a.delta_token];
            zz[i] = MODE == 0 && a.z ? (float)z[t * a.z_token] : 0.0f;
        }
        bool mark = false;
        if (a.start && lane < TQ && t0 + lane < stop) mark = a.start[b * a.start_row + (t0 + lane) * a.start_token] != 0;
        const unsigned long long marks = __ballot(mark);
        wave_sync();
#pragma unroll
        for (int e0 = 0; e0 < TQ * NP; e0 += 64) {
            const int e = e0 + lane, i = e / NP, s = e % NP;
            if (TQ * NP >= 64 || e < TQ * NP) {
                const bool in = t0 + i < stop && s < a.N;
                tile[wave][i][0][s] = in ? (float)Bm[(t0 + i) * a.B_token + s] : 0.0f;
                if (MODE == 0) tile[wave][i][1][s] = in ? (float)Cm[(t0 + i) * a.C_token + s] : 0.0f;
            }
        }
        wave_sync();
#pragma unroll
        for (int i = 0; i < TQ; ++i) {
            if (t0 + i < stop) {
                if (marks >> i & 1) {
                    cut = true;
#pragma unroll
                    for (int j = 0; j < NPL; ++j) h[j] = 0.0f;
                }
                const float dt = step_width(dd[i] + bias, a.softplus), du = dt * uu[i];
                if (MODE == 1) sum_dt += dt;
                float acc = 0.0f;
#pragma unroll
                for (int j = 0; j < NPL; ++j) {
                    const float e = exp2_hw(dt * A2[j]);
                    h[j] = fmaf(e, h[j], du * tile[wave][i][0][q * NPL + j]);
                    if (MODE == 0) acc = fmaf(h[j], tile[wave][i][1][q * NPL + j], acc);
                }
                if (MODE == 0) {
                    acc = lane_sum<0, (S >= 16 ? 4 : S >= 8 ? 3 : S >= 4 ? 2 : S >= 2 ? 1 : 0)>(acc);
                    acc = fmaf(skip, uu[i], acc);
                    if (a.z) acc *= zz[i] * sigmoid_f(zz[i]);
                    if (live && q == 0) y[(t0 + i) * a.y_token] = (T)acc;
                }
            }
        }
    }
    if (MODE == 1) {
        if (live) {
            const int64_t o = ((chunk * a.B + b) * a.D + d) * NP + q * NPL;
#pragma unroll
            for (int j = 0; j < NPL; ++j) {
                a.chunk_state[o + j] = h[j];
                a.chunk_decay[o + j] = cut ? 0.0f : exp2_hw(sum_dt * A2[j]);
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
        for (int64_t t = t_begin > n ? t_begin : n; t < t_end; ++t) y[t * a.y_token] = (T)0.0f;
}

// Joins the chunks of a row: chunk_state[c] becomes the state the chunk starts from (forwards from `state`) or, going
// backwards, the gradient that reaches the chunk's last state from behind (from the gradient of the states handed on,
// which lands in dstate at the front).  A workgroup takes 64 numbers and splits the chunks over 16 rows of threads.
constexpr int kJoinRows = 16;
struct JoinArgs {
    float *chunk_state, *chunk_decay;
    const float* first;     // [B,D,N] or null
    float* last;            // [B,D,N] or null
    int64_t chunks, count;  // count = B D NP
    int32_t N, NP, reverse;
};
__global__ __launch_bounds__(64 * kJoinRows) void k_scan_join(JoinArgs a) {
    __shared__ float hs[kJoinRows][64], ps[kJoinRows][64];
    const int lane = threadIdx.x & 63, row = threadIdx.x >> 6;
    const int64_t i = (int64_t)blockIdx.x * 64 + lane;
    const bool live = i < a.count;
    const int64_t per = (a.chunks + kJoinRows - 1) / kJoinRows;
    const int64_t c0 = row * per < a.chunks ? row * per : a.chunks, c1 = c0 + per < a.chunks ? c0 + per : a.chunks;
    auto at = [&](int64_t c) { return (a.reverse ? a.chunks - 1 - c : c) * a.count + i; };
    // a decay of exactly 0 cuts: whatever came before (also an infinity) has no part in what follows
    auto join = [](float p, float x, float s) { return p == 0.0f ? s : fmaf(p, x, s); };
    float h = 0.0f, p = 1.0f;
    if (live) {
#pragma unroll 4
        for (int64_t c = c0; c < c1; ++c) {
            const float s = a.chunk_state[at(c)], q = a.chunk_decay[at(c)];
            h = join(q, h, s);
            p *= q;
        }
    }
    hs[row][lane] = h;
    ps[row][lane] = p;
    __syncthreads();
    if (!live) return;
    const int64_t bd = i / a.NP;
    const int s = (int)(i - bd * a.NP);
    float x = a.first && s < a.N ? a.first[bd * a.N + s] : 0.0f;
    for (int r = 0; r < row; ++r) x = join(ps[r][lane], x, hs[r][lane]);
#pragma unroll 4
    for (int64_t c = c0; c < c1; ++c) {
        const float e = a.chunk_state[at(c)], q = a.chunk_decay[at(c)];
        a.chunk_state[at(c)] = x;
        x = join(q, x, e);
    }
    if (a.last && s < a.N && row == kJoinRows - 1) a.last[bd * a.N + s] = x;
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
template <int S>
constexpr int scan_back_waves() { return S <= 4 ? 8 : 4; }
template <int S>
constexpr size_t scan_back_lds() {
    constexpr int NP = 4 * S, CW = 64 / S, W = scan_back_waves<S>();
    // per wave: dt, u, g, - of 16 tokens x CW channels; B and C of 16 tokens; sums of 16 tokens
    return (size_t)W * 4 * (16 * CW * 4 + 16 * 2 * NP + 16 * 2 * NP);
}

// MODE 0: gradients.  MODE 1: from zero at the end of each chunk, only the carry at its front and its decay.
template <class T, int S, int MODE>
__global__ __launch_bounds__(scan_back_waves<S>() * 64) void k_scan_backward(ScanArgs a) {
    constexpr int NP = 4 * S, CW = 64 / S, W = scan_back_waves<S>(), Q = kSegment, KT = Q / S;
    constexpr int SB = S >= 16 ? 4 : S >= 8 ? 3 : S >= 4 ? 2 : S >= 2 ? 1 : 0;
    static_assert(S <= Q, "every lane of a channel has a token of its own to finish");
    extern __shared__ __align__(16) float lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int q = lane % S, c = lane / S;
    float(*const elem)[CW][4] = reinterpret_cast<float(*)[CW][4]>(lds + (size_t)wave * Q * CW * 4);
    float(*const bc)[2][NP] = reinterpret_cast<float(*)[2][NP]>(lds + (size_t)W * Q * CW * 4 + (size_t)wave * Q * 2 * NP);
    float* const red = lds + (size_t)W * (Q * CW * 4 + Q * 2 * NP);   // [wave][token][2][NP]

    const int64_t Dg = a.D / a.G;
    const int tiles = (int)((Dg + CW - 1) / CW);             // waves a group's channels take
    const int per = tiles < W ? tiles : W, units = W / per;  // ... of them in this workgroup; rows side by side in it
    const int blocks = (tiles + per - 1) / per;
    const int unit = wave / per, ct = (int)(blockIdx.y % blocks) * per + wave % per;
    const int64_t g = blockIdx.y / blocks;
    const int tb = blockIdx.y % blocks;
    const bool working = unit < units;
    const bool live = working && ct * CW + c < Dg;
    const int64_t d = g * Dg + (live ? ct * CW + c : Dg - 1);

    float A[4], A2[4], dA[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int s = q * 4 + j;
        A[j] = s < a.N ? a.A[d * a.N + s] : 0.0f;
        A2[j] = A[j] * kLog2e;
        dA[j] = 0.0f;
    }
    const float bias = a.bias ? a.bias[d] : 0.0f, skip = a.Dv ? a.Dv[d] : 0.0f;
    float dD = 0.0f, dbias = 0.0f;

    const int64_t groups = (a.B + units - 1) / units;
    for (int64_t item = blockIdx.x; item < groups * a.chunks; item += gridDim.x) {
        const int64_t chunk = item / groups;
        const int64_t row = (item % groups) * units + unit;
        const bool on = working && row < a.B;                  // the same for all lanes of a wave
        const int64_t b = row < a.B ? row : a.B - 1;
        const int64_t n = on ? row_length(a.lengths, b, a.L) : 0;
        const int64_t t_begin = chunk * a.chunk, t_end = t_begin + a.chunk < a.L ? t_begin + a.chunk : a.L;
        const T* const u = (const T*)a.u + b * a.u_row + d;
        const T* const delta = (const T*)a.delta + b * a.delta_row + d;
        const T* const z = (const T*)a.z + b * a.z_row + d;
        const T* const dy = (const T*)a.dy + b * a.dy_row + d;
        const T* const Bm = (const T*)a.Bm + b * a.B_row + g * a.B_group;
        const T* const Cm = (const T*)a.Cm + b * a.C_row + g * a.C_group;
        float carry[4];
        float sum_dt = 0.0f;
        bool cut = false;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int s = q * 4 + j;
            carry[j] = 0.0f;
            if (MODE == 0 && on) {
                if (a.chunks > 1) carry[j] = a.chunk_state[((chunk * a.B + b) * a.D + d) * NP + s];
                else if (a.dnew_state && s < a.N) carry[j] = a.dnew_state[(b * a.D + d) * a.N + s];
            }
        }
        for (int64_t t0 = (t_end - 1) / Q * Q; t0 >= t_begin; t0 -= Q) {
            const int here = t0 >= n ? 0 : n - t0 < Q ? (int)(n - t0) : Q;   // tokens of this row in the tile
            bool mark = false;
            if (a.start && lane < here) mark = a.start[b * a.start_row + (t0 + lane) * a.start_token] != 0;
            const unsigned long long marks = __ballot(mark);
            // element-wise part: lane q of a channel takes every S-th token
            float out[KT], zz[KT], slope[KT], uu[KT], gg[KT];
            wave_sync();
#pragma unroll
            for (int k = 0; k < KT; ++k) {
                const int i = k * S + q;
                const int64_t t = i < here ? t0 + i : n > 0 ? n - 1 : 0;
                const float raw = (float)delta[t * a.delta_token] + bias;
                const float dt = step_width(raw, a.softplus);
                out[k] = (float)dy[t * a.dy_token];
                zz[k] = a.z ? (float)z[t * a.z_token] : 0.0f;
                slope[k] = step_slope(raw, a.softplus);
                uu[k] = MODE == 0 ? (float)u[t * a.u_token] : 0.0f;
                gg[k] = a.z ? out[k] * (zz[k] * sigmoid_f(zz[k])) : out[k];
                *reinterpret_cast<float4*>(&elem[i][c][0]) = make_float4(dt, uu[k], gg[k], dt * uu[k]);
            }
            for (int e = lane; e < Q * NP; e += 64) {
                const int i = e / NP, s = e % NP;
                const bool in = i < here && s < a.N;
                bc[i][0][s] = in && MODE == 0 ? (float)Bm[(t0 + i) * a.B_token + s] : 0.0f;
                bc[i][1][s] = in ? (float)Cm[(t0 + i) * a.C_token + s] : 0.0f;
            }
            wave_sync();
            float s1[KT], s2[KT], yy[KT];
            if (MODE == 1) {
#pragma unroll
                for (int i = Q - 1; i >= 0; --i) {
                    if (i < here) {
                        const float4 el = *reinterpret_cast<const float4*>(&elem[i][c][0]);
                        sum_dt += el.x;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            carry[j] = fmaf(el.z, bc[i][1][q * 4 + j], carry[j]) * exp2_hw(el.x * A2[j]);
                        if (marks >> i & 1) {
                            cut = true;
#pragma unroll
                            for (int j = 0; j < 4; ++j) carry[j] = 0.0f;
                        }
                    }
                }
                continue;
            }
            // the states of the tile's tokens, from the one kept before it
            float hist[Q + 1][4];
            if (here > 0) {
                const float4 h0 = *reinterpret_cast<const float4*>(
                    a.segments + ((b * ((a.L + Q - 1) / Q) + t0 / Q) * a.D + d) * NP + q * 4);
                hist[0][0] = h0.x, hist[0][1] = h0.y, hist[0][2] = h0.z, hist[0][3] = h0.w;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) hist[0][j] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < Q; ++i) {
                if (i < here) {
                    const float4 el = *reinterpret_cast<const float4*>(&elem[i][c][0]);
                    const bool fresh = marks >> i & 1;
                    float acc = 0.0f;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float before = fresh ? 0.0f : hist[i][j];
                        hist[i + 1][j] = fmaf(exp2_hw(el.x * A2[j]), before, el.w * bc[i][0][q * 4 + j]);
                        acc = fmaf(hist[i + 1][j], bc[i][1][q * 4 + j], acc);
                    }
                    acc = lane_sum<0, SB>(acc);
                    if (i % S == q) yy[i / S] = acc;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) hist[i + 1][j] = hist[i][j];
                    if (i % S == q) yy[i / S] = 0.0f;
                }
            }
#pragma unroll
            for (int i = Q - 1; i >= 0; --i) {
                float db[4], dc[4];
                float p1 = 0.0f, p2 = 0.0f;
                if (i < here) {
                    const float4 el = *reinterpret_cast<const float4*>(&elem[i][c][0]);
                    const bool fresh = marks >> i & 1;
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float dh = fmaf(el.z, bc[i][1][q * 4 + j], carry[j]);
                        dc[j] = el.z * hist[i + 1][j];
                        db[j] = dh * el.w;
                        p1 = fmaf(dh, bc[i][0][q * 4 + j], p1);
                        carry[j] = fresh ? 0.0f : dh * exp2_hw(el.x * A2[j]);
                        const float through = fresh ? 0.0f : carry[j] * hist[i][j];
                        p2 = fmaf(through, A[j], p2);
                        dA[j] = fmaf(through, el.x, dA[j]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j) db[j] = dc[j] = 0.0f;
                }
                p1 = lane_sum<0, SB>(p1);
                p2 = lane_sum<0, SB>(p2);
                if (i % S == q) s1[i / S] = p1, s2[i / S] = p2;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    db[j] = lane_sum<SB, 6>(live ? db[j] : 0.0f);
                    dc[j] = lane_sum<SB, 6>(live ? dc[j] : 0.0f);
                }
                if (c == 0) {
                    float* const to = red + ((size_t)(wave * Q + i) * 2) * NP + q * 4;
                    *reinterpret_cast<float4*>(to) = make_float4(db[0], db[1], db[2], db[3]);
                    *reinterpret_cast<float4*>(to + NP) = make_float4(dc[0], dc[1], dc[2], dc[3]);
                }
            }
            if (live && on) {
#pragma unroll
                for (int k = 0; k < KT; ++k) {
                    const int i = k * S + q;
                    const int64_t t = t0 + i;
                    if (t < t_end) {
                        const bool in = i < here;
                        const float dt = elem[i][c][0];
                        const float draw = in ? fmaf(s1[k], uu[k], s2[k]) * slope[k] : 0.0f;
                        const float gu = in ? fmaf(s1[k], dt, gg[k] * skip) : 0.0f;
                        ((T*)a.du + b * a.du_row + d)[t * a.du_token] = (T)gu;
                        ((T*)a.ddelta + b * a.ddelta_row + d)[t * a.ddelta_token] = (T)draw;
                        if (a.z) {
                            const float sg = sigmoid_f(zz[k]);
                            const float gz = in ? out[k] * fmaf(skip, uu[k], yy[k]) * (sg * fmaf(zz[k], 1.0f - sg, 1.0f)) : 0.0f;
                            ((T*)a.dz + b * a.dz_row + d)[t * a.dz_token] = (T)gz;
                        }
                        dbias += draw;
                        if (in) dD = fmaf(gg[k], uu[k], dD);
                    }
                }
            }
            __syncthreads();
            for (int e = threadIdx.x; e < units * Q * 2 * NP; e += W * 64) {
                const int un = e / (Q * 2 * NP), i = e / (2 * NP) % Q, which = e / NP % 2, s = e % NP;
                const int64_t br = (item % groups) * units + un, t = t0 + i;
                if (br < a.B && t < t_end && s < a.N) {
                    float sum = 0.0f;
                    for (int w = 0; w < per; ++w) sum += red[((size_t)((un * per + w) * Q + i) * 2 + which) * NP + s];
                    if (a.bc_partial)
                        a.bc_partial[((((int64_t)tb * a.B + br) * a.L + t) * a.G + g) * 2 * NP + which * NP + s] = sum;
                    else if (which == 0)
                        ((T*)a.dB + br * a.dB_row + t * a.dB_token + g * a.dB_group)[s] = (T)sum;
                    else
                        ((T*)a.dC + br * a.dC_row + t * a.dC_token + g * a.dC_group)[s] = (T)sum;
                }
            }
            __syncthreads();
        }
        if (MODE == 1) {
            if (live && on) {
                const int64_t o = ((chunk * a.B + b) * a.D + d) * NP + q * 4;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    a.chunk_state[o + j] = carry[j];
                    a.chunk_decay[o + j] = cut ? 0.0f : exp2_hw(sum_dt * A2[j]);
                }
            }
        } else if (a.dstate && a.chunks == 1 && live && on) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (q * 4 + j < a.N) a.dstate[(b * a.D + d) * a.N + q * 4 + j] = carry[j];
        }
    }
    if (MODE == 1) return;
    if (working) {
        const int64_t K = a.N + 2;
        // the lanes of a channel finished different tokens: their dD and dbias add up
        dD = lane_sum<0, SB>(dD);
        dbias = lane_sum<0, SB>(dbias);
        float* const rec = a.partial + (((int64_t)blockIdx.x * units + unit) * a.D + d) * K;
        if (live) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (q * 4 + j < a.N) rec[q * 4 + j] = dA[j];
            if (q == 0) {
                rec[a.N] = dD;
                rec[a.N + 1] = dbias;
            }
        }
    }
}

// dB and dC of groups wider than one workgroup: the workgroups' sums in ascending order, rounded once.
template <class T>
__global__ __launch_bounds__(256) void k_scan_sum_bc(ScanArgs a, int NP, int blocks) {
    const int64_t count = a.B * a.L * a.G * 2 * NP;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
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
// lane holds 4 states, S lanes a channel, so that a wave reads 1 KiB of adjacent states per load.  state and new_state
// may be the same memory: a lane writes only what it alone has read.
// ----------------------------------------------------------------------------------------------------------------
template <class T, int S, bool WHOLE>   // WHOLE: N = 4 S and everything a lane loads in fours is aligned for it
__global__ __launch_bounds__(256) void k_scan_step(ScanArgs a) {
    constexpr int SB = S >= 16 ? 4 : S >= 8 ? 3 : S >= 4 ? 2 : S >= 2 ? 1 : 0;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / S;   // (row, channel)
    const int q = threadIdx.x % S;
    const bool live = i < a.B * a.D;
    const int64_t b = live ? i / a.D : 0, d = live ? i - b * a.D : 0;
    const int64_t g = d / (a.D / a.G);
    float h[4], A[4], Bv[4], Cv[4];
    const T* const Bm = (const T*)a.Bm + b * a.B_row + g * a.B_group + q * 4;
    const T* const Cm = (const T*)a.Cm + b * a.C_row + g * a.C_group + q * 4;
    const int64_t o = (b * a.D + d) * a.N + q * 4;
    if (WHOLE) {
        load<float, 4>(a.state + o, h);
        load<float, 4>(a.A + d * a.N + q * 4, A);
        load<T, 4>(Bm, Bv);
        load<T, 4>(Cm, Cv);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const bool in = q * 4 + j < a.N;
            h[j] = in ? a.state[o + j] : 0.0f;
            A[j] = in ? a.A[d * a.N + q * 4 + j] : 0.0f;
            Bv[j] = in ? (float)Bm[j] : 0.0f;
            Cv[j] = in ? (float)Cm[j] : 0.0f;
        }
    }
    if (a.start && a.start[b * a.start_row]) {
#pragma unroll
        for (int j = 0; j < 4; ++j) h[j] = 0.0f;
    }
    const float u = (float)((const T*)a.u)[b * a.u_row + d];
    const float dt = step_width((float)((const T*)a.delta)[b * a.delta_row + d] + (a.bias ? a.bias[d] : 0.0f), a.softplus);
    float acc = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        h[j] = fmaf(exp2_hw(dt * (A[j] * kLog2e)), h[j], dt * u * Bv[j]);
        acc = fmaf(h[j], Cv[j], acc);
    }
    acc = lane_sum<0, SB>(acc);
    if (!live) return;
    if (WHOLE) store<float, 4>(a.new_state + o, h);
    else
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (q * 4 + j < a.N) a.new_state[o + j] = h[j];
    if (q == 0) {
        acc = fmaf(a.Dv ? a.Dv[d] : 0.0f, u, acc);
        if (a.z) {
            const float z = (float)((const T*)a.z)[b * a.z_row + d];
            acc *= z * sigmoid_f(z);
        }
        ((T*)a.y)[b * a.y_row + d] = (T)acc;
    }
}

}  // namespace seq
}  // namespace auv
