// The norms round a block, with its gate, its scale and the residual sum between them, in one pass over the rows:
//
//   n  = y rsqrt(mean(y^2) + eps) post_weight          (post_weight absent: n = y)
//   x' = x + scale act(gate) n                         (scale, gate absent: 1; act: none, SiLU, sigmoid)
//   h  = x' rsqrt(mean(x'^2) + eps) pre_weight         (the next block's input; pre_weight absent: not formed)
//
// y absent: only h = x rsqrt(mean(x^2) + eps) pre_weight, the norm before the first block.
//
// Bound by memory: every element of x, y and gate is read once and of x' and h written once, against some 12
// operations.  A row stays in registers between its two sums: TPR lanes share it, 8 elements each, so rows of up to
// 128, 512, 2,048 and 8,192 channels take 16, 64, 256 and 1,024 lanes.
#pragma once

#include "auv_seq.hpp"

namespace auv {
namespace seq {

struct NormArgs {
    int64_t B, L, D;
    const void *x, *y, *gate;
    int64_t x_row, x_token, y_row, y_token, gate_row, gate_token;
    const float *post_weight, *pre_weight, *scale;
    float eps;
    int32_t act;             // AUV_GATE_*
    void *x_out, *h_out;     // [B, L, D] at x's and h's strides
    int64_t x_out_row, x_out_token, h_row, h_token;
    // backward
    const void *gx, *gh;     // gradients of x' (null: 0) and h (null: 0)
    int64_t gx_row, gx_token, gh_row, gh_token;
    void *dx, *dy, *dgate;
    int64_t dx_row, dx_token, dy_row, dy_token, dgate_row, dgate_token;
    float* partial;          // [gridDim.x, D, 3]: post_weight, pre_weight, scale
};

constexpr int kNormLane = 8;   // elements of a row per lane
template <int TPR>
constexpr int norm_threads() { return TPR < 256 ? 256 : TPR; }

// The row's sum, in every lane that shares the row.  `buf`: one number per wave of the workgroup.  One barrier: the caller
// hands in another buffer for the next sum, and comes back to this one only behind a barrier in between.
template <int TPR, int NSUM>
__device__ __forceinline__ void row_sum(float (&v)[NSUM], float (*buf)[NSUM]) {
#pragma unroll
    for (int k = 0; k < NSUM; ++k) v[k] = lane_sum<(TPR >= 64 ? 6 : 4)>(v[k]);
    if constexpr (TPR > 64) {
        constexpr int W = TPR / 64;
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0)
#pragma unroll
            for (int k = 0; k < NSUM; ++k) buf[wave][k] = v[k];
        __syncthreads();
#pragma unroll
        for (int k = 0; k < NSUM; ++k) v[k] = 0.0f;
        for (int w = 0; w < W; ++w)
#pragma unroll
            for (int k = 0; k < NSUM; ++k) v[k] += buf[w][k];
    }
}

__device__ __forceinline__ float gate_value(float g, int act) {
    return act == 0 ? g : act == 1 ? g * sigmoid_f(g) : sigmoid_f(g);
}
__device__ __forceinline__ float gate_slope(float g, int act) {
    if (act == 0) return 1.0f;
    const float s = sigmoid_f(g);
    return act == 1 ? s * fmaf(g, 1.0f - s, 1.0f) : s * (1.0f - s);
}

template <class TR, class T, int V, int TPR>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_forward(NormArgs a) {
    constexpr int TH = norm_threads<TPR>(), ROWS = TH / TPR, K = kNormLane / V;
    __shared__ float buf[2][TH / 64][1];
    const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const int64_t rows = a.B * a.L, row = (int64_t)blockIdx.x * ROWS + slot;
    const bool on = row < rows;
    const int64_t b = on ? row / a.L : 0, l = on ? row - b * a.L : 0;
    const float inv = 1.0f / (float)a.D;
    float r[K][V], y[K][V];
    float sum[1] = {0.0f};
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int64_t d = ((int64_t)k * TPR + lane) * V;
#pragma unroll
        for (int v = 0; v < V; ++v) r[k][v] = y[k][v] = 0.0f;
        if (on && d < a.D) {
            load<TR, V>((const TR*)a.x + b * a.x_row + l * a.x_token + d, r[k]);
            if (a.y) {
                load<T, V>((const T*)a.y + b * a.y_row + l * a.y_token + d, y[k]);
#pragma unroll
                for (int v = 0; v < V; ++v) sum[0] = fmaf(y[k][v], y[k][v], sum[0]);
            }
        }
    }
    if (a.y) {
        float r1 = 1.0f;
        if (a.post_weight) {
            row_sum<TPR, 1>(sum, buf[0]);
            r1 = __builtin_amdgcn_rsqf(fmaf(sum[0], inv, a.eps));
        }
        sum[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t d = ((int64_t)k * TPR + lane) * V;
            if (on && d < a.D) {
                float m[V];
#pragma unroll
                for (int v = 0; v < V; ++v) m[v] = a.scale ? a.scale[d + v] : 1.0f;
                if (a.gate) {
                    float g[V];
                    load<T, V>((const T*)a.gate + b * a.gate_row + l * a.gate_token + d, g);
#pragma unroll
                    for (int v = 0; v < V; ++v) m[v] *= gate_value(g[v], a.act);
                }
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    const float n = a.post_weight ? y[k][v] * r1 * a.post_weight[d + v] : y[k][v];
                    r[k][v] = fmaf(m[v], n, r[k][v]);
                }
                if (a.x_out) store<TR, V>((TR*)a.x_out + b * a.x_out_row + l * a.x_out_token + d, r[k]);
            }
        }
    }
    if (!a.h_out) return;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) sum[0] = fmaf(r[k][v], r[k][v], sum[0]);
    row_sum<TPR, 1>(sum, buf[1]);
    const float r2 = __builtin_amdgcn_rsqf(fmaf(sum[0], inv, a.eps));
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int64_t d = ((int64_t)k * TPR + lane) * V;
        if (on && d < a.D) {
            float h[V];
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = r[k][v] * r2 * a.pre_weight[d + v];
            store<T, V>((T*)a.h_out + b * a.h_row + l * a.h_token + d, h);
        }
    }
}

// Gradients.  x' is formed again from x, y and gate in 32 bits (its stored form may be rounded), then
//
//   t = gh pre_weight            dr = gx + r2 t - x' r2^3 mean(t x')            dx = dr
//   dn = dr scale act(gate)      s = dn post_weight      dy = r1 s - y r1^3 mean(s y)
//   dgate = dr scale n act'(gate)    dscale += dr act(gate) n    dpost += dn y r1    dpre += gh x' r2
//
// A lane owns the same columns of every row its workgroup works on, so the three sums over rows stay in registers and
// leave as one record per workgroup.
template <class TR, class T, int V, int TPR>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_backward(NormArgs a) {
    constexpr int TH = norm_threads<TPR>(), ROWS = TH / TPR, K = kNormLane / V;
    // by sum and, turn about, by row: whichever sums a call leaves out, a barrier lies between two uses of a buffer
    __shared__ float buf_y[2][TH / 64][1], buf_x[2][TH / 64][2], buf_n[2][TH / 64][1];
    int turn = 0;
    __shared__ float fold[ROWS > 1 ? TH * kNormLane : 1];
    const int lane = threadIdx.x % TPR, slot = threadIdx.x / TPR;
    const int64_t rows = a.B * a.L;
    const float inv = 1.0f / (float)a.D;
    float w1[K][V], w2[K][V], sc[K][V], d1[K][V], d2[K][V], ds[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int64_t d = ((int64_t)k * TPR + lane) * V;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const bool in = d < a.D;
            w1[k][v] = in && a.post_weight ? a.post_weight[d + v] : 1.0f;
            w2[k][v] = in && a.pre_weight ? a.pre_weight[d + v] : 0.0f;
            sc[k][v] = in && a.scale ? a.scale[d + v] : 1.0f;
            d1[k][v] = d2[k][v] = ds[k][v] = 0.0f;
        }
    }
    for (int64_t row0 = (int64_t)blockIdx.x * ROWS; row0 < rows; row0 += (int64_t)gridDim.x * ROWS, turn ^= 1) {
        const int64_t row = row0 + slot;
        const bool on = row < rows;
        const int64_t b = on ? row / a.L : 0, l = on ? row - b * a.L : 0;
        float r[K][V], y[K][V], gt[K][V], dr[K][V], t[K][V];
        float s1[1] = {0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t d = ((int64_t)k * TPR + lane) * V;
#pragma unroll
            for (int v = 0; v < V; ++v) r[k][v] = y[k][v] = dr[k][v] = t[k][v] = 0.0f, gt[k][v] = 1.0f;
            if (on && d < a.D) {
                load<TR, V>((const TR*)a.x + b * a.x_row + l * a.x_token + d, r[k]);
                if (a.y) load<T, V>((const T*)a.y + b * a.y_row + l * a.y_token + d, y[k]);
                if (a.gate) load<T, V>((const T*)a.gate + b * a.gate_row + l * a.gate_token + d, gt[k]);
                if (a.gx) load<TR, V>((const TR*)a.gx + b * a.gx_row + l * a.gx_token + d, dr[k]);
                if (a.gh) load<T, V>((const T*)a.gh + b * a.gh_row + l * a.gh_token + d, t[k]);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) s1[0] = fmaf(y[k][v], y[k][v], s1[0]);
        }
        float r1 = 1.0f;
        if (a.post_weight) {
            row_sum<TPR, 1>(s1, buf_y[turn]);
            r1 = __builtin_amdgcn_rsqf(fmaf(s1[0], inv, a.eps));
        }
        float s2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float m = sc[k][v] * (a.gate ? gate_value(gt[k][v], a.act) : 1.0f);
                r[k][v] = fmaf(m, y[k][v] * r1 * w1[k][v], r[k][v]);
                s2[0] = fmaf(r[k][v], r[k][v], s2[0]);
                s2[1] = fmaf(t[k][v] * w2[k][v], r[k][v], s2[1]);
            }
        float r2 = 0.0f, back = 0.0f;
        if (a.gh) {
            row_sum<TPR, 2>(s2, buf_x[turn]);
            r2 = __builtin_amdgcn_rsqf(fmaf(s2[0], inv, a.eps));
            back = s2[1] * inv * r2 * r2 * r2;
        }
        s1[0] = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t d = ((int64_t)k * TPR + lane) * V;
            float dg[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (a.gh) {
                    d2[k][v] = fmaf(t[k][v], r[k][v] * r2, d2[k][v]);
                    dr[k][v] += fmaf(r2 * w2[k][v], t[k][v], -r[k][v] * back);
                }
                const float n = y[k][v] * r1 * w1[k][v];
                const float act = a.gate ? gate_value(gt[k][v], a.act) : 1.0f;
                ds[k][v] = fmaf(dr[k][v], act * n, ds[k][v]);
                dg[v] = a.gate ? dr[k][v] * sc[k][v] * n * gate_slope(gt[k][v], a.act) : 0.0f;
                t[k][v] = dr[k][v] * sc[k][v] * act;                     // dn
                d1[k][v] = fmaf(t[k][v], y[k][v] * r1, d1[k][v]);
                s1[0] = fmaf(t[k][v] * w1[k][v], y[k][v], s1[0]);
            }
            if (on && d < a.D) {
                if (a.dx) store<TR, V>((TR*)a.dx + b * a.dx_row + l * a.dx_token + d, dr[k]);
                if (a.dgate) store<T, V>((T*)a.dgate + b * a.dgate_row + l * a.dgate_token + d, dg);
            }
        }
        if (!a.dy) continue;
        float through = 0.0f;
        if (a.post_weight) {
            row_sum<TPR, 1>(s1, buf_n[turn]);
            through = s1[0] * inv * r1 * r1 * r1;
        }
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int64_t d = ((int64_t)k * TPR + lane) * V;
            float gy[V];
#pragma unroll
            for (int v = 0; v < V; ++v) gy[v] = fmaf(r1 * w1[k][v], t[k][v], -y[k][v] * through);
            if (on && d < a.D) store<T, V>((T*)a.dy + b * a.dy_row + l * a.dy_token + d, gy);
        }
    }
    if (!a.partial) return;
    auto leave = [&](const float (&v)[K][V], int which) {
        if (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < V; ++i) fold[threadIdx.x * kNormLane + k * V + i] = v[k][i];
            __syncthreads();
        }
        if (slot == 0) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
                const int64_t d = ((int64_t)k * TPR + lane) * V;
                if (d < a.D)
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        float s = ROWS > 1 ? 0.0f : v[k][i];
                        if (ROWS > 1)
                            for (int w = 0; w < ROWS; ++w) s += fold[(w * TPR + lane) * kNormLane + k * V + i];
                        a.partial[((int64_t)blockIdx.x * a.D + d + i) * 3 + which] = s;
                    }
            }
        }
    };
    leave(d1, 0);
    leave(d2, 1);
    leave(ds, 2);
}

}  // namespace seq
}  // namespace auv
