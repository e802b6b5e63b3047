// The norms round a block, with its gate, its scale and the residual sum between them, in one pass over the rows:
//
//   n  = y rsqrt(mean(y^2) + eps) post_weight          (post_weight absent: n = y)
//   x' = x + scale act(gate) n                         (scale, gate absent: 1; act: none, SiLU, sigmoid)
//   h  = x' rsqrt(mean(x'^2) + eps) pre_weight         (the next block's input; pre_weight absent: not formed)
//
// y absent: only h = x rsqrt(mean(x^2) + eps) pre_weight, the norm before the first block.
//
// Bound by memory: every element of x, y and gate is read once and of x' and h written once, against some 12
// operations.  A row stays in registers between its two sums: TPR lanes share it, 8 adjacent elements each (16 bytes of a
// 16-bit type), so rows of up to 32, 64, 128, 256, 512, 2,048 and 8,192 channels take 4, 8, 16, 32, 64, 256 and 1,024
// lanes.
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
template <int TPR>
constexpr int norm_bits() { return TPR >= 64 ? 6 : TPR == 32 ? 5 : TPR == 16 ? 4 : TPR == 8 ? 3 : 2; }

// The row's sum, in every lane that shares the row.  `buf`: one number per wave of the workgroup.  One barrier: the caller
// hands in another buffer for the next sum, and comes back to this one only behind a barrier in between.
template <int TPR, int NSUM>
__device__ __forceinline__ void row_sum(float (&v)[NSUM], float (*buf)[NSUM]) {
#pragma unroll
    for (int k = 0; k < NSUM; ++k) v[k] = lane_sum<norm_bits<TPR>()>(v[k]);
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

template <class T>
__device__ __forceinline__ float gate_value(float g, int act) {
    return act == 0 ? g : act == 1 ? g * sigmoid_f<T>(g) : sigmoid_f<T>(g);
}
template <class TR, class T, int TPR>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_forward(NormArgs a) {
    constexpr int TH = norm_threads<TPR>(), ROWS = TH / TPR, V = kNormLane;
    __shared__ float buf[2][TH / 64][1];
    const int d = threadIdx.x % TPR * V, slot = threadIdx.x / TPR;
    const int64_t rows = a.B * a.L, row = (int64_t)blockIdx.x * ROWS + slot;
    const int count = row < rows ? clamp_count(a.D - d, V) : 0;
    const int64_t b = row < rows ? row / a.L : 0, l = row < rows ? row - b * a.L : 0;
    const float inv = 1.0f / (float)a.D;
    Raw<TR, V> rx;
    Raw<T, V> ry = {}, rg = {};
    fetch(rx, (const TR*)a.x + b * a.x_row + l * a.x_token + d, count);
    if (a.y) fetch(ry, (const T*)a.y + b * a.y_row + l * a.y_token + d, count);
    if (a.gate) fetch(rg, (const T*)a.gate + b * a.gate_row + l * a.gate_token + d, count);
    float r[V], sum[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = rx.at(v);
    if (a.y) {
        float r1 = 1.0f;
        if (a.post_weight) {
#pragma unroll
            for (int v = 0; v < V; ++v) sum[0] = fmaf(ry.at(v), ry.at(v), sum[0]);
            row_sum<TPR, 1>(sum, buf[0]);
            r1 = __builtin_amdgcn_rsqf(fmaf(sum[0], inv, a.eps));
        }
        Raw<float, V> w, s;
        if (a.post_weight) fetch(w, a.post_weight + d, count);
        if (a.scale) fetch(s, a.scale + d, count);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float n = ry.at(v);
            if (a.post_weight) n *= r1 * w.at(v);
            if (a.gate) n *= gate_value<T>(rg.at(v), a.act);
            if (a.scale) n *= s.at(v);
            r[v] += n;
        }
        put((TR*)a.x_out + b * a.x_out_row + l * a.x_out_token + d, count, r);
    }
    if (!a.h_out) return;
    Raw<float, V> w;
    fetch(w, a.pre_weight + d, count);
    sum[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) sum[0] = fmaf(r[v], r[v], sum[0]);
    row_sum<TPR, 1>(sum, buf[1]);
    const float r2 = __builtin_amdgcn_rsqf(fmaf(sum[0], inv, a.eps));
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] *= r2 * w.at(v);
    put((T*)a.h_out + b * a.h_row + l * a.h_token + d, count, r);
}

// Gradients.  x' is formed again from x, y and gate in 32 bits (its stored form may be rounded), then
//
//   t = gh pre_weight            dr = gx + r2 t - x' r2^3 mean(t x')            dx = dr
//   dn = dr scale act(gate)      s = dn post_weight      dy = r1 s - y r1^3 mean(s y)
//   dgate = dr scale n act'(gate)    dscale += dr act(gate) n    dpost += dn y r1    dpre += gh x' r2
//
// A lane owns the same columns of every row its workgroup works on, so the three sums over rows stay in registers and
// leave as one record per workgroup.  The next row's elements are asked for before the sums of this one.
template <class TR, class T, int TPR>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_backward(NormArgs a) {
    constexpr int TH = norm_threads<TPR>(), ROWS = TH / TPR, V = kNormLane;
    // by sum and, turn about, by row: whichever sums a call leaves out, a barrier lies between two uses of a buffer
    __shared__ float buf_y[2][TH / 64][1], buf_x[2][TH / 64][2], buf_n[2][TH / 64][1];
    int turn = 0;
    __shared__ float fold[ROWS > 1 ? TH * V : 1];
    const int d = threadIdx.x % TPR * V, slot = threadIdx.x / TPR;
    const int64_t rows = a.B * a.L;
    const int mine = clamp_count(a.D - d, V);
    const float inv = 1.0f / (float)a.D;
    float w1[V], w2[V], sc[V], d1[V], d2[V], ds[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        w1[v] = v < mine && a.post_weight ? a.post_weight[d + v] : 1.0f;
        w2[v] = v < mine && a.pre_weight ? a.pre_weight[d + v] : 0.0f;
        sc[v] = v < mine && a.scale ? a.scale[d + v] : 1.0f;
        d1[v] = d2[v] = ds[v] = 0.0f;
    }
    Raw<TR, V> fx = {}, fgx = {};
    Raw<T, V> fy = {}, fg = {}, fgh = {};
    auto ask = [&](int64_t row) {
        const int count = row < rows ? mine : 0;
        const int64_t b = row < rows ? row / a.L : 0, l = row < rows ? row - b * a.L : 0;
        fetch(fx, (const TR*)a.x + b * a.x_row + l * a.x_token + d, count);
        if (a.y) fetch(fy, (const T*)a.y + b * a.y_row + l * a.y_token + d, count);
        if (a.gate) fetch(fg, (const T*)a.gate + b * a.gate_row + l * a.gate_token + d, count);
        if (a.gx) fetch(fgx, (const TR*)a.gx + b * a.gx_row + l * a.gx_token + d, count);
        if (a.gh) fetch(fgh, (const T*)a.gh + b * a.gh_row + l * a.gh_token + d, count);
    };
    const int64_t first = (int64_t)blockIdx.x * ROWS, step = (int64_t)gridDim.x * ROWS;
    ask(first + slot);
    for (int64_t row0 = first; row0 < rows; row0 += step, turn ^= 1) {
        const int64_t row = row0 + slot;
        const int count = row < rows ? mine : 0;
        const int64_t b = row < rows ? row / a.L : 0, l = row < rows ? row - b * a.L : 0;
        float r[V], y[V], dr[V], t[V], act[V], slope[V];
        float s1[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            r[v] = fx.at(v), y[v] = fy.at(v), dr[v] = fgx.at(v), t[v] = fgh.at(v);
            act[v] = slope[v] = 1.0f;
            s1[0] = fmaf(y[v], y[v], s1[0]);
        }
        if (a.gate) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float g = fg.at(v);
                act[v] = g;
                if (a.act != 0) {
                    const float s = sigmoid_f<T>(g);
                    act[v] = a.act == 1 ? g * s : s;
                    slope[v] = a.act == 1 ? s * fmaf(g, 1.0f - s, 1.0f) : s * (1.0f - s);
                }
            }
        }
        ask(row + step);
        float r1 = 1.0f;
        if (a.post_weight) {
            row_sum<TPR, 1>(s1, buf_y[turn]);
            r1 = __builtin_amdgcn_rsqf(fmaf(s1[0], inv, a.eps));
        }
        float s2[2] = {0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            r[v] = fmaf(sc[v] * act[v], y[v] * (r1 * w1[v]), r[v]);
            s2[0] = fmaf(r[v], r[v], s2[0]);
            s2[1] = fmaf(t[v] * w2[v], r[v], s2[1]);
        }
        if (a.gh) {
            row_sum<TPR, 2>(s2, buf_x[turn]);
            const float r2 = __builtin_amdgcn_rsqf(fmaf(s2[0], inv, a.eps));
            const float back = s2[1] * inv * r2 * r2 * r2;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                d2[v] = fmaf(t[v], r[v] * r2, d2[v]);
                dr[v] += fmaf(r2 * w2[v], t[v], -r[v] * back);
            }
        }
        if (a.dx) put((TR*)a.dx + b * a.dx_row + l * a.dx_token + d, count, dr);
        if (!a.dy) continue;
        s1[0] = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float n = y[v] * (r1 * w1[v]);
            ds[v] = fmaf(dr[v], act[v] * n, ds[v]);
            slope[v] *= dr[v] * sc[v] * n;                          // dgate
            t[v] = dr[v] * sc[v] * act[v];                          // dn
            d1[v] = fmaf(t[v], y[v] * r1, d1[v]);
            s1[0] = fmaf(t[v] * w1[v], y[v], s1[0]);
        }
        if (a.dgate) put((T*)a.dgate + b * a.dgate_row + l * a.dgate_token + d, count, slope);
        float through = 0.0f;
        if (a.post_weight) {
            row_sum<TPR, 1>(s1, buf_n[turn]);
            through = s1[0] * inv * r1 * r1 * r1;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) t[v] = fmaf(r1 * w1[v], t[v], -y[v] * through);
        put((T*)a.dy + b * a.dy_row + l * a.dy_token + d, count, t);
    }
    if (!a.partial) return;
    auto leave = [&](const float (&v)[V], int which) {
        if (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; ++i) fold[threadIdx.x * V + i] = v[i];
            __syncthreads();
        }
        if (slot == 0) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < mine) {
                    float s = ROWS > 1 ? 0.0f : v[i];
                    if (ROWS > 1)
                        for (int w = 0; w < ROWS; ++w) s += fold[w * TPR * V + d + i];
                    a.partial[((int64_t)blockIdx.x * a.D + d + i) * 3 + which] = s;
                }
        }
    };
    leave(d1, 0);
    leave(d2, 1);
    leave(ds, 2);
}

}  // namespace seq
}  // namespace auv
