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
// lanes.  65,536 rows of 128 channels, bf16 and 32-bit residuals: 21.5 us forwards, 5.4 TB/s.  Just above a step lanes lie
// idle (520 channels 3.1 TB/s forwards, 512 5.5), and with 1,024 lanes the backward pass has 128 registers and spills 72 to
// 129 (8,192 channels 3.0 TB/s forwards and backwards, 512 5.4).
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
    int64_t first;           // forwards: workgroup of this launch
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
// The columns of a lane.  It takes whole vectors: where V does not divide the channels, the last lane takes the last V,
// `shared` of which its neighbour has as well.  Both form and write the same values; the sums take them from the neighbour.
// Lanes without channels read what the last one reads, and rows behind the last what that one holds, so that no load is
// masked; they write nothing and count for nothing.  (Rows of up to 32 channels may have fewer than V: theirs are.)
// 262,144 rows of 250 channels, bf16 and 32-bit residuals: 198 us forwards and 345 us backwards with masked loads and
// stores for the last lane, 167 us (5.5 TB/s) and 280 us (5.1 TB/s) so.  65,536 rows of 128: 21 us forwards (5.5 TB/s).
template <int TPR>
struct Columns {
    static constexpr int V = kNormLane;
    int d, mine, shared;    // where the lane's vector begins, and how much of it is real
    __device__ __forceinline__ explicit Columns(int D) {
        const int at = threadIdx.x % TPR * V;
        mine = at >= D ? 0 : TPR > 4 || D >= V ? V : D;
        d = (TPR > 4 || mine == V) && at > D - V ? D - V : at;
        shared = at - d < V ? at - d : V;
    }
    __device__ __forceinline__ float once(int v, float x) const { return v >= shared ? x : 0.0f; }
};

// A lane's elements of a row: all of them where its vector is whole (rows of more than 32 channels), or the first `count`.
template <int TPR, class T, int V>
__device__ __forceinline__ void fetch_row(Raw<T, V>& out, const T* p, int count) {
    fetch(out, p, TPR > 4 ? V : count);
}
template <int TPR, class T, int V>
__device__ __forceinline__ void put_row(T* p, int count, const float (&in)[V]) {
    if constexpr (TPR > 4) {
        if (count) store<T, V>(p, in);
    } else {
        put(p, count, in);
    }
}

template <class TR, class T, int TPR>
__global__ __launch_bounds__(norm_threads<TPR>()) void k_norm_forward(NormArgs a) {
    constexpr int TH = norm_threads<TPR>(), ROWS = TH / TPR, V = kNormLane;
    __shared__ float buf[2][TH / 64][1];
    const Columns<TPR> me((int)a.D);
    const int d = me.d, slot = threadIdx.x / TPR;
    const int64_t rows = a.B * a.L, row = (a.first + blockIdx.x) * ROWS + slot, real = row < rows ? row : rows - 1;
    const int count = row < rows ? me.mine : 0;
    const int64_t b = real / a.L, l = real - b * a.L;
    const float inv = 1.0f / (float)a.D;
    Raw<TR, V> rx;
    Raw<T, V> ry = {}, rg = {};
    fetch_row<TPR>(rx, (const TR*)a.x + b * a.x_row + l * a.x_token + d, count);
    if (a.y) fetch_row<TPR>(ry, (const T*)a.y + b * a.y_row + l * a.y_token + d, count);
    if (a.gate) fetch_row<TPR>(rg, (const T*)a.gate + b * a.gate_row + l * a.gate_token + d, count);
    float r[V], sum[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] = rx.at(v);
    if (a.y) {
        float r1 = 1.0f;
        if (a.post_weight) {
#pragma unroll
            for (int v = 0; v < V; ++v) sum[0] = fmaf(me.once(v, ry.at(v)), ry.at(v), sum[0]);
            row_sum<TPR, 1>(sum, buf[0]);
            r1 = __builtin_amdgcn_rsqf(fmaf(sum[0], inv, a.eps));
        }
        Raw<float, V> w, s;
        if (a.post_weight) fetch_row<TPR>(w, a.post_weight + d, count);
        if (a.scale) fetch_row<TPR>(s, a.scale + d, count);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float n = ry.at(v);
            if (a.post_weight) n *= r1 * w.at(v);
            if (a.gate) n *= gate_value<T>(rg.at(v), a.act);
            if (a.scale) n *= s.at(v);
            r[v] += n;
        }
        put_row<TPR>((TR*)a.x_out + b * a.x_out_row + l * a.x_out_token + d, count, r);
    }
    if (!a.h_out) return;
    Raw<float, V> w;
    fetch_row<TPR>(w, a.pre_weight + d, count);
    sum[0] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) sum[0] = fmaf(me.once(v, r[v]), r[v], sum[0]);
    row_sum<TPR, 1>(sum, buf[1]);
    const float r2 = __builtin_amdgcn_rsqf(fmaf(sum[0], inv, a.eps));
#pragma unroll
    for (int v = 0; v < V; ++v) r[v] *= r2 * w.at(v);
    put_row<TPR>((T*)a.h_out + b * a.h_row + l * a.h_token + d, count, r);
}

// The kernel's arguments, read where they are used: some fifty addresses and strides held in scalar registers through the
// row loop would push each other out to vector lanes.
__device__ __forceinline__ NormArgs norm_args() {
    const __attribute__((address_space(4))) NormArgs* p = (const __attribute__((address_space(4))) NormArgs*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    NormArgs r;
    __builtin_memcpy(&r, (const NormArgs*)p, sizeof(NormArgs));
    return r;
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
__global__ __launch_bounds__(norm_threads<TPR>(), 2) void k_norm_backward(NormArgs a) {
    constexpr int TH = norm_threads<TPR>(), ROWS = TH / TPR, V = kNormLane;
    // by sum and, turn about, by row: whichever sums a call leaves out, a barrier lies between two uses of a buffer
    __shared__ float buf_y[2][TH / 64][1], buf_x[2][TH / 64][2], buf_n[2][TH / 64][1];
    int turn = 0;
    __shared__ float fold[ROWS > 1 ? TH * V : 1];
    const int D = (int)a.D, slot = threadIdx.x / TPR;
    const Columns<TPR> me(D);
    const int d = me.d, mine = me.mine;
    const int64_t rows = a.B * a.L;
    const float inv = 1.0f / (float)D;
    const bool with_y = a.y != nullptr, gated = a.gate != nullptr, post = a.post_weight != nullptr, with_h = a.gh != nullptr;
    const int kind = a.act;
    float w1[V], w2[V], sc[V], d1[V], d2[V], ds[V];
    auto column = [&](const float* from, float absent, float (&to)[V]) {
        Raw<float, V> t;
        if (from) fetch_row<TPR>(t, from + d, mine);
#pragma unroll
        for (int v = 0; v < V; ++v) to[v] = from ? t.at(v) : absent;
    };
    column(a.post_weight, 1.0f, w1);
    column(a.pre_weight, 0.0f, w2);
    column(a.scale, 1.0f, sc);
#pragma unroll
    for (int v = 0; v < V; ++v) d1[v] = d2[v] = ds[v] = 0.0f;
    // the row's place is moved on, not divided out of its number, from one row to the next
    const int64_t first = (int64_t)blockIdx.x * ROWS, step = (int64_t)gridDim.x * ROWS, step_b = step / a.L, step_l = step - step_b * a.L;
    int64_t b, l, next_b = (first + slot) / a.L, next_l = first + slot - next_b * a.L;
    Raw<TR, V> fx = {}, fgx = {};
    Raw<T, V> fy = {}, fg = {}, fgh = {};
    auto ask = [&](int64_t row) {
        const NormArgs r = norm_args();
        const int count = row < rows ? mine : 0;
        if (TPR > 4 && row >= rows) next_b = r.B - 1, next_l = r.L - 1;
        fetch_row<TPR>(fx, (const TR*)r.x + next_b * r.x_row + next_l * r.x_token + d, count);
        if (r.y) fetch_row<TPR>(fy, (const T*)r.y + next_b * r.y_row + next_l * r.y_token + d, count);
        if (r.gate) fetch_row<TPR>(fg, (const T*)r.gate + next_b * r.gate_row + next_l * r.gate_token + d, count);
        if (r.gx) fetch_row<TPR>(fgx, (const TR*)r.gx + next_b * r.gx_row + next_l * r.gx_token + d, count);
        if (r.gh) fetch_row<TPR>(fgh, (const T*)r.gh + next_b * r.gh_row + next_l * r.gh_token + d, count);
    };
    ask(first + slot);
    for (int64_t row0 = first; row0 < rows; row0 += step, turn ^= 1) {
        const int64_t row = row0 + slot;
        const int count = row < rows ? mine : 0;
        b = next_b, l = next_l;
        float r[V], y[V], dr[V], t[V], act[V], slope[V];
        float s1[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            r[v] = fx.at(v), y[v] = fy.at(v), dr[v] = count ? fgx.at(v) : 0.0f, t[v] = count ? fgh.at(v) : 0.0f;
            act[v] = slope[v] = 1.0f;
            s1[0] = fmaf(me.once(v, y[v]), y[v], s1[0]);
        }
        if (gated && kind == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) act[v] = fg.at(v);
        } else if (gated) {
            const bool silu = kind == 1;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float g = fg.at(v), s = sigmoid_f<T>(g);
                act[v] = s * (silu ? g : 1.0f);
                slope[v] = fmaf(act[v], 1.0f - s, silu ? s : 0.0f);    // SiLU: s (1 + g (1 - s)); sigmoid: s (1 - s)
            }
        }
        next_b += step_b, next_l += step_l;
        if (next_l >= a.L) next_l -= a.L, ++next_b;
        ask(row + step);
        float r1 = 1.0f;
        if (post) {
            row_sum<TPR, 1>(s1, buf_y[turn]);
            r1 = __builtin_amdgcn_rsqf(fmaf(s1[0], inv, a.eps));
        }
#pragma unroll
        for (int v = 0; v < V; ++v) r[v] = fmaf(sc[v] * act[v], y[v] * (r1 * w1[v]), r[v]);
        if (with_h) {
            float s2[2] = {0.0f, 0.0f};
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float once = me.once(v, r[v]);
                s2[0] = fmaf(once, r[v], s2[0]);
                s2[1] = fmaf(t[v] * w2[v], once, s2[1]);
            }
            row_sum<TPR, 2>(s2, buf_x[turn]);
            const float r2 = __builtin_amdgcn_rsqf(fmaf(s2[0], inv, a.eps));
            const float back = s2[1] * inv * r2 * r2 * r2;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                d2[v] = fmaf(t[v], r[v] * r2, d2[v]);
                dr[v] += fmaf(r2 * w2[v], t[v], -r[v] * back);
            }
        }
        const NormArgs to = norm_args();
        if (to.dx) put_row<TPR>((TR*)to.dx + b * to.dx_row + l * to.dx_token + d, count, dr);
        if (!with_y) continue;
        s1[0] = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float n = y[v] * (r1 * w1[v]);
            ds[v] = fmaf(dr[v], act[v] * n, ds[v]);
            slope[v] *= dr[v] * sc[v] * n;                          // dgate
            t[v] = dr[v] * sc[v] * act[v];                          // dn
            d1[v] = fmaf(t[v], y[v] * r1, d1[v]);
            s1[0] = fmaf(t[v] * w1[v], me.once(v, y[v]), s1[0]);
        }
        if (to.dgate) put_row<TPR>((T*)to.dgate + b * to.dgate_row + l * to.dgate_token + d, count, slope);
        float through = 0.0f;
        if (post) {
            row_sum<TPR, 1>(s1, buf_n[turn]);
            through = s1[0] * inv * r1 * r1 * r1;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) t[v] = fmaf(r1 * w1[v], t[v], -y[v] * through);
        put_row<TPR>((T*)to.dy + b * to.dy_row + l * to.dy_token + d, count, t);
    }
    if (!a.partial) return;
    auto leave = [&](const float (&v)[V], int which) {
        float* const to = a.partial + (int64_t)blockIdx.x * a.D * 3 + which;
        if constexpr (ROWS > 1) {
            __syncthreads();
#pragma unroll
            for (int i = 0; i < V; ++i) fold[threadIdx.x * V + i] = v[i];
            __syncthreads();
#pragma unroll 1
            for (int e = threadIdx.x; e < TPR * V; e += TH) {
                // element e % V of lane e / V, whose vector may have moved up from where it belongs
                const int at = e / V * V, from = D >= V && at > D - V ? D - V : at, column = from + e % V;
                if (at >= D || column < at || column >= D) continue;
                float sum = 0.0f;
                for (int w = 0; w < ROWS; ++w) sum += fold[w * TPR * V + e];
                to[(int64_t)column * 3] = sum;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i >= me.shared && i < mine) to[(int64_t)(d + i) * 3] = v[i];
        }
    };
    leave(d1, 0);
    leave(d2, 1);
    leave(ds, 2);
}

}  // namespace seq
}  // namespace auv
