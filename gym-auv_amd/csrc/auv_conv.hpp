// The short causal convolution along time, channel by channel, with an optional SiLU:
//
//   pre[b,l,d] = bias[d] + sum_{j<W} weight[d,j] x~[b, l-(W-1)+j, d],     y = pre or pre sigmoid(pre)
//
// x~ is x within the token's own episode and 0 before it: a token marked in `start` opens an episode, tokens before the
// row's first come from `state` (0 without one).  Tokens at and behind lengths[b] are not read; their outputs are 0.
//
// Bound by memory: one read and one write per element against 2 W + 6 operations.  A thread therefore takes a run of
// tokens of V adjacent channels (one 16-byte access per token) and keeps the W - 1 earlier tokens in registers, so that
// every element is read once, but for W - 1 tokens at the start of each run, which the run before has just read.
#pragma once

#include "auv_seq.hpp"

namespace auv {
namespace seq {

struct ConvArgs {
    int64_t B, L, D;
    const void* x;
    int64_t x_row, x_token;
    const float* weight;
    const float* bias;
    const uint8_t* start;
    int64_t start_row, start_token;
    const int32_t* lengths;
    const void* state;      // [B, W-1, D]
    void* new_state;        // [B, W-1, D]
    void* y;
    int64_t y_row, y_token;
    const void* dy;
    int64_t dy_row, dy_token;
    const void* dnew_state; // [B, W-1, D]
    void* dx;
    int64_t dx_row, dx_token;
    void* dstate;           // [B, W-1, D]
    float* partial;         // [gridDim.x, D, W + 1]
    int32_t silu;
    int32_t run;            // tokens per thread
    int32_t lanes;          // channel vectors side by side in a workgroup
};

__device__ __forceinline__ int64_t row_length(const int32_t* lengths, int64_t b, int64_t L) {
    if (!lengths) return L;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > L ? L : n;
}

constexpr int kConvThreads = 256;

// The W - 1 tokens before `l0` of row b, oldest first, zeroed where an episode starts in between; `since` counts the
// tokens from the last start to l0 - 1 (W or more: none in sight).
template <class T, int W, int V>
__device__ __forceinline__ void conv_halo(const ConvArgs& a, int64_t b, int64_t l0, int64_t d, float (&win)[W - 1][V], int& since) {
    since = W;
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t t = l0 - (W - 1) + i;
        if (t < 0) {
            if (a.state) load<T, V>((const T*)a.state + (b * (W - 1) + (t + W - 1)) * a.D + d, win[i]);
            else
#pragma unroll
                for (int v = 0; v < V; ++v) win[i][v] = 0.0f;
        } else {
            if (a.start && a.start[b * a.start_row + t * a.start_token]) {
                since = 0;
#pragma unroll
                for (int k = 0; k < i; ++k)
#pragma unroll
                    for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
            }
            load<T, V>((const T*)a.x + b * a.x_row + t * a.x_token + d, win[i]);
        }
        ++since;
    }
}

template <class T, int W, int V>
__global__ __launch_bounds__(kConvThreads) void k_conv_forward(ConvArgs a) {
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
    const int slots = kConvThreads / a.lanes;
    const int64_t d = ((int64_t)blockIdx.y * a.lanes + lane) * V;
    if (slot >= slots || d >= a.D) return;
    const int64_t runs = (a.L + a.run - 1) / a.run;
    float w[W][V], bias[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = a.bias ? a.bias[d + v] : 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) w[j][v] = a.weight[(d + v) * W + j];
    }
    for (int64_t r = (int64_t)blockIdx.x * slots + slot; r < a.B * runs; r += (int64_t)gridDim.x * slots) {
        const int64_t b = r % a.B, l0 = (r / a.B) * a.run;   // rows side by side: adjacent in a time-major rollout
        const int64_t n = row_length(a.lengths, b, a.L);
        const int64_t end = l0 + a.run < a.L ? l0 + a.run : a.L;
        const int64_t stop = end < n ? end : n;
        T* const y = (T*)a.y + b * a.y_row + d;
        if (l0 < n || l0 == 0) {
            float win[W - 1][V];
            int since;
            conv_halo<T, W, V>(a, b, l0, d, win, since);
            const T* const x = (const T*)a.x + b * a.x_row + d;
            constexpr int kAhead = 4;
            for (int64_t t0 = l0; t0 < stop; t0 += kAhead) {
                float in[kAhead][V];
                bool fresh[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int64_t t = t0 + i < stop ? t0 + i : stop - 1;
                    load<T, V>(x + t * a.x_token, in[i]);
                    fresh[i] = a.start && a.start[b * a.start_row + t * a.start_token];
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    if (t0 + i < stop) {
                        if (fresh[i]) {
#pragma unroll
                            for (int k = 0; k < W - 1; ++k)
#pragma unroll
                                for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
                        }
                        float out[V];
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            float pre = bias[v];
#pragma unroll
                            for (int k = 0; k < W - 1; ++k) pre = fmaf(win[k][v], w[k][v], pre);
                            pre = fmaf(in[i][v], w[W - 1][v], pre);
                            out[v] = a.silu ? pre * sigmoid_f(pre) : pre;
#pragma unroll
                            for (int k = 0; k < W - 2; ++k) win[k][v] = win[k + 1][v];
                            win[W - 2][v] = in[i][v];
                        }
                        store<T, V>(y + (t0 + i) * a.y_token, out);
                    }
                }
            }
            // the run that holds the row's last token hands on what the next call would look back at
            if (a.new_state && (stop == n) && (l0 < n || n == 0)) {
#pragma unroll
                for (int i = 0; i < W - 1; ++i) store<T, V>((T*)a.new_state + (b * (W - 1) + i) * a.D + d, win[i]);
            }
        }
        float zero[V] = {};
        for (int64_t t = l0 > n ? l0 : n; t < end; ++t) store<T, V>(y + t * a.y_token, zero);
    }
}

// Gradients.  With g = dy silu'(pre):  dx[t-k] += weight[W-1-k] g[t],  dweight[W-1-k] += g[t] x~[t-k],  dbias += g, each
// only where t - k and t lie in one episode (at most `since` tokens back).  pre is formed again from x.  A run goes
// forwards over its tokens and the W - 1 behind them (those need g too), holding the W unfinished dx in registers; the
// sums over tokens stay in registers over all of a thread's runs and leave through one record per workgroup.
template <class T, int W, int V>
__global__ __launch_bounds__(kConvThreads) void k_conv_backward(ConvArgs a) {
    extern __shared__ float lds[];   // [slots][lanes][V][W + 1]
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
    const int slots = kConvThreads / a.lanes;
    const int64_t d = ((int64_t)blockIdx.y * a.lanes + lane) * V;
    const bool live = slot < slots && d < a.D;
    const int64_t runs = (a.L + a.run - 1) / a.run;
    float w[W][V], bias[V], dw[W][V], db[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        bias[v] = live && a.bias ? a.bias[d + v] : 0.0f;
        db[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            w[j][v] = live ? a.weight[(d + v) * W + j] : 0.0f;
            dw[j][v] = 0.0f;
        }
    }
    for (int64_t r = (int64_t)blockIdx.x * slots + slot; live && r < a.B * runs; r += (int64_t)gridDim.x * slots) {
        const int64_t b = r % a.B, l0 = (r / a.B) * a.run;
        const int64_t n = row_length(a.lengths, b, a.L);
        const int64_t end = l0 + a.run < a.L ? l0 + a.run : a.L;
        const int64_t own = end < n ? end : n;                              // tokens whose g counts for dweight here
        const int64_t stop = end + W - 1 < n ? end + W - 1 : n;             // tokens whose g reaches into [l0, end)
        T* const dx = (T*)a.dx + b * a.dx_row + d;
        if (l0 < n || l0 == 0) {
            float win[W - 1][V], pend[W][V];   // pend[k]: dx of the token k before the current one
            int since;
            conv_halo<T, W, V>(a, b, l0, d, win, since);
#pragma unroll
            for (int k = 0; k < W; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) pend[k][v] = 0.0f;
            auto emit = [&](int64_t t, const float (&g)[V]) {   // dx of token t is complete
                if (t >= l0) {
                    if (t < own) store<T, V>(dx + t * a.dx_token, g);
                } else if (l0 == 0 && a.dstate) {
                    if (t >= -(int64_t)(W - 1)) store<T, V>((T*)a.dstate + (b * (W - 1) + (t + W - 1)) * a.D + d, g);
                }
            };
            const T* const x = (const T*)a.x + b * a.x_row + d;
            const T* const dy = (const T*)a.dy + b * a.dy_row + d;
            constexpr int kAhead = 4;
            for (int64_t t0 = l0; t0 < stop; t0 += kAhead) {
                float in[kAhead][V], gin[kAhead][V];
                bool fresh[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int64_t t = t0 + i < stop ? t0 + i : stop - 1;
                    load<T, V>(x + t * a.x_token, in[i]);
                    load<T, V>(dy + t * a.dy_token, gin[i]);
                    fresh[i] = a.start && a.start[b * a.start_row + t * a.start_token];
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {
                    const int64_t t = t0 + i;
                    if (t < stop) {
                        if (fresh[i]) {
                            since = 0;
#pragma unroll
                            for (int k = 0; k < W - 1; ++k)
#pragma unroll
                                for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
                        }
                        float g[V];
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            float pre = bias[v];
#pragma unroll
                            for (int k = 0; k < W - 1; ++k) pre = fmaf(win[k][v], w[k][v], pre);
                            pre = fmaf(in[i][v], w[W - 1][v], pre);
                            const float s = sigmoid_f(pre);
                            g[v] = a.silu ? gin[i][v] * (s * fmaf(pre, 1.0f - s, 1.0f)) : gin[i][v];
                            pend[0][v] = fmaf(w[W - 1][v], g[v], pend[0][v]);
                        }
                        if (t < own) {
#pragma unroll
                            for (int v = 0; v < V; ++v) {
                                db[v] += g[v];
                                dw[W - 1][v] = fmaf(g[v], in[i][v], dw[W - 1][v]);
#pragma unroll
                                for (int k = 0; k < W - 1; ++k) dw[k][v] = fmaf(g[v], win[k][v], dw[k][v]);
                            }
                        }
#pragma unroll
                        for (int k = 1; k < W; ++k)
                            if (k <= since) {
#pragma unroll
                                for (int v = 0; v < V; ++v) pend[k][v] = fmaf(w[W - 1 - k][v], g[v], pend[k][v]);
                            }
                        ++since;
                        if (t == n - 1 && a.dnew_state) {   // the handed-on state is a copy of the last W - 1 tokens
#pragma unroll
                            for (int k = 0; k < W - 1; ++k)
                                if (k < since) {
                                    float g1[V];
                                    load<T, V>((const T*)a.dnew_state + (b * (W - 1) + (W - 2 - k)) * a.D + d, g1);
#pragma unroll
                                    for (int v = 0; v < V; ++v) pend[k][v] += g1[v];
                                }
                        }
                        emit(t - (W - 1), pend[W - 1]);
#pragma unroll
                        for (int v = 0; v < V; ++v) {
#pragma unroll
                            for (int k = W - 1; k > 0; --k) pend[k][v] = pend[k - 1][v];
                            pend[0][v] = 0.0f;
#pragma unroll
                            for (int k = 0; k < W - 2; ++k) win[k][v] = win[k + 1][v];
                            win[W - 2][v] = in[i][v];
                        }
                    }
                }
            }
            if (n == 0 && a.dnew_state) {   // a row without tokens hands its state on as it came
#pragma unroll
                for (int k = 1; k < W; ++k) load<T, V>((const T*)a.dnew_state + (b * (W - 1) + (W - 1 - k)) * a.D + d, pend[k]);
            }
            // pend[k] is now dx of token stop - k
#pragma unroll
            for (int k = W - 1; k > 0; --k) emit(stop - k, pend[k]);
        }
        float zero[V] = {};
        for (int64_t t = l0 > n ? l0 : n; t < end; ++t) store<T, V>(dx + t * a.dx_token, zero);
    }
    if (!a.partial) return;
    constexpr int K = W + 1;
    if (live) {
        float* const mine = lds + (size_t)(slot * a.lanes + lane) * V * K;
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int j = 0; j < W; ++j) mine[v * K + j] = dw[j][v];
            mine[v * K + W] = db[v];
        }
    }
    __syncthreads();
    const int row = a.lanes * V * K;
    for (int i = threadIdx.x; i < row; i += kConvThreads) {
        const int64_t chan = (int64_t)blockIdx.y * a.lanes * V + i / K;
        if (chan >= a.D) continue;
        float t = 0.0f;
        for (int s = 0; s < slots; ++s) t += lds[(size_t)s * row + i];
        a.partial[((int64_t)blockIdx.x * a.D + chan) * K + i % K] = t;
    }
}

// One token per row: the state's rows move up by one, in place or into new_state.  A thread reads what it replaces
// before it writes, so both may be the same memory.
template <class T, int W, int V>
__global__ __launch_bounds__(kConvThreads) void k_conv_step(ConvArgs a) {
    const int64_t dv = a.D / V;
    const int64_t i = (int64_t)blockIdx.x * kConvThreads + threadIdx.x;
    if (i >= a.B * dv) return;
    const int64_t b = i / dv, d = (i - b * dv) * V;
    const bool fresh = a.start && a.start[b * a.start_row];
    float win[W][V];
#pragma unroll
    for (int k = 0; k < W - 1; ++k) load<T, V>((const T*)a.state + (b * (W - 1) + k) * a.D + d, win[k]);
    load<T, V>((const T*)a.x + b * a.x_row + d, win[W - 1]);
    if (fresh) {
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
    }
    float out[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float pre = a.bias ? a.bias[d + v] : 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) pre = fmaf(win[k][v], a.weight[(d + v) * W + k], pre);
        out[v] = a.silu ? pre * sigmoid_f(pre) : pre;
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) store<T, V>((T*)a.new_state + (b * (W - 1) + k) * a.D + d, win[k + 1]);
    store<T, V>((T*)a.y + b * a.y_row + d, out);
}

}  // namespace seq
}  // namespace auv
