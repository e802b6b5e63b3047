// The short causal convolution along time, channel by channel, with an optional SiLU:
//
//   pre[b,l,d] = bias[d] + sum_{j<W} weight[d,j] x~[b, l-(W-1)+j, d],     y = pre or pre sigmoid(pre)
//
// x~ is x within the token's own episode and 0 before it: a token marked in `start` opens an episode, tokens before the
// row's first come from `state` (0 without one).  Tokens at and behind lengths[b] are not read; their outputs are 0.
//
// Bound by memory: one read and one write per element against 2 W + 20 operations.  A thread therefore takes a run of
// tokens of 8 (32-bit types: 4) adjacent channels, one 16-byte access per token at any alignment, and keeps the W - 1 earlier tokens in registers, so that
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
    int32_t lanes;          // vectors of channels side by side in a workgroup
};

__device__ __forceinline__ int64_t row_length(const int32_t* lengths, int64_t b, int64_t L) {
    if (!lengths) return L;
    const int64_t n = lengths[b];
    return n < 0 ? 0 : n > L ? L : n;
}

constexpr int kConvThreads = 256;
constexpr int kConvAhead = 4;   // tokens asked for together, one such group ahead of the one at work
template <class T>
constexpr int conv_vector() { return 16 / (int)sizeof(T); }   // channels per lane: one 16-byte access

// weight[d .. d + V) with W taps each, and bias; zeros behind the last channel
template <int W, int V>
__device__ __forceinline__ void conv_taps(const ConvArgs& a, int64_t d, int count, float (&w)[V * W], float (&bias)[V]) {
    Raw<float, V * W> t;
    fetch(t, a.weight + d * W, count == V ? V * W : 0);
#pragma unroll
    for (int i = 0; i < V * W; ++i) w[i] = t.at(i);
    if (count < V)
        for (int i = 0; i < V * W; ++i) w[i] = i < count * W ? a.weight[d * W + i] : 0.0f;
    Raw<float, V> s = {};
    if (a.bias) fetch(s, a.bias + d, count);
#pragma unroll
    for (int v = 0; v < V; ++v) bias[v] = s.at(v);
}

// The W - 1 tokens before `l0` of row b, oldest first, zeroed where an episode starts in between; `since` counts the
// tokens from the last start to l0 - 1 (W or more: none in sight).
template <class T, int W, int V>
__device__ __forceinline__ void conv_halo(const ConvArgs& a, int64_t b, int64_t l0, int64_t d, int count, float (&win)[W - 1][V],
                                          int& since) {
    since = W;
    Raw<T, V> t[W - 1] = {};
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t l = l0 - (W - 1) + i;
        if (l >= 0) fetch(t[i], (const T*)a.x + b * a.x_row + l * a.x_token + d, count);
        else if (a.state) fetch(t[i], (const T*)a.state + (b * (W - 1) + (l + W - 1)) * a.D + d, count);
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t l = l0 - (W - 1) + i;
        if (l >= 0 && a.start && a.start[b * a.start_row + l * a.start_token]) {
            since = 0;
#pragma unroll
            for (int k = 0; k < i; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) win[i][v] = t[i].at(v);
        ++since;
    }
}

template <class T, int W>
__global__ __launch_bounds__(kConvThreads) void k_conv_forward(ConvArgs a) {
    constexpr int V = conv_vector<T>();
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
    const int slots = kConvThreads / a.lanes;
    const int64_t d = ((int64_t)blockIdx.y * a.lanes + lane) * V;
    if (slot >= slots || d >= a.D) return;
    const int count = clamp_count(a.D - d, V);
    const int64_t runs = (a.L + a.run - 1) / a.run;
    float w[V * W], bias[V];
    conv_taps<W, V>(a, d, count, w, bias);
    for (int64_t r = (int64_t)blockIdx.x * slots + slot; r < a.B * runs; r += (int64_t)gridDim.x * slots) {
        const int64_t b = r % a.B, l0 = (r / a.B) * a.run;   // rows side by side: adjacent in a time-major rollout
        const int64_t n = row_length(a.lengths, b, a.L);
        const int64_t end = l0 + a.run < a.L ? l0 + a.run : a.L;
        const int64_t stop = end < n ? end : n;
        T* const y = (T*)a.y + b * a.y_row + d;
        if (l0 < n || l0 == 0) {
            const T* const x = (const T*)a.x + b * a.x_row + d;
            const uint8_t* const start = a.start ? a.start + b * a.start_row : nullptr;
            Raw<T, V> ahead[kConvAhead] = {};
            uint8_t marks[kConvAhead] = {};
            auto ask = [&](int64_t t0) {
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i)
                    if (t0 + i < stop) {
                        fetch(ahead[i], x + (t0 + i) * a.x_token, count);
                        if (start) marks[i] = start[(t0 + i) * a.start_token];
                    }
            };
            ask(l0);
            float win[W - 1][V];
            int since;
            conv_halo<T, W, V>(a, b, l0, d, count, win, since);
            for (int64_t t0 = l0; t0 < stop; t0 += kConvAhead) {
                Raw<T, V> in[kConvAhead];
                bool fresh[kConvAhead];
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i) in[i] = ahead[i], fresh[i] = marks[i] != 0;
                ask(t0 + kConvAhead);
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i) {
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
                            const float x1 = in[i].at(v);
                            float pre = bias[v];
#pragma unroll
                            for (int k = 0; k < W - 1; ++k) pre = fmaf(win[k][v], w[v * W + k], pre);
                            pre = fmaf(x1, w[v * W + W - 1], pre);
                            out[v] = a.silu ? pre * sigmoid_f(pre) : pre;
#pragma unroll
                            for (int k = 0; k < W - 2; ++k) win[k][v] = win[k + 1][v];
                            win[W - 2][v] = x1;
                        }
                        put(y + (t0 + i) * a.y_token, count, out);
                    }
                }
            }
            // the run that holds the row's last token hands on what the next call would look back at
            if (a.new_state && (stop == n) && (l0 < n || n == 0)) {
#pragma unroll
                for (int i = 0; i < W - 1; ++i) put((T*)a.new_state + (b * (W - 1) + i) * a.D + d, count, win[i]);
            }
        }
        float zero[V] = {};
        for (int64_t t = l0 > n ? l0 : n; t < end; ++t) put(y + t * a.y_token, count, zero);
    }
}

// Gradients.  With g = dy silu'(pre):  dx[t-k] += weight[W-1-k] g[t],  dweight[W-1-k] += g[t] x~[t-k],  dbias += g, each
// only where t - k and t lie in one episode (at most `since` tokens back).  pre is formed again from x.  A run goes
// forwards over its tokens and the W - 1 behind them (those need g too), holding the W unfinished dx in registers; the
// sums over tokens stay in registers over all of a thread's runs and leave through one record per workgroup.
template <class T, int W>
__global__ __launch_bounds__(kConvThreads) void k_conv_backward(ConvArgs a) {
    constexpr int V = conv_vector<T>();
    extern __shared__ float lds[];   // [slots][lanes][V][W + 1]
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
    const int slots = kConvThreads / a.lanes;
    const int64_t d = ((int64_t)blockIdx.y * a.lanes + lane) * V;
    const int count = slot < slots ? clamp_count(a.D - d, V) : 0;
    const bool live = count > 0;
    const int64_t runs = (a.L + a.run - 1) / a.run;
    float w[V * W] = {}, bias[V] = {}, dw[V * W], db[V];
    if (live) conv_taps<W, V>(a, d, count, w, bias);
#pragma unroll
    for (int i = 0; i < V * W; ++i) dw[i] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) db[v] = 0.0f;
    for (int64_t r = (int64_t)blockIdx.x * slots + slot; live && r < a.B * runs; r += (int64_t)gridDim.x * slots) {
        const int64_t b = r % a.B, l0 = (r / a.B) * a.run;
        const int64_t n = row_length(a.lengths, b, a.L);
        const int64_t end = l0 + a.run < a.L ? l0 + a.run : a.L;
        const int64_t own = end < n ? end : n;                              // tokens whose g counts for dweight here
        const int64_t stop = end + W - 1 < n ? end + W - 1 : n;             // tokens whose g reaches into [l0, end)
        T* const dx = (T*)a.dx + b * a.dx_row + d;
        if (l0 < n || l0 == 0) {
            const T* const x = (const T*)a.x + b * a.x_row + d;
            const T* const dy = (const T*)a.dy + b * a.dy_row + d;
            const uint8_t* const start = a.start ? a.start + b * a.start_row : nullptr;
            Raw<T, V> ahead[kConvAhead] = {}, gahead[kConvAhead] = {};
            uint8_t marks[kConvAhead] = {};
            auto ask = [&](int64_t t0) {
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i)
                    if (t0 + i < stop) {
                        fetch(ahead[i], x + (t0 + i) * a.x_token, count);
                        fetch(gahead[i], dy + (t0 + i) * a.dy_token, count);
                        if (start) marks[i] = start[(t0 + i) * a.start_token];
                    }
            };
            ask(l0);
            float win[W - 1][V], pend[W][V];   // pend[k]: dx of the token k before the current one
            int since;
            conv_halo<T, W, V>(a, b, l0, d, count, win, since);
#pragma unroll
            for (int k = 0; k < W; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) pend[k][v] = 0.0f;
            auto emit = [&](int64_t t, const float (&g)[V]) {   // dx of token t is complete
                if (t >= l0) {
                    if (t < own) put(dx + t * a.dx_token, count, g);
                } else if (l0 == 0 && a.dstate) {
                    if (t >= -(int64_t)(W - 1)) put((T*)a.dstate + (b * (W - 1) + (t + W - 1)) * a.D + d, count, g);
                }
            };
            for (int64_t t0 = l0; t0 < stop; t0 += kConvAhead) {
                Raw<T, V> in[kConvAhead], gin[kConvAhead];
                bool fresh[kConvAhead];
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i) in[i] = ahead[i], gin[i] = gahead[i], fresh[i] = marks[i] != 0;
                ask(t0 + kConvAhead);
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i) {
                    const int64_t t = t0 + i;
                    if (t < stop) {
                        if (fresh[i]) {
                            since = 0;
#pragma unroll
                            for (int k = 0; k < W - 1; ++k)
#pragma unroll
                                for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
                        }
                        float g[V], x1[V];
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            x1[v] = in[i].at(v);
                            g[v] = gin[i].at(v);
                            if (a.silu) {
                                float pre = bias[v];
#pragma unroll
                                for (int k = 0; k < W - 1; ++k) pre = fmaf(win[k][v], w[v * W + k], pre);
                                pre = fmaf(x1[v], w[v * W + W - 1], pre);
                                const float s = sigmoid_f(pre);
                                g[v] *= s * fmaf(pre, 1.0f - s, 1.0f);
                            }
                            pend[0][v] = fmaf(w[v * W + W - 1], g[v], pend[0][v]);
                        }
                        if (t < own) {
#pragma unroll
                            for (int v = 0; v < V; ++v) {
                                db[v] += g[v];
                                dw[v * W + W - 1] = fmaf(g[v], x1[v], dw[v * W + W - 1]);
#pragma unroll
                                for (int k = 0; k < W - 1; ++k) dw[v * W + k] = fmaf(g[v], win[k][v], dw[v * W + k]);
                            }
                        }
                        if (since >= W - 1) {
#pragma unroll
                            for (int k = 1; k < W; ++k)
#pragma unroll
                                for (int v = 0; v < V; ++v) pend[k][v] = fmaf(w[v * W + W - 1 - k], g[v], pend[k][v]);
                        } else {
#pragma unroll
                            for (int k = 1; k < W; ++k)
                                if (k <= since) {
#pragma unroll
                                    for (int v = 0; v < V; ++v) pend[k][v] = fmaf(w[v * W + W - 1 - k], g[v], pend[k][v]);
                                }
                        }
                        ++since;
                        if (t == n - 1 && a.dnew_state) {   // the handed-on state is a copy of the last W - 1 tokens
#pragma unroll
                            for (int k = 0; k < W - 1; ++k)
                                if (k < since) {
                                    Raw<T, V> g1;
                                    fetch(g1, (const T*)a.dnew_state + (b * (W - 1) + (W - 2 - k)) * a.D + d, count);
#pragma unroll
                                    for (int v = 0; v < V; ++v) pend[k][v] += g1.at(v);
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
                            win[W - 2][v] = x1[v];
                        }
                    }
                }
            }
            if (n == 0 && a.dnew_state) {   // a row without tokens hands its state on as it came
#pragma unroll
                for (int k = 1; k < W; ++k) {
                    Raw<T, V> g1;
                    fetch(g1, (const T*)a.dnew_state + (b * (W - 1) + (W - 1 - k)) * a.D + d, count);
#pragma unroll
                    for (int v = 0; v < V; ++v) pend[k][v] = g1.at(v);
                }
            }
            // pend[k] is now dx of token stop - k
#pragma unroll
            for (int k = W - 1; k > 0; --k) emit(stop - k, pend[k]);
        }
        float zero[V] = {};
        for (int64_t t = l0 > n ? l0 : n; t < end; ++t) put(dx + t * a.dx_token, count, zero);
    }
    if (!a.partial) return;
    constexpr int K = W + 1;
    if (live) {
        float* const mine = lds + (size_t)(slot * a.lanes + lane) * V * K;
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll
            for (int j = 0; j < W; ++j) mine[v * K + j] = dw[v * W + j];
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
// before it writes, so both may be the same memory.  It keeps its channels' taps (as many bytes as a row's elements) for
// all the rows it takes.
template <class T, int W>
__global__ __launch_bounds__(kConvThreads) void k_conv_step(ConvArgs a) {
    constexpr int V = conv_vector<T>();
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
    const int slots = kConvThreads / a.lanes;
    const int64_t d = ((int64_t)blockIdx.y * a.lanes + lane) * V;
    if (slot >= slots || d >= a.D) return;
    const int count = clamp_count(a.D - d, V);
    float w[V * W], bias[V];
    conv_taps<W, V>(a, d, count, w, bias);
    for (int64_t b = (int64_t)blockIdx.x * slots + slot; b < a.B; b += (int64_t)gridDim.x * slots) {
        Raw<T, V> t[W];
#pragma unroll
        for (int k = 0; k < W - 1; ++k) fetch(t[k], (const T*)a.state + (b * (W - 1) + k) * a.D + d, count);
        fetch(t[W - 1], (const T*)a.x + b * a.x_row + d, count);
        const bool fresh = a.start && a.start[b * a.start_row];
        float win[W][V], out[V];
#pragma unroll
        for (int k = 0; k < W; ++k)
#pragma unroll
            for (int v = 0; v < V; ++v) win[k][v] = fresh && k < W - 1 ? 0.0f : t[k].at(v);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float pre = bias[v];
#pragma unroll
            for (int k = 0; k < W; ++k) pre = fmaf(win[k][v], w[v * W + k], pre);
            out[v] = a.silu ? pre * sigmoid_f(pre) : pre;
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) put((T*)a.new_state + (b * (W - 1) + k) * a.D + d, count, win[k + 1]);
        put((T*)a.y + b * a.y_row + d, count, out);
    }
}

}  // namespace seq
}  // namespace auv
