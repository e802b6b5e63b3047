// The short causal convolution along time, channel by channel, with an optional SiLU:
//
//   pre[b,l,d] = bias[d] + sum_{j<W} weight[d,j] x~[b, l-(W-1)+j, d],     y = pre or pre sigmoid(pre)
//
// x~ is x within the token's own episode and 0 before it: a token marked in `start` opens an episode, tokens before the
// row's first come from `state` (0 without one).  Tokens at and behind lengths[b] are not read; their outputs are 0.
//
// Bound by memory: one read and one write per element against 2 W + 20 operations.  A thread therefore takes a run of
// tokens of 8 (32-bit types: 4) adjacent channels, one 16-byte access per token at any alignment, and keeps the W - 1
// earlier tokens in registers, so that every element is read once, but for W - 1 tokens at the start of each run, which the
// run before has just read.  bf16, width 4: 4,096 rows x 128 tokens x 128 channels 66 us forwards (268 MB, 4.1 TB/s) and 103
// us backwards (403 MB, 3.9 TB/s; 255 registers, four spilled, two waves per SIMD); a step of 65,536 rows 24 us (134 MB, 5.6
// TB/s).
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
// Whole rows of rollouts take V channels per lane without exception: where V does not divide the channels, the last lane
// takes the last V of them, some of which its neighbour has as well and writes the same values to.  (V = 1 for fewer than
// V channels.  A step may work in place, where that would read what the neighbour has written: its last lane takes fewer.)

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

// The W - 1 tokens before `l0` of row b, oldest first, zeroed where an episode starts in between.
template <class T, int W, int V>
__device__ __forceinline__ void conv_halo(const ConvArgs& a, int64_t b, int64_t l0, int64_t d, float (&win)[W - 1][V]) {
    Raw<T, V> t[W - 1] = {};
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t l = l0 - (W - 1) + i;
        if (l >= 0) fetch(t[i], (const T*)a.x + b * a.x_row + l * a.x_token + d, V);
        else if (a.state) fetch(t[i], (const T*)a.state + (b * (W - 1) + (l + W - 1)) * a.D + d, V);
    }
#pragma unroll
    for (int i = 0; i < W - 1; ++i) {
        const int64_t l = l0 - (W - 1) + i;
        if (l >= 0 && a.start && a.start[b * a.start_row + l * a.start_token]) {
#pragma unroll
            for (int k = 0; k < i; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) win[k][v] = 0.0f;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) win[i][v] = t[i].at(v);
    }
}

// One pre-activation per channel: xs holds the last four tokens, token t in place t % 4, so that no token is ever moved
// (i: the current one's place, a compile-time number).
template <int W, int V>
__device__ __forceinline__ float conv_pre(const float (&xs)[4][V], const float (&w)[V * W], const float (&bias)[V], int i, int v) {
    float pre = bias[v];
#pragma unroll
    for (int k = 0; k < W; ++k) pre = fmaf(xs[(i + 4 - (W - 1) + k) % 4][v], w[v * W + k], pre);
    return pre;
}

// Tokens of a run are counted from its first, in 32 bits: `tokens` of the run in the row at all, of them and of those
// behind `real` (below 1 where the row has ended before).
struct ConvRun {
    int64_t b, l0, n;
    int tokens, real;
};
__device__ __forceinline__ ConvRun conv_run_of(const ConvArgs& a, int64_t r) {
    ConvRun c;
    c.b = r % a.B, c.l0 = (r / a.B) * a.run;   // rows side by side: adjacent in a time-major rollout
    c.n = row_length(a.lengths, c.b, a.L);
    c.tokens = a.L - c.l0 < a.run ? (int)(a.L - c.l0) : a.run;
    const int64_t left = c.n - c.l0;
    c.real = left > 2 * a.run ? 2 * a.run : left < 0 ? 0 : (int)left;
    return c;
}

template <class T, int W, int V>
__global__ __launch_bounds__(kConvThreads) void k_conv_forward(ConvArgs a) {
    static_assert(kConvAhead == 4 && W <= 4, "a group of tokens goes once round xs");
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
    const int slots = kConvThreads / a.lanes;
    const int64_t d_lane = ((int64_t)blockIdx.y * a.lanes + lane) * V, d = d_lane < a.D - V ? d_lane : a.D - V;
    if (slot >= slots || d_lane >= a.D) return;
    const int64_t runs = (a.L + a.run - 1) / a.run;
    float w[V * W], bias[V];
    conv_taps<W, V>(a, d, V, w, bias);
    for (int64_t r = (int64_t)blockIdx.x * slots + slot; r < a.B * runs; r += (int64_t)gridDim.x * slots) {
        const ConvRun c = conv_run_of(a, r);
        const int stop = c.tokens < c.real ? c.tokens : c.real;
        T* y = (T*)a.y + c.b * a.y_row + c.l0 * a.y_token + d;
        float win[W - 1][V];
        if (stop > 0) {
            const T* x = (const T*)a.x + c.b * a.x_row + c.l0 * a.x_token + d;
            const uint8_t* start = a.start ? a.start + c.b * a.start_row + c.l0 * a.start_token : nullptr;
            Raw<T, V> ahead[kConvAhead] = {};
            uint8_t marks[kConvAhead] = {};
            auto ask = [&](int i, int t) {      // token t, i behind the group's first
                if (t < stop) {
                    fetch(ahead[i % kConvAhead], x + i * a.x_token, V);
                    if (start) marks[i % kConvAhead] = start[i * a.start_token];
                }
            };
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) ask(i, i);
            conv_halo<T, W, V>(a, c.b, c.l0, d, win);
            float xs[4][V];
#pragma unroll
            for (int k = 0; k < W - 1; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) xs[4 - (W - 1) + k][v] = win[k][v];
            for (int t0 = 0; t0 < stop; t0 += kConvAhead) {
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i) {
                    if (t0 + i < stop) {
                        if (marks[i]) {
#pragma unroll
                            for (int k = 1; k < 4; ++k)
#pragma unroll
                                for (int v = 0; v < V; ++v) xs[(i + k) % 4][v] = 0.0f;
                        }
#pragma unroll
                        for (int v = 0; v < V; ++v) xs[i][v] = ahead[i].at(v);
                        ask(i + kConvAhead, t0 + i + kConvAhead);     // into the place this token has left
                        float out[V];
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            const float pre = conv_pre<W, V>(xs, w, bias, i, v);
                            out[v] = a.silu ? pre * sigmoid_f<T>(pre) : pre;
                        }
                        put(y, V, out);
                        y += a.y_token;
                    }
                }
                x += kConvAhead * a.x_token;
                if (start) start += kConvAhead * a.start_token;
            }
        }
        // the run that holds the row's last token hands on what the next call would look back at
        if (a.new_state && stop == c.real && (stop > 0 || (c.n == 0 && c.l0 == 0))) {
            conv_halo<T, W, V>(a, c.b, c.n, d, win);
#pragma unroll
            for (int i = 0; i < W - 1; ++i) put((T*)a.new_state + (c.b * (W - 1) + i) * a.D + d, V, win[i]);
        }
        float zero[V] = {};
        for (int t = stop; t < c.tokens; ++t, y += a.y_token) put(y, V, zero);
    }
}

// Gradients.  With g = dy silu'(pre):  dx[s] = sum over k < W of weight[W-1-k] g[s+k],  dweight[W-1-k] += g[t] x~[t-k],
// dbias += g, each only where both tokens lie in one episode.  pre is formed again from x.  A run goes forwards over its
// tokens and the W - 1 behind them (those need g too), keeps the last four tokens' x and g, and at token t finishes dx of
// token t - (W-1).  Tokens behind the row's end count as g = 0.  The sums over tokens stay in registers over all of a
// thread's runs and leave through one record per workgroup.
template <class T, int W, int V>
__global__ __launch_bounds__(kConvThreads, 2) void k_conv_backward(ConvArgs a) {
    extern __shared__ float lds[];   // [slots][lanes][V][W + 1]
    const int lane = threadIdx.x % a.lanes, slot = threadIdx.x / a.lanes;
    const int slots = kConvThreads / a.lanes;
    const int64_t d_lane = ((int64_t)blockIdx.y * a.lanes + lane) * V, d = d_lane < a.D - V ? d_lane : a.D - V;
    const bool live = slot < slots && d_lane < a.D;
    const int64_t runs = (a.L + a.run - 1) / a.run;
    float w[V * W] = {}, bias[V] = {}, dw[V * W], db[V];
    if (live) conv_taps<W, V>(a, d, V, w, bias);
#pragma unroll
    for (int i = 0; i < V * W; ++i) dw[i] = 0.0f;
#pragma unroll
    for (int v = 0; v < V; ++v) db[v] = 0.0f;
    for (int64_t r = (int64_t)blockIdx.x * slots + slot; live && r < a.B * runs; r += (int64_t)gridDim.x * slots) {
        const ConvRun c = conv_run_of(a, r);
        const int own = c.tokens < c.real ? c.tokens : c.real;              // tokens whose g counts for dweight here
        T* dx = (T*)a.dx + c.b * a.dx_row + c.l0 * a.dx_token + d;          // of the token to be finished next
        if (own > 0 || c.l0 == 0) {
            const int last = own + W - 1;                                   // one behind the last token gone over
            const int stop = last < c.real ? last : c.real;
            const int state_from = c.n - c.l0 < 2 * a.run ? (int)(c.n - c.l0) - (W - 1) : 2 * a.run;   // first of the row's last W - 1
            const T* x = (const T*)a.x + c.b * a.x_row + c.l0 * a.x_token + d;
            const T* dy = (const T*)a.dy + c.b * a.dy_row + c.l0 * a.dy_token + d;
            const uint8_t* start = a.start ? a.start + c.b * a.start_row + c.l0 * a.start_token : nullptr;
            Raw<T, V> ahead[kConvAhead], gahead[kConvAhead];
            uint8_t marks[kConvAhead];
            auto ask = [&](int i, int t) {      // token t, i behind the group's first
                const int at = i % kConvAhead;
                ahead[at] = gahead[at] = {};
                marks[at] = 0;
                if (t < stop) {
                    fetch(ahead[at], x + i * a.x_token, V);
                    fetch(gahead[at], dy + i * a.dy_token, V);
                    if (start) marks[at] = start[i * a.start_token];
                }
            };
#pragma unroll
            for (int i = 0; i < kConvAhead; ++i) ask(i, i);
            float win[W - 1][V], xs[4][V], gs[4][V];
            conv_halo<T, W, V>(a, c.b, c.l0, d, win);
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) xs[k][v] = gs[k][v] = 0.0f;
#pragma unroll
            for (int k = 0; k < W - 1; ++k)
#pragma unroll
                for (int v = 0; v < V; ++v) xs[4 - (W - 1) + k][v] = win[k][v];
            unsigned opened = 0;      // bit j: the token j before the current one opened an episode
#pragma unroll 1
            for (int t0 = 0; t0 < last; t0 += kConvAhead) {
#pragma unroll
                for (int i = 0; i < kConvAhead; ++i) {
                    const int t = t0 + i;
                    if (t < last) {
                        opened = opened << 1 | (marks[i] ? 1u : 0u);
                        if (marks[i]) {
#pragma unroll
                            for (int k = 1; k < 4; ++k)
#pragma unroll
                                for (int v = 0; v < V; ++v) xs[(i + k) % 4][v] = 0.0f;
                        }
                        float out[V];
#pragma unroll
                        for (int v = 0; v < V; ++v) xs[i][v] = ahead[i].at(v), out[v] = gahead[i].at(v);
                        ask(i + kConvAhead, t + kConvAhead);          // into the place this token has left
#pragma unroll
                        for (int v = 0; v < V; ++v) {
                            float g = out[v];
                            if (a.silu) {
                                const float pre = conv_pre<W, V>(xs, w, bias, i, v), s = sigmoid_f<T>(pre);
                                g *= s * fmaf(pre, 1.0f - s, 1.0f);
                            }
                            gs[i][v] = t < c.real ? g : 0.0f;
                        }
                        // (those behind `own` are left out: 0 times an x that is infinite would be no 0)
                        if (t < own) {
#pragma unroll
                            for (int v = 0; v < V; ++v) {
                                db[v] += gs[i][v];
#pragma unroll
                                for (int k = 0; k < W; ++k) dw[v * W + k] = fmaf(gs[i][v], xs[(i + 4 - (W - 1) + k) % 4][v], dw[v * W + k]);
                            }
                        }
                        // dx of token s = t - (W-1), whose g lies in place (i + 5 - W) % 4; token s + k's start is bit W-1-k
                        const int s = t - (W - 1);
                        const unsigned between = opened & ((1u << (W - 1)) - 1);
#pragma unroll
                        for (int v = 0; v < V; ++v) out[v] = w[v * W + W - 1] * gs[(i + 5 - W) % 4][v];
                        if (between == 0) {
#pragma unroll
                            for (int v = 0; v < V; ++v)
#pragma unroll
                                for (int k = 1; k < W; ++k) out[v] = fmaf(w[v * W + W - 1 - k], gs[(i + 5 - W + k) % 4][v], out[v]);
                        } else {
#pragma unroll
                            for (int k = 1; k < W; ++k)
                                if ((between >> (W - 1 - k)) == 0) {
#pragma unroll
                                    for (int v = 0; v < V; ++v) out[v] = fmaf(w[v * W + W - 1 - k], gs[(i + 5 - W + k) % 4][v], out[v]);
                                }
                        }
                        // the handed-on state is a copy of the row's last W - 1 tokens, as far as no episode starts behind them
                        if (a.dnew_state && s >= state_from && (between >> (s - state_from + 1)) == 0) {
                            Raw<T, V> g1;
                            fetch(g1, (const T*)a.dnew_state + (c.b * (W - 1) + (s - state_from)) * a.D + d, V);
#pragma unroll
                            for (int v = 0; v < V; ++v) out[v] += g1.at(v);
                        }
                        if (s >= 0) {
                            if (s < own) {
                                put(dx, V, out);
                                dx += a.dx_token;
                            }
                        } else if (c.l0 == 0 && a.dstate) {
                            put((T*)a.dstate + (c.b * (W - 1) + (s + W - 1)) * a.D + d, V, out);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                x += kConvAhead * a.x_token;
                dy += kConvAhead * a.dy_token;
                if (start) start += kConvAhead * a.start_token;
            }
        }
        float zero[V] = {};
        for (int t = own > 0 ? own : 0; t < c.tokens; ++t, dx += a.dx_token) put(dx, V, zero);
    }
    if (!a.partial) return;
    constexpr int K = W + 1;
    if (live) {
        // (channel d_lane + v, that is; those of the last lane that its neighbour has too fall to the neighbour)
        float* const mine = lds + (size_t)(slot * a.lanes + lane) * V * K;
        const int shared = (int)(d_lane - d);
#pragma unroll
        for (int v = 0; v < V; ++v)
            if (v >= shared) {
#pragma unroll
                for (int j = 0; j < W; ++j) mine[(v - shared) * K + j] = dw[v * W + j];
                mine[(v - shared) * K + W] = db[v];
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
            out[v] = a.silu ? pre * sigmoid_f<T>(pre) : pre;
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) put((T*)a.new_state + (b * (W - 1) + k) * a.D + d, count, win[k + 1]);
        put((T*)a.y + b * a.y_row + d, count, out);
    }
}

}  // namespace seq
}  // namespace auv
