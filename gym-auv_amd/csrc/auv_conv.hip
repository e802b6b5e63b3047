// auv_causal_conv: checks, launch rules and launches of auv_conv.hpp.
#include "auv_seq_host.hpp"

#include "auv_conv.hpp"

namespace auv {
namespace seq {
namespace {
thread_local char g_seq_error[512];

// Tokens per thread.  A run re-reads the W - 1 tokens before it, so long runs read less; short ones give a small batch
// more threads.  Runs of 32 wherever that leaves two waves per SIMD of the 256 CUs (131,072 threads), down to 8.  4,096
// rows x 128 tokens x 128 channels, bf16, forwards and backwards: 167 us in runs of 32, 190 in runs of 16, 214 in runs of 8
// (156 in runs of 64); 5 rows of up to 4,001 tokens x 90 channels forwards: 15.7, 9.8 and 7.0 us.
int conv_run(int64_t B, int64_t L, int64_t vectors) {
    int run = 32;
    while (run > 8 && B * ceil_div(L, run) * vectors < 131072) run /= 2;
    return run;
}

// Records of a backward pass (each the sums of one workgroup over its runs): enough workgroups to fill the chip, few
// enough that the records stay small beside the activations.
int64_t conv_records(int64_t channels) {
    const int64_t most = ((int64_t)1 << 20) / channels;
    return most < 1 ? 1 : most > 2048 ? 2048 : most;
}

struct Plan {
    int64_t V, lanes, grid_x, grid_y;
    int run;
};

Plan conv_plan(const auv_conv_args& p, int32_t pass) {
    Plan r;
    r.V = 16 / type_size(p.dtype);
    if (pass != AUV_SEQ_STEP && p.channels < r.V) r.V = 1;
    const int64_t vectors = ceil_div(p.channels, r.V);
    r.run = conv_run(p.batch, p.length, vectors);
    r.lanes = vectors < kConvThreads ? vectors : kConvThreads;
    r.grid_y = ceil_div(vectors, r.lanes);
    const int64_t slots = kConvThreads / r.lanes;
    const int64_t want = ceil_div(p.batch * ceil_div(p.length, r.run), slots);
    // forwards: a workgroup per set of runs; backwards a workgroup takes several, because each leaves a record of sums;
    // a step's takes several rows, because it loads its taps first (65,536 rows of 128 channels: 23.8 us, 25.1 us with a
    // workgroup for every 16 rows)
    const int64_t cap = pass == AUV_SEQ_BACKWARD ? conv_records(p.channels) : pass == AUV_SEQ_STEP ? 1024 : (int64_t)1 << 22;
    r.grid_x = want < cap ? want : cap;
    return r;
}

int check(const auv_conv_args& p, int32_t pass) {
    const char* who = "auv_causal_conv";
    if (pass < AUV_SEQ_FORWARD || pass > AUV_SEQ_STEP) return seq_fail(AUV_ERR_ARG, "%s: unknown pass %d", who, pass);
    if (const int rc = check_rows(who, p.batch, p.length, p.channels, p.device, p.dtype)) return rc;
    if (p.width < 2 || p.width > 4) return seq_fail(AUV_ERR_ARG, "%s: width must be 2, 3 or 4, got %lld", who, (long long)p.width);
    if (pass == AUV_SEQ_STEP && p.length != 1) return seq_fail(AUV_ERR_ARG, "%s: a step takes one token per row", who);
    if (p.channels > (int64_t)256 * 4 * 65535) return seq_fail(AUV_ERR_ARG, "%s: too many channels", who);
    return AUV_OK;
}

template <class T, int W, int V>
int launch(const auv_conv_args& p, int32_t pass, const Plan& r, ConvArgs a, hipStream_t stream) {
    const dim3 grid((unsigned)r.grid_x, (unsigned)r.grid_y), block(kConvThreads);
    if (pass == AUV_SEQ_FORWARD) {
        hipLaunchKernelGGL((k_conv_forward<T, W, V>), grid, block, 0, stream, a);
        return launched("k_conv_forward");
    }
    if (pass == AUV_SEQ_STEP) {
        hipLaunchKernelGGL((k_conv_step<T, W>), grid, block, 0, stream, a);
        return launched("k_conv_step");
    }
    const size_t lds = (size_t)(kConvThreads / r.lanes) * r.lanes * V * (W + 1) * sizeof(float);
    hipLaunchKernelGGL((k_conv_backward<T, W, V>), grid, block, lds, stream, a);
    if (const int rc = launched("k_conv_backward")) return rc;
    if (!a.partial) return AUV_OK;
    SumArgs s{};
    s.src = a.partial;
    s.slices = r.grid_x;
    s.stride = s.count = p.channels * (W + 1);
    s.inner = W + 1;
    s.n[0] = W;
    s.n[1] = 1;
    s.dst[0] = p.d_weight;
    s.dst[1] = p.d_bias;
    return in_slices(ceil_div(s.count, kSumOutputs), kSumOutputs * kSumLanes, [&](int64_t first, int64_t count) {
        s.first = first;
        hipLaunchKernelGGL(k_seq_sum, dim3((unsigned)count), dim3(kSumOutputs * kSumLanes), 0, stream, s);
        return launched("k_seq_sum");
    });
}

template <class T, int W>
int by_vector(const auv_conv_args& p, int32_t pass, const Plan& r, const ConvArgs& a, hipStream_t stream) {
    return r.V == 1 ? launch<T, W, 1>(p, pass, r, a, stream) : launch<T, W, conv_vector<T>()>(p, pass, r, a, stream);
}
template <class T>
int by_width(const auv_conv_args& p, int32_t pass, const Plan& r, const ConvArgs& a, hipStream_t stream) {
    if (p.width == 2) return by_vector<T, 2>(p, pass, r, a, stream);
    return p.width == 3 ? by_vector<T, 3>(p, pass, r, a, stream) : by_vector<T, 4>(p, pass, r, a, stream);
}
}  // namespace

int seq_fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(g_seq_error, sizeof g_seq_error, fmt, ap);
    va_end(ap);
    return code;
}
}  // namespace seq
}  // namespace auv

using namespace auv::seq;

extern "C" {

const char* auv_seq_last_error(void) { return g_seq_error; }

int64_t auv_causal_conv_workspace(const auv_conv_args* p, int32_t pass) {
    if (!p) return seq_fail(AUV_ERR_ARG, "auv_causal_conv_workspace: null argument");
    if (const int rc = check(*p, pass)) return rc;
    if (pass != AUV_SEQ_BACKWARD || p->batch == 0 || p->length == 0) return 0;
    return conv_plan(*p, pass).grid_x * p->channels * (p->width + 1) * (int64_t)sizeof(float);
}

int auv_causal_conv(const auv_conv_args* p, int32_t pass, void* stream) {
    if (!p) return seq_fail(AUV_ERR_ARG, "auv_causal_conv: null argument");
    if (const int rc = check(*p, pass)) return rc;
    if (!p->weight) return seq_fail(AUV_ERR_ARG, "auv_causal_conv: null weight");
    const bool empty = p->batch == 0 || p->length == 0;
    if (!empty && !p->x) return seq_fail(AUV_ERR_ARG, "auv_causal_conv: null x");
    if (empty) {
        if (pass == AUV_SEQ_BACKWARD || p->new_state) return seq_fail(AUV_ERR_ARG, "auv_causal_conv: nothing to do for an empty batch");
        return AUV_OK;
    }
    if (pass != AUV_SEQ_BACKWARD && !p->y) return seq_fail(AUV_ERR_ARG, "auv_causal_conv: null y");
    if (pass == AUV_SEQ_STEP && (!p->state || !p->new_state)) return seq_fail(AUV_ERR_ARG, "auv_causal_conv: a step needs state and new_state");
    if (pass == AUV_SEQ_FORWARD && p->new_state && p->new_state == p->state)
        return seq_fail(AUV_ERR_ARG, "auv_causal_conv: new_state must not be state's memory");
    if (pass == AUV_SEQ_BACKWARD && (!p->d_y || !p->d_x)) return seq_fail(AUV_ERR_ARG, "auv_causal_conv: null d_y or d_x");
    const bool sums = pass == AUV_SEQ_BACKWARD && (p->d_weight || p->d_bias);
    const Plan r = conv_plan(*p, pass);
    if (sums && (!p->workspace || p->workspace_bytes < r.grid_x * p->channels * (p->width + 1) * (int64_t)sizeof(float)))
        return seq_fail(AUV_ERR_MEMORY, "auv_causal_conv: the workspace holds %lld bytes, too few", (long long)p->workspace_bytes);
    DeviceScope scope(p->device);
    if (!scope.ok()) return seq_fail(AUV_ERR_DEVICE, "auv_causal_conv: no HIP device %lld", (long long)p->device);
    ConvArgs a{};
    a.B = p->batch, a.L = p->length, a.D = p->channels;
    a.x = p->x, a.x_row = p->x_row, a.x_token = p->x_token;
    a.weight = p->weight, a.bias = p->bias;
    a.start = p->start, a.start_row = p->start_row, a.start_token = p->start_token;
    a.lengths = p->lengths;
    a.state = p->state, a.new_state = p->new_state;
    a.y = p->y, a.y_row = p->y_row, a.y_token = p->y_token;
    a.dy = p->d_y, a.dy_row = p->d_y_row, a.dy_token = p->d_y_token;
    a.dnew_state = p->d_new_state;
    a.dx = p->d_x, a.dx_row = p->d_x_row, a.dx_token = p->d_x_token;
    a.dstate = p->d_state;
    a.partial = sums ? (float*)p->workspace : nullptr;
    a.silu = p->silu != 0;
    a.run = r.run, a.lanes = (int32_t)r.lanes;
    const hipStream_t st = (hipStream_t)stream;
    if (p->dtype == AUV_F32) return by_width<float>(*p, pass, r, a, st);
    return p->dtype == AUV_BF16 ? by_width<bf16>(*p, pass, r, a, st) : by_width<f16>(*p, pass, r, a, st);
}

}  // extern "C"
