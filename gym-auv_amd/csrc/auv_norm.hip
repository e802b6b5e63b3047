// auv_residual_norm: checks, launch rules and launches of auv_norm.hpp.
#include "auv_seq_host.hpp"

#include <cfloat>

#include "auv_norm.hpp"

namespace auv {
namespace seq {
namespace {

int64_t lanes_of(int64_t channels) {
    for (int64_t lanes : {4, 8, 16, 32, 64, 256})
        if (channels <= lanes * kNormLane) return lanes;
    return 1024;
}
int64_t rows_of(int64_t lanes) { return lanes < 256 ? 256 / lanes : 1; }

// Workgroups of a backward pass: each leaves one record of column sums, so a workgroup takes many rows.  512 of 256
// threads are two per CU, all that the registers hold (262,144 rows of 250 channels, forward and backward: 450 us; with
// 768, the last of which start when the first end, 455 us, with 256 440 us; 16,384 rows of 1,024 channels 172, 171 and 175
// us).  256 of 1,024 threads are one per CU (8,192 rows of 4,096 channels 631 us; 128 857 us, 512 653 us).
int64_t back_blocks(int64_t rows, int64_t channels) {
    const int64_t lanes = lanes_of(channels), want = ceil_div(rows, rows_of(lanes)), cap = lanes == 1024 ? 256 : 512;
    return want < cap ? want : cap;
}

int check(const auv_norm_args& p, int32_t pass) {
    const char* who = "auv_residual_norm";
    if (pass != AUV_SEQ_FORWARD && pass != AUV_SEQ_BACKWARD) return seq_fail(AUV_ERR_ARG, "%s: unknown pass %d", who, pass);
    if (const int rc = check_rows(who, p.batch, p.length, p.channels, p.device, p.dtype)) return rc;
    if (p.residual_dtype != p.dtype && p.residual_dtype != AUV_F32)
        return seq_fail(AUV_ERR_ARG, "%s: the residual stream is f32 or of the block's type", who);
    if (p.channels > AUV_NORM_MAX_CHANNELS)
        return seq_fail(AUV_ERR_ARG, "%s: at most %d channels, got %lld", who, AUV_NORM_MAX_CHANNELS, (long long)p.channels);
    // (as a normal number of 32 bits: a row of zeros rests on it)
    if (!((float)p.eps >= FLT_MIN)) return seq_fail(AUV_ERR_ARG, "%s: eps must be positive in 32 bits", who);
    if (p.gate_act < AUV_GATE_PLAIN || p.gate_act > AUV_GATE_SIGMOID) return seq_fail(AUV_ERR_ARG, "%s: unknown gate activation", who);
    return AUV_OK;
}

template <class TR, class T, int TPR>
int launch(const auv_norm_args& p, int32_t pass, NormArgs a, int64_t blocks, hipStream_t stream) {
    constexpr int TH = norm_threads<TPR>();
    if (pass == AUV_SEQ_FORWARD) {
        return in_slices(blocks, TH, [&](int64_t first, int64_t count) {
            a.first = first;
            hipLaunchKernelGGL((k_norm_forward<TR, T, TPR>), dim3((unsigned)count), dim3(TH), 0, stream, a);
            return launched("k_norm_forward");
        });
    }
    hipLaunchKernelGGL((k_norm_backward<TR, T, TPR>), dim3((unsigned)blocks), dim3(TH), 0, stream, a);
    if (const int rc = launched("k_norm_backward")) return rc;
    if (!a.partial) return AUV_OK;
    SumArgs s{};
    s.src = a.partial;
    s.slices = blocks;
    s.stride = s.count = p.channels * 3;
    s.inner = 3;
    s.n[0] = s.n[1] = s.n[2] = 1;
    s.dst[0] = p.d_post_weight, s.dst[1] = p.d_pre_weight, s.dst[2] = p.d_scale;
    return in_slices(ceil_div(s.count, kSumOutputs), kSumOutputs * kSumLanes, [&](int64_t first, int64_t count) {
        s.first = first;
        hipLaunchKernelGGL(k_seq_sum, dim3((unsigned)count), dim3(kSumOutputs * kSumLanes), 0, stream, s);
        return launched("k_seq_sum");
    });
}

template <class TR, class T>
int by_shape(const auv_norm_args& p, int32_t pass, const NormArgs& a, int64_t blocks, hipStream_t stream) {
    switch (lanes_of(p.channels)) {
        case 4: return launch<TR, T, 4>(p, pass, a, blocks, stream);
        case 8: return launch<TR, T, 8>(p, pass, a, blocks, stream);
        case 16: return launch<TR, T, 16>(p, pass, a, blocks, stream);
        case 32: return launch<TR, T, 32>(p, pass, a, blocks, stream);
        case 64: return launch<TR, T, 64>(p, pass, a, blocks, stream);
        case 256: return launch<TR, T, 256>(p, pass, a, blocks, stream);
        default: return launch<TR, T, 1024>(p, pass, a, blocks, stream);
    }
}
}  // namespace
}  // namespace seq
}  // namespace auv

using namespace auv::seq;

extern "C" {

int64_t auv_residual_norm_workspace(const auv_norm_args* p, int32_t pass) {
    if (!p) return seq_fail(AUV_ERR_ARG, "auv_residual_norm_workspace: null argument");
    if (const int rc = check(*p, pass)) return rc;
    if (pass == AUV_SEQ_FORWARD || p->batch == 0 || p->length == 0) return 0;
    return back_blocks(p->batch * p->length, p->channels) * p->channels * 3 * (int64_t)sizeof(float);
}

int auv_residual_norm(const auv_norm_args* p, int32_t pass, void* stream) {
    if (!p) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: null argument");
    if (const int rc = check(*p, pass)) return rc;
    if (p->batch == 0 || p->length == 0) {
        if (pass == AUV_SEQ_BACKWARD) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: nothing to do for an empty batch");
        return AUV_OK;
    }
    if (!p->x) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: null x");
    if (!p->y && (p->gate || p->scale || p->post_weight))
        return seq_fail(AUV_ERR_ARG, "auv_residual_norm: gate, scale and post_weight belong to y, which is absent");
    if (pass == AUV_SEQ_FORWARD) {
        if ((p->y != nullptr) != (p->x_out != nullptr)) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: x_out goes with y");
        if ((p->pre_weight != nullptr) != (p->h != nullptr)) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: h goes with pre_weight");
        if (!p->x_out && !p->h) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: neither y nor pre_weight");
    } else {
        if (!p->d_x || (p->y && !p->d_y) || (p->gate && !p->d_gate)) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: null gradient");
        if (!p->d_x_out && !p->d_h) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: neither d_x_out nor d_h");
        if (p->d_h && !p->pre_weight) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: d_h goes with pre_weight");
    }
    const int64_t rows = p->batch * p->length;
    const bool sums = pass == AUV_SEQ_BACKWARD && (p->d_post_weight || p->d_pre_weight || p->d_scale);
    const int64_t blocks = pass == AUV_SEQ_FORWARD ? ceil_div(rows, rows_of(lanes_of(p->channels))) : back_blocks(rows, p->channels);
    if (blocks > 0x7fffffff) return seq_fail(AUV_ERR_ARG, "auv_residual_norm: too many rows");
    if (sums && (!p->workspace || p->workspace_bytes < blocks * p->channels * 3 * (int64_t)sizeof(float)))
        return seq_fail(AUV_ERR_MEMORY, "auv_residual_norm: the workspace holds %lld bytes, too few", (long long)p->workspace_bytes);
    DeviceScope scope(p->device);
    if (!scope.ok()) return seq_fail(AUV_ERR_DEVICE, "auv_residual_norm: no HIP device %lld", (long long)p->device);
    NormArgs a{};
    a.B = p->batch, a.L = p->length, a.D = p->channels;
    a.x = p->x, a.x_row = p->x_row, a.x_token = p->x_token;
    a.y = p->y, a.y_row = p->y_row, a.y_token = p->y_token;
    a.gate = p->gate, a.gate_row = p->gate_row, a.gate_token = p->gate_token;
    a.post_weight = p->post_weight, a.pre_weight = p->pre_weight, a.scale = p->scale;
    a.eps = (float)p->eps;
    a.act = (int32_t)p->gate_act;
    a.x_out = p->x_out, a.x_out_row = p->x_out_row, a.x_out_token = p->x_out_token;
    a.h_out = p->h, a.h_row = p->h_row, a.h_token = p->h_token;
    a.gx = p->d_x_out, a.gx_row = p->d_x_out_row, a.gx_token = p->d_x_out_token;
    a.gh = p->d_h, a.gh_row = p->d_h_row, a.gh_token = p->d_h_token;
    a.dx = p->d_x, a.dx_row = p->d_x_row, a.dx_token = p->d_x_token;
    a.dy = p->d_y, a.dy_row = p->d_y_row, a.dy_token = p->d_y_token;
    a.dgate = p->d_gate, a.dgate_row = p->d_gate_row, a.dgate_token = p->d_gate_token;
    a.partial = sums ? (float*)p->workspace : nullptr;
    const hipStream_t st = (hipStream_t)stream;
    if (p->dtype == AUV_F32) return by_shape<float, float>(*p, pass, a, blocks, st);
    if (p->dtype == AUV_BF16)
        return p->residual_dtype == AUV_F32 ? by_shape<float, bf16>(*p, pass, a, blocks, st) : by_shape<bf16, bf16>(*p, pass, a, blocks, st);
    return p->residual_dtype == AUV_F32 ? by_shape<float, f16>(*p, pass, a, blocks, st) : by_shape<f16, f16>(*p, pass, a, blocks, st);
}

}  // extern "C"
