// auv_selective_scan: checks, launch rules and launches of auv_scan.hpp.
#include "auv_seq_host.hpp"

#include <atomic>

#include "auv_scan.hpp"

namespace auv {
namespace seq {
namespace {

constexpr int64_t kMaxGrid = 0x7fffffff;   // waves, numbered in 32 bits, and workgroups, over all launches of a kernel

// States are padded to 4, 8, 16, 32 or 64: lanes per channel of the backward and step kernels, four states each.
int lanes_of(int64_t states) { return states <= 4 ? 1 : states <= 8 ? 2 : states <= 16 ? 4 : states <= 32 ? 8 : 16; }

int64_t tiles_of(const auv_scan_args& p, int64_t lanes) { return ceil_div(p.channels / p.groups, 64 / lanes); }

struct Chunks {
    int64_t length, count;
};
// Splits the time axis when the rows alone leave the chip short of waves: fewer than `enough`, which is one wave per SIMD
// of the 256 CUs forwards and two backwards.  A split pays for itself only when it brings at least three chunks: every
// element is then gone over twice.  16 states, 128 channels, 512 tokens, bf16: forwards 64 rows 64 us in chunks and 84 whole,
// 128 rows (1,024 waves) 106 and 85; forwards and backwards 128 rows 327 us with the backward pass in chunks and 486 whole,
// 192 rows (1,536 waves) 537 and 511.
Chunks split(int64_t L, int64_t waves, int64_t enough) {
    constexpr int64_t kTarget = 4096;   // four waves per SIMD (10,075 tokens x 128 forwards: 35.6 us, 34.7 for two, 38.7 for eight)
    if (waves >= enough || waves == 0 || L == 0) return {L, 1};     // (an empty batch has no waves)
    const int64_t want = ceil_div(kTarget, waves);
    int64_t length = ceil_div(ceil_div(L, want), kSegment) * kSegment;
    const int64_t count = ceil_div(L, length);
    return count < 3 ? Chunks{L, 1} : Chunks{length, count};
}

struct Forward {
    // four states per lane instead of sixteen: four times the waves for small batches.  16 states, 128 channels, 512 tokens,
    // bf16: 512 rows 179 us narrow, 249 us wide; 768 rows 272 and 321; 1,024 rows (two wide waves per SIMD) 344 and 324.
    bool narrow;
    int64_t waves;   // without chunks
    Chunks chunks;
};
Forward forward_plan(const auv_scan_args& p) {
    const int S = lanes_of(p.states);
    Forward f;
    const int64_t wide = tiles_of(p, S > 4 ? S / 4 : 1) * p.groups * p.batch;
    f.narrow = S > 1 && wide < 2048;
    f.waves = f.narrow ? tiles_of(p, S) * p.groups * p.batch : wide;
    f.chunks = split(p.length, f.waves, 1024);
    return f;
}

struct Backward {
    int64_t per, units, blocks, grid_x, grid_y;   // as in k_scan_backward
    Chunks chunks;
    int64_t chunk_bytes, record_bytes, bc_bytes;
};
Backward backward_plan(const auv_scan_args& p) {
    const int S = lanes_of(p.states);
    const int64_t waves = S <= 4 ? 8 : 4 /* scan_back_waves */, tiles = tiles_of(p, S);
    Backward r;
    r.per = tiles < waves ? tiles : waves;
    r.units = waves / r.per;
    r.blocks = ceil_div(tiles, r.per);
    r.grid_y = r.blocks * p.groups;
    const int64_t groups = ceil_div(p.batch, r.units);
    r.chunks = split(p.length, groups * r.grid_y * waves, 2048);
    // each workgroup leaves one record of sums per row it works on side by side: as many as fill the chip, not more
    // (4,096 rows x 64 tokens x 128 channels, 16 states, forwards and backwards: 825 us; with half of them 838, with twice as
    // many 822, with four times 836)
    const int64_t cap = r.grid_y < 1024 ? 1024 / r.grid_y : 1;
    r.grid_x = groups * r.chunks.count < cap ? groups * r.chunks.count : cap;
    const int64_t NP = 4 * S;
    r.chunk_bytes = r.chunks.count > 1 ? 2 * r.chunks.count * p.batch * p.channels * NP * 4 : 0;
    r.record_bytes = r.grid_x * r.units * p.channels * (p.states + 2) * 4;
    r.bc_bytes = r.blocks > 1 ? r.blocks * p.batch * p.length * p.groups * 2 * NP * 4 : 0;
    return r;
}

int check(const auv_scan_args& p, int32_t pass) {
    const char* who = "auv_selective_scan";
    if (pass < AUV_SEQ_FORWARD || pass > AUV_SEQ_STEP) return seq_fail(AUV_ERR_ARG, "%s: unknown pass %d", who, pass);
    if (const int rc = check_rows(who, p.batch, p.length, p.channels, p.device, p.dtype)) return rc;
    if (p.states < 1 || p.states > 64) return seq_fail(AUV_ERR_ARG, "%s: states must be in 1..64, got %lld", who, (long long)p.states);
    if (p.groups < 1 || p.channels % p.groups)
        return seq_fail(AUV_ERR_ARG, "%s: %lld groups do not divide %lld channels", who, (long long)p.groups, (long long)p.channels);
    if (pass == AUV_SEQ_STEP && p.length != 1) return seq_fail(AUV_ERR_ARG, "%s: a step takes one token per row", who);
    if (pass == AUV_SEQ_BACKWARD && backward_plan(p).grid_y > 65535) return seq_fail(AUV_ERR_ARG, "%s: too many channels or groups", who);
    return AUV_OK;
}

ScanArgs fill(const auv_scan_args& p) {
    ScanArgs a{};
    a.B = p.batch, a.L = p.length, a.D = p.channels, a.G = p.groups;
    a.N = (int32_t)p.states, a.softplus = p.softplus != 0;
    a.u = p.u, a.u_row = p.u_row, a.u_token = p.u_token;
    a.delta = p.delta, a.delta_row = p.delta_row, a.delta_token = p.delta_token;
    a.z = p.z, a.z_row = p.z_row, a.z_token = p.z_token;
    a.Bm = p.B, a.B_row = p.B_row, a.B_token = p.B_token, a.B_group = p.B_group;
    a.Cm = p.C, a.C_row = p.C_row, a.C_token = p.C_token, a.C_group = p.C_group;
    a.A = p.A, a.Dv = p.D, a.bias = p.delta_bias;
    a.start = p.start, a.start_row = p.start_row, a.start_token = p.start_token;
    a.lengths = p.lengths;
    a.state = p.state, a.new_state = p.new_state;
    a.y = p.y, a.y_row = p.y_row, a.y_token = p.y_token;
    a.segments = p.segments;
    a.dy = p.d_y, a.dy_row = p.d_y_row, a.dy_token = p.d_y_token;
    a.dnew_state = p.d_new_state;
    a.du = p.d_u, a.du_row = p.d_u_row, a.du_token = p.d_u_token;
    a.ddelta = p.d_delta, a.ddelta_row = p.d_delta_row, a.ddelta_token = p.d_delta_token;
    a.dz = p.d_z, a.dz_row = p.d_z_row, a.dz_token = p.d_z_token;
    a.dB = p.d_B, a.dB_row = p.d_B_row, a.dB_token = p.d_B_token, a.dB_group = p.d_B_group;
    a.dC = p.d_C, a.dC_row = p.d_C_row, a.dC_token = p.d_C_token, a.dC_group = p.d_C_group;
    a.dstate = p.d_state;
    return a;
}

int join(const ScanArgs& a, int NP, bool reverse, hipStream_t stream) {
    JoinArgs j{};
    j.chunk_state = a.chunk_state, j.chunk_decay = a.chunk_decay;
    j.first = reverse ? a.dnew_state : a.state;
    j.last = reverse ? a.dstate : nullptr;
    j.chunks = a.chunks, j.count = a.B * a.D * NP;
    j.N = a.N, j.NP = NP, j.reverse = reverse;
    // 64 numbers a workgroup, or 16 where they are few and the chunks enough for four in each of its 64 rows.  Whole forward
    // passes of 315 chunks: 1,024 numbers 29.1 us in 16s and 35.8 in 64s, 2,048 numbers 35.3 and 36.3; of 256 chunks: 512
    // numbers 23.2 and 29.2, 4,096 numbers 33.6 and 31.9, 8,192 numbers 59.2 and 54.9; of 63 chunks: 5,040 numbers 24.5 and 21.4
    if (j.count < 4096 && j.chunks >= 4 * 64) hipLaunchKernelGGL(k_scan_join<16>, dim3((unsigned)ceil_div(j.count, 16)), dim3(kJoinThreads), 0, stream, j);
    else hipLaunchKernelGGL(k_scan_join<64>, dim3((unsigned)ceil_div(j.count, 64)), dim3(kJoinThreads), 0, stream, j);
    return launched("k_scan_join");
}

template <class T, int NPL, int S>
int run_forward(ScanArgs a, const Forward& f, hipStream_t stream) {
    const int64_t blocks = ceil_div(f.waves * f.chunks.count, kScanWaves);
    const dim3 block(kScanWaves * 64);
    if (f.chunks.count > 1) {       // (there are few waves then)
        hipLaunchKernelGGL((k_scan_forward<T, NPL, S, 1>), dim3((unsigned)blocks), block, 0, stream, a);
        if (const int rc = launched("k_scan_forward")) return rc;
        if (const int rc = join(a, NPL * S, false, stream)) return rc;
    }
    return in_slices(blocks, kScanWaves * 64, [&](int64_t first, int64_t count) {
        a.first = first;
        hipLaunchKernelGGL((k_scan_forward<T, NPL, S, 0>), dim3((unsigned)count), block, 0, stream, a);
        return launched("k_scan_forward");
    });
}

template <class T, int S, bool TAIL>
int run_backward(ScanArgs a, const auv_scan_args& p, const Backward& r, hipStream_t stream) {
    static_assert(scan_back_lds<S>(scan_back_waves<S>()) <= 160 * 1024, "the tile's elements and sums must fit the CU's LDS");
    const size_t lds = scan_back_lds<S>((int)r.units);
    constexpr int threads = scan_back_waves<S>() * 64;
    static std::atomic<uint64_t> allowed{0};   // devices on which these kernels may take that much LDS
    const uint64_t bit = (uint64_t)1 << (p.device & 63);
    if (lds > 64 * 1024 && (p.device > 63 || !(allowed.load() & bit))) {
        for (const void* k : {reinterpret_cast<const void*>(&k_scan_backward<T, S, 0, TAIL>), reinterpret_cast<const void*>(&k_scan_backward<T, S, 1, true>)}) {
            const hipError_t e = hipFuncSetAttribute(k, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                     (int)scan_back_lds<S>(scan_back_waves<S>()));
            if (e != hipSuccess) return seq_fail(AUV_ERR_DEVICE, "k_scan_backward: %zu B of LDS refused: %s", lds, hipGetErrorString(e));
        }
        allowed.fetch_or(bit);
    }
    const dim3 grid((unsigned)r.grid_x, (unsigned)r.grid_y), block(threads);
    if (r.chunks.count > 1) {
        const dim3 all((unsigned)(ceil_div(a.B, r.units) * r.chunks.count), (unsigned)r.grid_y);
        hipLaunchKernelGGL((k_scan_backward<T, S, 1, true>), all, block, lds, stream, a);
        if (const int rc = launched("k_scan_backward")) return rc;
        if (const int rc = join(a, 4 * S, true, stream)) return rc;
    }
    hipLaunchKernelGGL((k_scan_backward<T, S, 0, TAIL>), grid, block, lds, stream, a);
    if (const int rc = launched("k_scan_backward")) return rc;
    if (a.bc_partial) {
        const int rc = in_slices(ceil_div(a.B * a.L * a.G * 2 * 4 * S, 256), 256, [&](int64_t first, int64_t count) {
            a.first = first;
            hipLaunchKernelGGL((k_scan_sum_bc<T>), dim3((unsigned)count), dim3(256), 0, stream, a, 4 * S, (int)r.blocks);
            return launched("k_scan_sum_bc");
        });
        if (rc) return rc;
    }
    SumArgs s{};
    s.src = a.partial;
    s.slices = r.grid_x * r.units;
    s.stride = s.count = a.D * (a.N + 2);
    s.inner = a.N + 2;
    s.n[0] = a.N, s.n[1] = s.n[2] = 1;
    s.dst[0] = p.d_A, s.dst[1] = p.d_D, s.dst[2] = p.d_delta_bias;
    return in_slices(ceil_div(s.count, kSumOutputs), kSumOutputs * kSumLanes, [&](int64_t first, int64_t count) {
        s.first = first;
        hipLaunchKernelGGL(k_seq_sum, dim3((unsigned)count), dim3(kSumOutputs * kSumLanes), 0, stream, s);
        return launched("k_seq_sum");
    });
}

template <class T, int S>
int by_tail(const ScanArgs& a, const auv_scan_args& p, const Backward& r, hipStream_t stream) {
    // (4,096 rows x 64 tokens x 128 channels, 16 states: 822 us without the masks for rows that end within a tile, 870 with)
    return p.lengths || p.length % kSegment ? run_backward<T, S, true>(a, p, r, stream) : run_backward<T, S, false>(a, p, r, stream);
}

template <class T, int S>
int run_step(ScanArgs a, hipStream_t stream) {
    const int64_t lanes = a.D * S < kStepThreads ? a.D * S : kStepThreads, tiles = ceil_div(a.D * S, lanes);
    a.lanes = (int32_t)lanes;
    // eight workgroups per CU, each with as many rows as it takes (65,536 rows of 64 channels, 16 states: 125 us; two per CU
    // 148 us; a workgroup for every row 168 us)
    const int64_t want = ceil_div(a.B, kStepThreads / lanes), most = ceil_div(2048, tiles);
    const dim3 grid((unsigned)(want < most ? want : most), (unsigned)tiles), block(kStepThreads);
    hipLaunchKernelGGL((k_scan_step<T, S>), grid, block, 0, stream, a);
    return launched("k_scan_step");
}

template <class T>
int by_states(const auv_scan_args& p, int32_t pass, ScanArgs a, hipStream_t stream) {
    const int S = lanes_of(p.states);
    if (pass == AUV_SEQ_STEP) {
        switch (S) {
            case 1: return run_step<T, 1>(a, stream);
            case 2: return run_step<T, 2>(a, stream);
            case 4: return run_step<T, 4>(a, stream);
            case 8: return run_step<T, 8>(a, stream);
            default: return run_step<T, 16>(a, stream);
        }
    }
    if (pass == AUV_SEQ_FORWARD) {
        const Forward f = forward_plan(p);
        a.chunk = f.chunks.length, a.chunks = f.chunks.count;
        a.chunk_state = (float*)p.workspace;
        a.chunk_decay = a.chunk_state + a.chunks * a.B * a.D * 4 * S;
        switch (S) {
            case 1: return run_forward<T, 4, 1>(a, f, stream);
            case 2: return f.narrow ? run_forward<T, 4, 2>(a, f, stream) : run_forward<T, 8, 1>(a, f, stream);
            case 4: return f.narrow ? run_forward<T, 4, 4>(a, f, stream) : run_forward<T, 16, 1>(a, f, stream);
            case 8: return f.narrow ? run_forward<T, 4, 8>(a, f, stream) : run_forward<T, 16, 2>(a, f, stream);
            default: return f.narrow ? run_forward<T, 4, 16>(a, f, stream) : run_forward<T, 16, 4>(a, f, stream);
        }
    }
    const Backward r = backward_plan(p);
    Width fours(4);
    fours.stride(a.D / a.G);
    for (const void* q : {a.u, a.delta, a.z, a.dy, (const void*)a.du, (const void*)a.ddelta, (const void*)a.dz}) fours.pointer(q, sizeof(T));
    if (a.B > 1)
        for (int64_t s : {a.u_row, a.delta_row, a.z_row, a.dy_row, a.du_row, a.ddelta_row, a.dz_row}) fours.stride(s);
    if (a.L > 1)
        for (int64_t s : {a.u_token, a.delta_token, a.z_token, a.dy_token, a.du_token, a.ddelta_token, a.dz_token}) fours.stride(s);
    a.whole = fours.elements() == 4;
    a.chunk = r.chunks.length, a.chunks = r.chunks.count;
    char* w = (char*)p.workspace;
    a.chunk_state = (float*)w;
    a.chunk_decay = (float*)(w + r.chunk_bytes / 2);
    a.partial = (float*)(w + r.chunk_bytes);
    a.bc_partial = r.bc_bytes ? (float*)(w + r.chunk_bytes + r.record_bytes) : nullptr;
    switch (S) {
        case 1: return by_tail<T, 1>(a, p, r, stream);
        case 2: return by_tail<T, 2>(a, p, r, stream);
        case 4: return by_tail<T, 4>(a, p, r, stream);
        case 8: return by_tail<T, 8>(a, p, r, stream);
        default: return by_tail<T, 16>(a, p, r, stream);
    }
}

int64_t workspace(const auv_scan_args& p, int32_t pass) {
    if (p.batch == 0 || p.length == 0 || pass == AUV_SEQ_STEP) return 0;
    if (pass == AUV_SEQ_FORWARD) {
        const Chunks c = forward_plan(p).chunks;
        return c.count > 1 ? 2 * c.count * p.batch * p.channels * 4 * lanes_of(p.states) * 4 : 0;
    }
    const Backward r = backward_plan(p);
    return r.chunk_bytes + r.record_bytes + r.bc_bytes;
}

int launches_fit(const auv_scan_args& p, int32_t pass) {
    const int S = lanes_of(p.states);
    // (states of 4 TiB would not fit the device either)
    int64_t most = p.batch * p.channels > ((int64_t)1 << 40) / p.states ? kMaxGrid + 1 : 0;
    if (pass == AUV_SEQ_STEP && ceil_div(p.channels * S, kStepThreads) > 65535) return seq_fail(AUV_ERR_ARG, "auv_selective_scan: too many channels");
    if (pass == AUV_SEQ_FORWARD) {
        const Forward f = forward_plan(p);
        if (f.waves * f.chunks.count > kMaxGrid) most = kMaxGrid + 1;   // numbered in 32 bits
    }
    if (pass == AUV_SEQ_BACKWARD) {
        const Backward r = backward_plan(p);
        if (r.bc_bytes && ceil_div(p.batch * p.length * p.groups * 8 * S, 256) > kMaxGrid) most = kMaxGrid + 1;
    }
    return most > kMaxGrid ? seq_fail(AUV_ERR_ARG, "auv_selective_scan: batch too large") : AUV_OK;
}
}  // namespace
}  // namespace seq
}  // namespace auv

using namespace auv::seq;

extern "C" {

int64_t auv_selective_scan_segments(const auv_scan_args* p) {
    if (!p) return seq_fail(AUV_ERR_ARG, "auv_selective_scan_segments: null argument");
    if (const int rc = check(*p, AUV_SEQ_FORWARD)) return rc;
    return p->batch * ceil_div(p->length, kSegment) * p->channels * 4 * lanes_of(p->states) * (int64_t)sizeof(float);
}

int64_t auv_selective_scan_workspace(const auv_scan_args* p, int32_t pass) {
    if (!p) return seq_fail(AUV_ERR_ARG, "auv_selective_scan_workspace: null argument");
    if (const int rc = check(*p, pass)) return rc;
    return workspace(*p, pass);
}

int auv_selective_scan(const auv_scan_args* p, int32_t pass, void* stream) {
    if (!p) return seq_fail(AUV_ERR_ARG, "auv_selective_scan: null argument");
    if (const int rc = check(*p, pass)) return rc;
    if (p->batch == 0 || p->length == 0) {
        if (pass == AUV_SEQ_BACKWARD || p->new_state) return seq_fail(AUV_ERR_ARG, "auv_selective_scan: nothing to do for an empty batch");
        return AUV_OK;
    }
    if (!p->u || !p->delta || !p->B || !p->C || !p->A) return seq_fail(AUV_ERR_ARG, "auv_selective_scan: null argument");
    if (pass != AUV_SEQ_BACKWARD && !p->y) return seq_fail(AUV_ERR_ARG, "auv_selective_scan: null y");
    if (pass == AUV_SEQ_STEP && (!p->state || !p->new_state)) return seq_fail(AUV_ERR_ARG, "auv_selective_scan: a step needs state and new_state");
    if (pass == AUV_SEQ_FORWARD && p->new_state && p->new_state == p->state)
        return seq_fail(AUV_ERR_ARG, "auv_selective_scan: new_state must not be state's memory");
    if (pass == AUV_SEQ_BACKWARD && (!p->segments || !p->d_y || !p->d_u || !p->d_delta || !p->d_B || !p->d_C || (p->z && !p->d_z)))
        return seq_fail(AUV_ERR_ARG, "auv_selective_scan: null gradient or segments");
    for (const void* q : {(const void*)p->segments, (const void*)p->workspace})
        if ((uintptr_t)q % 16) return seq_fail(AUV_ERR_ARG, "auv_selective_scan: segments and workspace must be 16-byte aligned");
    if (const int rc = launches_fit(*p, pass)) return rc;
    const int64_t need = workspace(*p, pass);
    if (need && (!p->workspace || p->workspace_bytes < need))
        return seq_fail(AUV_ERR_MEMORY, "auv_selective_scan: the workspace holds %lld bytes, %lld are needed", (long long)p->workspace_bytes, (long long)need);
    DeviceScope scope(p->device);
    if (!scope.ok()) return seq_fail(AUV_ERR_DEVICE, "auv_selective_scan: no HIP device %lld", (long long)p->device);
    const ScanArgs a = fill(*p);
    const hipStream_t st = (hipStream_t)stream;
    if (p->dtype == AUV_F32) return by_states<float>(*p, pass, a, st);
    return p->dtype == AUV_BF16 ? by_states<bf16>(*p, pass, a, st) : by_states<f16>(*p, pass, a, st);
}

}  // extern "C"
