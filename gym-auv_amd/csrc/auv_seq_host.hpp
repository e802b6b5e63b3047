// Host side shared by the sequence operators' entry points: the calling thread's last error, the device of the call,
// and the checks of shapes, types and alignment that come before any launch.  Nothing here throws.
#pragma once

#include "../../include/auvsim.h"
#include "auv_slices.hpp"

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

namespace auv {
namespace seq {

int seq_fail(int code, const char* fmt, ...);   // auv_conv.hip; returns `code`

// Makes `device` current for the scope and puts the caller's device back.
class DeviceScope {
public:
    explicit DeviceScope(int64_t device) {
        if (hipGetDevice(&old_) != hipSuccess) return;
        ok_ = old_ == device || hipSetDevice((int)device) == hipSuccess;
        moved_ = ok_ && old_ != device;
    }
    ~DeviceScope() {
        if (moved_) (void)hipSetDevice(old_);
    }
    bool ok() const { return ok_; }

private:
    int old_ = 0;
    bool ok_ = false, moved_ = false;
};

inline int64_t type_size(int64_t dtype) { return dtype == AUV_F32 ? 4 : (dtype == AUV_BF16 || dtype == AUV_F16) ? 2 : 0; }
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// The widest access, up to `most` elements, that an address and a set of element strides allow.
class Width {
public:
    Width(int64_t most) : bits_((uint64_t)most) {}
    void pointer(const void* p, int64_t size) {
        if (p) bits_ |= (uint64_t)((uintptr_t)p / (uintptr_t)size);
        if (p && (uintptr_t)p % (uintptr_t)size) bits_ |= 1;
    }
    void stride(int64_t elements) { bits_ |= (uint64_t)elements; }
    int64_t elements() const { return (int64_t)(bits_ & (~bits_ + 1)); }

private:
    uint64_t bits_;
};

inline int launched(const char* what) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? AUV_OK : seq_fail(AUV_ERR_DEVICE, "%s launch failed: %s", what, hipGetErrorString(e));
}

// Sizes and counts common to the rows of activations; B L D stays far below 2^62, so products of them fit 64 bits.
inline int check_rows(const char* who, int64_t B, int64_t L, int64_t D, int64_t device, int64_t dtype) {
    constexpr int64_t kMost = (int64_t)1 << 40;
    if (B < 0 || L < 0 || D < 1 || D > ((int64_t)1 << 24) || B > kMost || L > kMost || (L > 0 && B > kMost / L) ||
        (B * L > 0 && D > ((int64_t)1 << 46) / (B * L)))
        return seq_fail(AUV_ERR_ARG, "%s: bad shape [%lld, %lld, %lld]", who, (long long)B, (long long)L, (long long)D);
    if (!type_size(dtype)) return seq_fail(AUV_ERR_ARG, "%s: activations must be f32, bf16 or f16, got type %lld", who, (long long)dtype);
    if (device < 0) return seq_fail(AUV_ERR_ARG, "%s: bad device %lld", who, (long long)device);
    return AUV_OK;
}

}  // namespace seq
}  // namespace auv
