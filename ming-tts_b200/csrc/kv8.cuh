// kv8.cuh -- shared by the 8-bit key/value cache kernels (kv8.cu, kv8_attention.cu).
#pragma once

#include "common.cuh"

namespace mt {

// A request's rows, read by every kernel of a call: its first position and how many rows are its own
// (0 for an idle request: a position below `base`, or positions that would pass 2^31 - 1).
struct Kv8Rows {
    const int* positions;
    const int* counts;  // optional
    int rows, base;
};
struct Kv8Span {
    int pos, count;
};
__device__ __forceinline__ Kv8Span kv8_span(const Kv8Rows& a, int request) {
    Kv8Span s;
    s.pos = a.positions[request];
    s.count = a.counts ? min(max(a.counts[request], 0), a.rows) : a.rows;
    if (s.pos < a.base || s.pos > 0x7FFFFFFF - a.rows) s.count = 0;
    return s;
}

// Host-side checks that the entry points share. `what` names the entry point.
mt_status kv8_check_cache(mt_ctx* ctx, const char* what, const mt_kv8_cache* c, int requests);
mt_status kv8_check_rows(mt_ctx* ctx, const char* what, int requests, int rows, int hq, int hkv);

// Makes a device current for a call and puts the caller's back.
struct DeviceGuard {
    int before = -1;
    cudaError_t err;
    explicit DeviceGuard(int device) {
        err = cudaGetDevice(&before);
        if (err == cudaSuccess && before != device)
            err = cudaSetDevice(device);
        else
            before = -1;
    }
    ~DeviceGuard() {
        if (before >= 0) cudaSetDevice(before);
    }
};

}  // namespace mt
