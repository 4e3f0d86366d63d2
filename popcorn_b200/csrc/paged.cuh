// paged.cuh — a request of a paged step and the keys its tokens see, as the
// attention kernels read them from the lengths on the device.
#pragma once

#include <stdint.h>

#include "dtype.cuh"
#include "launch.hpp"

namespace popcorn {
namespace launch {

// Two floats -> one word of two 16-bit values (lo, hi), to nearest even; a
// NaN stays one (the bit-level bf16 rule of dtype.cuh carries it over to 0).
template <class T>
__device__ __forceinline__ uint32_t cvt_pair(float lo, float hi) {
    uint32_t d;
    if constexpr (T::code == TBF16::code) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
template <class T>
__device__ __forceinline__ void store_one(void* p, int64_t i, float x) {
    if constexpr (T::code == TF32::code) static_cast<float*>(p)[i] = x;
    else static_cast<uint16_t*>(p)[i] = static_cast<uint16_t>(cvt_pair<T>(x, 0.f));
}

struct Request {
    int64_t t0, n;  // first token of the step, new tokens
    int64_t len;    // keys, the new ones included
};

// Request r, with every length brought into range: tokens inside [0, T),
// keys inside the block table's row.
__device__ __forceinline__ Request request(const PagedAttention& p, int r) {
    int64_t a = p.query_start[r], b = p.query_start[r + 1], len = p.seq_lens[r];
    a = a < 0 ? 0 : (a > p.T ? p.T : a);
    b = b < a ? a : (b > p.T ? p.T : b);
    const int64_t most = p.W * p.ps;
    len = len < 0 ? 0 : (len > most ? most : len);
    return Request{a, b - a, len};
}

// The keys that the query at position pos sees: [0, sink) and [lo, hi).
struct Span {
    int64_t sink, lo, hi;
};
__device__ __forceinline__ Span visible(const PagedAttention& p, const Request& r, int64_t pos) {
    Span v{0, 0, r.len};
    if (p.mask_kind != 2) v.hi = pos + 1 < 0 ? 0 : (pos + 1 < r.len ? pos + 1 : r.len);
    if (p.mask_kind == 1) {
        v.lo = pos - p.window + 1;
        if (v.lo < 0) v.lo = 0;
        if (v.lo > v.hi) v.lo = v.hi;
        v.sink = p.sinks < v.lo ? p.sinks : v.lo;
    }
    return v;
}

}  // namespace launch
}  // namespace popcorn
