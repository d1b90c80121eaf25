// kv8.h -- the paged KV cache held in 8 bits, as its writer and its reader share it.
//
// A page of a head is block_size rows of head_dim e4m3 numbers and one exponent byte b:
// an element stands for half(e4m3 * 2^(b - 127)).  The scale is a power of two because
// e4m3 is a floating type: a finer scale would move the numbers within their binade and
// gain no precision but near the type's subnormals.  Then scaling is exact both ways, a
// page's exponent can be raised without its source, and the hardware's conversion applies it.
#pragma once

#include "mi_device.h"
#include "mi_kernels.h"

namespace mi {

constexpr int kKv8Segs = 8;
constexpr int kE8Bias = 127;

struct Kv8Segs {
    int n;
    int64_t off[kKv8Segs], B[kKv8Segs], S[kKv8Segs], mb[kKv8Segs];
    const int* bt[kKv8Segs];
    const int* sl[kKv8Segs];
    const int* sp[kKv8Segs];
};

// 2^(byte - 127) as the conversion instructions take it: they read an fp32's exponent.
__device__ __forceinline__ float e8_scale(int byte) {
    return __builtin_bit_cast(float, byte << 23);
}

// Checks segments of a call over T tokens and fills sg; token ranges are disjoint.
// MI_OK or an entry point's status (kv8.hip).
int kv8_segments(const mi_kv_segment* segments, int num_segments, int64_t T, Kv8Segs& sg);

}  // namespace mi
