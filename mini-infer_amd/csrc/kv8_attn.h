// kv8_attn.h -- what the two kernels of attention over the 8-bit cache share: a call's
// arguments, the keys of a tile of query rows, and the join of partial sums.
#pragma once

#include "kv8.h"

namespace mi {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr float kPShift = 10.0f;  // the softmax's weights are rounded to fp16 times 2^10
constexpr float kSlack = 5.0f;   // how far, in powers of two, a maximum may rise before the sums are scaled again
constexpr int kMaxSplits = 64;

struct Kv8Attn {
    const half_t* q;
    half_t* out;
    const uint8_t *kc, *vc, *ks, *vs;
    int64_t qs, os, num_blocks, layer;
    int Hq, Hkv, G, hd, bs, window;
    float c;   // |scale| * log2(e), above 0: a hidden score times it stays -inf
    bool neg;  // scale < 0: q is negated
    float* part;      // the workspace: partial sums of the splits
    unsigned* count;  // and how many of a tile's splits are done
    Kv8Segs sg;
    int tiles[kKv8Segs], nsplit[kKv8Segs];
    int64_t first[kKv8Segs + 1];            // a segment's first workgroup
    int64_t part0[kKv8Segs], cnt0[kKv8Segs];  // its places in the workspace, where it is in splits
};

// What a tile of rows attends to.
struct TileKeys {
    int S, r0, rows;       // the sequence's tokens; first row, rows of the tile
    int64_t sp, sl;        // the sequence's start position and length
    int64_t lo, hi;        // keys that some live row sees
    int64_t base;          // lo, down to a block of 16
    int steps, per, used;  // steps of KEYS keys from base; steps of a split, splits in use
};

// ROWS rows in a tile, KEYS keys in a step, at least LEAST steps in a split (a multiple of it).
template <int ROWS, int KEYS, int LEAST>
__device__ __forceinline__ TileKeys tile_keys(const Kv8Attn& a, int g, int64_t b, int tile) {
    TileKeys t;
    t.S = static_cast<int>(a.sg.S[g]);
    t.r0 = tile * ROWS;
    const int all = t.S * a.G;
    t.rows = min(ROWS, all - t.r0);
    t.sp = a.sg.sp[g][b];
    t.sl = a.sg.sl[g][b];
    const int64_t first = max<int64_t>(t.sp + t.r0 / a.G, 0);
    const int64_t last = min(t.sp + (t.r0 + t.rows - 1) / a.G, t.sl - 1);
    t.hi = min<int64_t>(last + 1, a.sg.mb[g] * a.bs);
    t.lo = a.window > 0 ? max<int64_t>(first - a.window + 1, 0) : 0;
    if (last < first) t.hi = t.lo = 0;
    t.base = t.lo & ~int64_t{15};
    t.steps = t.hi > t.lo && a.num_blocks > 0 ? static_cast<int>((t.hi - t.base + KEYS - 1) / KEYS) : 0;
    const int ns = a.nsplit[g];
    t.per = max((t.steps + ns - 1) / ns, LEAST);
    t.per = (t.per + LEAST - 1) / LEAST * LEAST;
    t.used = (t.steps + t.per - 1) / t.per;
    return t;
}

// id % d; id becomes id / d.
__device__ __forceinline__ int divmod(uint32_t& id, int d) {
    const uint32_t q = id / static_cast<uint32_t>(d), r = id - q * static_cast<uint32_t>(d);
    id = q;
    return static_cast<int>(r);
}

__device__ __forceinline__ float max_over_groups(float v) {
    uint32_t a, b;
    pair_xor16(__builtin_bit_cast(uint32_t, v), a, b);
    v = fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
    pair_xor32(__builtin_bit_cast(uint32_t, v), a, b);
    return fmaxf(__builtin_bit_cast(float, a), __builtin_bit_cast(float, b));
}
__device__ __forceinline__ float sum_over_groups(float v) {
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

// What a partial sum with maximum m and sum of weights l counts, beside the maximum ref;
// one that saw nothing counts nothing, and one of NaN alone (m stays -inf) must not be lost.
__device__ __forceinline__ float join_weight(float m, float l, float ref) {
    return m == -INFINITY ? (l == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m - ref);
}

__device__ __forceinline__ void store_agent(float* p, float v) {
    __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float load_agent(const float* p) {
    return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <int W>
__device__ __forceinline__ void load_words(uint32_t* to, const uint8_t* p) {
    typedef uint32_t vec __attribute__((ext_vector_type(W)));
    const vec v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) to[i] = v[i];
}

// All bits of the bytes of w that are NaN.
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) {
    const uint32_t top = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
    return top | (top - (top >> 7));
}

// Segments of many query rows (kv8_prompt.hip), already planned.
void kv8_prompt_launch(const Kv8Attn& a, hipStream_t s);
constexpr int kPromptRows = 128;   // query rows of its tile
constexpr int kPromptSplits = 32;  // at most
constexpr int kPromptLeast = 16;   // tiles of keys of a split: the join of many small ones costs more

}  // namespace mi
