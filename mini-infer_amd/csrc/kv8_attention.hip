// kv8_attention.hip -- causal attention over the paged cache held in 8 bits (kv8.h).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[t, h] . k_j - max),
//   j over the token's own position and those before it (the last `window` of them)
//
// in one pass over the keys with the running maximum and sum of the softmax.  e4m3 times a
// power of two is an fp16 number, so the products are fp16 MFMAs of exact inputs with
// fp32 sums; q is used as it is, p is rounded to fp16 (2^-11 relative, as the output's own
// rounding) after scaling by 2^14, so that weights down to 2^-28 keep their bits.
//
// Matrix layout.  The scores are made transposed, S^T = K Q^T: a lane then holds scores of
// one query column only, and the second product O^T = V^T P^T takes them as its operand
// from the registers they are in -- no shuffle, no LDS.  Which 16 keys a product's rows
// stand for is free: of 64 keys in four 16-key blocks, tile t takes keys 4t .. 4t + 3 of
// each block, so lane group g (lane / 16) ends up with all 16 keys of block g, and needs V
// of that block alone.  The same freedom in d lets a lane read K and V in runs of 16 and 8
// bytes (head_dim 128) straight from the pages.
#include <algorithm>
#include <cmath>

#include "kv8.h"
#include "mi_host.h"

namespace mi {

typedef float f4 __attribute__((ext_vector_type(4)));

constexpr int kRows = 16;      // query rows of a tile: (token, head of the KV head's group)
constexpr int kKeys = 64;      // keys of a wave's step
constexpr int kWaves = 4;      // waves of a workgroup, each on every fourth step
constexpr float kPShift = 14.0f;
constexpr int64_t kMaxSplits = 128;

struct Kv8Attn {
    const half_t* q;
    half_t* out;
    const uint8_t *kc, *vc, *ks, *vs;
    int64_t qs, os, num_blocks, layer;
    int Hq, Hkv, G, hd, bs, window;
    float c;  // scale * log2(e)
    float* part;  // [slot][row][hd + 2]: sums, then maximum and sum of weights
    Kv8Segs sg;
    int tiles[kKv8Segs], nsplit[kKv8Segs];
    int64_t first[kKv8Segs + 1];  // a segment's first workgroup, and its first slot
    int64_t group0[kKv8Segs + 1]; // a segment's first (sequence, tile, KV head)
};

// What a tile of rows attends to.
struct TileKeys {
    int S, r0, rows;       // the sequence's tokens; first row, rows of the tile
    int64_t sp, sl;        // the sequence's start position and length
    int64_t lo, hi;        // keys that some live row sees
    int64_t base;          // lo, down to a block of 16
    int steps, per, used;  // steps of 64 keys from base; steps of a split, splits in use
};

__device__ __forceinline__ TileKeys tile_keys(const Kv8Attn& a, int g, int64_t b, int tile) {
    TileKeys t;
    t.S = static_cast<int>(a.sg.S[g]);
    t.r0 = tile * kRows;
    const int all = t.S * a.G;
    t.rows = min(kRows, all - t.r0);
    t.sp = a.sg.sp[g][b];
    t.sl = a.sg.sl[g][b];
    const int64_t first = max<int64_t>(t.sp + t.r0 / a.G, 0);
    const int64_t last = min(t.sp + (t.r0 + t.rows - 1) / a.G, t.sl - 1);
    t.hi = min<int64_t>(last + 1, a.sg.mb[g] * a.bs);
    t.lo = a.window > 0 ? max<int64_t>(first - a.window + 1, 0) : 0;
    if (last < first) t.hi = t.lo = 0;
    t.base = t.lo & ~int64_t{15};
    t.steps = t.hi > t.lo ? static_cast<int>((t.hi - t.base + kKeys - 1) / kKeys) : 0;
    const int ns = a.nsplit[g];
    t.per = max((t.steps + ns - 1) / ns, kWaves);
    t.per = (t.per + kWaves - 1) / kWaves * kWaves;
    t.used = (t.steps + t.per - 1) / t.per;
    return t;
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

// Loads of W dwords where `ok`, zeros elsewhere.
template <int W>
__device__ __forceinline__ void load_words(uint32_t* to, const uint8_t* p, bool ok) {
    typedef uint32_t vec __attribute__((ext_vector_type(W)));
    vec v = vec(0);
    if (ok) v = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int i = 0; i < W; ++i) to[i] = v[i];
}

template <int HD>
struct Tile {
    static constexpr int kSteps = HD / 32;   // MFMA steps of q . k
    static constexpr int kD = HD / 16;       // tiles of d; consecutive d of a lane in V
    static constexpr int kKw = HD / 16;      // dwords of K a lane holds per tile of 16 keys
    static constexpr int kVw = HD / 64;      // dwords of V a lane holds per key
};

// V's d column `j` of keys 8m .. 8m + 7 of the lane's block, as an MFMA operand.
template <int HD>
__device__ __forceinline__ void v_pair(const uint32_t (&raw)[16][Tile<HD>::kVw], int m, int word, int hi,
                                       float scale, h8& even, h8& odd) {
    uint32_t e[4], o[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int k = 8 * m + 2 * p;
        h2 a, b;
        if (hi) {
            a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[k][word], scale, true);
            b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[k + 1][word], scale, true);
        } else {
            a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[k][word], scale, false);
            b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(raw[k + 1][word], scale, false);
        }
        const uint32_t ua = __builtin_bit_cast(uint32_t, a), ub = __builtin_bit_cast(uint32_t, b);
        e[p] = __builtin_amdgcn_perm(ub, ua, 0x05040100u);
        o[p] = __builtin_amdgcn_perm(ub, ua, 0x07060302u);
    }
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    even = __builtin_bit_cast(h8, u4{e[0], e[1], e[2], e[3]});
    odd = __builtin_bit_cast(h8, u4{o[0], o[1], o[2], o[3]});
}

// NaN elements of v to 0, and ones in their places in `nan`.
__device__ __forceinline__ void split_nan(h8& v, h8& nan) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool is = v[i] != v[i];
        nan[i] = is ? (half_t)1.0f : (half_t)0.0f;
        if (is) v[i] = (half_t)0.0f;
    }
}

// One workgroup: a tile of 16 rows of one sequence and KV head, over one split of its keys.
// A wave's step of 64 keys: K's bytes to fp16 and the scores; the softmax's step; V's bytes
// to fp16, transposed in pairs by byte permutes, and the sums.  K of the next step is
// read once the scores are made, V of the next after the sums, so a wave always has half a
// step (8 KB at head_dim 128) in flight while it computes.
template <int HD>
__global__ __launch_bounds__(256, 2) void kv8_attn_kernel(Kv8Attn a) {
    using L = Tile<HD>;
    __shared__ float s_ml[kWaves][2][kRows];
    __shared__ float s_o[kWaves][kRows][HD + 4];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    int64_t id = blockIdx.x;
    int g = 0;
    while (id >= a.first[g + 1]) ++g;
    id -= a.first[g];
    const int h = static_cast<int>(id % a.Hkv);
    id /= a.Hkv;
    const int split = static_cast<int>(id % a.nsplit[g]);
    id /= a.nsplit[g];
    const int tile = static_cast<int>(id % a.tiles[g]);
    const int64_t b = id / a.tiles[g];
    const TileKeys t = tile_keys(a, g, b, tile);
    if (split >= max(t.used, 1)) return;
    const int col = lane & 15, grp = lane >> 4;
    const int64_t tok0 = a.sg.off[g] + b * t.S;

    // this lane's query column
    const int row = t.r0 + col, s = row / a.G, head = h * a.G + (row - s * a.G);
    const int64_t pos = t.sp + s;
    const bool live = col < t.rows && pos >= 0 && pos < t.sl;
    const int64_t row_hi = live ? min(pos + 1, t.hi) : 0;
    const int64_t row_lo = a.window > 0 ? max<int64_t>(pos - a.window + 1, 0) : 0;
    h8 qf[L::kSteps];
#pragma unroll
    for (int i = 0; i < L::kSteps; ++i) {
        const int d = grp * (HD / 4) + i * 8;
        qf[i] = h8(0);
        if (live && d < a.hd) qf[i] = ld8(a.q + (tok0 + s) * a.qs + head * a.hd + d);
    }

    // the page of a 16-key block, -1 where it has none
    const int* const table = a.sg.bt[g] + b * a.sg.mb[g];
    const int sub = a.bs >> 4;  // 16-key blocks of a page
    const float inv_sub = 1.0f / static_cast<float>(sub);
    const auto page_of = [&](int step, int blk, int& in_page) {
        const int64_t key = t.base + static_cast<int64_t>(step) * kKeys + blk * 16;
        const int k16 = static_cast<int>(key >> 4);  // < 2^22
        const int idx = small_div(k16, inv_sub);
        in_page = (k16 - idx * sub) * 16;
        if (key >= t.hi) return -1;
        const int phys = table[idx];
        return phys >= 0 && phys < a.num_blocks ? phys : -1;
    };
    const auto at = [&](int phys) { return (a.layer * a.num_blocks + phys) * a.Hkv + h; };

    uint32_t kr[4][L::kKw], vr[16][L::kVw];
    float kscale = 1.0f, vscale = 1.0f;
    const auto load_k = [&](int step) {
        int in_page;
        const int phys = page_of(step, col >> 2, in_page);
        const int64_t pg = at(max(phys, 0));
        const uint8_t* p = a.kc + (pg * a.bs + in_page + (col & 3)) * a.hd + grp * (HD / 4);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int w = 0; w < L::kKw; w += 4)
                load_words<4>(&kr[i][w], p + i * 4 * a.hd + w * 4, phys >= 0 && grp * (HD / 4) + w * 4 < a.hd);
        kscale = phys >= 0 ? e8_scale(a.ks[pg]) : 1.0f;
    };
    int vphys = -1;
    const auto load_v = [&](int step) {
        int in_page;
        vphys = page_of(step, grp, in_page);
        const int64_t pg = at(max(vphys, 0));
        const uint8_t* p = a.vc + (pg * a.bs + in_page) * a.hd + col * L::kD;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            load_words<L::kVw>(vr[i], p + i * a.hd, vphys >= 0 && col * L::kD < a.hd);
        vscale = vphys >= 0 ? e8_scale(a.vs[pg]) : 1.0f;
    };

    f4 o[L::kD];
#pragma unroll
    for (int j = 0; j < L::kD; ++j) o[j] = f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    // every row sees every key of a step that lies in [all_lo, all_hi)
    const int64_t all_hi = min<int64_t>(max<int64_t>(t.sp + t.r0 / a.G, 0) + 1, t.hi);
    const int64_t all_lo = a.window > 0 ? max<int64_t>(t.sp + (t.r0 + t.rows - 1) / a.G - a.window + 1, t.lo) : 0;
    const bool one_pos = t.r0 / a.G == (t.r0 + t.rows - 1) / a.G;
    const int end = min((split + 1) * t.per, t.steps);
    int step = split * t.per + wave;
    if (step < end) {
        load_k(step);
        load_v(step);
    }
    for (; step < end; step += kWaves) {
        // scores: tile i's row 4 g + e is key 4 i + e of block g
        f4 sc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            sc[i] = f4{0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < L::kSteps; ++w) {
                const h2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kr[i][2 * w], kscale, false);
                const h2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kr[i][2 * w], kscale, true);
                const h2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kr[i][2 * w + 1], kscale, false);
                const h2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kr[i][2 * w + 1], kscale, true);
                const h8 kf = {x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
                sc[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[w], sc[i], 0, 0, 0);
            }
        }
        const int next = step + kWaves;
        if (next < end) load_k(next);
        const int64_t key0 = t.base + static_cast<int64_t>(step) * kKeys;
        const bool masked = key0 + kKeys > all_hi || key0 < all_lo || key0 < t.lo || __any(vphys < 0);
        uint32_t seen = 0xFFFF;  // of the lane's 16 keys, those that its row sees
        bool nan_path = false;
        float x[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = sc[i >> 2][i & 3] * a.c;
        if (masked) {
            seen = 0;
            uint32_t some = 0;  // and those that any row may see
            const int64_t k0 = key0 + grp * 16;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (vphys >= 0 && k0 + i < row_hi && k0 + i >= row_lo) seen |= 1u << i;
                if (vphys >= 0 && k0 + i < t.hi && k0 + i >= t.lo) some |= 1u << i;
                if (!(seen & (1u << i))) x[i] = -INFINITY;
            }
            // what no row sees may hold anything, NaN too: 0 times it must be 0
            uint32_t nan = vphys >= 0 && (__builtin_bit_cast(uint32_t, vscale) >> 23) == 255 ? some : 0;
#pragma unroll
            for (int i = 0; i < 16; ++i)
#pragma unroll
                for (int w = 0; w < L::kVw; ++w) {
                    if (!(some & (1u << i))) vr[i][w] = 0;
                    nan |= ((vr[i][w] & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                }
            // a NaN that some rows see and others do not
            nan_path = !one_pos && __any(nan != 0);
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < 16; ++i) mx = fmaxf(mx, x[i]);
        const float mn = fmaxf(m, max_over_groups(mx));
        if (__any(mn > m)) {
            const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= by;
#pragma unroll
            for (int j = 0; j < L::kD; ++j) o[j] *= by;
            m = mn;
        }
        const float ref = (m == -INFINITY ? 0.0f : m) - kPShift;
        h8 p[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float w = __builtin_amdgcn_exp2f(x[i] - ref);
            l += w;
            p[i >> 3][i & 7] = (half_t)w;
        }
        if (!nan_path) {
#pragma unroll
            for (int j = 0; j < L::kD; j += 2)
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    h8 even, odd;
                    v_pair<HD>(vr, k, j >> 2, (j >> 1) & 1, vscale, even, odd);
                    o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p[k], o[j], 0, 0, 0);
                    o[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p[k], o[j + 1], 0, 0, 0);
                }
        } else {
            h8 see[2];
#pragma unroll
            for (int i = 0; i < 16; ++i) see[i >> 3][i & 7] = (half_t)(seen & (1u << i) ? 1.0f : 0.0f);
#pragma unroll
            for (int j = 0; j < L::kD; j += 2) {
                f4 n0 = f4{0, 0, 0, 0}, n1 = n0;
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    h8 even, odd, ne, no;
                    v_pair<HD>(vr, k, j >> 2, (j >> 1) & 1, vscale, even, odd);
                    split_nan(even, ne);
                    split_nan(odd, no);
                    o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p[k], o[j], 0, 0, 0);
                    o[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p[k], o[j + 1], 0, 0, 0);
                    n0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(ne, see[k], n0, 0, 0, 0);
                    n1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(no, see[k], n1, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (n0[e] > 0.0f) o[j][e] = __builtin_nanf("");
                    if (n1[e] > 0.0f) o[j + 1][e] = __builtin_nanf("");
                }
            }
        }
        if (next < end) load_v(next);
    }

    // the four waves' sums, joined
    l = sum_over_groups(l);
    if (grp == 0) {
        s_ml[wave][0][col] = m;
        s_ml[wave][1][col] = l;
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int j = 0; j < L::kD; ++j) s_o[wave][col][(4 * grp + e) * L::kD + j] = o[j][e];
    __syncthreads();
    const int64_t slot = a.first[g] + ((b * a.tiles[g] + tile) * a.Hkv + h) * a.nsplit[g] + split;
    const float inv_hd = 1.0f / static_cast<float>(a.hd);
    for (int i = threadIdx.x; i < t.rows * a.hd; i += 256) {
        const int r = small_div(i, inv_hd), d = i - r * a.hd;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, s_ml[w][0][r]);
        float sum = 0.0f, tot = 0.0f;
        if (mm > -INFINITY) {
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                if (s_ml[w][0][r] == -INFINITY && s_ml[w][1][r] == 0.0f) continue;  // saw nothing
                const float by = __builtin_amdgcn_exp2f(s_ml[w][0][r] - mm);
                sum = fmaf(s_o[w][r][d], by, sum);
                tot = fmaf(s_ml[w][1][r], by, tot);
            }
        } else {  // nothing seen, or NaN alone
#pragma unroll
            for (int w = 0; w < kWaves; ++w) tot += s_ml[w][1][r], sum += s_o[w][r][d];
        }
        const int rr = t.r0 + r, rs = rr / a.G;
        const int64_t rp = t.sp + rs;
        if (t.used <= 1) {
            const bool rl = rp >= 0 && rp < t.sl && tot != 0.0f;
            a.out[(tok0 + rs) * a.os + (h * a.G + rr - rs * a.G) * a.hd + d] = (half_t)(rl ? sum / tot : 0.0f);
        } else {
            float* const p = a.part + (slot * kRows + r) * (a.hd + 2);
            p[d] = sum;
            if (d == 0) {
                p[a.hd] = mm;
                p[a.hd + 1] = tot;
            }
        }
    }
}

// The splits of a tile, joined: one workgroup per (sequence, tile, KV head).
__global__ __launch_bounds__(256) void kv8_join_kernel(Kv8Attn a) {
    int64_t id = blockIdx.x;
    int g = 0;
    while (id >= a.group0[g + 1]) ++g;
    id -= a.group0[g];
    const int h = static_cast<int>(id % a.Hkv);
    const int64_t bt = id / a.Hkv;
    const int tile = static_cast<int>(bt % a.tiles[g]);
    const int64_t b = bt / a.tiles[g];
    const TileKeys t = tile_keys(a, g, b, tile);
    if (t.used <= 1) return;
    const float* const part = a.part + (a.first[g] + (bt * a.Hkv + h) * a.nsplit[g]) * kRows * (a.hd + 2);
    const int64_t step = static_cast<int64_t>(kRows) * (a.hd + 2);
    for (int i = threadIdx.x; i < t.rows * a.hd; i += 256) {
        const int r = i / a.hd, d = i - r * a.hd;
        const float* const p = part + static_cast<int64_t>(r) * (a.hd + 2);
        float mm = -INFINITY;
        for (int s = 0; s < t.used; ++s) mm = fmaxf(mm, p[s * step + a.hd]);
        float sum = 0.0f, tot = 0.0f;
        for (int s = 0; s < t.used; ++s) {
            const float ms = p[s * step + a.hd], ls = p[s * step + a.hd + 1];
            if (ms == -INFINITY && ls == 0.0f) continue;
            const float by = mm == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ms - mm);
            sum = fmaf(p[s * step + d], by, sum);
            tot = fmaf(ls, by, tot);
        }
        const int rr = t.r0 + r, rs = rr / a.G;
        const int64_t rp = t.sp + rs;
        const bool live = rp >= 0 && rp < t.sl && tot != 0.0f;
        a.out[(a.sg.off[g] + b * t.S + rs) * a.os + (h * a.G + rr - rs * a.G) * a.hd + d] =
            (half_t)(live ? sum / tot : 0.0f);
    }
}

// Tiles, splits and slots of a call; what the launch and the workspace's size go by.
static int kv8_attn_plan(Kv8Attn& a, int64_t& slots) {
    const int64_t kWant = 2048;  // workgroups that fill the GPU a few times over
    slots = 0;
    for (int i = 0; i < a.sg.n; ++i) {
        const int64_t tiles = ceil_div(a.sg.S[i] * a.G, kRows);
        const int64_t groups = a.sg.B[i] * tiles * a.Hkv;
        const int64_t ns = std::clamp<int64_t>(kWant / std::max<int64_t>(groups, 1), 1,
                                               std::min<int64_t>(a.sg.mb[i], kMaxSplits));
        a.tiles[i] = static_cast<int>(tiles);
        a.nsplit[i] = static_cast<int>(ns);
        a.first[i + 1] = a.first[i] + groups * ns;
        a.group0[i + 1] = a.group0[i] + groups;
        if (ns > 1) slots = a.first[i + 1];
    }
    return a.first[a.sg.n] <= kMaxGridX ? MI_OK : MI_ERR_UNSUPPORTED;
}

static int kv8_attn_shape(int64_t T, int64_t Hq, int64_t Hkv, int64_t hd,
                          const mi_kv_segment* segments, int num_segments, Kv8Attn& a) {
    if (T < 0 || Hq < 0 || Hkv < 0 || hd < 0) return MI_ERR_INVALID_ARGUMENT;
    const int st = kv8_segments(segments, num_segments, T, a.sg);
    if (st != MI_OK) return st;
    if (T == 0 || Hq == 0 || hd == 0 || a.sg.n == 0) {
        a.sg.n = 0;
        return MI_OK;
    }
    if (Hkv == 0 || Hq % Hkv != 0) return MI_ERR_INVALID_ARGUMENT;
    if (hd % 16 != 0 || hd > 256 || Hq > 1024 || T > (int64_t{1} << 24)) return MI_ERR_UNSUPPORTED;
    a.Hq = static_cast<int>(Hq);
    a.Hkv = static_cast<int>(Hkv);
    a.G = static_cast<int>(Hq / Hkv);
    a.hd = static_cast<int>(hd);
    return MI_OK;
}

}  // namespace mi

extern "C" int64_t mi_kv8_attention_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t head_dim,
                                                    const mi_kv_segment* segments, int num_segments) {
    using namespace mi;
    Kv8Attn a{};
    int64_t slots = 0, T = 0;
    for (int i = 0; i < num_segments && segments; ++i) {  // any packing of the segments
        const mi_kv_segment& g = segments[i];
        if (g.B > 0 && g.S > 0 && g.B < (int64_t{1} << 31) && g.S < (int64_t{1} << 31) && g.token_offset >= 0 &&
            g.token_offset < (int64_t{1} << 31))
            T = std::max(T, g.token_offset + g.B * g.S);
    }
    const int st = kv8_attn_shape(T, Hq, Hkv, head_dim, segments, num_segments, a);
    if (st != MI_OK) return st;
    const int pl = kv8_attn_plan(a, slots);
    if (pl != MI_OK) return pl;
    return slots * kRows * (head_dim + 2) * 4;
}

extern "C" int mi_kv8_attention_f16(const void* q, int64_t q_stride, const void* k_cache,
                                    const void* v_cache, const void* k_scale, const void* v_scale,
                                    void* out, int64_t out_stride, int64_t T, int64_t Hq,
                                    int64_t Hkv, int64_t head_dim, float scale, int64_t window,
                                    int64_t layer, int64_t num_blocks, int64_t block_size,
                                    const mi_kv_segment* segments, int num_segments,
                                    void* workspace, int64_t workspace_bytes, void* stream) {
    using namespace mi;
    if (q_stride < 0 || out_stride < 0 || window < 0 || layer < 0 || layer >= (int64_t{1} << 62) ||
        num_blocks < 0 || block_size <= 0 || !std::isfinite(scale))
        return MI_ERR_INVALID_ARGUMENT;
    Kv8Attn a{};
    const int st = kv8_attn_shape(T, Hq, Hkv, head_dim, segments, num_segments, a);
    if (st != MI_OK) return st;
    if (a.sg.n == 0) return MI_OK;
    // a step's keys are whole 16-key blocks of pages; block numbers stay below 2^22
    if (block_size % 16 != 0 || block_size > 4096) return MI_ERR_UNSUPPORTED;
    for (int i = 0; i < a.sg.n; ++i)
        if (a.sg.mb[i] > (int64_t{1} << 22) || a.sg.mb[i] * block_size > (int64_t{1} << 25))
            return MI_ERR_UNSUPPORTED;
    a.bs = static_cast<int>(block_size);
    if (!q || !out || !k_cache || !v_cache || !k_scale || !v_scale) return MI_ERR_INVALID_ARGUMENT;
    const int64_t row = Hq * head_dim;
    if (T > 1 && (q_stride < row || out_stride < row)) return MI_ERR_INVALID_ARGUMENT;
    if (num_blocks > (int64_t{1} << 31) - 1 || !product_fits({T, q_stride, 2}) ||
        !product_fits({T, out_stride, 2}) ||
        !product_fits({layer + 1, std::max<int64_t>(num_blocks, 1), Hkv * head_dim, block_size}))
        return MI_ERR_INVALID_ARGUMENT;
    if (!aligned16(q) || !aligned16(k_cache) || !aligned16(v_cache) || (T > 1 && q_stride % 8 != 0) ||
        (reinterpret_cast<uintptr_t>(out) & 1))
        return MI_ERR_UNSUPPORTED;
    const int64_t cells = (layer + 1) * num_blocks * Hkv;
    const int64_t qb = 2 * ((T - 1) * q_stride + row), ob = 2 * ((T - 1) * out_stride + row);
    int64_t slots = 0;
    const int pl = kv8_attn_plan(a, slots);
    if (pl != MI_OK) return pl;
    const int64_t need = slots * kRows * (head_dim + 2) * 4;
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return MI_ERR_INVALID_ARGUMENT;
    const void* bufs[6] = {k_cache, v_cache, k_scale, v_scale, q, workspace};
    const int64_t lens[6] = {cells * block_size * head_dim, cells * block_size * head_dim, cells, cells, qb, need};
    for (int i = 0; i < 6; ++i) {
        if (overlaps(bufs[i], lens[i], out, ob)) return MI_ERR_ALIASING;
        if (i < 5 && overlaps(bufs[i], lens[i], workspace, need)) return MI_ERR_ALIASING;
    }
    a.q = static_cast<const half_t*>(q);
    a.out = static_cast<half_t*>(out);
    a.kc = static_cast<const uint8_t*>(k_cache);
    a.vc = static_cast<const uint8_t*>(v_cache);
    a.ks = static_cast<const uint8_t*>(k_scale);
    a.vs = static_cast<const uint8_t*>(v_scale);
    a.qs = q_stride;
    a.os = out_stride;
    a.layer = layer;
    a.num_blocks = num_blocks;
    a.window = static_cast<int>(std::min<int64_t>(window, int64_t{1} << 30));
    a.c = scale * 1.4426950408889634f;
    a.part = static_cast<float*>(workspace);
    const hipStream_t s = as_stream(stream);
    const dim3 grid(static_cast<unsigned>(a.first[a.sg.n])), block(256);
    if (head_dim <= 64) kv8_attn_kernel<64><<<grid, block, 0, s>>>(a);
    else if (head_dim <= 128) kv8_attn_kernel<128><<<grid, block, 0, s>>>(a);
    else kv8_attn_kernel<256><<<grid, block, 0, s>>>(a);
    if (slots > 0) kv8_join_kernel<<<dim3(static_cast<unsigned>(a.group0[a.sg.n])), block, 0, s>>>(a);
    return launch_status();
}
