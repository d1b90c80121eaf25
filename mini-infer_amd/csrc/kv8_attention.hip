// kv8_attention.hip -- causal attention over the paged cache held in 8 bits (kv8.h).
//
//   out[t, h] = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q[t, h] . k_j - max),
//   j over the token's own position and those before it (the last `window` of them)
//
// in one pass over the keys with the running maximum and sum of the softmax.  e4m3 times a
// power of two is an fp16 number, so the products are fp16 MFMAs of exact inputs with
// fp32 sums; q is used as it is, p is rounded to fp16 (2^-11 relative, as the output's own
// rounding) after scaling by 2^10.  The reference maximum may lag the true one by 2^5, so a weight is at
// most 2^15, and those down to 2^-24 of the reference keep their bits.
//
// Matrix layout.  The scores are made transposed, S^T = K Q^T: a lane then holds scores of
// one query column only, and the second product O^T = V^T P^T takes them as its operand
// from the registers they are in -- no shuffle, no LDS.  Which 16 keys a product's rows
// stand for is free: of 64 keys in four 16-key blocks, tile t takes keys 4t .. 4t + 3 of
// each block, so lane group g (lane / 16) ends up with all 16 keys of block g, and needs V
// of that block alone.  The same freedom in d lets a lane read K and V in runs of 16 and 8
// bytes (head_dim 128) straight from the pages.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "kv8_attn.h"
#include "mi_host.h"

namespace mi {

// Which of the two kernels a segment takes.  Tiles of 16 rows read their keys once each, tiles of
// 128 once for all, but leave CUs idle where there are few.  By the number of 16-row tiles; tiles
// of 16 against 128 (us), 28 heads on 4 of 128: a chunk at 8000 228 tiles 75 / 84, 452 117 / 124, 900 226 / 138;
// 16 chunks at 4000 256 tiles 52 / 62, 512 75 / 70; 64 at 500 1024 53 / 23.  16 heads of 64: 544 tiles
// 38 / 41, 768 67 / 78, 1056 67 / 57.  16 heads on 8 of 256: 528 tiles 112 / 121, 640 203 / 184, 1056 81 / 62.
constexpr int kFewRows = 32;  // that always go in tiles of 16 (64 sequences of 18 rows, 8 of 256: 58 / 77)
constexpr int64_t few_tiles(int64_t hd) { return hd <= 64 ? 800 : hd <= 128 ? 480 : 600; }
std::atomic<int> g_kv8_tile{0};  // mi_kv8_attention_test_tile
constexpr int kRows = 16;      // query rows of a tile: (token, head of the KV head's group)
// Workgroups that a segment of few rows is split into: two for each CU, which holds one at a time.
// Uniform lengths would take one (64 sequences of 5000: 66 us with 256, 76 with 512, 83 with 1024),
// ragged ones need the second (100 to 12000: 105, 90, 107).
constexpr int64_t kWant = 512;
// Tiles of a call from which a workgroup has four waves, two workgroups to a CU: one's loads go on while the
// other begins and ends.  1024 tiles (128 sequences, 8 KV heads of 128) of 1000 keys 50 us, 62 with eight
// waves, of 100 to 12000 289 and 298; fewer tiles of ragged lengths want the longest one's keys on eight waves
// (512 tiles of 100 to 12000: 184 and 150).
constexpr int64_t kFill = 1024;
// And one of many rows: what the CUs hold at once, 3, 2 and 1 each.  A chunk of 1024 at 12000, 16 heads of 64: 137
// us with 512, 115 with 768; 32 on 8 of 128: 274 with 512, 313 with 768; 16 on 8 of 256: 440 with 256, 506 with 512.
constexpr int64_t prompt_want(int64_t hd) { return hd <= 64 ? 768 : hd <= 128 ? 512 : 256; }
constexpr int64_t kCounters = kKv8Segs * 1024;  // at the head of the workspace, zeros between calls

template <int HD, int WAVES>
struct Tile {
    static constexpr int kWaves = WAVES;         // of a workgroup, each on every WAVES-th step; two a SIMD
    static constexpr int kLeast = 2 * kWaves;    // steps of a split, and what they are a multiple of
    static constexpr int kKl = HD > 128 ? 8 : 16;  // keys of a step that a lane group has
    static constexpr int kKeys = 4 * kKl;            // keys of a wave's step
    static constexpr int kSteps = HD / 32;   // MFMA steps of q . k
    static constexpr int kD = HD / 16;       // tiles of d; consecutive d of a lane in V
    static constexpr int kKw = HD / 16;      // dwords of K a lane holds per tile of 16 keys
    static constexpr int kVw = HD / 64;      // dwords of V a lane holds per key
};

// V's d column `j` of keys 8m .. 8m + 7 of the lane's block, as an MFMA operand.
template <int KL, int VW>
__device__ __forceinline__ void v_pair(const uint32_t (&raw)[KL][VW], int m, int word, int hi,
                                       float scale, h8& even, h8& odd) {
    uint32_t e[4], o[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const int k = 8 * m + 2 * p;
        // two keys' bytes of d and of d + 1, side by side
        const uint32_t w = __builtin_amdgcn_perm(raw[k + 1][word], raw[k][word], hi ? 0x07030602u : 0x05010400u);
        e[p] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, false));
        o[p] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, scale, true));
    }
    typedef uint32_t u4 __attribute__((ext_vector_type(4)));
    even = __builtin_bit_cast(h8, u4{e[0], e[1], e[2], e[3]});
    odd = __builtin_bit_cast(h8, u4{o[0], o[1], o[2], o[3]});
}

// One workgroup: a tile of 16 rows of one sequence and KV head, over one split of its keys.
// A wave's step of 64 keys: K's bytes to fp16 and the scores; the softmax's step; V's bytes
// to fp16, transposed in pairs by byte permutes, and the sums.  K of the next step is
// read once the scores are made, V of the next after the sums, so a wave always has half a
// step (8 KB at head_dim 128) in flight while it computes.
//
// Bound by HBM where the caches are long: 64 sequences of 100 to 28000 tokens, 28 query heads on 4,
// head_dim 128, 0.92 GB in 179 us, 5.1 TB/s, what a large copy reaches; 24 sequences in a
// window of 1024, head_dim 256, 50 MB in 20 us.  Short ones are bound by the chain from the sequence's
// length to the join: one sequence of 517 tokens 11.3 us (14.4 with four waves to a workgroup).  At
// least two steps a wave in a split: with one the window takes 28 us, with four 26.
template <int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void kv8_attn_kernel(Kv8Attn a) {
    using L = Tile<HD, WAVES>;
    constexpr int kWaves = L::kWaves, kThreads = kWaves * 64, KL = L::kKl, NT = KL / 4, kKeys = L::kKeys;
    __shared__ float s_ml[kWaves][2][kRows];
    __shared__ float s_o[kWaves][kRows][HD + 4];
    __shared__ bool s_last;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    uint32_t id = blockIdx.x;
    int g = 0;
    while (id >= static_cast<uint32_t>(a.first[g + 1])) ++g;
    id -= static_cast<uint32_t>(a.first[g]);
    // splits outermost: those that a short sequence leaves empty are whole runs of workgroups (every
    // eighth of them in use, and all of those fell to a quarter of the CUs: 37 us where 18 do)
    const int h = divmod(id, a.Hkv);
    const int tile = divmod(id, a.tiles[g]);
    const int64_t b = divmod(id, static_cast<int>(a.sg.B[g]));
    const int split = static_cast<int>(id);
    const TileKeys t = tile_keys<kRows, kKeys, L::kLeast>(a, g, b, tile);
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
        if (a.neg) qf[i] = -qf[i];
    }

    // The page of a 16-key block, -1 where it has none.  Every load is unconditional --
    // of the table's entry 0 or of page 0 where there is none, of the row's first bytes
    // where head_dim ends before the lane's -- since a load in a branch is waited for there.
    const int* const table = a.sg.bt[g] + b * a.sg.mb[g];
    const int sub = a.bs >> 4;  // 16-key blocks of a page
    const float inv_sub = 1.0f / static_cast<float>(sub);
    const int nb = static_cast<int>(a.num_blocks);
    const int end = min((split + 1) * t.per, t.steps);
    const int base32 = static_cast<int>(t.base);  // <= 2^25
    const int hi32 = min(static_cast<int>(t.hi), base32 + end * kKeys);
    const auto page_of = [&](int step, int blk, int& in_page) {
        const int key = base32 + step * kKeys + blk * 16;
        const int k16 = key >> 4;  // < 2^22
        const int idx = small_div(k16, inv_sub);
        in_page = (k16 - idx * sub) * 16;
        const int phys = table[key < hi32 ? idx : 0];
        return key < hi32 && static_cast<uint32_t>(phys) < static_cast<uint32_t>(nb) ? phys : -1;
    };
    const int64_t page0 = a.layer * a.num_blocks;
    uint32_t kr[NT][L::kKw], vr[KL][L::kVw];
    int kbyte = 0, vbyte = 0, kphys = -1, vphys = -1, kin = 0, vin = 0, vnext = -1, vnin = 0;
    // a lane group's keys of a step: all 16 of a block, or half of one
    const int kgrp = col >> 2;  // the group whose keys this lane's row of K stands for
    const auto blk_of = [](int group) { return KL == 16 ? group : group >> 1; };
    const auto in_blk = [](int group) { return KL == 16 ? 0 : (group & 1) * 8; };
    const auto find_k = [&](int step) { kphys = page_of(step, blk_of(kgrp), kin); };
    const auto find_v = [&](int step) { vnext = page_of(step, blk_of(grp), vnin); };
    const auto load_k = [&] {
        const int64_t pg = (page0 + max(kphys, 0)) * a.Hkv + h;
        const uint8_t* const p = a.kc + (pg * a.bs + kin + in_blk(kgrp) + (col & 3)) * a.hd;
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int w = 0; w < L::kKw; w += 4) {
                const int d = grp * (HD / 4) + w * 4;
                load_words<4>(&kr[i][w], p + i * 4 * a.hd + (d < a.hd ? d : 0));
            }
        kbyte = a.ks[pg];
    };
    const auto load_v = [&] {
        vphys = vnext;
        vin = vnin;
        const int64_t pg = (page0 + max(vphys, 0)) * a.Hkv + h;
        const uint8_t* const p = a.vc + (pg * a.bs + vin + in_blk(grp)) * a.hd + (col * L::kD < a.hd ? col * L::kD : 0);
#pragma unroll
        for (int i = 0; i < KL; ++i) load_words<L::kVw>(vr[i], p + i * a.hd);
        vbyte = a.vs[pg];
    };

    f4 o[L::kD];
#pragma unroll
    for (int j = 0; j < L::kD; ++j) o[j] = f4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    // every row sees every key of a step that lies in [all_lo, all_hi)
    const int64_t all_hi = min<int64_t>(max<int64_t>(t.sp + t.r0 / a.G, 0) + 1, t.hi);
    const int64_t all_lo = a.window > 0 ? max<int64_t>(t.sp + (t.r0 + t.rows - 1) / a.G - a.window + 1, t.lo) : 0;
    const bool one_pos = t.r0 / a.G == (t.r0 + t.rows - 1) / a.G;
    int step = split * t.per + wave;
    if (step < end) {
        find_k(step);
        find_v(step);
        load_k();
        load_v();
        find_k(step + kWaves);
        find_v(step + kWaves);
    }
    for (; step < end; step += kWaves) {
        const float kscale = e8_scale(kbyte);
        // scores: tile i's row 4 g + e is key 4 i + e of block g
        f4 sc[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
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
        load_k();  // of the next step; behind the last, of whatever page find_k names
        find_k(step + 2 * kWaves);
        float vscale = e8_scale(vbyte);
        const int64_t key0 = t.base + static_cast<int64_t>(step) * kKeys;
        const bool masked = key0 + kKeys > all_hi || key0 < all_lo || key0 < t.lo || __any(vphys < 0);
        uint32_t seen_by_any = 0, seen = 0xFFFF;  // of the lane's keys, those that its row sees
        bool nan_path = false;
        float x[KL];
#pragma unroll
        for (int i = 0; i < KL; ++i) x[i] = sc[i >> 2][i & 3] * a.c;
        if (masked) {
            seen = 0;
            uint32_t some = 0;  // and those that any row may see
            const int64_t k0 = key0 + grp * KL;
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                if (vphys >= 0 && k0 + i < row_hi && k0 + i >= row_lo) seen |= 1u << i;
                if (vphys >= 0 && k0 + i < t.hi && k0 + i >= t.lo) some |= 1u << i;
                if (!(seen & (1u << i))) x[i] = -INFINITY;
            }
            // what no row sees may hold anything, NaN too: 0 times it must be 0
            uint32_t nan = vphys >= 0 && vbyte == 255 ? some : 0;
#pragma unroll
            for (int i = 0; i < KL; ++i)
#pragma unroll
                for (int w = 0; w < L::kVw; ++w) {
                    if (!(some & (1u << i))) vr[i][w] = 0;
                    nan |= nan_bytes(vr[i][w]);
                }
            // a NaN that some rows see and others do not
            nan_path = !one_pos && __any(nan != 0);
            seen_by_any = some;
            if (vbyte == 255 && (nan_path || some == 0)) vscale = 1.0f;
        }
        float mx = x[0];
#pragma unroll
        for (int i = 1; i < KL; ++i) mx = fmaxf(mx, x[i]);
        const float mn = fmaxf(m, max_over_groups(mx));
        if (__any(mn > m + kSlack)) {
            const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= by;
#pragma unroll
            for (int j = 0; j < L::kD; ++j) o[j] *= by;
            m = mn;
        }
        const float ref = (m == -INFINITY ? 0.0f : m) - kPShift;
        h8 p[KL / 8];
#pragma unroll
        for (int i = 0; i < KL; ++i) {
            const float w = __builtin_amdgcn_exp2f(x[i] - ref);
            l += w;
            p[i >> 3][i & 7] = (half_t)w;
        }
        if (nan_path) {
#pragma unroll
            for (int i = 0; i < KL; ++i)
#pragma unroll
                for (int w = 0; w < L::kVw; ++w) vr[i][w] = vbyte == 255 ? 0u : vr[i][w] & ~nan_bytes(vr[i][w]);
        }
#pragma unroll
        for (int j = 0; j < L::kD; j += 2)
#pragma unroll
            for (int k = 0; k < KL / 8; ++k) {
                h8 even, odd;
                v_pair(vr, k, j >> 2, (j >> 1) & 1, vscale, even, odd);
                o[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, p[k], o[j], 0, 0, 0);
                o[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, p[k], o[j + 1], 0, 0, 0);
            }
        if (nan_path) {  // the rows that see one of the NaN: V again, as ones in their places
            const int64_t pg = (page0 + max(vphys, 0)) * a.Hkv + h;
            const uint8_t* const q = a.vc + (pg * a.bs + vin + in_blk(grp)) * a.hd + (col * L::kD < a.hd ? col * L::kD : 0);
            h8 see[KL / 8];
#pragma unroll
            for (int i = 0; i < KL; ++i) {
                load_words<L::kVw>(vr[i], q + i * a.hd);
                see[i >> 3][i & 7] = (half_t)(seen & (1u << i) ? 1.0f : 0.0f);
            }
#pragma unroll
            for (int i = 0; i < KL; ++i)
#pragma unroll
                for (int w = 0; w < L::kVw; ++w)  // 0x38: one
                    vr[i][w] = seen_by_any & (1u << i) ? 0x38383838u & (vbyte == 255 ? ~0u : nan_bytes(vr[i][w])) : 0u;
#pragma unroll
            for (int j = 0; j < L::kD; j += 2) {
                f4 n0 = f4{0, 0, 0, 0}, n1 = n0;
#pragma unroll
                for (int k = 0; k < KL / 8; ++k) {
                    h8 even, odd;
                    v_pair(vr, k, j >> 2, (j >> 1) & 1, 1.0f, even, odd);
                    n0 = __builtin_amdgcn_mfma_f32_16x16x32_f16(even, see[k], n0, 0, 0, 0);
                    n1 = __builtin_amdgcn_mfma_f32_16x16x32_f16(odd, see[k], n1, 0, 0, 0);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (n0[e] > 0.0f) o[j][e] = __builtin_nanf("");
                    if (n1[e] > 0.0f) o[j + 1][e] = __builtin_nanf("");
                }
            }
        }
        load_v();
        find_v(step + 2 * kWaves);
    }

    // the waves' sums, joined
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
    const float inv_hd = 1.0f / static_cast<float>(a.hd);
    const int64_t group = (b * a.tiles[g] + tile) * a.Hkv + h;
    // [split][row][hd + 2]: sums, then the maximum and the sum of the weights
    float* const part = a.part + a.part0[g] + group * a.nsplit[g] * kRows * (a.hd + 2);
    const int64_t apart = static_cast<int64_t>(kRows) * (a.hd + 2);
    const auto put = [&](int r, int d, float sum, float tot) {
        const int rr = t.r0 + r, rs = rr / a.G;
        const int64_t rp = t.sp + rs;
        const bool rl = rp >= 0 && rp < t.sl && tot != 0.0f;
        a.out[(tok0 + rs) * a.os + (h * a.G + rr - rs * a.G) * a.hd + d] = (half_t)(rl ? sum / tot : 0.0f);
    };
    for (int i = threadIdx.x; i < t.rows * a.hd; i += kThreads) {
        const int r = small_div(i, inv_hd), d = i - r * a.hd;
        float mm = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, s_ml[w][0][r]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        float sum = 0.0f, tot = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {  // a wave that saw nothing: exp2(-inf) = 0 of zeros
            const float by = join_weight(s_ml[w][0][r], s_ml[w][1][r], ref);
            sum = fmaf(s_o[w][r][d], by, sum);
            tot = fmaf(s_ml[w][1][r], by, tot);
        }
        if (t.used <= 1) {
            put(r, d, sum, tot);
        } else {
            float* const p = part + split * apart + r * (a.hd + 2);
            store_agent(p + d, sum);
            if (d == 0) {
                store_agent(p + a.hd, mm);
                store_agent(p + a.hd + 1, tot);
            }
        }
    }
    if (t.used <= 1) return;
    // The tile's last workgroup joins the splits, in their order.  The partial sums went through
    // to memory and are read from there (agent scope), so no cache has to be written back.
    __builtin_amdgcn_s_waitcnt(kDrainVmem);
    __syncthreads();
    unsigned* const counter = a.count + a.cnt0[g] + group;
    if (threadIdx.x == 0)
        s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 static_cast<unsigned>(t.used - 1);
    __syncthreads();
    if (!s_last) return;
    if (threadIdx.x == 0) *counter = 0;  // for the next call
    float* const w_of = &s_o[0][0][0];   // [split][row], then the rows' sums
    static_assert(kMaxSplits * kRows * 2 <= kWaves * kRows * (HD + 4), "the splits' weights fit");
    float* const l_of = w_of + kMaxSplits * kRows;
    for (int i = threadIdx.x; i < t.used * t.rows; i += kThreads) {
        const int sp = i / t.rows, r = i - sp * t.rows;
        w_of[sp * kRows + r] = load_agent(part + sp * apart + r * (a.hd + 2) + a.hd);
        l_of[sp * kRows + r] = load_agent(part + sp * apart + r * (a.hd + 2) + a.hd + 1);
    }
    // the first splits' sums are asked for before their weights are known
    constexpr int kAhead = 8;
    float ahead[kAhead];
    const int r0 = small_div(threadIdx.x, inv_hd), d0 = threadIdx.x - r0 * a.hd;
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
        ahead[k] = load_agent(part + min(k, t.used - 1) * apart + (r0 < t.rows ? r0 * (a.hd + 2) + d0 : 0));
    __syncthreads();
    if (threadIdx.x < t.rows) {
        const int r = threadIdx.x;
        float mm = -INFINITY, tot = 0.0f;
        for (int sp = 0; sp < t.used; ++sp) mm = fmaxf(mm, w_of[sp * kRows + r]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
        for (int sp = 0; sp < t.used; ++sp) {
            const float l1 = l_of[sp * kRows + r], by = join_weight(w_of[sp * kRows + r], l1, ref);
            w_of[sp * kRows + r] = by;
            tot = fmaf(l1, by, tot);
        }
        s_ml[0][0][r] = tot;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < t.rows * a.hd; i += kThreads) {
        const int r = small_div(i, inv_hd), d = i - r * a.hd;
        const float* const p = part + r * (a.hd + 2) + d;
        float sum = 0.0f;
        int sp = 0;
        if (i == static_cast<int>(threadIdx.x)) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
                if (k < t.used) sum = fmaf(ahead[k], w_of[k * kRows + r], sum);
            sp = min(kAhead, t.used);
        }
        for (; sp + 8 <= t.used; sp += 8) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = load_agent(p + (sp + k) * apart);
#pragma unroll
            for (int k = 0; k < 8; ++k) sum = fmaf(v[k], w_of[(sp + k) * kRows + r], sum);
        }
        for (; sp < t.used; ++sp) sum = fmaf(load_agent(p + sp * apart), w_of[sp * kRows + r], sum);
        put(r, d, sum, s_ml[0][0][r]);
    }
}

// The segments of a call, those of few query rows in `few` and the others in `many`, with
// their tiles and splits (a segment of few tiles is split over its keys) and what they need of the
// workspace.  By the segments' B, S and table width alone.
static int kv8_attn_plan(const Kv8Attn& all, Kv8Attn& few, Kv8Attn& many, int64_t& bytes) {
    few = many = all;
    few.sg.n = many.sg.n = 0;
    int64_t floats = 0, counters = 0;
    const int asked = g_kv8_tile.load(std::memory_order_relaxed);
    for (int i = 0; i < all.sg.n; ++i) {
        const int64_t rows = all.sg.S[i] * all.G;
        const int64_t tiles16 = all.sg.B[i] * ceil_div(rows, kRows) * all.Hkv;
        const bool wide = asked == 0 ? rows > kFewRows && tiles16 >= few_tiles(all.hd) : asked != kRows;
        Kv8Attn& a = wide ? many : few;
        const int n = a.sg.n++;
        a.sg.off[n] = all.sg.off[i];
        a.sg.B[n] = all.sg.B[i];
        a.sg.S[n] = all.sg.S[i];
        a.sg.mb[n] = all.sg.mb[i];
        a.sg.bt[n] = all.sg.bt[i];
        a.sg.sl[n] = all.sg.sl[i];
        a.sg.sp[n] = all.sg.sp[i];
        const int64_t tile = wide ? kPromptRows : kRows, tiles = ceil_div(rows, tile);
        const int64_t groups = a.sg.B[n] * tiles * a.Hkv;
        const int64_t ns = std::clamp<int64_t>((wide ? prompt_want(all.hd) : kWant) / std::max<int64_t>(groups, 1), 1,
                                               std::min<int64_t>(a.sg.mb[n], wide ? kPromptSplits : kMaxSplits));
        a.tiles[n] = static_cast<int>(tiles);
        a.nsplit[n] = static_cast<int>(ns);
        a.first[n + 1] = a.first[n] + groups * ns;
        a.part0[n] = floats;
        a.cnt0[n] = counters;
        if (ns > 1) {
            floats += groups * ns * tile * (a.hd + 2);
            counters += groups;
        }
    }
    bytes = floats > 0 ? 4 * (kCounters + floats) : 0;
    return few.first[few.sg.n] <= kMaxGridX && many.first[many.sg.n] <= kMaxGridX ? MI_OK : MI_ERR_UNSUPPORTED;
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
    for (int i = 0; i < a.sg.n; ++i)  // a sequence's rows are numbered in 31 bits
        if (a.sg.S[i] * (Hq / Hkv) > INT32_MAX - kPromptRows) return MI_ERR_UNSUPPORTED;
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
    Kv8Attn a{}, few, many;
    int64_t bytes = 0, T = 0;
    for (int i = 0; i < num_segments && segments; ++i) {  // any packing of the segments
        const mi_kv_segment& g = segments[i];
        if (g.B > 0 && g.S > 0 && g.B < (int64_t{1} << 31) && g.S < (int64_t{1} << 31) && g.token_offset >= 0 &&
            g.token_offset < (int64_t{1} << 31))
            T = std::max(T, g.token_offset + g.B * g.S);
    }
    const int st = kv8_attn_shape(T, Hq, Hkv, head_dim, segments, num_segments, a);
    if (st != MI_OK) return st;
    const int pl = kv8_attn_plan(a, few, many, bytes);
    return pl != MI_OK ? pl : bytes;
}

extern "C" int mi_kv8_attention_test_tile(int rows) {
    if (rows != 0 && rows != mi::kRows && rows != mi::kPromptRows) return MI_ERR_INVALID_ARGUMENT;
    return mi::g_kv8_tile.exchange(rows);
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
    a.c = std::max(std::fabs(scale) * 1.4426950408889634f, 1e-37f);
    a.neg = scale < 0.0f;
    a.count = static_cast<unsigned*>(workspace);
    a.part = static_cast<float*>(workspace) + kCounters;
    Kv8Attn few, many;
    int64_t need = 0;
    const int pl = kv8_attn_plan(a, few, many, need);
    if (pl != MI_OK) return pl;
    if (need > 0 && (!workspace || workspace_bytes < need || !aligned16(workspace))) return MI_ERR_INVALID_ARGUMENT;
    const void* bufs[6] = {k_cache, v_cache, k_scale, v_scale, q, workspace};
    const int64_t lens[6] = {cells * block_size * head_dim, cells * block_size * head_dim, cells, cells, qb, need};
    for (int i = 0; i < 6; ++i) {
        if (overlaps(bufs[i], lens[i], out, ob)) return MI_ERR_ALIASING;
        if (i < 5 && overlaps(bufs[i], lens[i], workspace, need)) return MI_ERR_ALIASING;
    }
    const hipStream_t s = as_stream(stream);
    if (many.sg.n > 0) kv8_prompt_launch(many, s);
    if (few.sg.n > 0) {
        const dim3 grid(static_cast<unsigned>(few.first[few.sg.n]));
        int64_t groups = 0;
        for (int i = 0; i < few.sg.n; ++i) groups += few.sg.B[i] * few.tiles[i] * few.Hkv;
        const auto launch = [&](auto width) {
            constexpr int HD = decltype(width)::value;
            if (groups < kFill) kv8_attn_kernel<HD, 8><<<grid, dim3(512), 0, s>>>(few);
            else kv8_attn_kernel<HD, 4><<<grid, dim3(256), 0, s>>>(few);
        };
        if (head_dim <= 64) launch(std::integral_constant<int, 64>{});
        else if (head_dim <= 128) launch(std::integral_constant<int, 128>{});
        else launch(std::integral_constant<int, 256>{});
    }
    return launch_status();
}
