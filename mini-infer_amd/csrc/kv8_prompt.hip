// kv8_prompt.hip -- attention of many query rows over the 8-bit cache: prompts and chunks of
// prompts.  The mathematics and the roundings are kv8_attention.hip's.
//
// Bound by the matrix and vector units, not by HBM: a workgroup's 128 rows -- (token, query head
// of the KV head) -- share every key, so K and V are converted to fp16 once per workgroup, into LDS
// (the next tile's while this one is computed), and a wave multiplies 32 rows by tiles of
// 32x32x16.  As there, the scores are made transposed and their registers are the second
// product's operand: row r of a 32-key subtile stands for the key that puts a lane's eight
// scores of an operand in key order, so V^T is read from LDS in plain order.
//
// Two prompts of 3000 tokens, 28 query heads on 4, head_dim 128: 129 GFLOP in 168 us, 770 TFLOP/s, 69%
// of a large matrix product's rate here; one of 8192 tokens 481 GFLOP in 580 us, 830.  The matrix units
// are busy for a third of that, the vector units for somewhat more than half (a wave's step of 64
// keys: 32 products, and some 300 vector instructions: 32 exponentials, as many fmas, and the
// conversion of its share of K and V), and with two waves to a SIMD, what 241 registers leave, the two
// overlap little.  Tiles of 256 rows, which halve the conversions of a row, take as long: their
// one workgroup per CU has all its waves at the same stage.  Conversions placed among the second product's
// instructions cost 3%.
#include <type_traits>

#include "kv8_attn.h"
#include "mi_host.h"

namespace mi {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Keys of a tile: what two LDS buffers of K and V and two workgroups per CU allow.
template <int HD>
constexpr int prompt_keys() { return HD > 128 ? 32 : 64; }

// LDS reads 256 bytes a clock, 16 lanes of 16 bytes.  The 16-byte pieces of a row of K [key][HD] and
// of V^T [d][KT] are exchanged within the row so that 16 lanes on consecutive rows fall on
// different banks (with eight lanes apart only, every read took half as long again).
template <int HD>
__device__ __forceinline__ int k_piece(int key, int c) { return c ^ (HD == 64 ? key >> 1 & 7 : key & 15); }
template <int KT>
__device__ __forceinline__ int v_piece(int d, int c) {
    if constexpr (KT == 64) return c ^ ((d >> 1 & 7) ^ (d >> 4 & 1));
    else return c ^ (d >> 2 & 3);
}

// A vector register's offset, for a load relative to scalar registers: what the compiler knows to be
// uniform it reads through the scalar cache, and a scalar load is waited for together with LDS.
__device__ __forceinline__ uint32_t in_vgpr(uint32_t v) {
    asm("" : "+v"(v));
    return v;
}

// The next `n` instructions of a kind, in the scheduler's order.
constexpr int kMfma = 0x8, kDsRead = 0x100;
template <int KIND>
__device__ __forceinline__ void order(int n) {
#pragma unroll
    for (int i = 0; i < n; ++i) __builtin_amdgcn_sched_group_barrier(KIND, 1, 0);
}

template <int HD, bool WHOLE>
__global__ __launch_bounds__(256, HD > 128 ? 1 : 2) void kv8_prompt_kernel(Kv8Attn a) {
    constexpr int KT = prompt_keys<HD>();
    constexpr int kSub = KT / 32;             // 32-key subtiles
    constexpr int kSteps = HD / 16;           // MFMA steps of q . k
    constexpr int kDt = HD / 32;              // 32-wide tiles of d
    constexpr int kKu = KT * HD / 16 / 256;   // 16-byte units of K a lane converts
    constexpr int kTileBytes = KT * HD * 2;
    // two tiles of K and of V; afterwards the rows of the output
    __shared__ __attribute__((aligned(16))) uint8_t s_mem[4 * kTileBytes];
    const auto s_k = reinterpret_cast<half_t(*)[KT * HD]>(s_mem);
    const auto s_v = reinterpret_cast<half_t(*)[KT * HD]>(s_mem + 2 * kTileBytes);
    __shared__ int s_ok[2][KT / 16];
    __shared__ __attribute__((aligned(8))) int s_mark[2][2];  // the tile that has a block without a page; that has a NaN
    __shared__ __attribute__((aligned(4))) uint8_t s_bits[2][KT / 8][HD];  // V's NaN: a bit per key
    __shared__ bool s_last;
    const int hd = WHOLE ? HD : a.hd;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hf = lane >> 5;
    uint32_t id = blockIdx.x;
    int g = 0;
    while (id >= static_cast<uint32_t>(a.first[g + 1])) ++g;
    id -= static_cast<uint32_t>(a.first[g]);
    const int h = divmod(id, a.Hkv);
    const int64_t b = divmod(id, static_cast<int>(a.sg.B[g]));
    const int tile = a.tiles[g] - 1 - divmod(id, a.tiles[g]);  // a sequence's last tiles have the most keys: first
    const int split = static_cast<int>(id);  // outermost, as in kv8_attention.hip
    const TileKeys t = tile_keys<kPromptRows, KT, kPromptLeast>(a, g, b, tile);
    if (split >= max(t.used, 1)) return;
    const int64_t tok0 = a.sg.off[g] + b * t.S;

    // this lane's query column
    const int w0 = t.r0 + wave * 32;  // the wave's first row
    const int row = w0 + col, s = row / a.G, head = h * a.G + (row - s * a.G);
    const int64_t pos = t.sp + s;
    const bool live = wave * 32 + col < t.rows && pos >= 0 && pos < t.sl;
    const int row_hi = live ? static_cast<int>(min(pos + 1, t.hi)) : 0;
    const int row_lo = a.window > 0 ? static_cast<int>(min<int64_t>(max<int64_t>(pos - a.window + 1, 0), INT32_MAX)) : 0;
    h8 qf[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int d = i * 16 + hf * 8;
        qf[i] = h8(0);
        if (live && d < hd) qf[i] = ld8(a.q + (tok0 + s) * a.qs + head * hd + d);
        if (a.neg) qf[i] = -qf[i];
    }
    // keys that every live row of the wave sees, and that any does
    const int64_t wp0 = max<int64_t>(t.sp + w0 / a.G, 0);
    const int64_t wp1 = min(t.sp + (w0 + 31) / a.G, t.sl - 1);
    const int all_hi = static_cast<int>(min(wp0 + 1, t.hi)), any_hi = static_cast<int>(min(wp1 + 1, t.hi));
    const int all_lo = a.window > 0 ? static_cast<int>(min<int64_t>(max<int64_t>(wp1 - a.window + 1, 0), INT32_MAX)) : 0;
    const int any_lo = a.window > 0 ? static_cast<int>(max<int64_t>(wp0 - a.window + 1, 0)) : 0;
    const bool some_row = wave * 32 < t.rows && wp1 >= wp0;

    const int* const table = a.sg.bt[g] + b * a.sg.mb[g];
    const int sub = a.bs >> 4;
    const int nb = static_cast<int>(a.num_blocks);
    const int end = min((split + 1) * t.per, t.steps);
    const int base32 = static_cast<int>(t.base), lo32 = static_cast<int>(t.lo);
    const int hi32 = min(static_cast<int>(t.hi), base32 + end * KT);
    const int64_t page0 = a.layer * a.num_blocks;
    const int last_entry = static_cast<int>((t.hi - 1) >> 4) / sub;
    const uint64_t inv_sub = ((uint64_t{1} << 40) + sub - 1) / static_cast<uint32_t>(sub);
    // What a wave brings of a tile: of one 16-key block (half of one where a tile has two) K in units
    // of 16 bytes of a key, and V in units of four d of eight keys.  The block's page, scales and place
    // are found by the scalar unit, once for both; a lane adds offsets that never change.
    constexpr int kBlocks = KT / 16, kOwn = 4 / kBlocks;  // blocks of a tile; waves of a block
    constexpr int kKeysW = 16 / kOwn;                      // keys of a wave
    static_assert(kBlocks * kOwn == 4 && kKeysW * HD / 16 == 64 * kKu, "four waves bring a tile");
    const int blk = wave / kOwn, kw = wave % kOwn * kKeysW;  // the wave's block, its first key there
    const int vk = kKeysW == 16 ? (lane / (HD / 4) & 1) * 8 : 0, vd = lane % (HD / 4) * 4;  // of the wave's keys
    const bool has_v = HD >= 128 || lane < 32;  // heads of 64: 32 lanes hold 16 keys of V
    const int64_t page_bytes = static_cast<int64_t>(a.Hkv) * a.bs * hd;
    const uint8_t* const kbase = a.kc + (page0 * a.Hkv + h) * a.bs * hd + kw * hd;
    const uint8_t* const vbase = a.vc + (page0 * a.Hkv + h) * a.bs * hd + kw * hd;
    uint32_t koff[kKu];
#pragma unroll
    for (int u = 0; u < kKu; ++u) {
        const int key = (lane + u * 64) / (HD / 16), d = (lane + u * 64) % (HD / 16) * 16;
        koff[u] = key * hd + (d < hd ? d : 0);
    }
    const uint32_t voff = vk * hd + (vd < hd ? vd : 0);
    uint32_t kraw[kKu][4], vraw[8];
    int kb = 0, vb = 0, phys = -1, entry = 0, in_page = 0;
    bool in_split = false;
    // The table's entry of the wave's block of a tile, read a tile before its page is.
    const auto find = [&](int step) {
        const int key = base32 + step * KT + blk * 16;
        const uint32_t k16 = static_cast<uint32_t>(key) >> 4;  // < 2^22, sub <= 256: the quotient is exact
        const int idx = static_cast<int>(k16 * inv_sub >> 40);
        in_page = static_cast<int>(k16 - idx * sub) * 16;
        in_split = key < hi32;
        entry = *reinterpret_cast<const int*>(reinterpret_cast<const uint8_t*>(table) + in_vgpr(4u * min(idx, last_entry)));
    };
    const auto load = [&] {
        const int e = __builtin_amdgcn_readfirstlane(entry);
        phys = in_split && static_cast<uint32_t>(e) < static_cast<uint32_t>(nb) ? e : -1;
        const int64_t pg = max(phys, 0), at = pg * page_bytes + in_page * hd, cell = (page0 + pg) * a.Hkv + h;
        const uint8_t *const kp = kbase + at, *const vp = vbase + at;
        const uint32_t ko = in_vgpr(koff[0]), vo = in_vgpr(voff);
#pragma unroll
        for (int u = 0; u < kKu; ++u)
            load_words<4>(kraw[u], WHOLE ? kp + ko + u * (1024 / HD) * HD : kp + in_vgpr(koff[u]));
        kb = a.ks[cell];
#pragma unroll
        for (int i = 0; i < 8; ++i) load_words<1>(&vraw[i], WHOLE ? vp + vo + i * HD : vp + in_vgpr(voff + i * hd));
        vb = a.vs[cell];
    };
    const auto store = [&](int step, int buf) {
#pragma unroll
        for (int u = 0; u < kKu; ++u) {
            const int key = blk * 16 + kw + (lane + u * 64) / (HD / 16), c = (lane + u * 64) % (HD / 16) * 2;
            const float scale = e8_scale(kb);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const h2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i], scale, false);
                const h2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i], scale, true);
                const h2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i + 1], scale, false);
                const h2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i + 1], scale, true);
                *reinterpret_cast<h8*>(&s_k[buf][key * HD + k_piece<HD>(key, c + i) * 8]) =
                    h8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
            }
        }
        // V: what no row may see is zero, whatever it holds, and NaN is zero with its place kept
        // in s_bits
        const int tile0 = base32 + step * KT, vkey = blk * 16 + kw + vk, key0 = tile0 + vkey;
        float scale = e8_scale(vb);
        uint32_t nan = vb == 255 ? 0x80u : 0u, bits = 0;
        if (tile0 + KT > hi32 || tile0 < lo32 || phys < 0) {
            const bool ok = phys >= 0 && key0 < hi32 && key0 + 8 > lo32;
            if (!ok) scale = 1.0f, nan = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!ok || key0 + i >= hi32 || key0 + i < lo32) vraw[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) nan |= (vraw[i] & 0x7F7F7F7Fu) + 0x01010101u;
        if (__any(nan & 0x80808080u)) {
            const bool all_nan = __builtin_bit_cast(uint32_t, scale) >> 23 == 255;
            if (all_nan) scale = 1.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const bool in = key0 + i < hi32 && key0 + i >= lo32;
                const uint32_t n = all_nan ? (in ? ~0u : 0u) : nan_bytes(vraw[i]);
                bits |= (n & 0x01010101u) << i;
                vraw[i] &= ~n;
            }
        }
        if (has_v) {
            uint32_t w[4][4];  // [d][pair of keys]
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {  // two keys' bytes of d and of d + 1, side by side
                    const uint32_t x = __builtin_amdgcn_perm(vraw[2 * i + 1], vraw[2 * i], j ? 0x07030602u : 0x05010400u);
                    w[2 * j][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, false));
                    w[2 * j + 1][i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, scale, true));
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<u4*>(&s_v[buf][(vd + i) * KT + v_piece<KT>(vd + i, vkey >> 3) * 8]) =
                    u4{w[i][0], w[i][1], w[i][2], w[i][3]};
            *reinterpret_cast<uint32_t*>(&s_bits[buf][vkey >> 3][vd]) = bits;
            if (vd == 0) s_ok[buf][blk] = phys >= 0;
            if (phys < 0) s_mark[buf][0] = step;
            if (bits) s_mark[buf][1] = step;
        }
    };

    f16v o[kDt];
#pragma unroll
    for (int j = 0; j < kDt; ++j) o[j] = f16v(0);
    float m = -INFINITY, l = 0.0f;
    int step = split * t.per;
    if (tid < 4) s_mark[tid >> 1][tid & 1] = -1;
    __syncthreads();
    if (step < end) {
        find(step);
        load();
        find(step + 1);
        store(step, 0);
    }
    __syncthreads();
    for (int buf = 0; step < end; ++step, buf ^= 1) {
        load();  // of the next tile; behind the last, of whatever page find names
        find(step + 2);
        const int key0 = base32 + step * KT;
        const half_t *const sk = s_k[buf], *const sv = s_v[buf];
        if (some_row && key0 < any_hi && key0 + KT > any_lo) {
            // Each fragment is asked for while the products before it run: LDS answers in some
            // 100 cycles, a product takes 32.
            const int2 mark = *reinterpret_cast<const int2*>(s_mark[buf]);
            f16v sc[kSub];
            h8 kf[2][kSteps], vf[2][kSub * 2];
            const auto k_read = [&](int ks) {
                // row 16 i + 8 j + 4 f + e of the subtile stands for key 16 i + 8 f + 4 j + e
                const int key = ks * 32 + (col & 0x13) + ((col & 4) << 1) + ((col & 8) >> 1);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) kf[ks & 1][i] = ld8(sk + key * HD + k_piece<HD>(key, 2 * i + hf) * 8);
            };
            const auto v_read = [&](int j) {
                const int d = j * 32 + col;
#pragma unroll
                for (int k = 0; k < kSub * 2; ++k) vf[j & 1][k] = ld8(sv + d * KT + v_piece<KT>(d, 2 * k + hf) * 8);
            };
            k_read(0);
#pragma unroll
            for (int ks = 0; ks < kSub; ++ks) {
                if (ks + 1 < kSub) k_read(ks + 1);
                else v_read(0);
                sc[ks] = f16v(0);
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
                    sc[ks] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[ks & 1][i], qf[i], sc[ks], 0, 0, 0);
            }
            order<kDsRead>(kSteps);
#pragma unroll
            for (int i = 0; i < kSub * kSteps; ++i) {
                order<kMfma>(1);
                order<kDsRead>(1);
            }
            const bool masked = key0 + KT > all_hi || key0 < all_lo ||
                                __builtin_amdgcn_readfirstlane(mark.x) == step;
            const bool marked = __builtin_amdgcn_readfirstlane(mark.y) == step;
            if (masked) {
#pragma unroll
                for (int ks = 0; ks < kSub; ++ks)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int key = key0 + ks * 32 + (i >> 3) * 16 + hf * 8 + (i & 7);
                        if (!(s_ok[buf][ks * 2 + (i >> 3)] && key < row_hi && key >= row_lo)) sc[ks][i] = -INFINITY;
                    }
            }
            float mx = sc[0][0];
#pragma unroll
            for (int ks = 0; ks < kSub; ++ks)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[ks][i]);
            uint32_t pa, pb;
            pair_xor32(__builtin_bit_cast(uint32_t, mx), pa, pb);
            mx = fmaxf(__builtin_bit_cast(float, pa), __builtin_bit_cast(float, pb));
            const float mn = fmaxf(m, mx * a.c);  // a.c > 0
            // the reference follows the maximum only where the weights would grow past 2^15
            if (__any(mn > m + kSlack)) {
                const float by = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
                l *= by;
#pragma unroll
                for (int j = 0; j < kDt; ++j) o[j] *= by;
                m = mn;
            }
            const float ref = kPShift - (m == -INFINITY ? 0.0f : m);
            h8 p[kSub * 2];
#pragma unroll
            for (int ks = 0; ks < kSub; ++ks)
#pragma unroll
                for (int i = 0; i < 16; i += 2) {
                    const h2 w = {(half_t)__builtin_amdgcn_exp2f(fmaf(sc[ks][i], a.c, ref)),
                                  (half_t)__builtin_amdgcn_exp2f(fmaf(sc[ks][i + 1], a.c, ref))};
                    p[ks * 2 + (i >> 3)][i & 7] = w[0];
                    p[ks * 2 + (i >> 3)][(i & 7) + 1] = w[1];
                    // their sum, of the weights as rounded
                    l = __builtin_amdgcn_fdot2(w, h2{(half_t)1.0f, (half_t)1.0f}, l, false);
                }
#pragma unroll
            for (int j = 0; j < kDt; ++j) {
                if (j + 1 < kDt) v_read(j + 1);
#pragma unroll
                for (int k = 0; k < kSub * 2; ++k)
                    o[j] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vf[j & 1][k], p[k], o[j], 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < kDt * kSub * 2; ++i) {
                order<kMfma>(1);
                order<kDsRead>(1);
            }
            if (marked) {  // rare: a NaN reaches the rows that see its key, and no other
                uint8_t see[KT / 8];
#pragma unroll
                for (int c = 0; c < KT / 8; ++c) {
                    see[c] = 0;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int key = key0 + c * 8 + i;
                        if (s_ok[buf][c >> 1] && key < row_hi && key >= row_lo) see[c] |= 1u << i;
                    }
                }
#pragma unroll
                for (int j = 0; j < kDt; ++j)
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const int d = j * 32 + (i >> 2) * 8 + hf * 4 + (i & 3);
                        uint32_t hit = 0;
#pragma unroll
                        for (int c = 0; c < KT / 8; ++c) hit |= s_bits[buf][c][d] & see[c];
                        if (hit) o[j][i] = __builtin_nanf("");
                    }
            }
        }
        if (step + 1 < end) store(step + 1, buf ^ 1);
        __syncthreads();
    }

    l += __shfl_xor(l, 32, kWave);
    const auto out_row = [&](int r) {  // of row r of the tile
        const int rr = t.r0 + r, rs = rr / a.G;
        return a.out + (tok0 + rs) * a.os + (h * a.G + rr - rs * a.G) * hd;
    };
    if (t.used <= 1) {
        // By way of LDS, half of d at a time, so that a row leaves in runs of 16 bytes and more.
        const bool some = live && l != 0.0f;
        const float inv = some ? 1.0f / l : 0.0f;
        constexpr int kPitch = HD / 2 + 8;  // halves of a row, off the banks of the one before
        static_assert(kPromptRows * kPitch * 2 <= 4 * kTileBytes, "the rows fit");
        half_t* const rows = reinterpret_cast<half_t*>(s_mem) + wave * 32 * kPitch;
        typedef _Float16 h4 __attribute__((ext_vector_type(4)));
        const bool vec = (reinterpret_cast<uintptr_t>(a.out) & 15) == 0 && (a.os & 7) == 0;
#pragma unroll
        for (int part = 0; part < 2; ++part) {
#pragma unroll
            for (int jj = 0; jj < kDt / 2; ++jj)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const int j = part * (kDt / 2) + jj;
                    h4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = (half_t)(some ? o[j][i + e] * inv : 0.0f);
                    *reinterpret_cast<h4*>(rows + col * kPitch + jj * 32 + (i >> 2) * 8 + hf * 4) = v;
                }
            __builtin_amdgcn_wave_barrier();  // a wave's own rows: its LDS accesses keep their order
#pragma unroll
            for (int i = 0; i < 32 * HD / 2 / 8 / 64; ++i) {
                const int u = i * 64 + lane, r = u / (HD / 16), d = u % (HD / 16) * 8, dd = part * (HD / 2) + d;
                const h8 v = *reinterpret_cast<const h8*>(rows + r * kPitch + d);
                if (wave * 32 + r < t.rows && dd < hd) {
                    half_t* const to = out_row(wave * 32 + r) + dd;
                    if (vec) {
                        *reinterpret_cast<h8*>(to) = v;
                    } else {
#pragma unroll
                        for (int e = 0; e < 8; ++e) to[e] = v[e];
                    }
                }
            }
            __builtin_amdgcn_wave_barrier();
        }
        return;
    }
    // Partial sums [split][row][hd], then the rows' maxima and sums of weights; written through to
    // memory and read from there (agent scope), joined by the tile's last workgroup in their order.
    const int64_t group = (b * a.tiles[g] + tile) * a.Hkv + h;
    const int64_t apart = static_cast<int64_t>(kPromptRows) * (hd + 2);
    float* const part = a.part + a.part0[g] + group * a.nsplit[g] * apart;
    {
        const int r = wave * 32 + col;
        float* const to = part + split * apart + static_cast<int64_t>(r) * hd;
        float* const ml = part + split * apart + static_cast<int64_t>(kPromptRows) * hd + 2 * r;
#pragma unroll
        for (int j = 0; j < kDt; ++j)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const int d = j * 32 + (i >> 2) * 8 + hf * 4;
                if (d < hd)
                    st8_stream_wt(reinterpret_cast<half_t*>(to + d),
                                  __builtin_bit_cast(h8, f4{o[j][i], o[j][i + 1], o[j][i + 2], o[j][i + 3]}));
            }
        if (hf == 0) {
            store_agent(ml, m);
            store_agent(ml + 1, l);
        }
    }
    __builtin_amdgcn_s_waitcnt(kDrainVmem);
    __syncthreads();
    unsigned* const counter = a.count + a.cnt0[g] + group;
    if (tid == 0)
        s_last = __hip_atomic_fetch_add(counter, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
                 static_cast<unsigned>(t.used - 1);
    __syncthreads();
    if (!s_last) return;
    if (tid == 0) *counter = 0;  // for the next call
    float* const w_of = reinterpret_cast<float*>(s_mem);  // [split][row]: what a split's sums count
    static_assert((kPromptSplits + 1) * kPromptRows * 4 <= 4 * kTileBytes, "the weights of kPromptSplits splits fit");
    float* const tot_of = w_of + kPromptSplits * kPromptRows;
    if (tid < kPromptRows) {
        const float* const ml = part + static_cast<int64_t>(kPromptRows) * hd + 2 * tid;
        float mm = -INFINITY, tot = 0.0f;
        for (int sp = 0; sp < t.used; ++sp) mm = fmaxf(mm, load_agent(ml + sp * apart));
        const float ref = mm == -INFINITY ? 0.0f : mm;
        for (int sp = 0; sp < t.used; ++sp) {
            const float l1 = load_agent(ml + sp * apart + 1), by = join_weight(load_agent(ml + sp * apart), l1, ref);
            w_of[sp * kPromptRows + tid] = by;
            tot = fmaf(l1, by, tot);
        }
        const int64_t rp = t.sp + (t.r0 + tid) / a.G;
        tot_of[tid] = rp >= 0 && rp < t.sl ? tot : 0.0f;
    }
    __syncthreads();
    const int pieces = hd >> 3;  // of eight d
    const float inv_pieces = 1.0f / static_cast<float>(pieces);
    for (int i = tid; i < t.rows * pieces; i += 256) {
        const int r = small_div(i, inv_pieces), d = (i - r * pieces) * 8;
        const uint64_t* const from = reinterpret_cast<const uint64_t*>(part + static_cast<int64_t>(r) * hd + d);
        float sum[8] = {};
        for (int sp = 0; sp < t.used; ++sp) {
            const float w = w_of[sp * kPromptRows + r];
            uint64_t v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = __hip_atomic_load(from + sp * (apart / 2) + e, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                sum[2 * e] = fmaf(__builtin_bit_cast(float, static_cast<uint32_t>(v[e])), w, sum[2 * e]);
                sum[2 * e + 1] = fmaf(__builtin_bit_cast(float, static_cast<uint32_t>(v[e] >> 32)), w, sum[2 * e + 1]);
            }
        }
        const float tot = tot_of[r];
        half_t* const to = out_row(r) + d;
#pragma unroll
        for (int e = 0; e < 8; ++e) to[e] = (half_t)(tot != 0.0f ? sum[e] / tot : 0.0f);
    }
}

void kv8_prompt_launch(const Kv8Attn& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.first[a.sg.n])), block(256);
    const auto launch = [&](auto width) {
        constexpr int HD = decltype(width)::value;
        if (a.hd == HD) kv8_prompt_kernel<HD, true><<<grid, block, 0, s>>>(a);
        else kv8_prompt_kernel<HD, false><<<grid, block, 0, s>>>(a);
    };
    if (a.hd <= 64) launch(std::integral_constant<int, 64>{});
    else if (a.hd <= 128) launch(std::integral_constant<int, 128>{});
    else launch(std::integral_constant<int, 256>{});
}

}  // namespace mi
