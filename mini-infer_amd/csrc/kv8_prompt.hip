// kv8_prompt.hip -- attention of many query rows over the 8-bit cache: prompts and chunks of
// prompts.  The mathematics and the roundings are kv8_attention.hip's.
//
// Bound by the matrix and vector units, not by HBM: a workgroup's 128 rows -- (token, query head
// of the KV head) -- share every key, so K and V are converted to fp16 once per workgroup, into LDS
// (the next tile's while this one is computed), and a wave multiplies 32 rows by tiles of
// 32x32x16.  As there, the scores are made transposed and their registers are the second
// product's operand: row r of a 32-key subtile stands for the key that puts a lane's eight
// scores of an operand in key order, so V^T is read from LDS in plain order.
#include "kv8_attn.h"
#include "mi_host.h"

namespace mi {

typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Keys of a tile: what two LDS buffers of K and V and two workgroups per CU allow.
template <int HD>
constexpr int prompt_keys() { return HD > 128 ? 32 : 64; }

// 16-byte pieces of a row of K [key][HD] and of V^T [d][keys] are exchanged within groups of
// eight (four for rows of 64 bytes) so that lanes on consecutive rows fall on different banks.
__device__ __forceinline__ int k_piece(int key, int c) { return c ^ ((key & 3) | ((key >> 1) & 4)); }
template <int KT>
__device__ __forceinline__ int v_piece(int d, int c) {
    if constexpr (KT == 64) return c ^ (((d >> 2) & 7) ^ ((d & 3) << 1));
    else return c ^ (((d >> 2) & 3) ^ (d & 2));
}

// The next `n` instructions of a kind, in the scheduler's order.
constexpr int kMfma = 0x8, kDsRead = 0x100;
template <int KIND>
__device__ __forceinline__ void order(int n) {
#pragma unroll
    for (int i = 0; i < n; ++i) __builtin_amdgcn_sched_group_barrier(KIND, 1, 0);
}

template <int HD, int WAVES>
__global__ __launch_bounds__(WAVES * 64, HD > 128 ? WAVES / 4 : 2) void kv8_prompt_kernel(Kv8Attn a) {
    constexpr int KT = prompt_keys<HD>();
    constexpr int kRowsT = WAVES * 32;        // query rows
    constexpr bool kRoles = WAVES == 8;       // the first four waves bring K, the others V
    constexpr int kSub = KT / 32;             // 32-key subtiles
    constexpr int kSteps = HD / 16;           // MFMA steps of q . k
    constexpr int kDt = HD / 32;              // 32-wide tiles of d
    constexpr int kKu = KT * HD / 16 / 256;   // 16-byte units of K a lane converts
    constexpr bool kAllV = KT / 8 * (HD / 4) >= 256;
    __shared__ __attribute__((aligned(16))) half_t s_k[2][KT * HD];
    __shared__ __attribute__((aligned(16))) half_t s_v[2][KT * HD];
    __shared__ int s_ok[2][KT / 16], s_nan[2];
    __shared__ __attribute__((aligned(4))) uint8_t s_bits[2][KT / 8][HD];  // V's NaN: a bit per key
    __shared__ bool s_last;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, hf = lane >> 5;
    uint32_t id = blockIdx.x;
    int g = 0;
    while (id >= static_cast<uint32_t>(a.first[g + 1])) ++g;
    id -= static_cast<uint32_t>(a.first[g]);
    const int h = divmod(id, a.Hkv);
    const int split = divmod(id, a.nsplit[g]);
    // a sequence's last tiles have the most keys: first
    const int64_t b = id % static_cast<uint32_t>(a.sg.B[g]);
    const int tile = a.tiles[g] - 1 - static_cast<int>(id / static_cast<uint32_t>(a.sg.B[g]));
    const TileKeys t = tile_keys<kRowsT, KT, 4>(a, g, b, tile);
    if (split >= max(t.used, 1)) return;
    const int64_t tok0 = a.sg.off[g] + b * t.S;

    // this lane's query column
    const int w0 = t.r0 + wave * 32;  // the wave's first row
    const int row = w0 + col, s = row / a.G, head = h * a.G + (row - s * a.G);
    const int64_t pos = t.sp + s;
    const bool mine = wave * 32 + col < t.rows, live = mine && pos >= 0 && pos < t.sl;
    const int row_hi = live ? static_cast<int>(min(pos + 1, t.hi)) : 0;
    const int row_lo = a.window > 0 ? static_cast<int>(min<int64_t>(max<int64_t>(pos - a.window + 1, 0), INT32_MAX)) : 0;
    h8 qf[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int d = i * 16 + hf * 8;
        qf[i] = h8(0);
        if (live && d < a.hd) qf[i] = ld8(a.q + (tok0 + s) * a.qs + head * a.hd + d);
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
    const float inv_sub = 1.0f / static_cast<float>(sub);
    const int nb = static_cast<int>(a.num_blocks);
    const int end = min((split + 1) * t.per, t.steps);
    const int base32 = static_cast<int>(t.base), lo32 = static_cast<int>(t.lo);
    const int hi32 = min(static_cast<int>(t.hi), base32 + end * KT);
    const int64_t page0 = a.layer * a.num_blocks;
    const auto page_of = [&](int key, int& in_page) {  // as in kv8_attention.hip: every load is made
        const int k16 = key >> 4;
        const int idx = small_div(k16, inv_sub);
        in_page = (k16 - idx * sub) * 16;
        const int phys = table[key < hi32 ? idx : 0];
        return key < hi32 && static_cast<uint32_t>(phys) < static_cast<uint32_t>(nb) ? phys : -1;
    };

    // what this lane brings of a tile: of K, units of 16 bytes of a key; of V, four d of eight keys
    const int lid = kRoles ? tid & 255 : tid;
    const bool has_k = !kRoles || wave < 4;
    const int vk = lid / (HD / 4) * 8, vd = lid % (HD / 4) * 4;
    const bool has_v = (!kRoles || wave >= 4) && (kAllV || vk < KT);
    const uint32_t page_bytes = static_cast<uint32_t>(a.Hkv * a.bs * a.hd);  // of all heads: < 2^31
    const uint8_t* const kbase = a.kc + (page0 * a.Hkv + h) * a.bs * a.hd;
    const uint8_t* const vbase = a.vc + (page0 * a.Hkv + h) * a.bs * a.hd + (vk & 8) * a.hd + (vd < a.hd ? vd : 0);
    const uint8_t *const ksc = a.ks + page0 * a.Hkv + h, *const vsc = a.vs + page0 * a.Hkv + h;
    int koff[kKu];
#pragma unroll
    for (int u = 0; u < kKu; ++u) {
        const int key = (lid + u * 256) / (HD / 16) & 15, d = (lid + u * 256) % (HD / 16) * 16;
        koff[u] = key * a.hd + (d < a.hd ? d : 0);
    }
    uint32_t kraw[kKu][4], vraw[8];
    int kb[kKu], vb = 0, vphys = -1, vfound = -1, vin = 0, kphys[kKu], kin[kKu];
    const auto find = [&](int step) {
        const int key0 = base32 + step * KT;
        if (has_k) {
#pragma unroll
            for (int u = 0; u < kKu; ++u) kphys[u] = page_of(key0 + ((lid + u * 256) / (HD / 16) & ~15), kin[u]);
        }
        // every lane, as it also says which blocks of the tile have a page
        vfound = page_of(key0 + ((kAllV || vk < KT ? vk : 0) & ~15), vin);
    };
    const auto load = [&] {
        vphys = vfound;
        if (has_k) {
#pragma unroll
            for (int u = 0; u < kKu; ++u) {
                const uint32_t pg = max(kphys[u], 0);
                load_words<4>(kraw[u], kbase + static_cast<uint64_t>(pg) * page_bytes + (kin[u] * a.hd + koff[u]));
                kb[u] = ksc[static_cast<uint64_t>(pg) * static_cast<uint32_t>(a.Hkv)];
            }
        }
        if (!kRoles || wave >= 4) {
            const uint32_t pg = max(vphys, 0);
            const uint8_t* p = vbase + static_cast<uint64_t>(pg) * page_bytes + vin * a.hd;
#pragma unroll
            for (int i = 0; i < 8; ++i, p += a.hd) load_words<1>(&vraw[i], p);
            vb = vsc[static_cast<uint64_t>(pg) * static_cast<uint32_t>(a.Hkv)];
        }
    };
    const auto store = [&](int step, int buf) {
        if (has_k) {
#pragma unroll
            for (int u = 0; u < kKu; ++u) {
                const int key = (lid + u * 256) / (HD / 16), c = (lid + u * 256) % (HD / 16) * 2;
                const float scale = e8_scale(kb[u]);
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const h2 x0 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i], scale, false);
                    const h2 x1 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i], scale, true);
                    const h2 x2 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i + 1], scale, false);
                    const h2 x3 = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(kraw[u][2 * i + 1], scale, true);
                    *reinterpret_cast<h8*>(&s_k[buf][key * HD + k_piece(key, c + i) * 8]) =
                        h8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
                }
            }
        }
        if (has_v) {
            // what no row may see is zero, whatever it holds, and NaN is zero with its place
            // kept in s_bits
            const int tile0 = base32 + step * KT, key0 = tile0 + vk;
            float scale = e8_scale(vb);
            uint32_t nan = vb == 255 ? 0x80u : 0u, bits = 0;
            if (tile0 + KT > hi32 || tile0 < lo32 || __any(vphys < 0)) {
                const bool ok = vphys >= 0 && key0 < hi32 && key0 + 8 > lo32;
                if (!ok) scale = 1.0f, nan = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (!ok || key0 + i >= hi32 || key0 + i < lo32) vraw[i] = 0;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) nan |= (vraw[i] & 0x7F7F7F7Fu) + 0x01010101u;
            if (nan & 0x80808080u) {
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
            uint32_t w[4][4];  // [d][pair of keys]
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const h2 x = j ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vraw[2 * i], scale, true)
                                   : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vraw[2 * i], scale, false);
                    const h2 y = j ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vraw[2 * i + 1], scale, true)
                                   : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(vraw[2 * i + 1], scale, false);
                    const uint32_t ux = __builtin_bit_cast(uint32_t, x), uy = __builtin_bit_cast(uint32_t, y);
                    w[2 * j][i] = __builtin_amdgcn_perm(uy, ux, 0x05040100u);
                    w[2 * j + 1][i] = __builtin_amdgcn_perm(uy, ux, 0x07060302u);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<u4*>(&s_v[buf][(vd + i) * KT + v_piece<KT>(vd + i, vk >> 3) * 8]) =
                    u4{w[i][0], w[i][1], w[i][2], w[i][3]};
            if (vd == 0 && (vk & 8) == 0) s_ok[buf][vk >> 4] = vphys >= 0;
            *reinterpret_cast<uint32_t*>(&s_bits[buf][vk >> 3][vd]) = bits;
            if (bits) s_nan[buf] = step;
        }
    };

    f16v o[kDt];
#pragma unroll
    for (int j = 0; j < kDt; ++j) o[j] = f16v(0);
    float m = -INFINITY, l = 0.0f;
    int step = split * t.per;
    if (tid < 2) s_nan[tid] = -1;
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
            f16v sc[kSub];
            h8 kf[2][kSteps], vf[2][kSub * 2];
            const auto k_read = [&](int ks) {
                // row 16 i + 8 j + 4 f + e of the subtile stands for key 16 i + 8 f + 4 j + e
                const int key = ks * 32 + (col & 0x13) + ((col & 4) << 1) + ((col & 8) >> 1);
#pragma unroll
                for (int i = 0; i < kSteps; ++i) kf[ks & 1][i] = ld8(sk + key * HD + k_piece(key, 2 * i + hf) * 8);
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
            int in_cache = 1;
#pragma unroll
            for (int i = 0; i < KT / 16; ++i) in_cache &= s_ok[buf][i];
            const bool masked = key0 + KT > all_hi || key0 < all_lo || __builtin_amdgcn_readfirstlane(in_cache) == 0;
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
            // the reference follows the maximum only where the weights would grow past 2^15.5
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
                for (int i = 0; i < 16; ++i) {
                    const float w = __builtin_amdgcn_exp2f(fmaf(sc[ks][i], a.c, ref));
                    l += w;
                    p[ks * 2 + (i >> 3)][i & 7] = (half_t)w;
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
            if (__builtin_amdgcn_readfirstlane(s_nan[buf]) == step) {  // rare: a NaN reaches the rows that see its key, and no other
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
    const auto out_row = [&](int r) {  // of the tile, and whether it is live
        const int rr = t.r0 + r, rs = rr / a.G;
        const int64_t rp = t.sp + rs;
        half_t* const to = a.out + (tok0 + rs) * a.os + (h * a.G + rr - rs * a.G) * a.hd;
        return std::pair<half_t*, bool>(to, rp >= 0 && rp < t.sl);
    };
    if (t.used <= 1) {
        if (!mine) return;
        const auto [to, on] = out_row(wave * 32 + col);
        const bool some = on && l != 0.0f;
        const float inv = some ? 1.0f / l : 0.0f;
#pragma unroll
        for (int j = 0; j < kDt; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int d = j * 32 + (i >> 2) * 8 + hf * 4 + (i & 3);
                if (d < a.hd) to[d] = (half_t)(some ? o[j][i] * inv : 0.0f);
            }
        return;
    }
    // partial sums [split][d, maximum, sum][row]
    const int64_t group = (b * a.tiles[g] + tile) * a.Hkv + h;
    const int64_t apart = static_cast<int64_t>(kRowsT) * (a.hd + 2);
    float* const part = a.part + a.part0[g] + group * a.nsplit[g] * apart;
    {
        float* const to = part + split * apart + wave * 32 + col;
#pragma unroll
        for (int j = 0; j < kDt; ++j)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int d = j * 32 + (i >> 2) * 8 + hf * 4 + (i & 3);
                if (d < a.hd) store_agent(to + d * kRowsT, o[j][i]);
            }
        if (hf == 0) {
            store_agent(to + a.hd * kRowsT, m);
            store_agent(to + (a.hd + 1) * kRowsT, l);
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
    if (tid == 0) *counter = 0;
    const int r = tid & (kRowsT - 1);
    if (r >= t.rows) return;
    const float* const from = part + r;
    float mm = -INFINITY, tot = 0.0f;
    for (int sp = 0; sp < t.used; ++sp) mm = fmaxf(mm, load_agent(from + sp * apart + a.hd * kRowsT));
    const float ref = mm == -INFINITY ? 0.0f : mm;
    const auto weight = [&](int sp) {
        return join_weight(load_agent(from + sp * apart + a.hd * kRowsT),
                           load_agent(from + sp * apart + (a.hd + 1) * kRowsT), ref);
    };
    for (int sp = 0; sp < t.used; ++sp)
        tot = fmaf(load_agent(from + sp * apart + (a.hd + 1) * kRowsT), weight(sp), tot);
    const auto [to, on] = out_row(r);
    const bool some = on && tot != 0.0f;
    for (int d = tid / kRowsT * 8; d < a.hd; d += 16) {  // two lanes per row
        float sum[8] = {};
        for (int sp = 0; sp < t.used; ++sp) {
            const float w = weight(sp);
            float v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = load_agent(from + sp * apart + (d + e) * kRowsT);
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] = fmaf(v[e], w, sum[e]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) to[d + e] = (half_t)(some ? sum[e] / tot : 0.0f);
    }
}

template <int WAVES>
static void prompt_go(const Kv8Attn& a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.first[a.sg.n])), block(WAVES * 64);
    if (a.hd <= 64) kv8_prompt_kernel<64, WAVES><<<grid, block, 0, s>>>(a);
    else if (a.hd <= 128) kv8_prompt_kernel<128, WAVES><<<grid, block, 0, s>>>(a);
    else kv8_prompt_kernel<256, WAVES><<<grid, block, 0, s>>>(a);
}

void kv8_prompt_launch(const Kv8Attn& a, hipStream_t s) {
    if (a.rows == 256) prompt_go<8>(a, s);
    else prompt_go<4>(a, s);
}

}  // namespace mi
