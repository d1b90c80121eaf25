// kv8.hip -- K and V rows into the paged cache held in 8 bits (kv8.h).
//
// A page's exponent is the least e in [-32, 8] with |x| <= 448 * 2^e for the page's
// finite values (448: e4m3's largest number; fp16 needs no more than that range).  At
// e = 8 values are held to 61440, the largest of the page's numbers that fp16 has too;
// infinities and NaN become NaN.  A call's tokens of one page are known together, so
// a page that the call begins (it writes slot 0) gets the exponent of all of them; a page
// that holds tokens already keeps at least its exponent, and where the new ones need a
// larger one, its other slots are requantised by 2^(old - new), rounded again to nearest even.
#include <algorithm>

#include "kv8.h"
#include "mi_host.h"

namespace mi {

constexpr int kE8Min = -32, kE8Max = 8;

struct Kv8Write {
    const half_t* src[2];
    uint8_t* cache[2];
    uint8_t* scale[2];
    int64_t stride[2];
    int64_t layer, num_blocks, T;
    int Hkv, hd, bs;
    Kv8Segs sg;
    int64_t first[kKv8Segs + 1];  // a segment's first task: pages that B * S tokens can touch, x heads
    int pages[kKv8Segs];          // pages that one sequence's S tokens can touch
};

template <int VW>
using hv = _Float16 __attribute__((ext_vector_type(VW)));

// The exponent that amplitudes up to amax need (amax >= 0, finite).
__device__ __forceinline__ int e8_of(float amax) {
    // amax = m * 2^x, 1 <= m < 2, 448 = 1.75 * 2^8; fp16's subnormals are normal in fp32
    const int bits = __builtin_bit_cast(int, amax);
    const int e = (bits >> 23) - kE8Bias - 8 + ((bits & 0x7fffff) > 0x600000 ? 1 : 0);
    return min(max(e, kE8Min), kE8Max);  // 0 gives the least
}

// VW elements to e4m3, scaled by 2^-e and held to `most`; infinities become NaN.
template <int VW>
__device__ __forceinline__ void quantise(const hv<VW>& x, float inv, float most, uint8_t* to) {
    float f[VW];
#pragma unroll
    for (int i = 0; i < VW; ++i) {
        const float v = (float)x[i];
        const float t = fminf(fmaxf(v * inv, -most), most);
        f[i] = fabsf(v) <= 65504.0f ? t : __builtin_nanf("");
    }
    if constexpr (VW >= 4) {
        uint32_t w[VW / 4];
#pragma unroll
        for (int i = 0; i < VW / 4; ++i) {
            int p = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i], f[4 * i + 1], 0, false);
            w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * i + 2], f[4 * i + 3], p, true);
        }
        if constexpr (VW == 8) {
            typedef uint32_t u2 __attribute__((ext_vector_type(2)));
            *reinterpret_cast<u2*>(to) = u2{w[0], w[1]};
        } else {
            *reinterpret_cast<uint32_t*>(to) = w[0];
        }
    } else {
#pragma unroll
        for (int i = 0; i < VW; ++i)
            to[i] = static_cast<uint8_t>(__builtin_amdgcn_cvt_pk_fp8_f32(f[i], 0.0f, 0, false));
    }
}

// One wave per (page, head) of K or of V: it alone writes that page's exponent, so nothing
// is exchanged and no order decides a result.  VW elements per lane and access (8, or 1 for
// heads or rows that 16-byte accesses do not fit); the first R accesses of the new rows stay
// in registers between the maximum and the rounding.
//
// Bound by a chain of dependent reads (the sequence's length, the table's entry, the page's
// exponent), each of which waits for the memory: 64 single tokens 4.1 us in a graph, 6064 tokens
// (two prompts and 64 single tokens, 18.6 MB) 7.7 us, where a copy of as much takes 5.  The new rows are
// asked for before the chain's answers (8.3 us otherwise).
template <int VW>
__global__ __launch_bounds__(256) void kv8_write_kernel(Kv8Write a) {
    constexpr int R = 4;
    const int lane = threadIdx.x & 63;
    const uint32_t task = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // < 2^31
    if (task >= static_cast<uint32_t>(a.first[a.sg.n])) return;
    int g = 0;
    while (task >= static_cast<uint32_t>(a.first[g + 1])) ++g;
    uint32_t t = task - static_cast<uint32_t>(a.first[g]);
    const int which = static_cast<int>(t & 1);
    t >>= 1;
    const int h = static_cast<int>(t % static_cast<uint32_t>(a.Hkv));
    t /= static_cast<uint32_t>(a.Hkv);
    const int pg = static_cast<int>(t % static_cast<uint32_t>(a.pages[g]));
    const int64_t b = t / static_cast<uint32_t>(a.pages[g]);
    // the sequence's new positions [p0, p1), and this page's part of them
    const int64_t sp = a.sg.sp[g][b];
    const int64_t p0 = max<int64_t>(sp, 0), p1 = min<int64_t>(sp + a.sg.S[g], a.sg.sl[g][b]);
    const int64_t blk = static_cast<uint32_t>(p0) / static_cast<uint32_t>(a.bs) + pg;  // 0 <= p0 < 2^31
    const int64_t lo = max(p0, blk * a.bs), hi = min(p1, (blk + 1) * a.bs);
    if (lo >= hi || blk >= a.sg.mb[g]) return;
    const int64_t phys = a.sg.bt[g][b * a.sg.mb[g] + blk];
    const half_t* const src = a.src[which] + (a.sg.off[g] + b * a.sg.S[g] + (lo - sp)) * a.stride[which] + h * a.hd;
    const int slot = static_cast<int>(lo - blk * a.bs), n = static_cast<int>(hi - lo);
    const int vph = a.hd / VW, nv = n * vph;
    const float inv_vph = 1.0f / static_cast<float>(vph);
    const auto load = [&](int v) {
        const int r = small_div(v, inv_vph);
        return __builtin_nontemporal_load(
            reinterpret_cast<const hv<VW>*>(src + r * a.stride[which] + (v - r * vph) * VW));
    };
    hv<VW> x[R];
    float amax = 0.0f;
    const auto take = [&](const hv<VW>& v) {
#pragma unroll
        for (int i = 0; i < VW; ++i) {
            const float f = fabsf((float)v[i]);
            amax = fmaxf(amax, f <= 65504.0f ? f : 0.0f);
        }
    };
#pragma unroll
    for (int r = 0; r < R; ++r) x[r] = lane + r * 64 < nv ? load(lane + r * 64) : hv<VW>(0);
    // the rows are asked for before the table's answer is needed
    if (phys < 0 || phys >= a.num_blocks) return;
    const int64_t page = (a.layer * a.num_blocks + phys) * a.Hkv + h;
    uint8_t* const rows = a.cache[which] + page * a.bs * a.hd;
    uint8_t* const scale = a.scale[which] + page;
    const int old = slot > 0 ? static_cast<int>(*scale) - kE8Bias : -1000;
#pragma unroll
    for (int r = 0; r < R; ++r) take(x[r]);
    for (int v = lane + R * 64; v < nv; v += 64) take(load(v));
    amax = group_max<64>(amax);
    const int e = max(e8_of(amax), old);
    const float inv = ldexpf(1.0f, -e), most = fminf(448.0f, ldexpf(61440.0f, -e));
    const auto put = [&](int v, const hv<VW>& w) {
        const int r = small_div(v, inv_vph);
        quantise<VW>(w, inv, most, rows + static_cast<int64_t>(slot + r) * a.hd + (v - r * vph) * VW);
    };
#pragma unroll
    for (int r = 0; r < R; ++r)
        if (lane + r * 64 < nv) put(lane + r * 64, x[r]);
    for (int v = lane + R * 64; v < nv; v += 64) put(v, load(v));
    if (slot > 0 && e > old) {  // the page's other slots, from their old exponent to e
        const float by = ldexpf(1.0f, old - e);
        const int64_t all = static_cast<int64_t>(a.bs) * a.hd, from = static_cast<int64_t>(slot) * a.hd,
                      to = from + static_cast<int64_t>(n) * a.hd;
        constexpr int B = VW == 8 ? 4 : 1;  // bytes at a time: hd is a multiple of it
        for (int64_t i = static_cast<int64_t>(lane) * B; i < all; i += 64 * B) {
            if (i >= from && i < to) continue;
            uint32_t w = 0;
            if constexpr (B == 4) w = *reinterpret_cast<const uint32_t*>(rows + i);
            else w = rows[i];
            int y = 0;
            const auto f0 = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
            y = __builtin_amdgcn_cvt_pk_fp8_f32(f0[0] * by, f0[1] * by, y, false);
            if constexpr (B == 4) {
                const auto f1 = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
                y = __builtin_amdgcn_cvt_pk_fp8_f32(f1[0] * by, f1[1] * by, y, true);
                *reinterpret_cast<uint32_t*>(rows + i) = y;
            } else {
                rows[i] = static_cast<uint8_t>(y);
            }
        }
    }
    if (lane == 0) *scale = static_cast<uint8_t>(e + kE8Bias);
}

int kv8_segments(const mi_kv_segment* segments, int num_segments, int64_t T, Kv8Segs& sg) {
    if (num_segments < 0 || (num_segments > 0 && !segments)) return MI_ERR_INVALID_ARGUMENT;
    if (num_segments > kKv8Segs) return MI_ERR_UNSUPPORTED;
    sg = Kv8Segs{};
    for (int i = 0; i < num_segments; ++i) {
        const mi_kv_segment& g = segments[i];
        if (g.token_offset < 0 || g.token_offset > T || g.B < 0 || g.S < 0) return MI_ERR_INVALID_ARGUMENT;
        if (g.B == 0 || g.S == 0) continue;
        if (g.B > T || g.S > T || g.B * g.S > T - g.token_offset || !g.block_table || !g.seq_len ||
            !g.start_pos || g.max_blocks_per_seq <= 0 || !product_fits({g.B, g.max_blocks_per_seq, 4}))
            return MI_ERR_INVALID_ARGUMENT;
        for (int j = 0; j < sg.n; ++j)
            if (g.token_offset < sg.off[j] + sg.B[j] * sg.S[j] && sg.off[j] < g.token_offset + g.B * g.S)
                return MI_ERR_UNSUPPORTED;
        const int n = sg.n++;
        sg.off[n] = g.token_offset;
        sg.B[n] = g.B;
        sg.S[n] = g.S;
        sg.mb[n] = g.max_blocks_per_seq;
        sg.bt[n] = g.block_table;
        sg.sl[n] = g.seq_len;
        sg.sp[n] = g.start_pos;
    }
    return MI_OK;
}

}  // namespace mi

extern "C" int mi_kv8_scatter_f16(const void* k, const void* v, int64_t k_stride, int64_t v_stride,
                                  int64_t T, int64_t Hkv, int64_t head_dim, void* k_cache,
                                  void* v_cache, void* k_scale, void* v_scale, int64_t layer,
                                  int64_t num_blocks, int64_t block_size,
                                  const mi_kv_segment* segments, int num_segments, void* stream) {
    using namespace mi;
    if (T < 0 || Hkv < 0 || head_dim < 0 || k_stride < 0 || v_stride < 0 || layer < 0 ||
        layer >= (int64_t{1} << 62) || num_blocks < 0 || block_size <= 0)
        return MI_ERR_INVALID_ARGUMENT;
    Kv8Write a{};
    const int st = kv8_segments(segments, num_segments, T, a.sg);
    if (st != MI_OK) return st;
    if (T == 0 || Hkv == 0 || head_dim == 0 || num_blocks == 0 || a.sg.n == 0) return MI_OK;
    if (!k || !v || !k_cache || !v_cache || !k_scale || !v_scale) return MI_ERR_INVALID_ARGUMENT;
    if (Hkv > 1024 || head_dim > 512 || block_size > 4096 || T > kMaxGridX) return MI_ERR_UNSUPPORTED;
    const int64_t row = Hkv * head_dim;
    if (T > 1 && (k_stride < row || v_stride < row)) return MI_ERR_INVALID_ARGUMENT;
    if (!product_fits({T, k_stride, 2}) || !product_fits({T, v_stride, 2}) ||
        !product_fits({layer + 1, num_blocks, row, block_size}))
        return MI_ERR_INVALID_ARGUMENT;
    if (((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 1) != 0)
        return MI_ERR_INVALID_ARGUMENT;
    const int64_t cells = (layer + 1) * num_blocks * Hkv;
    const void* bufs[6] = {k_cache, v_cache, k_scale, v_scale, k, v};
    const int64_t lens[6] = {cells * block_size * head_dim, cells * block_size * head_dim, cells, cells,
                             2 * ((T - 1) * k_stride + row), 2 * ((T - 1) * v_stride + row)};
    for (int i = 0; i < 4; ++i)  // k and v may be slices of one product
        for (int j = i + 1; j < 6; ++j)
            if (overlaps(bufs[i], lens[i], bufs[j], lens[j])) return MI_ERR_ALIASING;
    a.src[0] = static_cast<const half_t*>(k);
    a.src[1] = static_cast<const half_t*>(v);
    a.cache[0] = static_cast<uint8_t*>(k_cache);
    a.cache[1] = static_cast<uint8_t*>(v_cache);
    a.scale[0] = static_cast<uint8_t*>(k_scale);
    a.scale[1] = static_cast<uint8_t*>(v_scale);
    a.stride[0] = k_stride;
    a.stride[1] = v_stride;
    a.layer = layer;
    a.num_blocks = num_blocks;
    a.T = T;
    a.Hkv = static_cast<int>(Hkv);
    a.hd = static_cast<int>(head_dim);
    a.bs = static_cast<int>(block_size);
    for (int i = 0; i < a.sg.n; ++i) {
        a.pages[i] = static_cast<int>((a.sg.S[i] + block_size - 2) / block_size + 1);
        a.first[i + 1] = a.first[i] + a.sg.B[i] * a.pages[i] * Hkv * 2;
    }
    const int64_t groups = ceil_div(a.first[a.sg.n], 4);
    if (groups > kMaxGridX / 4) return MI_ERR_UNSUPPORTED;
    const bool vec = head_dim % 8 == 0 && aligned16(k) && aligned16(v) && aligned16(k_cache) &&
                     aligned16(v_cache) && (T == 1 || (k_stride % 8 == 0 && v_stride % 8 == 0));
    const dim3 grid(static_cast<unsigned>(groups)), block(256);
    if (vec) kv8_write_kernel<8><<<grid, block, 0, as_stream(stream)>>>(a);
    else kv8_write_kernel<1><<<grid, block, 0, as_stream(stream)>>>(a);
    return launch_status();
}
