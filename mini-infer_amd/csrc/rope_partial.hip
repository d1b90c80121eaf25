// rope_partial.hip -- rotary positions beyond the reference's form: either layout
// (halves, or interleaved pairs), the first rot elements of each head, any inverse
// frequencies (scaled for long contexts) and a factor on both cos and sin, over rows
// that may be slices of a fused QKV product, in place or into other tensors.
//
//   (c, s) = mscale * (cos, sin)(pos * f_i),  y1 = x1 c - x2 s,  y2 = x2 c + x1 s
//   halves: (x1, x2) = x[i], x[i + rot/2];  interleaved: x[2i], x[2i+1];  i < rot/2
//
// The angle is the exact product of the position and the fp32 frequency, reduced in
// fp64 (positions up to 2^52): at position 100000 an fp32 angle is off by 0.004, more
// than fp16's own step.  cos and sin stay in fp32, each output is rounded once.
#include <algorithm>
#include <cmath>

#include "mi_host.h"
#include "rope_math.h"

namespace mi {

struct RopePartial {
    const half_t *q, *k;
    half_t *qo, *ko;
    const int64_t* positions;
    int64_t T, qs, ks, qos, kos;  // rows of a token, in elements apart
    int Hq, Hkv, hd, rot, tpw;
    float mscale;
};

// cos and sin of pos * f: the product as a double and its error, times 2/pi as a
// double and a correction, so that the reduced argument keeps 50 bits.
__device__ __forceinline__ void far_sincos(int64_t pos, float f, float* s, float* c) {
#pragma clang fp contract(off)  // t - n fused with t's product would count te twice
    const double kTwoOverPi = 0x1.45f306dc9c883p-1, kTwoOverPiLo = -0x1.6b01ec5417056p-55;
    const double p = static_cast<double>(pos), fd = static_cast<double>(f);
    const double a = p * fd, ae = fma(p, fd, -a);
    const double t = a * kTwoOverPi;
    const double te = fma(a, kTwoOverPi, -t) + fma(a, kTwoOverPiLo, ae * kTwoOverPi);
    const double n = rint(t);
    double sd, cd;
    rope_sincos_quadrant(((t - n) + te) * 0x1.921fb54442d18p+0,
                         static_cast<int>(static_cast<long long>(n) & 3), &sd, &cd);
    *s = static_cast<float>(sd);
    *c = static_cast<float>(cd);
}

template <int VW>
using hv = _Float16 __attribute__((ext_vector_type(VW)));

// A workgroup of 256 lanes takes tpw tokens: their cos/sin rows once, into LDS, then
// the tokens' units -- VW elements of each of a pair's halves, or VW / 2 interleaved
// pairs, or (COPY) VW elements behind the rotated part -- R per lane at a time, every
// load of a batch before its first use.  VW: the largest of 8, 4, 2, 1 that the head,
// the rotated part and the rows' places allow.
//
// Bound by HBM for many tokens: [8192, 28 + 4 heads of 128], pairs over half of each, 134 MB read
// or written in 25.2 us, 5.3 TB/s, as a copy of that size; by its launch for few: 64 tokens
// 3.1 us in a graph.  The fp64 angles are made once per token and frequency, under the loads.
template <int VW, bool INTER, bool COPY, int NF>
__global__ __launch_bounds__(256) void rope_partial_kernel(RopePartial a, InvFreqN<NF> inv) {
    extern __shared__ float cs[];  // cos [tpw][half], sin [tpw][half]
    constexpr int R = 4;
    const int half = a.rot >> 1;
    const int64_t tok0 = static_cast<int64_t>(blockIdx.x) * a.tpw;
    const int toks = static_cast<int>(min<int64_t>(a.tpw, a.T - tok0));
    const int rotu = INTER ? a.rot / VW : half / VW;
    const int uph = rotu + (COPY ? (a.hd - a.rot) / VW : 0);
    const int upt = uph * (a.Hq + a.Hkv), units = upt * toks;
    const float inv_upt = 1.0f / static_cast<float>(upt), inv_uph = 1.0f / static_cast<float>(uph);
    float* sn = cs + a.tpw * half;
    for (int base = 0; base < units; base += 256 * R) {
        hv<VW> x1[R], x2[R];
        half_t* dst[R];
        int at[R];  // the unit's first entry of the cos row; -1: copied; -2: none
#pragma unroll
        for (int r = 0; r < R; ++r) {
            const int u = base + r * 256 + static_cast<int>(threadIdx.x);
            x1[r] = x2[r] = hv<VW>(0);
            dst[r] = nullptr;
            at[r] = -2;
            if (u >= units) continue;
            const int t = small_div(u, inv_upt), v = u - t * upt;  // units < 2^22
            const int h = small_div(v, inv_uph), c = v - h * uph;
            const bool is_q = h < a.Hq;
            const int64_t tok = tok0 + t;
            const half_t* src = is_q ? a.q + tok * a.qs + h * a.hd : a.k + tok * a.ks + (h - a.Hq) * a.hd;
            dst[r] = is_q ? a.qo + tok * a.qos + h * a.hd : a.ko + tok * a.kos + (h - a.Hq) * a.hd;
            const bool copied = COPY && c >= rotu;
            const int o = copied ? a.rot + (c - rotu) * VW : c * VW;
            at[r] = copied ? -1 : t * half + (INTER ? o >> 1 : o);
            dst[r] += o;
            x1[r] = __builtin_nontemporal_load(reinterpret_cast<const hv<VW>*>(src + o));
            if (!INTER && !copied)
                x2[r] = __builtin_nontemporal_load(reinterpret_cast<const hv<VW>*>(src + o + half));
        }
        if (base == 0) {
            const float inv_half = 1.0f / static_cast<float>(half);
            for (int i = threadIdx.x; i < toks * half; i += 256) {
                const int t = small_div(i, inv_half);
                float s, c;
                far_sincos(a.positions[tok0 + t], inv.v[i - t * half], &s, &c);
                cs[i] = c * a.mscale;
                sn[i] = s * a.mscale;
            }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
            if (at[r] == -2) continue;
            hv<VW> y1 = x1[r], y2 = x2[r];
            if (at[r] >= 0) {
                if constexpr (INTER) {
#pragma unroll
                    for (int e = 0; e < VW; e += 2) {
                        const float c = cs[at[r] + (e >> 1)], s = sn[at[r] + (e >> 1)];
                        const float xa = (float)x1[r][e], xb = (float)x1[r][e + 1];
                        y1[e] = (half_t)(xa * c - xb * s);
                        y1[e + 1] = (half_t)(xb * c + xa * s);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < VW; ++e) {
                        const float c = cs[at[r] + e], s = sn[at[r] + e];
                        const float xa = (float)x1[r][e], xb = (float)x2[r][e];
                        y1[e] = (half_t)(xa * c - xb * s);
                        y2[e] = (half_t)(xb * c + xa * s);
                    }
                }
            }
            __builtin_nontemporal_store(y1, reinterpret_cast<hv<VW>*>(dst[r]));
            if (!INTER && at[r] >= 0)
                __builtin_nontemporal_store(y2, reinterpret_cast<hv<VW>*>(dst[r] + half));
        }
    }
}

template <int VW, bool INTER, bool COPY>
static void rope_partial_go(const RopePartial& a, const float* inv, int64_t groups, hipStream_t s) {
    const int half = a.rot / 2;
    const size_t lds = static_cast<size_t>(a.tpw) * half * 2 * sizeof(float);
    const auto go = [&](auto nf) {
        constexpr int NF = decltype(nf)::value;
        InvFreqN<NF> f{};
        std::copy(inv, inv + half, f.v);
        rope_partial_kernel<VW, INTER, COPY, NF>
            <<<dim3(static_cast<unsigned>(groups)), dim3(256), lds, s>>>(a, f);
    };
    if (half <= 64) go(std::integral_constant<int, 64>{});
    else go(std::integral_constant<int, kMaxHalf>{});
}

// Rows of two strided tensors: bytes [p + t * stride, + width) for t < T.
struct Rows {
    const void* p;
    int64_t stride, width;
};
// Whether any row of x shares a byte with a row of y.  Rows of one stride may lie
// between one another; of two strides, their whole extents are compared.
static bool rows_touch(const Rows& x, const Rows& y, int64_t T) {
    if (!overlaps(x.p, (T - 1) * x.stride + x.width, y.p, (T - 1) * y.stride + y.width)) return false;
    if (T == 1 || x.stride != y.stride) return true;
    const int64_t d = static_cast<int64_t>(reinterpret_cast<uintptr_t>(y.p) - reinterpret_cast<uintptr_t>(x.p));
    const int64_t m = ((d % x.stride) + x.stride) % x.stride;
    return m < x.width || x.stride - m < y.width;
}

}  // namespace mi

extern "C" int mi_rope_partial_qk_f16(const void* q, const void* k, void* q_out, void* k_out,
                                      const int64_t* positions, const float* inv_freq_host,
                                      int64_t T, int64_t Hq, int64_t Hkv, int64_t head_dim,
                                      int64_t rotary_dim, int64_t q_stride, int64_t k_stride,
                                      int64_t q_out_stride, int64_t k_out_stride, int interleaved,
                                      float mscale, void* stream) {
    using namespace mi;
    if (T < 0 || Hq < 0 || Hkv < 0 || head_dim < 0 || rotary_dim < 0 || q_stride < 0 || k_stride < 0 ||
        q_out_stride < 0 || k_out_stride < 0)
        return MI_ERR_INVALID_ARGUMENT;
    if (T == 0 || Hq + Hkv == 0) return MI_OK;
    if (!positions || !inv_freq_host || (Hq > 0 && (!q || !q_out)) || (Hkv > 0 && (!k || !k_out)) ||
        !std::isfinite(mscale) || head_dim == 0 || rotary_dim == 0 || rotary_dim % 2 != 0 ||
        rotary_dim > head_dim)
        return MI_ERR_INVALID_ARGUMENT;
    if (rotary_dim / 2 > kMaxHalf || head_dim > 4096 || Hq + Hkv > 1024 || T > kMaxGridX)
        return MI_ERR_UNSUPPORTED;
    const int64_t wq = Hq * head_dim, wk = Hkv * head_dim;
    if (T > 1 && (q_stride < wq || q_out_stride < wq || k_stride < wk || k_out_stride < wk))
        return MI_ERR_INVALID_ARGUMENT;
    for (int64_t st : {q_stride, k_stride, q_out_stride, k_out_stride})
        if (!product_fits({T, st, 2})) return MI_ERR_INVALID_ARGUMENT;
    for (int64_t i = 0; i < rotary_dim / 2; ++i)
        if (!std::isfinite(inv_freq_host[i])) return MI_ERR_INVALID_ARGUMENT;
    const Rows rows[4] = {{q, 2 * q_stride, 2 * wq}, {k, 2 * k_stride, 2 * wk},
                          {q_out, 2 * q_out_stride, 2 * wq}, {k_out, 2 * k_out_stride, 2 * wk}};
    for (int w = 2; w < 4; ++w)  // each output against every other tensor
        for (int r = 0; r < w; ++r) {
            if (rows[w].width == 0 || rows[r].width == 0) continue;
            const bool itself = r == w - 2 && rows[r].p == rows[w].p &&
                                (T == 1 || rows[r].stride == rows[w].stride);
            if (!itself && rows_touch(rows[r], rows[w], T)) return MI_ERR_ALIASING;
        }
    const bool in_place = (Hq == 0 || q == q_out) && (Hkv == 0 || k == k_out);
    // the widest vector that every place is a multiple of
    int vw = 8;
    const auto allows = [&](int v) {
        const int64_t part = interleaved ? rotary_dim : rotary_dim / 2;
        if (part % v || head_dim % v) return false;
        for (const Rows& r : rows)
            if (r.width && (reinterpret_cast<uintptr_t>(r.p) % (2 * v) || (T > 1 && r.stride % (2 * v))))
                return false;
        return true;
    };
    while (vw > 1 && !allows(vw)) vw >>= 1;
    if (!allows(1)) return MI_ERR_INVALID_ARGUMENT;  // fp16 at an odd address
    if (interleaved && vw < 2) return MI_ERR_UNSUPPORTED;  // pairs that no 4-byte access takes whole
    RopePartial a{};
    a.q = static_cast<const half_t*>(q);
    a.k = static_cast<const half_t*>(k);
    a.qo = static_cast<half_t*>(q_out);
    a.ko = static_cast<half_t*>(k_out);
    a.positions = positions;
    a.T = T;
    a.qs = q_stride;
    a.ks = k_stride;
    a.qos = q_out_stride;
    a.kos = k_out_stride;
    a.Hq = static_cast<int>(Hq);
    a.Hkv = static_cast<int>(Hkv);
    a.hd = static_cast<int>(head_dim);
    a.rot = static_cast<int>(rotary_dim);
    a.mscale = mscale;
    const int64_t rotu = (interleaved ? rotary_dim : rotary_dim / 2) / vw;
    const int64_t upt = (rotu + (in_place ? 0 : (head_dim - rotary_dim) / vw)) * (Hq + Hkv);
    if (upt >= (int64_t{1} << 22)) return MI_ERR_UNSUPPORTED;
    a.tpw = static_cast<int>(std::clamp<int64_t>(std::min(1024 / upt, T / 1024), 1, 8));
    const int64_t groups = ceil_div(T, a.tpw);
    const hipStream_t s = as_stream(stream);
    const auto go = [&](auto v) {
        constexpr int VW = decltype(v)::value;
        if (interleaved) {
            if constexpr (VW >= 2) {
                in_place ? rope_partial_go<VW, true, false>(a, inv_freq_host, groups, s)
                         : rope_partial_go<VW, true, true>(a, inv_freq_host, groups, s);
            }
        } else {
            in_place ? rope_partial_go<VW, false, false>(a, inv_freq_host, groups, s)
                     : rope_partial_go<VW, false, true>(a, inv_freq_host, groups, s);
        }
    };
    if (vw == 8) go(std::integral_constant<int, 8>{});
    else if (vw == 4) go(std::integral_constant<int, 4>{});
    else if (vw == 2) go(std::integral_constant<int, 2>{});
    else go(std::integral_constant<int, 1>{});
    return launch_status();
}
