// test_kv8 -- the C++ launchers of the 8-bit paged cache (host/kernels/kv8_kernel.h) on
// inputs whose results are known: small whole numbers, which e4m3 holds exactly, so a sequence of
// one token attends to its own V bit for bit and one of equal keys to the mean of its values.
//
// `test_kv8 --cpu` runs the refusals alone, which launch nothing (no GPU needed).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdio>
#include <cstring>
#include <functional>
#include <stdexcept>
#include <vector>

#include "kernels/kv8_kernel.h"

using namespace mini_infer::kernels;

static int g_failures = 0;
static void expect(bool ok, const char* what) {
    std::printf("  %-60s %s\n", what, ok ? "OK" : "FAIL");
    g_failures += !ok;
}

static bool throws(const std::function<void()>& f) {
    try {
        f();
    } catch (const std::runtime_error&) {
        return true;
    }
    return false;
}

static void hip(hipError_t e) {
    if (e != hipSuccess) throw std::runtime_error(hipGetErrorString(e));
}

// a device array, filled from the host
template <typename T>
struct Dev {
    T* p = nullptr;
    size_t n;
    explicit Dev(const std::vector<T>& h) : n(h.size()) {
        hip(hipMalloc(reinterpret_cast<void**>(&p), n * sizeof(T)));
        hip(hipMemcpy(p, h.data(), n * sizeof(T), hipMemcpyHostToDevice));
    }
    ~Dev() { (void)hipFree(p); }
    Dev(const Dev&) = delete;
    std::vector<T> host() const {
        std::vector<T> h(n);
        hip(hipDeviceSynchronize());
        hip(hipMemcpy(h.data(), p, n * sizeof(T), hipMemcpyDeviceToHost));
        return h;
    }
};

static float f(__half x) { return __half2float(x); }

static void refusals() {
    __half x[1]{};
    uint8_t c[1]{};
    int i[1]{};
    float w[1]{};
    int64_t pos[1]{};
    void* const bad = c;
    expect(throws([&] { launch_rope_partial_qk(x, x, pos, w, 1, 1, 1, 16, 3, 16, 16, false, 1.0f, nullptr); }),
           "rope: an odd rotary_dim throws");
    expect(throws([&] { launch_kv8_scatter(x, x, c, c, c, c, i, i, i, 1, 1, 0, 1, 1, 16, 0, 1, nullptr); }),
           "write: a block size of 0 throws");
    expect(throws([&] { kv8_attention_workspace_bytes(1, 1, 3, 2, 64, 1); }),
           "workspace: heads that are no multiple throw");
    expect(throws([&] {
               launch_kv8_attention(x, c, c, c, c, x, i, i, i, 1, 1, 1, 1, 8, 1.0f, 0, 0, 1, 16, 1, nullptr, 0,
                                    nullptr);
           }),
           "attention: a head_dim of 8 throws");
    expect(throws([&] { launch_kv_copy_pages(nullptr, 1, 4, i, i, 1, i, nullptr); }), "copy: no cache throws");
    expect(throws([&] { launch_kv_free(i, i, i, 1, 1, 1, nullptr, 1, nullptr); }), "free: no rows throw");
    expect(throws([&] { launch_kv_fork(i, i, i, 1, 1, 1, i, nullptr, 1, i, nullptr); }),
           "fork: no children throw");
    expect(throws([&] { launch_kv_reserve(nullptr, 0, i, i, i, 1, 1, 1, 0, i, i, 1, i, bad, 1, nullptr); }),
           "reserve: a block size of 0 throws");
    expect(throws([&] { launch_kv_compact(nullptr, 0, i, i, 1, 1, 1, i, nullptr, 0, nullptr); }),
           "compact: no workspace throws");
    expect(throws([&] { kv_pages_workspace_bytes(-1, 0); }), "pages: a negative size throws");
}

static void on_gpu() {
    // two rows of up to 4 blocks of 16 tokens, 8 pages; row 0: 20 tokens, row 1: 1 token
    const int B = 3, mb = 4, NB = 8, bs = 16, Hq = 4, Hkv = 2, hd = 64;
    Dev<int> table(std::vector<int>(B * mb, -1)), len(std::vector<int>(B, 0)), ref(std::vector<int>(NB, 0));
    const size_t bytes = static_cast<size_t>(NB) * Hkv * bs * hd, cells = static_cast<size_t>(NB) * Hkv;
    Dev<uint8_t> kc(std::vector<uint8_t>(bytes, 0x7F)), vc(std::vector<uint8_t>(bytes, 0x7F));
    Dev<uint8_t> ks(std::vector<uint8_t>(cells, 255)), vs(std::vector<uint8_t>(cells, 255));
    const mi_kv_pages caches[4] = {{kc.p, 1, Hkv * bs * hd}, {vc.p, 1, Hkv * bs * hd}, {ks.p, 1, Hkv}, {vs.p, 1, Hkv}};
    const int64_t wb = kv_pages_workspace_bytes(NB, 2);
    Dev<uint8_t> ws(std::vector<uint8_t>(wb, 1));
    Dev<int> rows(std::vector<int>{0, 1}), want(std::vector<int>{20, 1}), status(std::vector<int>(2, -1));
    launch_kv_reserve(caches, 4, table.p, len.p, ref.p, B, mb, NB, bs, rows.p, want.p, 2, status.p, ws.p, wb, nullptr);
    expect(table.host() == std::vector<int>{0, 1, -1, -1, 2, -1, -1, -1, -1, -1, -1, -1} &&
               status.host() == std::vector<int>{MI_KV_DONE, MI_KV_DONE},
           "reserve: the lowest pages");

    // row 0's prompt: equal keys, so each token's output is the mean of the values before it
    const int S = 20;
    std::vector<__half> k(S * Hkv * hd), v(S * Hkv * hd), q(S * Hq * hd, __float2half(1.0f));
    for (int t = 0; t < S; ++t)
        for (int i = 0; i < Hkv * hd; ++i) {
            k[t * Hkv * hd + i] = __float2half(static_cast<float>(i % 3));
            v[t * Hkv * hd + i] = __float2half(static_cast<float>((t + i) % 7 - 3));
        }
    Dev<__half> kd(k), vd(v), qd(q), od(std::vector<__half>(q.size()));
    Dev<int> start(std::vector<int>{0, 0, 0});
    launch_kv8_scatter(kd.p, vd.p, kc.p, vc.p, ks.p, vs.p, table.p, len.p, start.p, 1, S, 0, NB, Hkv, hd, bs, mb,
                       nullptr);
    const int64_t ab = kv8_attention_workspace_bytes(1, S, Hq, Hkv, hd, mb);
    Dev<uint8_t> aw(std::vector<uint8_t>(ab > 0 ? ab : 16, 0));
    auto attend = [&](int window, const int* tab, const int* ln, const int* st, int n) {
        launch_kv8_attention(qd.p, kc.p, vc.p, ks.p, vs.p, od.p, tab, ln, st, 1, n, Hq, Hkv, hd, 0.125f, window, 0, NB,
                             bs, mb, aw.p, ab, nullptr);
        return od.host();
    };
    const auto mean_ok = [&](const std::vector<__half>& o, int window) {
        for (int t = 0; t < S; ++t)
            for (int h = 0; h < Hq; ++h)
                for (int d = 0; d < hd; ++d) {
                    const int from = window > 0 ? std::max(0, t + 1 - window) : 0;
                    double sum = 0;
                    for (int j = from; j <= t; ++j) sum += f(v[(j * Hkv + h / (Hq / Hkv)) * hd + d]);
                    sum /= t + 1 - from;
                    // equal weights are exact in fp16 and cancel; one rounding of the output and the
                    // fp32 sums' 2^-20
                    if (std::fabs(f(o[(t * Hq + h) * hd + d]) - sum) > std::fabs(sum) * 0x1p-11 + 0x1p-20) return false;
                }
        return true;
    };
    expect(mean_ok(attend(0, table.p, len.p, start.p, S), 0), "attention: equal keys give the mean");
    expect(mean_ok(attend(1, table.p, len.p, start.p, S), 1), "attention: a window of 1 gives the token's own value");

    // a fork shares row 0's pages; making room copies the one that is partly full
    Dev<int> parent(std::vector<int>{0}), child(std::vector<int>{2}), to(std::vector<int>{21});
    launch_kv_fork(table.p, len.p, ref.p, B, mb, NB, parent.p, child.p, 1, status.p, nullptr);
    expect(ref.host() == std::vector<int>{2, 2, 1, 0, 0, 0, 0, 0}, "fork: pages with two holders");
    launch_kv_reserve(caches, 4, table.p, len.p, ref.p, B, mb, NB, bs, child.p, to.p, 1, status.p, ws.p, wb, nullptr);
    expect(table.host()[2 * mb + 1] == 3 && ref.host() == std::vector<int>{2, 1, 1, 1, 0, 0, 0, 0},
           "reserve: a page of its own");
    // row 2 written behind row 0's 20 tokens by its own page; row 0 reads as before
    Dev<int> at20(std::vector<int>{20});
    launch_kv8_scatter(kd.p, vd.p, kc.p, vc.p, ks.p, vs.p, table.p + 2 * mb, len.p + 2, at20.p, 1, 1, 0, NB, Hkv, hd,
                       bs, mb, nullptr);
    expect(mean_ok(attend(0, table.p, len.p, start.p, S), 0), "write behind a fork: the parent reads as before");

    // row 1 goes, the rest moves to the front
    launch_kv_free(table.p, len.p, ref.p, B, mb, NB, rows.p + 1, 1, nullptr);
    Dev<int> moved(std::vector<int>(NB, -2));
    launch_kv_compact(caches, 4, table.p, ref.p, B, mb, NB, moved.p, ws.p, wb, nullptr);
    expect(moved.host() == std::vector<int>{0, 1, -1, 2, -1, -1, -1, -1} && table.host()[2 * mb + 1] == 2,
           "free and compact: page 3 moves to 2");
    expect(mean_ok(attend(0, table.p + 2 * mb, len.p + 2, start.p, S), 0), "compact: the child's prefix reads as before");

    // a page over another
    Dev<int> src(std::vector<int>{0}), dst(std::vector<int>{5});
    launch_kv_copy_pages(caches, 4, NB, src.p, dst.p, 1, status.p, nullptr);
    const auto h = kc.host();
    expect(std::memcmp(h.data(), h.data() + 5 * Hkv * bs * hd, Hkv * bs * hd) == 0 && status.host()[0] == MI_KV_DONE,
           "copy: page 0 over page 5");

    // rotary positions: position 0 keeps everything, a half turn of the first pair negates it
    std::vector<__half> x(2 * hd, __float2half(1.0f));
    Dev<__half> xq(x), xk(x);
    std::vector<float> inv(hd / 4, 0.0f);
    inv[0] = 3.14159274f;
    Dev<int64_t> pos(std::vector<int64_t>{0, 1});
    launch_rope_partial_qk(xq.p, xk.p, pos.p, inv.data(), 2, 1, 1, hd, hd / 2, hd, hd, true, 1.0f, nullptr);
    const auto r = xq.host(), rk = xk.host();
    bool ok = std::memcmp(r.data(), rk.data(), r.size() * 2) == 0;
    for (int i = 0; i < 2 * hd; ++i) ok = ok && f(r[i]) == (i == hd || i == hd + 1 ? -1.0f : 1.0f);
    expect(ok, "rope: pairs, the elements behind rotary_dim kept");
}

int main(int argc, char** argv) {
    refusals();
    if (argc < 2 || std::strcmp(argv[1], "--cpu") != 0) on_gpu();
    std::printf(g_failures ? "%d FAILED\n" : "ALL OK\n", g_failures);
    return g_failures != 0;
}
