"""Rotary positions in other layouts (mi_rope_partial_qk_f16) against 64 bits.

Tolerance per element: each output is one rounding of a value made in fp32 from cos and sin
that are within 2^-23 of the exact ones: 2^-11 |y| for the rounding (2^-25 where fp16 has no
finer step), and 2^-22 (|x1 c| + |x2 s|) for the two products, the factor and their sum."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(x, pos, inv, inter, mscale):
    x = x.astype(np.float64)
    rot = 2 * len(inv)
    ang = np.array([int(p) for p in pos], object)[:, None] * np.array(
        [int(f * 2.0 ** 200) for f in inv.astype(np.float64)], object)[None, :]  # exact, times 2^200
    # reduced by 2 pi in whole numbers of 2^-200 (pi to 75 digits)
    two_pi = 2 * 3141592653589793238462643383279502884197169399375105820974944592307816406286 * 2 ** 200 // 10 ** 75
    a = np.array([[float(v % two_pi) * 2.0 ** -200 for v in row] for row in ang]).reshape(len(pos), -1)
    c, s = np.cos(a)[:, None] * mscale, np.sin(a)[:, None] * mscale
    first, second = (np.s_[..., 0:rot:2], np.s_[..., 1:rot:2]) if inter else \
        (np.s_[..., :rot // 2], np.s_[..., rot // 2:rot])
    y, tol = x.copy(), np.zeros_like(x)
    y[first] = x[first] * c - x[second] * s
    y[second] = x[second] * c + x[first] * s
    for f, g in ((first, second), (second, first)):
        tol[f] = 2.0 ** -11 * np.abs(y[f]) + 2.0 ** -25 + 2.0 ** -22 * (np.abs(x[f] * c) + np.abs(x[g] * s))
    return y, tol


def check(got, x, pos, inv, inter, mscale, what):
    y, tol = reference(x, pos, inv, inter, mscale)
    err = np.abs(got.astype(np.float64) - y)
    assert (err <= tol).all(), (what, float((err - tol).max()), np.argwhere(err > tol)[:4].tolist())


def make(rng, T, H, hd):
    return rng.standard_normal((T, H, hd)).astype(np.float16)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("T,Hq,Hkv,hd,rot", [(1, 28, 4, 128, 128), (65, 28, 4, 128, 64), (300, 32, 32, 80, 20),
                                             (77, 32, 32, 80, 40), (5, 14, 2, 64, 16), (2, 8, 4, 256, 256),
                                             (9, 1, 0, 6, 2), (3, 2, 1, 512, 512), (1500, 3, 1, 64, 64),
                                             (4, 3, 2, 66, 66), (2100, 71, 1, 64, 32)])
def test_in_place_and_out(mk, dev, T, Hq, Hkv, hd, rot, inter):
    rng = np.random.default_rng(T * 7 + hd)
    q, k = make(rng, T, Hq, hd), make(rng, T, max(Hkv, 1), hd)
    pos = rng.integers(0, 130000, T)
    inv, m = mk.rope_scaled_inv_freq(rot, 1e6, "yarn", 4.0)
    dp = torch.from_numpy(pos).to(dev)
    dq, dk = torch.from_numpy(q).to(dev), torch.from_numpy(k).to(dev) if Hkv else None
    oq, ok = torch.empty_like(dq), torch.empty_like(dk) if Hkv else None
    r = mk.rope_partial_qk(dq, dk, dp, inv, interleaved=inter, mscale=m, q_out=oq, k_out=ok)
    assert r[0] is oq and r[1] is ok
    check(oq.cpu().numpy(), q, pos, inv, inter, m, "q out")
    assert (dq.cpu().numpy() == q).all()
    r = mk.rope_partial_qk(dq, dk, dp, inv, interleaved=inter, mscale=m)
    assert r[0] is dq and torch.equal(dq, oq)
    if Hkv:
        check(ok.cpu().numpy(), k, pos, inv, inter, m, "k out")
        assert torch.equal(dk, ok)


@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 2, 4])
def test_slices_of_a_fused_product(mk, dev, inter, shift):
    """q and k as slices of rows that hold more, at any alignment that their layout allows."""
    T, Hq, Hkv, hd, rot = 37, 6, 2, 64, 32
    if inter and shift == 1:
        shift = 6
    rng = np.random.default_rng(shift)
    width = (Hq + 2 * Hkv) * hd + shift + (shift & 1)
    buf = rng.standard_normal((T, width)).astype(np.float16)
    db = torch.from_numpy(buf).to(dev)
    views = [t[:, shift:shift + Hq * hd].reshape(T, Hq, hd) if isinstance(t, np.ndarray) else
             t[:, shift:shift + Hq * hd].unflatten(1, (Hq, hd)) for t in (buf, db)]
    kv = [t[:, shift + Hq * hd:shift + (Hq + Hkv) * hd].reshape(T, Hkv, hd) if isinstance(t, np.ndarray) else
          t[:, shift + Hq * hd:shift + (Hq + Hkv) * hd].unflatten(1, (Hkv, hd)) for t in (buf, db)]
    pos = rng.integers(0, 5000, T)
    inv, _ = mk.rope_scaled_inv_freq(rot, 1e4)
    dp = torch.from_numpy(pos).to(dev)
    oq = torch.full((T, Hq, hd + 2), 7.0, dtype=torch.float16, device=dev)
    q_ref, k_ref = views[0].copy(), kv[0].copy()
    out = torch.empty((T, Hq, hd), dtype=torch.float16, device=dev)
    mk.rope_partial_qk(views[1], None, dp, inv, interleaved=inter, q_out=out)
    check(out.cpu().numpy(), q_ref, pos, inv, inter, 1.0, "out of the slice")
    assert torch.equal(db.cpu(), torch.from_numpy(buf))
    mk.rope_partial_qk(views[1], kv[1], dp, inv, interleaved=inter)  # in the product itself
    now = db.cpu().numpy()
    check(now[:, shift:shift + Hq * hd].reshape(T, Hq, hd), q_ref, pos, inv, inter, 1.0, "q")
    check(now[:, shift + Hq * hd:shift + (Hq + Hkv) * hd].reshape(T, Hkv, hd), k_ref, pos, inv, inter, 1.0, "k")
    rest = np.ones(width, bool)
    rest[shift:shift + (Hq + Hkv) * hd] = False
    assert (now[:, rest] == buf[:, rest]).all()
    with pytest.raises(ValueError, match="contiguous"):
        mk.rope_partial_qk(oq[:, :, :hd], None, dp, inv)


def test_one_of_two_in_place(mk, dev):
    rng = np.random.default_rng(3)
    q, k = make(rng, 19, 4, 64), make(rng, 19, 2, 64)
    pos = rng.integers(0, 99, 19)
    inv, _ = mk.rope_scaled_inv_freq(32)
    dq, dk = torch.from_numpy(q).to(dev), torch.from_numpy(k).to(dev)
    ok = torch.empty_like(dk)
    mk.rope_partial_qk(dq, dk, torch.from_numpy(pos).to(dev), inv, k_out=ok)
    check(dq.cpu().numpy(), q, pos, inv, False, 1.0, "q")
    check(ok.cpu().numpy(), k, pos, inv, False, 1.0, "k")
    assert (dk.cpu().numpy() == k).all()


@pytest.mark.parametrize("inter", [False, True])
def test_far_positions(mk, dev, inter):
    """Exact angles: negative positions, 2^31, 2^45, at every frequency."""
    rng = np.random.default_rng(5)
    pos = np.array([0, -1, 1, -70000, 1048575, 2 ** 24 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 12345, 2 ** 45 - 3])
    x = make(rng, len(pos), 2, 128)
    inv, _ = mk.rope_scaled_inv_freq(128, 1e6)
    d = torch.from_numpy(x).to(dev)
    mk.rope_partial_qk(d, None, torch.from_numpy(pos).to(dev), inv, interleaved=inter)
    check(d.cpu().numpy(), x, pos, inv, inter, 1.0, "far")


def test_the_whole_head_is_the_neox_form(mk, dev):
    """The half layout over whole heads at near positions: within a rounding of cos / sin tables
    in fp16 (2^-11 of each product) of rope_neox_qk."""
    rng = np.random.default_rng(8)
    x = make(rng, 33, 5, 128)
    pos = torch.arange(33, device=dev)
    inv, _ = mk.rope_scaled_inv_freq(128, 1e6)
    a, b = torch.from_numpy(x).to(dev), torch.from_numpy(x).to(dev)
    mk.rope_partial_qk(a, None, pos, inv)
    mk.rope_neox_qk(b, None, pos, inv)
    most = 2.0 ** -11 * 2 * np.abs(np.concatenate([x[..., 64:], x[..., :64]], -1)) + 2.0 ** -9 * np.abs(x) + 1e-6
    assert (np.abs(a.float().cpu().numpy() - b.float().cpu().numpy()) <= 2 * most).all()


def test_nan_and_infinities_stay_in_their_pair(mk, dev):
    x = np.ones((2, 1, 64), np.float16)
    x[0, 0, 3], x[1, 0, 40] = np.nan, np.inf
    pos = torch.tensor([5, 9], device=dev)
    inv, _ = mk.rope_scaled_inv_freq(64)
    for inter, pairs in ((False, ({3, 35}, {8, 40})), (True, ({2, 3}, {40, 41}))):
        d = torch.from_numpy(x.copy()).to(dev)
        mk.rope_partial_qk(d, None, pos, inv, interleaved=inter)
        for t in (0, 1):
            assert set(torch.nonzero(~torch.isfinite(d[t, 0].cpu())).view(-1).tolist()) == pairs[t]


def test_stream_and_graph(mk, dev):
    """On a stream of its own, captured, replayed over new inputs with eager work between."""
    rng = np.random.default_rng(9)
    T, inv = 50, mk.rope_scaled_inv_freq(64)[0]
    q, pos = torch.zeros((T, 4, 64), dtype=torch.float16, device=dev), torch.zeros(T, dtype=torch.int64, device=dev)
    out = torch.empty_like(q)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    mk.rope_partial_qk(q, None, pos, inv, q_out=out, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mk.rope_partial_qk(q, None, pos, inv, q_out=out)
    for i in range(3):
        x, p = make(rng, T, 4, 64), rng.integers(0, 9999, T)
        q.copy_(torch.from_numpy(x))
        pos.copy_(torch.from_numpy(p))
        graph.replay()
        check(out.cpu().numpy(), x, p, inv, False, 1.0, f"replay {i}")


def test_empty(mk, dev):
    inv = mk.rope_scaled_inv_freq(64)[0]
    q = torch.empty((0, 4, 64), dtype=torch.float16, device=dev)
    assert mk.rope_partial_qk(q, None, torch.empty(0, dtype=torch.int64, device=dev), inv)[0] is q
