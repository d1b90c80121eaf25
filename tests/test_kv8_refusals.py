"""What the 8-bit cache's, the pages' and the partial RoPE's entry points refuse: decided on the
host, before any HIP call (fake pointers), and the wrappers' own checks."""
import ctypes

import numpy as np
import pytest
import torch

import kv8_ref as R
import mi_kernels as mk

INVALID, UNSUPPORTED, ALIASING = -1, -2, -3


def P(v):
    return ctypes.c_void_p(v)


@pytest.fixture(scope="module")
def lib():
    return mk.load_library()


Q, K, QO, KO, POS = (0x10000000 * i for i in range(1, 6))


def rope(lib, q=Q, k=K, qo=QO, ko=KO, pos=POS, inv=None, T=4, Hq=8, Hkv=2, hd=64, rot=64, qs=512,
         ks=128, qos=512, kos=128, inter=0, mscale=1.0):
    f = (ctypes.c_float * 600)(*(inv if inv is not None else [0.5] * 600))
    return lib.mi_rope_partial_qk_f16(P(q), P(k), P(qo), P(ko), P(pos), f, T, Hq, Hkv, hd, rot, qs,
                                      ks, qos, kos, inter, mscale, None)


def test_rope_partial_refusals(lib):
    for bad in (dict(T=-1), dict(Hq=-1), dict(rot=63), dict(rot=66), dict(rot=0), dict(hd=0),
                dict(q=0), dict(ko=0), dict(pos=0), dict(qs=511), dict(kos=127),
                dict(mscale=float("nan")), dict(mscale=float("inf")), dict(q=Q + 1),
                dict(inv=[1.0, float("inf")] + [0.0] * 598), dict(inv=[float("nan")] * 600),
                dict(T=1 << 30, qs=1 << 40)):
        assert rope(lib, **bad) == INVALID, bad
    for bad in (dict(hd=2048, rot=1024, qs=1 << 14, ks=1 << 12, qos=1 << 14, kos=1 << 12),
                dict(inter=1, q=Q + 2), dict(Hq=2000, qs=1 << 17, qos=1 << 17)):
        assert rope(lib, **bad) == UNSUPPORTED, bad
    # outputs that are not the inputs may touch no other row
    for bad in (dict(qo=Q + 16), dict(qo=K), dict(ko=QO + 1024), dict(qo=Q, qos=1024),
                dict(qo=Q + 2 * 400, qs=1024, qos=1024)):
        assert rope(lib, **bad) == ALIASING, bad
    # nothing to do
    assert rope(lib, T=0) == 0
    assert rope(lib, Hq=0, Hkv=0) == 0


def seg(off=0, B=1, S=1, mb=4, bt=0x60000, sl=0x70000, sp=0x80000):
    g = mk.KvSegment()
    g.token_offset, g.B, g.S, g.max_blocks_per_seq = off, B, S, mb
    g.block_table, g.seq_len, g.start_pos = bt, sl, sp
    return g


def segs(*g):
    return (mk.KvSegment * max(1, len(g)))(*g)


def scatter(lib, k=0x10000000, v=0x20000000, ks=512, vs=512, T=8, H=4, hd=128, kc=0x30000000,
            vc=0x40000000, sk=0x50000000, sv=0x58000000, layer=0, NB=8, bs=16, g=None, n=None):
    g = segs(seg()) if g is None else g
    return lib.mi_kv8_scatter_f16(P(k), P(v), ks, vs, T, H, hd, P(kc), P(vc), P(sk), P(sv), layer,
                                  NB, bs, g, len(g) if n is None else n, None)


BAD_SEGMENTS = [dict(off=-1), dict(off=9), dict(B=-1), dict(S=-1), dict(B=3, S=3), dict(off=7, S=2),
                dict(B=1 << 40, S=1 << 40), dict(bt=None), dict(sl=None), dict(sp=None), dict(mb=0)]


def test_scatter_refusals(lib):
    for bad in (dict(T=-1), dict(H=-1), dict(hd=-1), dict(ks=-1), dict(ks=511), dict(vs=100),
                dict(layer=-1), dict(layer=(1 << 63) - 1), dict(NB=-1), dict(bs=0), dict(k=0),
                dict(v=0), dict(kc=0), dict(sv=0), dict(k=0x10000001), dict(NB=1 << 60), dict(n=-1),
                *(dict(g=segs(seg(**b))) for b in BAD_SEGMENTS)):
        assert scatter(lib, **bad) == INVALID, bad
    nine = segs(*(seg() for _ in range(9)))
    for bad in (dict(hd=513, ks=4096, vs=4096), dict(bs=4097), dict(H=1025, ks=1 << 18, vs=1 << 18),
                dict(g=nine), dict(g=segs(seg(0, 2, 2), seg(3, 1, 1)))):
        assert scatter(lib, **bad) == UNSUPPORTED, bad
    for bad in (dict(kc=0x40000000), dict(sk=0x40000010), dict(sv=0x50000000), dict(k=0x30000000),
                dict(vc=0x20000400)):
        assert scatter(lib, **bad) == ALIASING, bad
    for nothing in (dict(T=0, g=segs(), n=0), dict(H=0), dict(hd=0), dict(NB=0),
                    dict(g=segs(seg(B=0)))):
        assert scatter(lib, **nothing) == 0, nothing


def attend(lib, q=0x10000000, qs=1024, kc=0x30000000, vc=0x40000000, sk=0x50000000, sv=0x58000000,
           out=0x20000000, os=1024, T=8, Hq=8, Hkv=4, hd=128, scale=0.1, window=0, layer=0, NB=8,
           bs=16, g=None, n=None, ws=0x80000000, nbytes=1 << 30):
    g = segs(seg()) if g is None else g
    return lib.mi_kv8_attention_f16(P(q), qs, P(kc), P(vc), P(sk), P(sv), P(out), os, T, Hq, Hkv,
                                    hd, scale, window, layer, NB, bs, g,
                                    len(g) if n is None else n, P(ws), nbytes, None)


def test_attention_refusals(lib):
    for bad in (dict(T=-1), dict(Hq=-1), dict(Hkv=0), dict(Hq=6), dict(hd=-16), dict(qs=1023),
                dict(os=8), dict(scale=float("nan")), dict(scale=float("inf")), dict(window=-1),
                dict(layer=-1), dict(layer=(1 << 63) - 1), dict(NB=-1), dict(bs=0), dict(q=0),
                dict(out=0), dict(vc=0), dict(sk=0), dict(NB=1 << 40), dict(ws=0), dict(nbytes=100),
                dict(ws=0x80000008), dict(n=-1), *(dict(g=segs(seg(**b))) for b in BAD_SEGMENTS)):
        assert attend(lib, **bad) == INVALID, bad
    nine = segs(*(seg() for _ in range(9)))
    for bad in (dict(hd=24), dict(hd=272, qs=4096, os=4096), dict(bs=8), dict(bs=24), dict(bs=8192),
                dict(g=nine), dict(g=segs(seg(mb=1 << 23))), dict(g=segs(seg(mb=1 << 20)), bs=64),
                dict(q=0x10000008), dict(qs=1028), dict(kc=0x30000004), dict(out=0x20000001),
                dict(g=segs(seg(0, 2, 2), seg(3, 1, 1)))):
        assert attend(lib, **bad) == UNSUPPORTED, bad
    for bad in (dict(out=0x10000000), dict(out=0x30000000), dict(out=0x50000010),
                dict(out=0x80000000), dict(ws=0x10000000), dict(ws=0x40000010)):
        assert attend(lib, **bad) == ALIASING, bad
    for nothing in (dict(T=0, g=segs(), n=0), dict(Hq=0), dict(hd=0), dict(g=segs(seg(S=0)))):
        assert attend(lib, **nothing) == 0, nothing
    g = segs(seg(B=2, S=3, mb=64))
    need = lib.mi_kv8_attention_workspace_bytes(8, 4, 128, g, 1)
    assert need > 0 and attend(lib, g=g, nbytes=need - 1) == INVALID
    assert lib.mi_kv8_attention_workspace_bytes(8, 3, 128, g, 1) == INVALID
    assert lib.mi_kv8_attention_workspace_bytes(8, 4, 120, g, 1) == UNSUPPORTED
    assert lib.mi_kv8_attention_workspace_bytes(8, 4, 128, segs(), 0) == 0


def caches(*c):
    return (mk.KvPages * max(1, len(c)))(*(mk.KvPages(*x) for x in c))


TWO = ((0x10000000, 2, 1024), (0x20000000, 2, 4))


def test_pages_refusals(lib):
    S, D, ST = P(0x30000000), P(0x31000000), P(0x32000000)

    def copy(c=TWO, n_c=None, NB=16, src=S, dst=D, n=4, st=ST):
        return lib.mi_kv_pages_copy(caches(*c), len(c) if n_c is None else n_c, NB, src, dst, n, st, None)

    for bad in (dict(n=-1), dict(NB=-1), dict(n_c=-1), dict(src=None), dict(dst=None), dict(st=None),
                dict(c=((0, 2, 1024),)), dict(c=((1 << 20, -1, 4),)), dict(c=((1 << 20, 1, -4),)),
                dict(c=((1 << 20, 1 << 40, 1 << 40),))):
        assert copy(**bad) == INVALID, bad
    assert copy(c=(TWO * 5)[:9]) == UNSUPPORTED
    assert copy(n=1 << 21) == UNSUPPORTED and copy(NB=1 << 31) == UNSUPPORTED
    assert copy(c=(TWO[0], (0x10000400, 1, 4))) == ALIASING
    assert copy(n=0) == 0

    T, L, REF, ROWS, LEN, WS = (P(0x40000000 + (i << 24)) for i in range(6))

    def free(t=T, l=L, r=REF, B=4, mb=8, NB=16, rows=ROWS, n=2):
        return lib.mi_kv_pages_free(t, l, r, B, mb, NB, rows, n, None)

    def fork(t=T, l=L, r=REF, B=4, mb=8, NB=16, rows=ROWS, kids=LEN, n=2, st=ST):
        return lib.mi_kv_pages_fork(t, l, r, B, mb, NB, rows, kids, n, st, None)

    def reserve(c=TWO, t=T, l=L, r=REF, B=4, mb=8, NB=16, bs=16, rows=ROWS, lens=LEN, n=2, st=ST,
                ws=WS, nbytes=1 << 20):
        return lib.mi_kv_pages_reserve(caches(*c), len(c), t, l, r, B, mb, NB, bs, rows, lens, n,
                                       st, ws, nbytes, None)

    def compact(c=TWO, t=T, r=REF, B=4, mb=8, NB=16, moved=ST, ws=WS, nbytes=1 << 20):
        return lib.mi_kv_pages_compact(caches(*c), len(c), t, r, B, mb, NB, moved, ws, nbytes, None)

    for f in (free, fork, reserve, compact):
        for bad in (dict(t=None), dict(r=None), dict(B=-1), dict(mb=-1), dict(NB=-1)):
            assert f(**bad) == INVALID, (f, bad)
        assert f(B=1 << 31) == UNSUPPORTED and f(NB=1 << 31) == UNSUPPORTED
    for f in (free, fork, reserve):
        assert f(l=None) == INVALID and f(rows=None) == INVALID and f(n=-1) == INVALID
        assert f(n=1 << 21) == UNSUPPORTED and f(n=0) == 0
    for bad in (dict(kids=None), dict(st=None)):
        assert fork(**bad) == INVALID, bad
    need = lib.mi_kv_pages_workspace_bytes(16, 2)
    for bad in (dict(bs=0), dict(lens=None), dict(st=None), dict(ws=None), dict(nbytes=need - 1),
                dict(ws=P(0x45000002)), dict(c=((0, 2, 1024),))):
        assert reserve(**bad) == INVALID, bad
    assert reserve(n=1025) == UNSUPPORTED and reserve(mb=1 << 28, bs=16) == UNSUPPORTED
    for bad in (dict(moved=None), dict(ws=None), dict(nbytes=lib.mi_kv_pages_workspace_bytes(16, 0) - 1)):
        assert compact(**bad) == INVALID, bad
    assert compact(NB=0) == 0
    assert lib.mi_kv_pages_workspace_bytes(-1, 2) == INVALID


def test_wrappers_check_on_the_host():
    h = torch.zeros(4, 2, 64, dtype=torch.float16)
    pos = torch.zeros(4, dtype=torch.int64)
    inv = np.ones(32, np.float32)
    with pytest.raises(ValueError, match="GPU"):
        mk.rope_partial_qk(h, None, pos, inv)
    with pytest.raises(TypeError):
        mk.rope_partial_qk(h.numpy(), None, pos, inv)
    c = mk.kv8_cache(1, 4, 2, 16, 64, device="cpu")
    assert c[0].dtype == torch.float8_e4m3fn and c[2].shape == (1, 4, 2)
    with pytest.raises(ValueError, match="GPU"):
        mk.kv8_scatter(h, h, *c, layer=0, segments=[])
    with pytest.raises(ValueError, match="GPU"):
        mk.kv8_attention(h, *c, layer=0, segments=[])
    i = torch.zeros(4, dtype=torch.int32)
    for call in (lambda: mk.kv_free(i.view(2, 2), i[:2], i, i),
                 lambda: mk.kv_fork(i.view(2, 2), i[:2], i, i, i),
                 lambda: mk.kv_reserve([c[0]], i.view(2, 2), i[:2], i, i, i, 16),
                 lambda: mk.kv_compact([c[0]], i.view(2, 2), i),
                 lambda: mk.kv_copy_pages([c[0]], i, i)):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_scaled_frequencies():
    """Each scaling against its formula, and what they all keep: the highest frequency (but for
    linear's), the lowest divided by the factor."""
    f0, one = mk.rope_scaled_inv_freq(128, 1e6)
    i = np.arange(0, 128, 2) / 128
    np.testing.assert_allclose(f0, 1e6 ** -i, rtol=2.0 ** -23)
    assert one == 1.0 and f0.dtype == np.float32
    f, m = mk.rope_scaled_inv_freq(128, 1e6, "linear", 4.0)
    np.testing.assert_array_equal(f, (1e6 ** -i / 4).astype(np.float32))
    assert m == 1.0
    for kind in ("ntk", "bands", "yarn"):
        f, m = mk.rope_scaled_inv_freq(128, 1e6, kind, 8.0)
        assert f[0] == f0[0] and abs(f[-1] * 8 / f0[-1] - 1) < 1e-6, kind
        assert (f <= f0 * (1 + 2.0 ** -23)).all() and (f >= f0 / 8 * (1 - 2.0 ** -23)).all(), kind
    assert m == pytest.approx(0.1 * np.log(8.0) + 1)
    turns = 4096 * 1e6 ** -i / (2 * np.pi)
    f, _ = mk.rope_scaled_inv_freq(128, 1e6, "bands", 8.0, low=1.0, high=4.0)
    assert (f[turns < 1] == (1e6 ** -i / 8).astype(np.float32)[turns < 1]).all()
    assert (f[turns > 4] == f0[turns > 4]).all()
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and ((f < f0) & (f > f0 / 8))[mid].all()
    assert mk.rope_scaled_inv_freq(2, 1e4, "ntk", 4.0)[0].tolist() == [1.0]
    for bad in (dict(rotary_dim=3), dict(rotary_dim=0), dict(scaling="other"), dict(factor=0.5),
                dict(theta=1.0), dict(low=2.0, high=1.0)):
        with pytest.raises(ValueError):
            mk.rope_scaled_inv_freq(**{**dict(rotary_dim=64), **bad})


def test_the_plain_rounding():
    """to_e4m3 against torch's own conversion, and the exponent's rule at its steps."""
    x = np.concatenate([R._POS, (R._POS[1:] + R._POS[:-1]) / 2, np.random.default_rng(0).uniform(0, 448, 4000)])
    x = np.concatenate([x, -x])
    want = torch.from_numpy(x).to(torch.float64).to(torch.float32).to(torch.float8_e4m3fn)
    same = x.astype(np.float32) == x  # the way over fp32 rounds the others twice
    assert same.sum() > 500
    np.testing.assert_array_equal(R.to_e4m3(x)[same], want.view(torch.uint8).numpy()[same])
    assert [R.exponent(a) for a in (0.0, 448.0, 448.5, 2.0 ** -24, 65504.0, 57344.0)] == [-32, 0, 1, -32, 8, 7]


def test_attention_numbers_a_sequences_rows_in_31_bits(lib):
    """S tokens of Hq / Hkv heads each: 2^21 of 1024 are 2^31 rows."""
    most = ((1 << 31) - 1 - 128) // 1024
    for S, ok in ((1 << 24, False), (1 << 21, False), (most + 1, False), (most, True)):
        n = lib.mi_kv8_attention_workspace_bytes(1024, 1, 16, segs(seg(S=S)), 1)
        assert (n >= 0) if ok else (n == UNSUPPORTED), (S, n)
