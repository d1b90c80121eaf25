"""Writes into the 8-bit paged cache: bytes and exponents equal to the plain rule's (kv8_ref)."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


def segment(rng, B, S, mb, NB, off=0, starts=None, lens=None, used=None):
    """B sequences of S new tokens; pages that no other sequence of `used` has."""
    starts = np.asarray(rng.integers(0, 40, B) if starts is None else starts)
    lens = np.asarray(starts + S if lens is None else lens)
    used = set() if used is None else used
    free = [p for p in rng.permutation(NB) if p not in used]
    table = np.array([[free.pop() for _ in range(mb)] for _ in range(B)], np.int32).reshape(B, mb)
    used.update(table.reshape(-1).tolist())
    return dict(token_offset=off, S=S, block_table=table, seq_len=lens.astype(np.int32),
                start_pos=starts.astype(np.int32))


def run(mk, dev, k, v, cache, segs, layer, strided=False):
    kc, vc, ks, vs = cache
    d = [R.dev_cache(kc, dev), R.dev_cache(vc, dev), torch.from_numpy(ks.copy()).to(dev), torch.from_numpy(vs.copy()).to(dev)]
    if strided:
        both = torch.from_numpy(np.concatenate([k, v], 1)).to(dev)
        dk, dv = both[:, :k.shape[1]], both[:, k.shape[1]:]
    else:
        dk, dv = torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev)
    mk.kv8_scatter(dk, dv, *d, layer=layer, segments=R.dev_segments(segs, dev))
    return [R.cache_bytes(d[0]), R.cache_bytes(d[1]), d[2].cpu().numpy(), d[3].cpu().numpy()]


def same_bytes(got, want, what):
    nan = (got & 0x7F == 0x7F) & (want & 0x7F == 0x7F)  # a NaN's sign says nothing
    bad = (got != want) & ~nan
    assert not bad.any(), (what, int(bad.sum()), np.argwhere(bad)[:4].tolist())


def check(mk, dev, k, v, cache, segs, layer=0, strided=False):
    got = run(mk, dev, k, v, cache, segs, layer, strided)
    for src, (c, s), (gc, gs), what in ((k, cache[0::2], got[0::2], "k"), (v, cache[1::2], got[1::2], "v")):
        c, s = c.copy(), s.copy()
        R.scatter(src, c, s, layer, segs)
        same_bytes(gc, c, what)
        assert (gs == s).all(), (what, np.argwhere(gs != s)[:4].tolist())
    return got


def random_cache(rng, L, NB, H, bs, hd):
    k, ks = R.random_cache(rng, L, NB, H, bs, hd)
    v, vs = R.random_cache(rng, L, NB, H, bs, hd)
    return [k, v, ks, vs]


def rows(rng, T, H, hd, std=1.0):
    return (rng.standard_normal((T, H, hd)) * std * 2.0 ** rng.integers(-3, 4, (T, H, 1))).astype(np.float16)


@pytest.mark.parametrize("H,hd,bs", [(4, 128, 16), (2, 64, 32), (3, 80, 16), (1, 256, 64), (2, 20, 5), (1, 7, 3),
                                     (2, 512, 128), (5, 16, 1), (1, 8, 4096)])
@pytest.mark.parametrize("S", [1, 2, 33])
def test_shapes(mk, dev, H, hd, bs, S):
    rng = np.random.default_rng(H * 1000 + hd + S)
    B, mb = 3, -(-(40 + S) // bs)
    NB = B * mb + 2
    cache = random_cache(rng, 2, NB, H, bs, hd)
    segs = [segment(rng, B, S, mb, NB)]
    for strided in (False, True):
        check(mk, dev, rows(rng, B * S, H, hd), rows(rng, B * S, H, hd), cache, segs, 1, strided)


def test_mixed_batch_with_padding(mk, dev):
    """Decodes, a padded batch of prompts, tokens of no segment; tokens at or behind seq_len,
    before 0, or in pages that are none are passed over."""
    rng = np.random.default_rng(1)
    H, hd, bs, NB = 2, 64, 16, 60
    used = set()
    a = segment(rng, 5, 1, 6, NB, off=3, used=used)
    b = segment(rng, 3, 20, 3, NB, off=8, starts=[0, 15, -4], lens=[20, 22, 9], used=used)
    b["block_table"][1, 1], b["block_table"][2, 0] = -1, NB
    c = segment(rng, 2, 4, 1, NB, off=70, starts=[14, 0], lens=[18, 0], used=used)
    k, v = rows(rng, 80, H, hd), rows(rng, 80, H, hd)
    cache = random_cache(rng, 1, NB, H, bs, hd)
    got = check(mk, dev, k, v, cache, [a, b, c])
    assert (got[0] != cache[0]).any()


def test_a_sequence_of_appends(mk, dev):
    """A prompt, then single tokens that grow: each raises its page's exponent, and the page's
    former tokens are rounded again; the same twice changes nothing."""
    rng = np.random.default_rng(2)
    H, hd, bs, NB, mb = 2, 128, 16, 8, 4
    cache = random_cache(rng, 1, NB, H, bs, hd)
    table = np.array([[5, 0, 7, 2]], np.int32)
    at, size = 0, 2.0 ** -20
    raised = 0
    for S in [5] + [1] * 40:
        k, v = rows(rng, S, H, hd, size), rows(rng, S, H, hd, size)
        g = dict(token_offset=0, S=S, block_table=table, seq_len=np.array([at + S], np.int32),
                 start_pos=np.array([at], np.int32))
        before = cache
        cache = check(mk, dev, k, v, cache, [g])
        raised += int((cache[2] > before[2]).any())
        again = run(mk, dev, k, v, cache, [g], 0)
        for x, y in zip(again, cache):
            assert (x == y).all()
        at, size = at + S, size * 2.2
    # (the premise alone: the exponents themselves are compared above, step by step)
    assert raised > 5


def test_values_at_the_edges(mk, dev):
    """Zeros, subnormals, the steps of the exponent, fp16's largest, infinities, NaN."""
    rng = np.random.default_rng(3)
    edge = np.array([0.0, -0.0, 2.0 ** -24, -2.0 ** -24, 2.0 ** -14, 448, 448.25, 449, 464, 57344, 57376, 61440,
                     61472, 65504, -65504, 1.0, np.inf, -np.inf, np.nan, 240, 256], np.float16)
    H, hd, bs = 1, 16, 16
    T = 64
    k = rng.choice(edge, (T, H, hd))
    k[0:4] = 0  # a page of zeros
    k[4:8] = 2.0 ** -24
    k[8:12] = np.nan
    v = rng.choice(edge[:16], (T, H, hd))
    cache = random_cache(rng, 1, T + 1, H, bs, hd)
    segs = [segment(rng, T // 4, 4, 1, T, starts=rng.integers(0, 2, T // 4) * rng.integers(0, 12, T // 4))]
    got = check(mk, dev, k, v, cache, segs)
    # whatever is finite in a sequence's slots is a finite fp16 number (those behind hold anything)
    x = R.values(got[1], got[3])[0][segs[0]["block_table"][:, 0], 0]
    x = np.concatenate([p[:n] for p, n in zip(x, segs[0]["seq_len"])])
    assert (np.abs(x[np.isfinite(x)]) <= 65504).all()


def test_a_page_whose_scale_is_nan_stays_nan(mk, dev):
    rng = np.random.default_rng(4)
    cache = random_cache(rng, 1, 2, 1, 16, 16)
    cache[2][0, 1, 0] = 255
    segs = [segment(rng, 1, 2, 1, 1, starts=[3])]
    segs[0]["block_table"][:] = 1
    got = run(mk, dev, rows(rng, 2, 1, 16), rows(rng, 2, 1, 16), cache, segs, 0)
    assert got[2][0, 1, 0] == 255


def test_past_4_gib(mk, dev):
    """Rows whose offset passes 32 bits."""
    H, hd, bs, NB = 8, 128, 16, (1 << 32) // (8 * 128 * 16) + 3
    rng = np.random.default_rng(5)
    k, v = rows(rng, 2, H, hd), rows(rng, 2, H, hd)
    kc, vc = (torch.empty((1, NB, H, bs, hd), dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn) for _ in range(2))
    ks, vs = (torch.full((1, NB, H), 100, dtype=torch.uint8, device=dev) for _ in range(2))
    g = dict(token_offset=0, S=2, block_table=np.array([[NB - 1]], np.int32), seq_len=np.array([2]), start_pos=np.array([0]))
    kc.view(torch.uint8)[0, [0, 1, 2, NB - 1]] = 9
    mk.kv8_scatter(torch.from_numpy(k).to(dev), torch.from_numpy(v).to(dev), kc, vc, ks, vs, 0, R.dev_segments([g], dev))
    c, s = np.full((1, 1, H, bs, hd), 9, np.uint8), np.full((1, 1, H), 100, np.uint8)
    R.scatter(k, c, s, 0, [dict(g, block_table=np.array([[0]]))])
    got = kc.view(torch.uint8)[0, [0, 1, 2, NB - 1]].cpu().numpy()
    same_bytes(got[3], c[0, 0], "the last page")
    assert (got[:3] == 9).all() and (ks[0, -1].cpu().numpy() == s[0, 0]).all()
    assert (ks[0, :-1] == 100).all()


def test_stream_and_graph(mk, dev):
    rng = np.random.default_rng(6)
    H, hd, bs, NB, B = 2, 64, 16, 12, 4
    cache = random_cache(rng, 1, NB, H, bs, hd)
    segs = [segment(rng, B, 1, 3, NB, starts=[3, 16, 31, 0])]
    d = [R.dev_cache(cache[0], dev), R.dev_cache(cache[1], dev)] + [torch.from_numpy(c).to(dev) for c in cache[2:]]
    ds = R.dev_segments(segs, dev)
    k, v = (torch.zeros((B, H, hd), dtype=torch.float16, device=dev) for _ in range(2))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    mk.kv8_scatter(k, v, *d, layer=0, segments=ds, stream=side)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mk.kv8_scatter(k, v, *d, layer=0, segments=ds)
    for _ in range(3):
        hk, hv = rows(rng, B, H, hd), rows(rng, B, H, hd)
        now = [R.cache_bytes(d[0]), R.cache_bytes(d[1]), d[2].cpu().numpy(), d[3].cpu().numpy()]
        k.copy_(torch.from_numpy(hk))
        v.copy_(torch.from_numpy(hv))
        graph.replay()
        for src, c, s, dc, dsc in ((hk, now[0], now[2], d[0], d[2]), (hv, now[1], now[3], d[1], d[3])):
            R.scatter(src, c, s, 0, segs)
            same_bytes(R.cache_bytes(dc), c, "replay")
            assert (dsc.cpu().numpy() == s).all()
