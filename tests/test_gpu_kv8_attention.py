"""Attention over the 8-bit paged cache against 64 bits (kv8_ref.attention, which derives the
tolerance)."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu

NAN = 0x7F


@pytest.fixture(autouse=True, params=[0, 128], ids=["by shape", "tiles of 128"])
def tile(mk, request):
    """Every test in the tiles that its shapes choose, and in tiles of 128 query rows."""
    prev = mk.kv8_attention_test_tile(request.param)
    yield request.param
    mk.kv8_attention_test_tile(prev)


class Case:
    """A cache, its segments and queries; pages in random order, one owner each."""

    def __init__(self, seed, Hq, Hkv, hd, bs, parts, T=None, L=1, spare=3, qstd=2.0):
        """parts: lists of (start, length) per segment, with its S: [(S, [(start, len), ...]), ...]"""
        rng = self.rng = np.random.default_rng(seed)
        self.bs, self.L = bs, L
        need = [[max(0, -(-max(n, st + S) // bs)) for st, n in seqs] for S, seqs in parts]
        NB = self.NB = sum(map(sum, need)) + spare
        self.cache = [x for pair in zip(R.random_cache(rng, L, NB, Hkv, bs, hd), R.random_cache(rng, L, NB, Hkv, bs, hd))
                      for x in pair]  # k, v, ks, vs
        order = rng.permutation(NB).tolist()
        self.segs, at = [], 0
        for (S, seqs), pages in zip(parts, need):
            mb = max(pages + [1])
            table = np.full((len(seqs), mb), -1, np.int32)
            for b, n in enumerate(pages):
                table[b, :n] = [order.pop() for _ in range(n)]
            self.segs.append(dict(token_offset=at, S=S, block_table=table,
                                  seq_len=np.array([n for _, n in seqs], np.int32),
                                  start_pos=np.array([st for st, _ in seqs], np.int32)))
            at += len(seqs) * S
        T = at if T is None else T
        self.q = (rng.standard_normal((T, Hq, hd)) * qstd).astype(np.float16)
        self.out = rng.standard_normal((T, Hq, hd)).astype(np.float16)

    def unused(self, byte=NAN):
        """What no token may see -- slots behind a sequence's end, pages of nobody -- filled."""
        seen = np.zeros((self.NB, self.bs), bool)
        for g in self.segs:
            for b, n in enumerate(g["seq_len"]):
                last = min(n, g["start_pos"][b] + g["S"])
                for p in range(max(0, last)):
                    if p // self.bs < g["block_table"].shape[1] and 0 <= g["block_table"][b, p // self.bs] < self.NB:
                        seen[g["block_table"][b, p // self.bs], p % self.bs] = True
        for c in self.cache[:2]:
            c.transpose(0, 1, 3, 2, 4)[:, ~seen] = byte
        return self

    def run(self, mk, dev, layer=0, window=0, scale=None, ws=None, q=None, out=None, stream=None):
        hd = self.q.shape[2]
        d = [R.dev_cache(c, dev) for c in self.cache[:2]] + [torch.from_numpy(c).to(dev) for c in self.cache[2:]]
        q = torch.from_numpy(self.q).to(dev) if q is None else q
        out = torch.from_numpy(self.out.copy()).to(dev) if out is None else out
        mk.kv8_attention(q, *d, layer=layer, segments=R.dev_segments(self.segs, dev), scale=scale, window=window,
                         out=out, workspace=ws, stream=stream)
        return out

    def check(self, mk, dev, layer=0, window=0, scale=None, **kw):
        got = self.run(mk, dev, layer, window, scale, **kw).cpu().numpy()
        self.compare(got, layer, window, scale)
        return got

    def compare(self, got, layer=0, window=0, scale=None):
        s = self.q.shape[2] ** -0.5 if scale is None else scale
        want, tol = R.attention(self.q, *self.cache, layer, self.segs, s, window, self.out)
        err = np.abs(got.astype(np.float64) - want)
        assert (np.isnan(got) == np.isnan(want)).all(), np.argwhere(np.isnan(got) != np.isnan(want))[:5].tolist()
        bad = ~np.isnan(want) & ~(err <= tol)
        assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5].tolist(), float(np.nanmax(err)),
                               got[bad][:3], want[bad][:3])


HEADS = [(28, 4, 128), (14, 2, 64), (8, 4, 256), (4, 4, 80), (5, 1, 16), (34, 1, 128), (2, 2, 240)]


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
@pytest.mark.parametrize("window", [0, 1, 37])
def test_single_tokens(mk, dev, Hq, Hkv, hd, window):
    """Sequences of one token and of lengths around a block's and a step's ends; one that is empty."""
    lens = [1, 2, 15, 16, 17, 63, 64, 65, 130, 300, 0]
    c = Case(hd + window, Hq, Hkv, hd, 16, [(1, [(max(n - 1, 0), n) for n in lens])]).unused()
    c.check(mk, dev, window=window)


@pytest.mark.parametrize("bs", [16, 48, 64, 272])
def test_page_sizes(mk, dev, bs):
    c = Case(bs, 6, 2, 64, bs, [(1, [(n - 1, n) for n in (1, bs - 1, bs, bs + 1, 3 * bs + 5, 700)])]).unused()
    c.check(mk, dev)
    c.check(mk, dev, window=100)


@pytest.mark.parametrize("Hq,Hkv,hd", HEADS)
@pytest.mark.parametrize("S", [2, 5, 17, 70])
def test_several_tokens(mk, dev, Hq, Hkv, hd, S):
    """Prompts, and chunks behind a cached prefix."""
    c = Case(hd + S, Hq, Hkv, hd, 16, [(S, [(0, S), (13, 13 + S), (100, 100 + S)])]).unused()
    c.check(mk, dev)
    c.check(mk, dev, window=24)


@pytest.mark.parametrize("Hq,Hkv,hd", [(28, 4, 128), (8, 4, 64), (4, 2, 256), (3, 3, 80)])
def test_prompts_of_some_length(mk, dev, Hq, Hkv, hd):
    c = Case(hd, Hq, Hkv, hd, 16, [(333, [(0, 333), (200, 533)])]).unused()
    c.check(mk, dev)
    c.check(mk, dev, window=129)


@pytest.mark.parametrize("Hq,Hkv,hd,S,B", [(28, 4, 128, 65, 4), (16, 16, 64, 81, 8), (8, 4, 256, 129, 16),
                                           (28, 4, 128, 9, 30), (8, 4, 256, 100, 3)])
def test_either_side_of_the_choice(mk, dev, Hq, Hkv, hd, S, B):
    """About as many tiles of 16 rows as move a segment to tiles of 128, in one call with single tokens."""
    c = Case(S, Hq, Hkv, hd, 16, [(1, [(90, 91)]), (S, [(7 * b, 7 * b + S) for b in range(B)])]).unused()
    c.check(mk, dev)
    n = mk.kv8_attention_workspace_bytes(Hq, Hkv, hd, R.dev_segments(c.segs, dev))
    prev = mk.kv8_attention_test_tile(16)
    c.check(mk, dev)
    mk.kv8_attention_test_tile(prev)
    assert mk.kv8_attention_workspace_bytes(Hq, Hkv, hd, R.dev_segments(c.segs, dev)) == n


@pytest.mark.parametrize("Hq,Hkv,hd", [(16, 8, 64), (24, 8, 128), (16, 16, 80), (8, 8, 256)])
def test_many_sequences(mk, dev, Hq, Hkv, hd):
    """More tiles than the GPU holds workgroups, beside a few of a long sequence."""
    rng = np.random.default_rng(hd)
    lens = rng.integers(0, 300, 130).tolist() + [1, 64, 65]
    c = Case(hd, Hq, Hkv, hd, 16, [(1, [(max(n - 1, 0), n) for n in lens]), (2, [(1998, 2000)])]).unused()
    c.check(mk, dev)
    c.check(mk, dev, window=70)


@pytest.mark.parametrize("hd", [64, 128, 256])
def test_long_sequences_in_splits(mk, dev, hd):
    c = Case(hd, 4, 2, hd, 16, [(1, [(4999, 5000), (2300, 2301), (70, 71)])]).unused()
    c.check(mk, dev)
    c.check(mk, dev, window=1500)


def test_mixed_batch(mk, dev):
    """Decodes, a padded batch of prompts and a chunk in one call; rows in no segment stay, tokens
    behind their sequence's end or before position 0 get zeros."""
    c = Case(1, 12, 3, 128, 16, [(1, [(40, 41), (0, 1), (5, 5), (700, 701)]), (9, [(0, 9), (3, 8), (-2, 7), (0, 0)]),
                                 (50, [(61, 111)])], T=100).unused()
    got = c.check(mk, dev)
    assert (got[2] == 0).all() and (got[90:] == c.out[90:]).all() and (got[4 + 9 + 5:4 + 18] == 0).all()
    assert (got[4 + 18:4 + 20] == 0).all() and (got[4 + 27:4 + 36] == 0).all()


def test_pages_that_are_none(mk, dev):
    """Keys of entries outside the cache, or beyond the table, are left out; where that leaves
    nothing, the output is zero."""
    c = Case(2, 4, 2, 64, 16, [(1, [(200, 201), (30, 31), (90, 91)]), (20, [(60, 80)])])
    t = c.segs[0]["block_table"]
    t[0, [0, 3, 12]] = -1, c.NB, -7
    t[1, :2] = -1
    c.segs[1]["block_table"][0, 4] = 1 << 30
    c.segs[0]["seq_len"][2], c.segs[0]["start_pos"][2] = 100000, 5000  # far behind the table
    got = c.check(mk, dev)
    assert (got[1] == 0).all() and (got[2] != 0).any()


def test_nan_in_keys_and_values_of_later_tokens(mk, dev):
    """A NaN that a token's mask hides reaches no output of it, one that it sees reaches it."""
    c = Case(3, 4, 2, 128, 16, [(40, [(30, 70), (0, 40)]), (1, [(80, 81)])]).unused()
    t = c.segs[0]["block_table"]
    c.cache[1][0, t[0, 50 // 16], 1, 50 % 16, 7] = NAN   # v of position 50, one element, KV head 1
    c.cache[0][0, t[1, 20 // 16], 0, 20 % 16, 3] = 0xFF  # k of position 20
    got = c.check(mk, dev)
    assert np.isnan(got[20, 2, 7]) and not np.isnan(got[19]).any() and not np.isnan(got[20, 2, 8])
    assert np.isnan(got[60, 0]).all() and not np.isnan(got[59]).any()
    assert not np.isnan(got[80]).any()
    c.check(mk, dev, window=11)


def test_a_page_of_nan_scale(mk, dev):
    c = Case(4, 2, 1, 64, 16, [(1, [(100, 101), (100, 101)]), (30, [(20, 50)])])
    for g, b, blk in ((0, 0, 3), (1, 0, 2)):
        c.cache[3][0, c.segs[g]["block_table"][b, blk], 0] = 255
    got = c.check(mk, dev)
    assert np.isnan(got[0]).all() and not np.isnan(got[1]).any()


@pytest.mark.parametrize("qstd", [0.0, 60.0])
def test_flat_and_peaked(mk, dev, qstd):
    """Equal weights, and one key that takes all."""
    Case(5, 8, 2, 128, 16, [(1, [(2000, 2001), (33, 34)]), (20, [(0, 20)])], qstd=qstd).unused().check(mk, dev)


def test_scales_far_apart(mk, dev):
    """Pages whose exponents span what the writer makes, and keys so small that they count alike."""
    c = Case(6, 4, 4, 64, 16, [(1, [(400, 401)]), (25, [(90, 115)])], qstd=0.5).unused()
    rng = np.random.default_rng(0)
    c.cache[3][:] = rng.integers(127 - 32, 127 + 8, c.cache[3].shape)
    c.cache[1][:] = np.where(c.cache[3][..., None, None] > 127 + 6, c.cache[1] & 0xF7, c.cache[1])
    big = np.abs(R.values(c.cache[1], c.cache[3])) > 61440
    c.cache[1][big] = 0
    # such a cache's values are fp16 numbers but for those under its least step
    v = R.values(c.cache[1], c.cache[3])
    keep = v.astype(np.float16).astype(np.float64) == v
    c.cache[1][~keep & ~np.isnan(v)] = 0
    c.check(mk, dev)


def test_scale_zero_and_negative(mk, dev):
    c = Case(7, 4, 2, 64, 16, [(1, [(100, 101)]), (9, [(3, 12)])]).unused()
    c.check(mk, dev, scale=0.0)
    c.check(mk, dev, scale=-0.3)


def test_layers_strides_and_the_binding(mk, dev):
    c = Case(8, 6, 2, 64, 16, [(1, [(77, 78), (20, 21)]), (5, [(10, 15)])], L=3).unused()
    c.check(mk, dev, layer=2)
    T = c.q.shape[0]
    wide = torch.zeros((T, 10 * 64), dtype=torch.float16, device=dev)
    wide[:, 64:64 * 7] = torch.from_numpy(c.q.reshape(T, -1)).to(dev)
    o = torch.zeros((T, 7, 64), dtype=torch.float16, device=dev)
    got = c.run(mk, dev, layer=1, q=wide[:, 64:64 * 7].unflatten(1, (6, 64)), out=o[:, :6])
    c.compare(got.cpu().numpy(), layer=1)
    assert (o[:, 6] == 0).all()
    with pytest.raises(ValueError, match="head"):
        c.run(mk, dev, q=torch.zeros((T, 5, 64), dtype=torch.float16, device=dev))
    with pytest.raises(ValueError, match="layer"):
        c.run(mk, dev, layer=3)


def test_the_same_bits_each_time(mk, dev):
    """A sequence's output is the same from call to call."""
    c = Case(9, 28, 4, 128, 16, [(1, [(1500, 1501), (64, 65), (300, 301)]), (40, [(100, 140)])]).unused()
    a = c.check(mk, dev)
    b = c.run(mk, dev).cpu().numpy()
    assert (a.view(np.uint16) == b.view(np.uint16)).all()


def test_workspace_streams_and_graphs(mk, dev):
    """One workspace for calls of all shapes, two graphs among them, with eager work between."""
    shapes = [Case(10, 8, 2, 128, 16, [(1, [(900, 901), (10, 11)])]).unused(),
              Case(11, 8, 2, 128, 16, [(1, [(100, 101)] * 5), (30, [(50, 80)])]).unused()]
    n = max(mk.kv8_attention_workspace_bytes(8, 2, 128, R.dev_segments(c.segs, dev)) for c in shapes)
    ws = torch.zeros(n, dtype=torch.uint8, device=dev)
    for c in shapes:
        c.check(mk, dev, ws=ws)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = shapes[0].run(mk, dev, ws=ws, stream=side)
    side.synchronize()
    shapes[0].compare(got.cpu().numpy())
    held = []
    for c in shapes:
        d = [R.dev_cache(x, dev) for x in c.cache[:2]] + [torch.from_numpy(x).to(dev) for x in c.cache[2:]]
        q, out, segs = torch.from_numpy(c.q).to(dev), torch.from_numpy(c.out).to(dev), R.dev_segments(c.segs, dev)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mk.kv8_attention(q, *d, layer=0, segments=segs, out=out, workspace=ws)
        held.append((c, graph, d, q, out, segs))
    for i in range(3):
        for c, graph, d, q, out, segs in held:
            c.q = (c.rng.standard_normal(c.q.shape) * 2).astype(np.float16)
            q.copy_(torch.from_numpy(c.q))
            graph.replay()
            c.compare(out.cpu().numpy())
            shapes[i % 2].run(mk, dev, ws=ws)
            torch.cuda.synchronize()


def test_past_4_gib(mk, dev):
    """Pages whose offsets pass 32 bits: the same output as from a small cache."""
    c = Case(12, 8, 8, 128, 16, [(1, [(100, 101)]), (20, [(30, 50)])], spare=0).unused()
    first = (1 << 32) // (8 * 128 * 16) - 2  # the pages lie on both sides of 4 GiB
    NB = first + c.NB
    d = [torch.empty((1, NB, 8, 16, 128), dtype=torch.uint8, device=dev) for _ in range(2)]
    d += [torch.full((1, NB, 8), 255, dtype=torch.uint8, device=dev) for _ in range(2)]
    for big, small in zip(d, c.cache):
        big[:, first:] = torch.from_numpy(small).to(dev)
    d[:2] = [x.view(torch.float8_e4m3fn) for x in d[:2]]
    segs = [dict(g, block_table=np.where(g["block_table"] >= 0, g["block_table"] + first, -1)) for g in c.segs]
    out = torch.from_numpy(c.out).to(dev)
    mk.kv8_attention(torch.from_numpy(c.q).to(dev), *d, layer=0, segments=R.dev_segments(segs, dev), out=out)
    c.compare(out.cpu().numpy())


def test_new_output_and_nothing_to_do(mk, dev):
    c = Case(13, 4, 2, 64, 16, [(1, [(20, 21)])], T=3).unused()
    d = [R.dev_cache(x, dev) for x in c.cache[:2]] + [torch.from_numpy(x).to(dev) for x in c.cache[2:]]
    q = torch.from_numpy(c.q).to(dev)
    got = mk.kv8_attention(q, *d, layer=0, segments=R.dev_segments(c.segs, dev))
    assert (got[1:] == 0).all() and (got[0] != 0).any()
    assert (mk.kv8_attention(q, *d, layer=0, segments=[]) == 0).all()
    assert mk.kv8_attention(q[:0], *d, layer=0, segments=[]).shape == (0, 4, 64)
