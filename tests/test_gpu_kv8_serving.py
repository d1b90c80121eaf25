"""The 8-bit cache's operators together, as a serving loop uses them: room reserved, Q and K
rotated out of a fused product, K and V written, attention over the cache; sequences forked,
freed, the cache compacted; decodes and a padded batch of prompts in one step."""
import numpy as np
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu

L, HQ, HKV, HD, BS, NB, B, MB = 2, 6, 2, 64, 16, 40, 8, 6
WINDOWS = (0, 40)  # by layer


class Engine:
    def __init__(self, mk, dev):
        self.mk, self.dev = mk, dev
        self.rng = np.random.default_rng(0)
        self.cache = list(mk.kv8_cache(L, NB, HKV, BS, HD, device=dev))  # k, v, k_scale, v_scale
        self.table = torch.full((B, MB), -1, dtype=torch.int32, device=dev)
        self.seq = torch.zeros(B, dtype=torch.int32, device=dev)
        self.ref = torch.zeros(NB, dtype=torch.int32, device=dev)
        self.inv, self.mscale = mk.rope_scaled_inv_freq(32, 1e4, "yarn", 2.0, original_len=64)
        self.h_cache = [c.view(torch.uint8).cpu().numpy().copy() for c in self.cache]
        self.h_table, self.h_seq, self.h_ref = (t.cpu().numpy().copy() for t in (self.table, self.seq, self.ref))
        self.history = {r: [([], []) for _ in range(L)] for r in range(B)}

    def ints(self, v):
        return torch.tensor([int(x) for x in v], dtype=torch.int32, device=self.dev)

    def same(self, what):
        for d, h in ((self.table, self.h_table), (self.seq, self.h_seq), (self.ref, self.h_ref)):
            assert (d.cpu().numpy() == h).all(), what
        for d, h in zip(self.cache, self.h_cache):
            assert (d.view(torch.uint8).cpu().numpy() == h).all(), what

    def reserve(self, rows, lens):
        got = self.mk.kv_reserve(self.cache, self.table, self.seq, self.ref, self.ints(rows), self.ints(lens), BS)
        want = R.reserve(self.h_cache, self.h_table, self.h_seq, self.h_ref, rows, lens, BS)
        assert got.tolist() == want == [0] * len(rows)
        self.same("reserve")

    def fork(self, parents, kids):
        got = self.mk.kv_fork(self.table, self.seq, self.ref, self.ints(parents), self.ints(kids))
        assert got.tolist() == R.fork(self.h_table, self.h_seq, self.h_ref, parents, kids) == [0] * len(kids)
        for p, k in zip(parents, kids):
            self.history[k] = [(list(a), list(b)) for a, b in self.history[p]]
        self.same("fork")

    def free(self, rows):
        self.mk.kv_free(self.table, self.seq, self.ref, self.ints(rows))
        R.free(self.h_table, self.h_seq, self.h_ref, rows)
        for r in rows:
            self.history[r] = [([], []) for _ in range(L)]
        self.same("free")

    def compact(self):
        moved = self.mk.kv_compact(self.cache, self.table, self.ref)
        assert (moved.cpu().numpy() == R.compact(self.h_cache, self.h_table, self.h_ref)).all()
        self.same("compact")

    def step(self, groups):
        """groups: lists of (row, new tokens); a list's rows are padded to its longest."""
        rows = [r for g in groups for r, _ in g]
        start = {r: int(self.h_seq[r]) for r in rows}
        self.reserve(rows, [start[r] + n for g in groups for r, n in g])
        segs, hsegs, pos, at = [], [], [], 0
        for g in groups:
            S = max(n for _, n in g)
            idx = [r for r, _ in g]
            hsegs.append(dict(token_offset=at, S=S, block_table=self.h_table[idx], seq_len=self.h_seq[idx],
                              start_pos=np.array([start[r] for r in idx], np.int32)))
            segs.append(dict(token_offset=at, S=S, block_table=self.table[self.ints(idx).long()].contiguous(),
                             seq_len=self.seq[self.ints(idx).long()].contiguous(),
                             start_pos=self.ints(start[r] for r in idx)))
            pos += [start[r] + s for r in idx for s in range(S)]
            at += len(g) * S
        T = at
        for layer in range(L):
            std = 2.0 ** self.rng.integers(-2, 3)
            qkv = (self.rng.standard_normal((T, (HQ + 2 * HKV) * HD)) * std).astype(np.float16)
            d = torch.from_numpy(qkv).to(self.dev)
            q, k, v = (t.unflatten(1, (-1, HD)) for t in d.split([HQ * HD, HKV * HD, HKV * HD], 1))
            qr = torch.empty((T, HQ, HD), dtype=torch.float16, device=self.dev)
            self.mk.rope_partial_qk(q, k, torch.tensor(pos, device=self.dev), self.inv, mscale=self.mscale, q_out=qr,
                                    k_out=torch.empty_like(qr[:, :HKV]) if layer else None)
            if layer == 1:  # into a tensor of its own, then as the cache's source
                kr = torch.empty((T, HKV, HD), dtype=torch.float16, device=self.dev)
                self.mk.rope_partial_qk(q, k, torch.tensor(pos, device=self.dev), self.inv, mscale=self.mscale,
                                        q_out=qr, k_out=kr)
            else:           # in the product
                kr = k
            self.mk.kv8_scatter(kr, v, *self.cache, layer=layer, segments=segs)
            out = torch.full((T, HQ, HD), 5.0, dtype=torch.float16, device=self.dev)
            self.mk.kv8_attention(qr, *self.cache, layer=layer, segments=segs, window=WINDOWS[layer], out=out)
            hk, hv = kr.cpu().numpy(), v.cpu().numpy()
            for src, c, s in ((hk, 0, 2), (hv, 1, 3)):
                R.scatter(src, self.h_cache[c], self.h_cache[s], layer, hsegs)
            self.same("scatter")
            want, tol = R.attention(qr.cpu().numpy(), self.h_cache[0], self.h_cache[1], self.h_cache[2],
                                    self.h_cache[3], layer, hsegs, HD ** -0.5, WINDOWS[layer], np.zeros((T, HQ, HD)))
            assert (np.abs(out.cpu().numpy() - want) <= tol).all()
            for g, seg in zip(groups, hsegs):
                for i, (r, n) in enumerate(g):
                    t = seg["token_offset"] + i * seg["S"]
                    self.history[r][layer][0].extend(hk[t:t + n])
                    self.history[r][layer][1].extend(hv[t:t + n])
        self.check_history(rows)

    def check_history(self, rows):
        """Each row's pages hold its own tokens: rounded once to 4 bits (2^-4 of the value), and by at
        most half of the least step, 2^-10 of the scale, where a page's scale was raised (each
        raise doubles the scale at least, so all of them come to 2^-9 of the last)."""
        for r in rows:
            n = int(self.h_seq[r])
            at = np.arange(n)
            pages = self.h_table[r][at // BS]
            for layer in range(L):
                for i in (0, 1):
                    x = np.array(self.history[r][layer][i], np.float64)
                    assert x.shape == (n, HKV, HD)
                    scale = 2.0 ** (self.h_cache[2 + i][layer][pages].astype(np.float64) - 127)[..., None]
                    y = R.values(self.h_cache[i][layer], self.h_cache[2 + i][layer])[pages, :, at % BS]
                    assert (np.abs(y - x) <= 2.0 ** -4 * np.abs(x) + 2.0 ** -9 * scale).all(), (r, layer, i)


def test_serving(mk, dev):
    e = Engine(mk, dev)
    e.step([[(0, 37), (1, 50), (2, 1)]])           # a padded batch of prompts
    for _ in range(3):
        e.step([[(0, 1), (1, 1), (2, 1)]])
    e.fork([0, 0, 1], [3, 4, 5])                   # beams
    for _ in range(2):
        e.step([[(r, 1) for r in (0, 1, 2, 3, 4, 5)]])
    e.free([1, 4, 4])
    e.compact()
    e.step([[(r, 1) for r in (5, 3, 0, 2)], [(6, 33)], [(1, 17), (4, 5)]])  # a mixed step
    e.free([0, 2])
    e.fork([3], [0])
    e.compact()
    for _ in range(12):
        e.step([[(r, 1) for r in (0, 1, 3, 4, 5, 6)]])
    n = int((e.h_ref > 0).sum())
    e.free([0, 1, 2, 3, 4, 5, 6, 7])
    assert n > 0 and (e.h_ref == 0).all()


def test_what_a_call_on_another_stream_makes_is_made_there(mk, dev):
    """With the current stream busy, calls on another one without output, workspace or status."""
    rng = np.random.default_rng(3)
    NBK = 64
    cache = [R.random_cache(rng, 1, NBK, 2, 16, 64) for _ in range(2)]
    host = [x for pair in zip(*cache) for x in pair]  # k, v, ks, vs
    table = rng.permutation(NBK)[:2 * 31].reshape(2, 31).astype(np.int32)
    seg = dict(token_offset=0, S=1, block_table=table, seq_len=np.array([490, 201], np.int32),
               start_pos=np.array([489, 200], np.int32))
    q = rng.standard_normal((3, 4, 64)).astype(np.float16)
    d = [R.dev_cache(c, dev) for c in host[:2]] + [torch.from_numpy(c).to(dev) for c in host[2:]]
    qd, segs = torch.from_numpy(q).to(dev), R.dev_segments([seg], dev)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    pages, src, dst, rows, want = torch.zeros((1, NBK, 64), device=dev), i32([1]), i32([2]), i32([0, 1]), i32([40, 20])
    parent, child = i32([0]), i32([2])
    state = [i32([[-1] * 4] * 3), i32([0] * 3), i32([0] * NBK)]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(3):
        poison = torch.full((1 << 20,), 255, dtype=torch.uint8, device=dev)  # memory that the calls may be given
        torch.cuda._sleep(20_000_000)
        poison.fill_(255)
        del poison
        out = mk.kv8_attention(qd, *d, layer=0, segments=segs, stream=side)
        said = [mk.kv_copy_pages([pages], src, dst, stream=side),
                mk.kv_reserve([pages], *state, rows, want, 16, stream=side),
                mk.kv_fork(*state, parent, child, stream=side)]
        moved = mk.kv_compact([pages], state[0], state[2], stream=side)
        with torch.cuda.stream(side):
            got, said, moved = out.cpu().numpy(), [s.cpu().tolist() for s in said], moved.cpu().numpy()
            mk.kv_free(*state, rows, stream=side)
            mk.kv_free(*state, i32([2]), stream=side)
        want_o, tol = R.attention(q, *host, 0, [seg], 64 ** -0.5, 0, np.zeros_like(q))
        assert (np.abs(got.astype(np.float64) - want_o) <= tol).all()
        assert said == [[0], [0, 0], [0]] and (moved[:5] >= 0).all() and (moved[5:] == -1).all()
        torch.cuda.synchronize()
