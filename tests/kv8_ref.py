"""The 8-bit paged cache, its attention and its pages in plain Python and 64 bits, for the tests."""
import math

import numpy as np
import torch

# the 256 e4m3 bytes as numbers: sign, 4 bits of exponent (bias 7), 3 of mantissa, 0x7f NaN
E4M3 = np.array([math.nan if b & 0x7F == 0x7F else
                 (-1.0 if b & 0x80 else 1.0) * ((8 + (b & 7)) * 2.0 ** ((b >> 3 & 15) - 10)
                                                if b >> 3 & 15 else (b & 7) * 2.0 ** -9)
                 for b in range(256)])
_POS = E4M3[:127]


def to_e4m3(x):
    """Bytes of the nearest e4m3 values (ties to the even byte) of |x| <= 448; NaN stays."""
    x = np.asarray(x, np.float64)
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0)), 448.0)
    hi = np.clip(np.searchsorted(_POS, a), 1, 126)
    lo = hi - 1
    up, down = _POS[hi] - a, a - _POS[lo]
    b = np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    b = np.where(np.signbit(x), b | 0x80, b)
    return np.where(np.isnan(x), 0x7F, b).astype(np.uint8)


def exponent(amax):
    """The least e in -32 .. 8 with amax <= 448 * 2^e."""
    e = -32
    while e < 8 and amax > 448.0 * 2.0 ** e:
        e += 1
    return e


def write_page(page, byte, slot, x):
    """x [n, hd] into page [bs, hd] (bytes, in place) at `slot`, its exponent byte `byte`; the new one."""
    x = np.asarray(x, np.float64)
    fine = np.isfinite(x)
    e = exponent(np.abs(x[fine]).max() if fine.any() else 0.0)
    n = x.shape[0]
    if slot:
        old = int(byte) - 127
        e = max(e, old)
        if e > old:
            rest = [i for i in range(page.shape[0]) if not slot <= i < slot + n]
            page[rest] = to_e4m3(E4M3[page[rest]] * 2.0 ** (old - e))
    most = min(448.0, 61440.0 * 2.0 ** -e)
    q = np.clip(np.where(fine, x, math.nan) * 2.0 ** -e, -most, most)
    page[slot:slot + n] = to_e4m3(q)
    return e + 127


def scatter(src, cache, scale, layer, segments):
    """src [T, H, hd] into cache (bytes [L, NB, H, bs, hd]) and scale [L, NB, H], in place."""
    L, NB, H, bs, hd = cache.shape
    for g in segments:
        table, lens, starts = g["block_table"], g["seq_len"], g["start_pos"]
        for b in range(len(lens)):
            todo = {}
            for s in range(g["S"]):
                p = int(starts[b]) + s
                if p < 0 or p >= lens[b] or p // bs >= table.shape[1]:
                    continue
                phys = int(table[b, p // bs])
                if 0 <= phys < NB:
                    todo.setdefault((p // bs, phys), []).append((p % bs, g["token_offset"] + b * g["S"] + s))
            for (_, phys), rows in todo.items():
                for h in range(H):
                    scale[layer, phys, h] = write_page(cache[layer, phys, h], scale[layer, phys, h],
                                                       rows[0][0], src[[t for _, t in rows], h])


def values(cache, scale):
    e = np.where(scale == 255, math.nan, 2.0 ** (scale.astype(np.float64) - 127))
    return E4M3[cache] * e[..., None, None]


def attention(q, kc, vc, ks, vs, layer, segments, scale, window, out):
    """(out, tolerance) in 64 bits; `out` holds what rows outside the segments keep.

    The tolerance, per element with w the softmax's weights, n the keys, A = sum w |v|:
      fp16 weights: 2^-11 A, and 2^-35 max|v| for each of those too small for 11 bits (2^-25 on a
        scale of 2^10 or more for the largest weight; the weights' sum is at least that one's, 1);
      scores in fp32: each weight is off by the exponent's error, at most
        (hd + 4) 2^-24 scale sum |q k| <= d, in the weight and in the sum: 2 d A; the
        hardware's exp2 and the factor log2(e): 2^-21 each, of the exponent's size;
      sums of n terms in fp32, of weights and of products: 2 n 2^-24 A;
      the output's rounding: 2^-11 |out|, at least half fp16's least step, 2^-25.
    """
    L, NB, Hkv, bs, hd = kc.shape
    out = out.astype(np.float64).copy()
    tol = np.zeros_like(out)
    G = q.shape[1] // Hkv
    K, V = values(kc[layer], ks[layer]), values(vc[layer], vs[layer])
    for g in segments:
        for b in range(len(g["seq_len"])):
            for s in range(g["S"]):
                t = g["token_offset"] + b * g["S"] + s
                out[t] = 0.0
                p = int(g["start_pos"][b]) + s
                if p < 0 or p >= g["seq_len"][b]:
                    continue
                at = np.arange(max(0, p - window + 1) if window else 0, p + 1)
                at = at[at // bs < g["block_table"].shape[1]]
                phys = g["block_table"][b][at // bs]
                at, phys = at[(phys >= 0) & (phys < NB)], phys[(phys >= 0) & (phys < NB)]
                if not len(at):
                    continue
                for h in range(q.shape[1]):
                    k, v = K[phys, h // G, at % bs], V[phys, h // G, at % bs]
                    x = q[t, h].astype(np.float64)
                    sc = k @ x * scale
                    m = sc.max()
                    w = np.exp(sc - m)
                    tot = w.sum()
                    out[t, h] = w @ v / tot
                    A = w @ np.abs(v) / tot
                    n = len(at)
                    big = (np.abs(k) @ np.abs(x) * abs(scale)).max()
                    d = (hd + 4) * 2.0 ** -24 * big + 2.0 ** -21 * (1 + big)
                    tol[t, h] = (A * (2.0 ** -11 + 2 * d + 2 * n * 2.0 ** -24)
                                 + n * 2.0 ** -35 * np.nan_to_num(np.abs(v)).max() + 2.0 ** -11 * np.abs(out[t, h]) + 2.0 ** -25)
    return out, tol


def random_cache(rng, L, NB, Hkv, bs, hd):
    """Pages of numbers of unequal sizes: (bytes, scale bytes), values within about +-4."""
    x = rng.standard_normal((L, NB, Hkv, bs, hd))
    e = rng.integers(-9, -6, (L, NB, Hkv))
    return to_e4m3(np.clip(x * 100, -448, 448)), (e + 127).astype(np.uint8)


def dev_segments(segments, dev):
    return [dict(token_offset=g["token_offset"], S=g["S"],
                 **{n: torch.from_numpy(np.ascontiguousarray(g[n], np.int32)).to(dev)
                    for n in ("block_table", "seq_len", "start_pos")}) for g in segments]


def dev_cache(a, dev):
    return torch.from_numpy(a.copy()).to(dev).view(torch.float8_e4m3fn)


def cache_bytes(t):
    return t.view(torch.uint8).cpu().numpy()


# --- pages ---------------------------------------------------------------------

DONE, FULL, REFUSED = 0, 1, 2


def copy_pages(caches, src, dst):
    NB = caches[0].shape[1]
    status = []
    for i, (s, d) in enumerate(zip(src, dst)):
        bad = not (0 <= s < NB and 0 <= d < NB) or d in list(dst[:i]) or \
            any(src[j] == d for j in range(len(src)) if j != i)
        status.append(REFUSED if bad else DONE)
    before = [c.copy() for c in caches]
    for s, d, st in zip(src, dst, status):
        if st == DONE:
            for c, o in zip(caches, before):
                c[:, d] = o[:, s]
    return status


def free(table, seq, ref, rows):
    for r in dict.fromkeys(int(r) for r in rows):
        if not 0 <= r < len(table):
            continue
        for pg in table[r]:
            if 0 <= pg < len(ref):
                ref[pg] = max(ref[pg] - 1, 0)
        table[r] = -1
        seq[r] = 0


def fork(table, seq, ref, parents, kids):
    status = []
    start_t, start_s = table.copy(), seq.copy()
    for i, (a, b) in enumerate(zip(parents, kids)):
        ok = 0 <= a < len(table) and 0 <= b < len(table) and a not in kids and b not in list(kids[:i])
        ok = ok and start_s[b] == 0 and (start_t[b] < 0).all()
        status.append(DONE if ok else REFUSED)
        if ok:
            table[b], seq[b] = start_t[a], start_s[a]
            for pg in start_t[a]:
                if 0 <= pg < len(ref):
                    ref[pg] += 1
    return status


def reserve(caches, table, seq, ref, rows, lengths, bs):
    mb = table.shape[1]
    free_pages = [p for p in range(len(ref)) if ref[p] == 0]
    ref0 = ref.copy()
    taken, full, shared, status, copies = 0, False, {}, [], []
    for i, (r, n) in enumerate(zip(rows, lengths)):
        r, n = int(r), int(n)
        if not 0 <= r < len(table) or r in [int(x) for x in rows[:i]] or n < 0 or n > mb * bs or \
                not 0 <= seq[r] <= mb * bs:
            status.append(REFUSED)
            continue
        now = int(seq[r])
        have = -(-now // bs)
        want = max(have, -(-n // bs))
        cow = False
        if n > now and now % bs:
            last = int(table[r, have - 1])
            if not 0 <= last < len(ref):
                status.append(REFUSED)
                continue
            cow = shared.get(last, 0) < ref0[last] - 1
            shared[last] = shared.get(last, 0) + 1
        need = cow + want - have
        if full or taken + need > len(free_pages):
            full = True
            status.append(FULL)
            continue
        got = free_pages[taken:taken + need]
        taken += need
        for pg in got:
            ref[pg] = 1
        if cow:
            ref[last] -= 1
            table[r, have - 1] = got[0]
            copies.append((last, got[0]))
            got = got[1:]
        table[r, have:want] = got
        seq[r] = max(now, n)
        status.append(DONE)
    for s, d in copies:
        for c in caches:
            c[:, d] = c[:, s]
    return status


def compact(caches, table, ref):
    live = [p for p in range(len(ref)) if ref[p] > 0]
    n = len(live)
    holes = [p for p in range(n) if ref[p] <= 0]
    movers = [p for p in live if p >= n]
    moved = np.where(ref > 0, np.arange(len(ref)), -1).astype(np.int32)
    for s, d in zip(movers, holes):
        moved[s] = d
        ref[d], ref[s] = ref[s], 0
        for c in caches:
            c[:, d] = c[:, s]
    inside = (table >= 0) & (table < len(ref))
    table[:] = np.where(inside, moved[np.where(inside, table, 0)], -1)
    return moved
