"""The operators around a paged KV cache held in 8 bits, as a program that serves a
language model has them done.

A case is a dict with a "kind":

  rope     rotary positions of Q and K out of a fused QKV product: either layout, the
           whole head or a part of it, inverse frequencies scaled for long contexts
  write    a step's K and V into the 8-bit cache (e4m3 values, one power-of-two scale
           per page and head)
  attend   causal attention of a step's Q over that cache: decodes, prompts, chunks of
           prompts, with or without a sliding window
  beam     a step of a beam search: the old beams freed, the kept ones forked, each
           given room for its next token (copy on write)
  compact  a fragmented cache's live pages moved to its front
  copy     pages copied within a cache, by a list

With `own` false, run() computes the plain form in elementary torch operations; with
it true, it calls the library.
"""
import math
import sys
from pathlib import Path

import torch

own = False

F16, F32, F64, F8 = torch.float16, torch.float32, torch.float64, torch.float8_e4m3fn
E4M3_MAX = 448.0
E_MIN, E_MAX = -32, 8  # exponents that fp16 amplitudes need
HEADS = ((28, 4, 128), (32, 8, 128), (14, 2, 64), (8, 4, 256), (16, 16, 64), (32, 32, 80),
         (64, 8, 128))
MAX_START = 28000


_library = None


def _mk():
    global _library
    if _library is None:
        path = str(Path(__file__).resolve().parents[1] / "mini-infer_amd")
        if path not in sys.path:
            sys.path.insert(0, path)
        import mi_kernels
        _library = mi_kernels
    return _library


# --- the cases ---------------------------------------------------------------

def listed():
    return [
        # a decode batch's Q and K, a context scaled to four times its length
        dict(name="rope_decode_64", kind="rope", T=64, Hq=28, Hkv=4, hd=128, rot=128,
             interleaved=False, factor=4.0),
        # a long prompt, interleaved pairs over half of each head
        dict(name="rope_interleaved_8192", kind="rope", T=8192, Hq=28, Hkv=4, hd=128, rot=64,
             interleaved=True, factor=1.0),
        # one token for each of 64 sequences, into pages that are partly full
        dict(name="write_decode_64", kind="write", B=64, lo=100, hi=28000, S=0, Hkv=4, hd=128,
             bs=16),
        # the same beside two prompts: a step of continuous batching at full load
        dict(name="write_mixed_6064", kind="write", B=64, lo=100, hi=28000, S=3000, Hkv=4, hd=128,
             bs=16),
        # one user's next token in a short conversation: latency
        dict(name="attend_one_517", kind="attend", B=1, lo=517, hi=517, P=0, S=0, start=0, Hq=28,
             Hkv=4, hd=128, bs=16, window=0),
        # a decode batch of ragged lengths, seven query heads to a KV head
        dict(name="attend_decode_64", kind="attend", B=64, lo=100, hi=28000, P=0, S=0, start=0,
             Hq=28, Hkv=4, hd=128, bs=16, window=0),
        # a decode batch of wide heads with a sliding window
        dict(name="attend_decode_24_window", kind="attend", B=24, lo=700, hi=28000, P=0, S=0,
             start=0, Hq=8, Hkv=4, hd=256, bs=16, window=1024),
        # two prompts
        dict(name="attend_prompt_3000", kind="attend", B=0, lo=0, hi=0, P=2, S=3000, start=0,
             Hq=28, Hkv=4, hd=128, bs=16, window=0),
        # a chunk of a long prompt beside a decode batch
        dict(name="attend_chunk_1048", kind="attend", B=37, lo=300, hi=9001, P=1, S=1011,
             start=12345, Hq=32, Hkv=8, hd=128, bs=16, window=0),
        # eight requests of four beams each, a few hundred tokens in
        dict(name="beam_32", kind="beam", parents=8, width=4, lo=200, hi=900, L=28, Hkv=4, hd=128,
             bs=16),
        # half of the pages free, here and there
        dict(name="compact_8192", kind="compact", NB=8192, L=16, fill=0.5, B=64, Hkv=4, hd=128,
             bs=16),
        # a prompt's pages copied for a second owner
        dict(name="copy_190", kind="copy", NB=1024, n=190, L=28, Hkv=4, hd=128, bs=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_attend(rng):
    Hq, Hkv, hd = rng.choice(HEADS)
    form = rng.choice(("decode", "decode", "prompt", "chunk"))
    B = 0 if form == "prompt" else _log_int(rng, 1, 64)
    hi = _log_int(rng, 16, 28000) if B else 0
    P = 0 if form == "decode" else rng.choice((1, 1, 2, 3))
    return dict(kind="attend", B=B, lo=_log_int(rng, 1, hi) if B else 0, hi=hi, P=P,
                S=_log_int(rng, 2, 3000) if P else 0,
                start=_log_int(rng, 1, 20000) if form == "chunk" else 0, Hq=Hq, Hkv=Hkv, hd=hd,
                bs=rng.choice((16, 16, 32, 64)), window=rng.choice((0, 0, 0, 512, 1024, 4096)))


def draw(rng):
    kind = rng.choice(("rope", "write", "attend", "attend", "attend", "beam", "compact", "copy"))
    if kind == "rope":
        Hq, Hkv, hd = rng.choice(HEADS)
        # whole heads, halves and quarters of them
        return dict(kind=kind, T=_log_int(rng, 1, 8192 * 32 // max(32, (Hq + Hkv) * hd // 128)),
                    Hq=Hq, Hkv=Hkv, hd=hd, rot=rng.choice((hd, hd // 2, hd // 4)),
                    interleaved=rng.random() < 0.5, factor=rng.choice((1.0, 2.0, 4.0, 8.0)))
    if kind == "write":
        Hkv, hd = rng.choice(HEADS)[1:]
        most = 3000 * 4 * 128 // max(512, Hkv * hd)
        hi = _log_int(rng, 16, 28000)
        return dict(kind=kind, B=_log_int(rng, 1, 64), lo=_log_int(rng, 1, hi), hi=hi,
                    S=rng.choice((0, _log_int(rng, 2, most))), Hkv=Hkv, hd=hd,
                    bs=rng.choice((16, 16, 32, 64)))
    if kind == "attend":
        top = max(work(c)["flops"] for c in listed() if c["kind"] == "attend")
        top_bytes = max(work(c)["bytes"] for c in listed() if c["kind"] == "attend")
        while True:
            c = _draw_attend(rng)
            w = work(c)
            if w["flops"] <= top and w["bytes"] <= top_bytes:
                return c
    Hkv, hd = rng.choice(HEADS)[1:]
    row = max(512, Hkv * hd)
    if kind == "beam":
        hi = _log_int(rng, 16, 900)
        return dict(kind=kind, parents=_log_int(rng, 1, 16), width=rng.choice((1, 2, 3, 4)),
                    lo=_log_int(rng, 1, hi), hi=hi, L=_log_int(rng, 1, 28 * 512 // row), Hkv=Hkv,
                    hd=hd, bs=rng.choice((16, 16, 32)))
    if kind == "compact":
        return dict(kind=kind, NB=_log_int(rng, 64, 8192), L=_log_int(rng, 1, 16 * 512 // row),
                    fill=rng.uniform(0.2, 0.95), B=_log_int(rng, 1, 64), Hkv=Hkv, hd=hd, bs=16)
    NB = _log_int(rng, 16, 1024)
    return dict(kind=kind, NB=NB, n=_log_int(rng, 1, max(1, min(190, NB // 2))),
                L=_log_int(rng, 1, 28 * 512 // row), Hkv=Hkv, hd=hd, bs=rng.choice((16, 32)))


def _lengths(case):
    """The batch's context lengths, evenly over lo .. hi, the longest first."""
    B, lo, hi = case["B"], case["lo"], case["hi"]
    return [hi - (hi - lo) * b // max(1, B - 1) for b in range(B)]


def _keys(pos, window):
    return min(pos + 1, window) if window else pos + 1


def work(case):
    kind = case["kind"]
    if kind == "rope":
        heads = case["T"] * (case["Hq"] + case["Hkv"])
        return dict(bytes=4.0 * heads * case["hd"] + 8.0 * case["T"], flops=3.0 * heads * case["rot"])
    Hkv, hd, bs = case["Hkv"], case["hd"], case["bs"]
    if kind == "write":
        n = case["B"] + 2 * case["S"]
        return dict(bytes=2.0 * n * Hkv * hd * 3, flops=2.0 * n * Hkv * hd * 2)
    if kind == "attend":
        W, Hq = case["window"], case["Hq"]
        lens = _lengths(case)
        start, S, P = case["start"], case["S"], case["P"]
        pairs = sum(_keys(n - 1, W) for n in lens) + P * sum(_keys(start + s, W) for s in range(S))
        # the pages' keys that some query of the sequence sees
        read = sum(_keys(n - 1, W) for n in lens)
        read += P * (min(start + S, S + W - 1) if W else start + S)
        rows = case["B"] + P * S
        return dict(bytes=2.0 * read * Hkv * hd + 4.0 * rows * Hq * hd, flops=4.0 * hd * pairs * Hq)
    page = 2.0 * case["L"] * Hkv * (bs * hd + 1)
    if kind == "beam":
        # every beam takes a copy of its parent's last page where that is partly full
        copies = sum(case["width"] for n in _beam_lengths(case) if n % bs)
        pages = sum(-(-n // bs) for n in _beam_lengths(case)) * case["width"]
        return dict(bytes=2.0 * copies * page + 4.0 * 4 * pages, flops=1.0)
    if kind == "compact":
        moved = case["NB"] * case["fill"] * (1 - case["fill"])
        return dict(bytes=2.0 * moved * page + 16.0 * case["NB"], flops=1.0)
    return dict(bytes=2.0 * case["n"] * page + 8.0 * case["n"], flops=1.0)


# --- inputs ------------------------------------------------------------------

def _quantised(x):
    """Pages x [..., bs, hd] of values as (e4m3, scale byte), one exponent per page."""
    e = _exponent(x.abs().amax(dim=(-1, -2)))
    return torch.ldexp(x, -e[..., None, None]).to(F8), (e + 127).to(torch.uint8)


def _exponent(amax):
    """The least e in E_MIN .. E_MAX with amax <= 448 * 2^e, as int32."""
    m, x = torch.frexp(amax)  # amax = m * 2^x, m in [0.5, 1): 448 * 2^e = 0.875 * 2^(e + 9)
    e = x - 9 + (m > 0.875)
    return torch.where(amax > 0, e, torch.full_like(e, E_MIN)).clamp(E_MIN, E_MAX).to(torch.int32)


def _cache(gen, L, NB, Hkv, bs, hd, spread=2):
    """(e4m3 [L, NB, Hkv, bs, hd], scale bytes [L, NB, Hkv]) of pages of unequal sizes."""
    dev = gen.device
    q8 = torch.empty((L, NB, Hkv, bs, hd), dtype=F8, device=dev)
    sc = torch.empty((L, NB, Hkv), dtype=torch.uint8, device=dev)
    step = max(1, (1 << 27) // (Hkv * bs * hd))  # whole caches in fp32 would be large
    for layer in range(L):
        for a in range(0, NB, step):
            n = min(step, NB - a)
            x = torch.randn((n, Hkv, bs, hd), generator=gen, device=dev)
            x *= torch.exp2(torch.randint(-spread, 1, (n, Hkv, 1, 1), generator=gen, device=dev))
            q8[layer, a:a + n], sc[layer, a:a + n] = _quantised(x)
    return q8, sc


def _bytes_cache(gen, L, NB, Hkv, bs, hd):
    """The same of any bytes that are numbers: for what only moves them."""
    q8 = torch.randint(0, 256, (L, NB, Hkv, bs, hd), generator=gen, device=gen.device,
                       dtype=torch.uint8).bitwise_and_(0xBF)
    sc = torch.randint(100, 135, (L, NB, Hkv), generator=gen, device=gen.device, dtype=torch.uint8)
    return q8.view(F8), sc


def _tables(gen, lens, mb, NB):
    """A block table [len(lens), mb] of pages in random order, -1 behind each row's own."""
    dev = gen.device
    order = torch.randperm(NB, generator=gen, device=dev)
    n = torch.tensor([list(lens)], device=dev).view(-1, 1)
    col = torch.arange(mb, device=dev)[None, :]
    first = torch.cumsum(n, 0) - n
    at = (first + col).clamp(max=NB - 1)
    return torch.where(col < n, order[at], torch.full_like(at, -1)).to(torch.int32)


def _ints(v, dev, dtype=torch.int32):
    return torch.tensor(list(v), dtype=dtype, device=dev)


def _inv_freq(rot, factor):
    """Inverse frequencies for contexts `factor` times as long: low ones divided by it, high
    ones kept, a linear ramp between one and 32 turns over 4096 tokens."""
    i = torch.arange(0, rot, 2, dtype=F64)
    f = 1.0 / torch.pow(torch.tensor(1e6, dtype=F64), i / rot)
    turns = 4096.0 * f / (2 * math.pi)
    keep = ((turns - 1) / 31).clamp(0, 1)
    return (f * keep + f / factor * (1 - keep)).to(F32)


def _segments(case, table_of, dev):
    """(decodes, prompts) of a step: tokens first .. first + B * S of it, and their tables."""
    bs = case["bs"]
    lens = _lengths(case)
    P, S, start = case.get("P", 2), case["S"], case.get("start", 0)
    rows = []
    if lens:
        rows.append((0, 1, lens, [n - 1 for n in lens]))
    if S:
        rows.append((len(lens), S, [start + S] * P, [start] * P))
    need = [[-(-n // bs) for n in seq] for _, _, seq, _ in rows]
    tables = table_of(need)
    return [dict(token_offset=off, S=s, block_table=t, seq_len=_ints(seq, dev),
                 start_pos=_ints(at, dev))
            for (off, s, seq, at), t in zip(rows, tables)]


def _beam_lengths(case):
    P, lo, hi = case["parents"], case["lo"], case["hi"]
    return [hi - (hi - lo) * i // max(1, P - 1) for i in range(P)]


def prepare(case, seed):
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind = case["kind"]

    def r(shape, std=1.0):
        return torch.randn(shape, generator=gen, device=dev).mul_(std).to(F16)

    s = dict(case=case, kind=kind)
    if kind == "rope":
        T, Hq, Hkv, hd, rot = (case[n] for n in ("T", "Hq", "Hkv", "hd", "rot"))
        # the QKV product's output; Q and K are slices of its rows
        qkv = r((T, (Hq + 2 * Hkv) * hd))
        if T > 256:  # a prompt's positions, from a cached prefix on
            start = int(torch.randint(0, MAX_START, (1,), generator=gen, device=dev))
            pos = torch.arange(start, start + T, device=dev)
        else:  # a decode batch's
            pos = torch.randint(0, int(MAX_START * case["factor"]), (T,), generator=gen, device=dev)
        inv = _inv_freq(rot, case["factor"])
        s.update(q=qkv[:, :Hq * hd].view(T, Hq, hd),
                 k=qkv[:, Hq * hd:(Hq + Hkv) * hd].view(T, Hkv, hd), pos=pos, inv=inv.numpy(),
                 inv_dev=inv.to(dev), mscale=0.1 * math.log(case["factor"]) + 1.0,
                 q_out=torch.empty((T, Hq, hd), dtype=F16, device=dev),
                 k_out=torch.empty((T, Hkv, hd), dtype=F16, device=dev))
        return s
    Hkv, hd, bs = case["Hkv"], case["hd"], case["bs"]
    if kind in ("write", "attend"):
        pages = []

        def table_of(need):
            NB = sum(map(sum, need)) + 7
            pages.append(NB)
            flat = [n for row in need for n in row]
            mb = max(flat) + 1
            table = _tables(gen, flat, mb, NB)
            out, at = [], 0
            for row in need:
                out.append(table[at:at + len(row)].contiguous())
                at += len(row)
            return out

        s["segments"] = _segments(case, table_of, dev)
        T = sum(g["S"] * g["block_table"].shape[0] for g in s["segments"])
        s["kc"], s["ks"] = _cache(gen, 1, pages[0], Hkv, bs, hd)
        s["vc"], s["vs"] = _cache(gen, 1, pages[0], Hkv, bs, hd)
        if kind == "write":
            # rows of unequal sizes: some raise their page's scale
            big = torch.exp2(torch.randint(-1, 2, (T, Hkv, 1), generator=gen, device=dev))
            s.update(k=r((T, Hkv, hd)) * big.to(F16), v=r((T, Hkv, hd)) * big.to(F16))
        else:
            s.update(q=r((T, case["Hq"], hd), 2.0), out=torch.zeros((T, case["Hq"], hd), dtype=F16,
                                                                     device=dev))
        return s
    L = case["L"]
    if kind == "beam":
        lens = _beam_lengths(case)
        W = case["width"]
        need = [-(-n // bs) for n in lens]
        # the parents' pages, a page for each beam's copy and one for its next token, twice
        NB = sum(need) + 4 * len(lens) * W + 5
        mb = max(need) + 2
        table = _tables(gen, need + [0] * (len(lens) * W), mb, NB)
        ref = torch.zeros(NB, dtype=torch.int32, device=dev)
        used = table[table >= 0].long()
        ref[used] = 1
        kids = list(range(len(lens), len(lens) * (W + 1)))
        s.update(table=table, ref=ref, seq=_ints(lens + [0] * len(kids), dev),
                 parents=_ints([i for i in range(len(lens)) for _ in range(W)], dev),
                 kids=_ints(kids, dev), lens=_ints([n + 1 for n in lens for _ in range(W)], dev))
    elif kind == "compact":
        NB, B = case["NB"], case["B"]
        live = int(NB * case["fill"])
        share = [live // B + (b < live % B) for b in range(B)]
        table = _tables(gen, share, max(share) + 1, NB)
        ref = torch.zeros(NB, dtype=torch.int32, device=dev)
        ref[table[table >= 0].long()] = 1
        s.update(table0=table, ref0=ref, table=table.clone(), ref=ref.clone(),
                 moved=torch.empty(NB, dtype=torch.int32, device=dev))
    else:
        NB = case["NB"]
        order = torch.randperm(NB, generator=gen, device=dev).to(torch.int32)
        s.update(src=order[:case["n"]].contiguous(),
                 dst=order[case["n"]:2 * case["n"]].contiguous())
    kc, ks = _bytes_cache(gen, L, NB, Hkv, bs, hd)
    vc, vs = _bytes_cache(gen, L, NB, Hkv, bs, hd)
    s["caches"] = [kc, vc, ks, vs]
    return s


# --- the plain forms ---------------------------------------------------------

def _rope_plain(x, out, pos, inv, mscale, interleaved):
    rot = 2 * inv.numel()
    # a far position times a frequency needs more than 24 bits
    ang = pos.double()[:, None] * inv.double()[None, :]
    c = (torch.cos(ang) * mscale).float()[:, None, :]
    s = (torch.sin(ang) * mscale).float()[:, None, :]
    xr = x[..., :rot].float()
    out[..., rot:] = x[..., rot:]
    if interleaved:
        a, b = xr[..., 0::2], xr[..., 1::2]
        out[..., 0:rot:2] = (a * c - b * s).to(F16)
        out[..., 1:rot:2] = (b * c + a * s).to(F16)
    else:
        a, b = xr[..., :rot // 2], xr[..., rot // 2:]
        out[..., :rot // 2] = (a * c - b * s).to(F16)
        out[..., rot // 2:rot] = (b * c + a * s).to(F16)
    return out


def _token_places(segments, bs):
    """Page and slot of every token of the step, and whether it is its page's first here."""
    pages, slots = [], []
    for g in segments:
        s = torch.arange(g["S"], device=g["start_pos"].device)
        pos = g["start_pos"].long()[:, None] + s[None, :]
        pages.append(torch.gather(g["block_table"].long(), 1, pos // bs).reshape(-1))
        slots.append((pos % bs).reshape(-1))
    return torch.cat(pages), torch.cat(slots)


def _write_plain(x, cache, scales, page, slot):
    """x [T, H, hd] into cache [NB, H, bs, hd], scales [NB, H]."""
    NB, H, bs, hd = cache.shape
    held = cache.view(torch.uint8)
    x = x.float()
    tok = _exponent(x.abs().amax(-1))  # [T, H]: the page's exponent is the largest of its tokens'
    e = torch.full((NB, H), E_MIN, dtype=torch.int32, device=x.device)
    e = e.scatter_reduce(0, page[:, None].expand(-1, H), tok, "amax")
    begun = torch.ones(NB, dtype=torch.bool, device=x.device)
    begun[page[slot == 0]] = False  # slot 0 is written: the page begins here
    old = scales.int() - 127
    e = torch.where(begun[:, None], torch.maximum(e, old), e)
    e_tok, old_tok = e[page], old[page]  # [T, H]
    # the pages' other slots, as many times as the page has tokens here, the same each time
    kept = held[page].view(F8).float()
    again = torch.ldexp(kept, (old_tok - e_tok)[..., None, None])
    kept = torch.where(begun[page][:, None, None, None], again, kept).to(F8)
    held[page] = kept.view(torch.uint8)
    top = torch.exp2(torch.minimum(torch.full_like(e_tok, 16), 16 - e_tok).float())
    top = torch.minimum(torch.full_like(top, E4M3_MAX), top * 0.9375)  # 61440 in all, and 448
    q = torch.ldexp(x, -e_tok[..., None])
    q = torch.maximum(torch.minimum(q, top[..., None]), -top[..., None])
    held[page, :, slot] = q.to(F8).view(torch.uint8)
    scales[page] = (e_tok + 127).to(torch.uint8)


def _attend_plain(q, cache, kscale, vcache, vscale, g, out, window):
    """One segment: q and out [T, Hq, hd] of the step, cache [NB, Hkv, bs, hd]."""
    Hq, hd = q.shape[1:]
    table = g["block_table"].long().clamp(min=0)
    B, mb = table.shape
    _, Hkv, bs, _ = cache.shape
    S, G = g["S"], Hq // Hkv

    def keys(c, sc):
        x = c.view(torch.uint8)[table].view(F8).float()
        x = torch.ldexp(x, (sc[table].int() - 127)[..., None, None])
        return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, mb * bs, hd)

    part = slice(g["token_offset"], g["token_offset"] + B * S)
    x = q[part].float().view(B, S, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * S, hd)
    pos = g["start_pos"].long()[:, None] + torch.arange(S, device=q.device)[None, :]
    at = torch.arange(mb * bs, device=q.device)
    seen = at <= pos[..., None]
    if window:
        seen &= at > pos[..., None] - window
    hidden = ~seen[:, None, None].expand(B, 1, G, S, mb * bs).reshape(B, 1, G * S, mb * bs)
    score = torch.matmul(x, keys(cache, kscale).transpose(-1, -2).contiguous())
    score.mul_(1.0 / math.sqrt(hd)).masked_fill_(hidden, -math.inf)
    score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    y = torch.matmul(score, keys(vcache, vscale)) / total
    out[part] = y.view(B, Hkv, G, S, hd).permute(0, 3, 1, 2, 4).reshape(B * S, Hq, hd).to(F16)


def _free_plain(table, seq, ref, rows):
    gone = table[rows.long()]
    count = torch.zeros(ref.numel() + 1, dtype=torch.int32, device=ref.device)
    count.index_add_(0, torch.where(gone >= 0, gone, ref.numel()).long().view(-1),
                     torch.ones(gone.numel(), dtype=torch.int32, device=ref.device))
    ref.sub_(count[:-1])
    table[rows.long()] = -1
    seq[rows.long()] = 0


def _fork_plain(table, seq, ref, parents, kids):
    got = table[parents.long()]
    table[kids.long()] = got
    seq[kids.long()] = seq[parents.long()]
    count = torch.zeros(ref.numel() + 1, dtype=torch.int32, device=ref.device)
    count.index_add_(0, torch.where(got >= 0, got, ref.numel()).long().view(-1),
                     torch.ones(got.numel(), dtype=torch.int32, device=ref.device))
    ref.add_(count[:-1])


def _reserve_plain(caches, table, seq, ref, rows, lens, bs):
    """Room for lens[i] tokens in row rows[i]: new pages, and a copy of a shared last one."""
    rows, mb = rows.long(), table.shape[1]
    n = seq[rows].long()
    have, want = (n + bs - 1) // bs, (lens.long() + bs - 1) // bs
    last = torch.gather(table[rows].long(), 1, (have - 1).clamp(min=0)[:, None])[:, 0]
    part = (n % bs != 0) & (lens > n)
    same = (last[:, None] == last[None, :]) & part[None, :]
    rank = torch.tril(same, -1).sum(1)  # rows before this one that share its last page
    cow = part & (rank < ref[last.clamp(min=0)] - 1)
    need = cow.long() + (want - have).clamp(min=0)
    first = torch.cumsum(need, 0) - need
    free = torch.sort((ref != 0).int(), stable=True).indices  # free pages first, lowest first
    col = torch.arange(mb, device=table.device)[None, :]
    copy = cow[:, None] & (col == have[:, None] - 1)
    grow = (col >= have[:, None]) & (col < want[:, None])
    take = torch.where(copy, first[:, None], (first + cow.long() - have)[:, None] + col)
    page = free[take.clamp(0, free.numel() - 1)]
    fresh = copy | grow
    add = torch.zeros(ref.numel() + 1, dtype=torch.int32, device=ref.device)
    add.index_add_(0, torch.where(fresh, page, ref.numel()).view(-1),
                   torch.ones(page.numel(), dtype=torch.int32, device=ref.device))
    add.index_add_(0, torch.where(cow, last, ref.numel()),
                   torch.full((rows.numel(),), -1, dtype=torch.int32, device=ref.device))
    ref.add_(add[:-1])
    table[rows] = torch.where(fresh, page, table[rows].long()).to(torch.int32)
    seq[rows] = torch.maximum(seq[rows], lens)
    src = last[cow]
    dst = free[first[cow]]
    for c in caches:
        _copy_plain(c, src, dst)


def _copy_plain(cache, src, dst):
    c = cache.view(torch.uint8)
    c[:, dst] = c[:, src]


def _compact_plain(caches, table, ref):
    live = ref > 0
    page = torch.arange(ref.numel(), device=ref.device)
    n = live.sum()
    hole, mover = ~live & (page < n), live & (page >= n)
    dst, src = torch.nonzero(hole)[:, 0], torch.nonzero(mover)[:, 0]
    moved = torch.where(live, page, torch.full_like(page, -1))
    moved[src] = dst
    for c in caches:
        _copy_plain(c, src, dst)
    ref[dst] = ref[src]
    ref[src] = 0
    table.copy_(torch.where(table >= 0, moved[table.clamp(min=0).long()], -1))
    return moved.to(torch.int32)


def run(s):
    case, kind = s["case"], s["kind"]
    if kind == "rope":
        if own:
            q, k = _mk().rope_partial_qk(s["q"], s["k"], s["pos"], s["inv"],
                                         interleaved=case["interleaved"], mscale=s["mscale"],
                                         q_out=s["q_out"], k_out=s["k_out"])
        else:
            q, k = (_rope_plain(s[n], s[n + "_out"], s["pos"], s["inv_dev"], s["mscale"],
                                case["interleaved"]) for n in "qk")
        return dict(q=q, k=k)
    if kind == "write":
        if own:
            _mk().kv8_scatter(s["k"], s["v"], s["kc"], s["vc"], s["ks"], s["vs"], layer=0,
                              segments=s["segments"])
        else:
            page, slot = _token_places(s["segments"], case["bs"])
            _write_plain(s["k"], s["kc"][0], s["ks"][0], page, slot)
            _write_plain(s["v"], s["vc"][0], s["vs"][0], page, slot)
        return dict(kc=s["kc"], vc=s["vc"], ks=s["ks"], vs=s["vs"])
    if kind == "attend":
        if own:
            mk = _mk()
            if "ws" not in s:  # a program keeps it
                nbytes = mk.kv8_attention_workspace_bytes(case["Hq"], case["Hkv"], case["hd"],
                                                          s["segments"])
                s["ws"] = torch.zeros(max(16, nbytes), dtype=torch.uint8, device=s["q"].device)
            return mk.kv8_attention(s["q"], s["kc"], s["vc"], s["ks"], s["vs"], layer=0,
                                    segments=s["segments"], window=case["window"], out=s["out"],
                                    workspace=s["ws"])
        for g in s["segments"]:
            _attend_plain(s["q"], s["kc"][0], s["ks"][0], s["vc"][0], s["vs"][0], g, s["out"],
                          case["window"])
        return s["out"]
    caches = s["caches"]
    if kind == "beam":
        table, seq, ref = s["table"], s["seq"], s["ref"]
        if own:
            mk = _mk()
            mk.kv_free(table, seq, ref, s["kids"])
            mk.kv_fork(table, seq, ref, s["parents"], s["kids"])
            mk.kv_reserve(caches, table, seq, ref, s["kids"], s["lens"], case["bs"])
        else:
            _free_plain(table, seq, ref, s["kids"])
            _fork_plain(table, seq, ref, s["parents"], s["kids"])
            _reserve_plain(caches, table, seq, ref, s["kids"], s["lens"], case["bs"])
        return dict(caches=caches, table=table, seq=seq, ref=ref)
    if kind == "compact":
        # the fragmented state again (the moved pages' old places still hold them)
        s["table"].copy_(s["table0"])
        s["ref"].copy_(s["ref0"])
        if own:
            moved = _mk().kv_compact(caches, s["table"], s["ref"], moved=s["moved"])
        else:
            moved = _compact_plain(caches, s["table"], s["ref"])
        return dict(caches=caches, table=s["table"], ref=s["ref"], moved=moved)
    if own:
        _mk().kv_copy_pages(caches, s["src"], s["dst"])
    else:
        for c in caches:
            _copy_plain(c, s["src"].long(), s["dst"].long())
    return dict(caches=caches)


# --- the same in 64 bits -----------------------------------------------------

def _exact_rope(s):
    case = s["case"]
    freq = torch.from_numpy(s["inv"]).to(s["q"].device).to(F64)
    turn = torch.polar(torch.full((case["T"], 1, freq.numel()), s["mscale"], dtype=F64,
                                  device=freq.device),
                       (s["pos"].to(F64).view(-1, 1) * freq).unsqueeze(1))

    def rotated(x):
        x = x.to(F64)
        r = x[..., :case["rot"]]
        if case["interleaved"]:
            z = torch.view_as_complex(r.reshape(*r.shape[:-1], -1, 2).contiguous()) * turn
            y = torch.view_as_real(z).reshape(r.shape)
        else:
            z = torch.complex(*(t.contiguous() for t in r.chunk(2, -1))) * turn
            y = torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., case["rot"]:]), -1)

    return dict(q=rotated(s["q"]), k=rotated(s["k"]))


def _e4m3(x):
    """x in 64 bits, rounded to the nearest e4m3 value, ties to even."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_write(s):
    bs = s["case"]["bs"]
    out = {}
    for name in "kv":
        x = s[name].to(F64)
        cache, sc = s[name + "c"].to(F64), s[name + "s"].clone()
        for g in s["segments"]:
            table, starts = g["block_table"].tolist(), g["start_pos"].tolist()
            for b, (row, p0) in enumerate(zip(table, starts)):
                t0 = g["token_offset"] + b * g["S"]
                p = p0
                while p < p0 + g["S"]:  # a page of the sequence at a time
                    end = min(p0 + g["S"], (p // bs + 1) * bs)
                    new = x[t0 + p - p0:t0 + end - p0].transpose(0, 1)  # [H, n, hd]
                    page, slot = row[p // bs], p % bs
                    amax = new.abs().amax(dim=(1, 2))
                    e = torch.ceil(torch.log2(amax.clamp(min=2.0 ** -40) / 448)).clamp(-32, 8)
                    if slot:
                        old = sc[0, page].to(F64) - 127
                        e = torch.maximum(e, old)
                        cache[0, page] = _e4m3(cache[0, page] * torch.exp2(old - e)[:, None, None])
                    q = new * torch.exp2(-e)[:, None, None]
                    most = torch.clamp(61440 * torch.exp2(-e), max=448)[:, None, None]
                    cache[0, page][:, slot:slot + end - p] = _e4m3(torch.minimum(
                        torch.maximum(q, -most), most))
                    sc[0, page] = (e + 127).to(torch.uint8)
                    p = end
        out[name + "c"] = cache
    return dict(kc=out["kc"], vc=out["vc"], ks=None, vs=None)


def _exact_attend(s):
    case = s["case"]
    bs, W, G, hd = case["bs"], case["window"], case["Hq"] // case["Hkv"], case["hd"]
    out = torch.zeros(s["q"].shape, dtype=F64, device=s["q"].device)
    for g in s["segments"]:
        lens, starts = g["seq_len"].tolist(), g["start_pos"].tolist()
        for b, (n, p0) in enumerate(zip(lens, starts)):
            lo = max(0, p0 - W + 1) // bs if W else 0  # the first page that a query sees
            pages = g["block_table"][b, lo:-(-n // bs)].long()
            kv = []
            for c, sc in ((s["kc"], s["ks"]), (s["vc"], s["vs"])):
                x = c[0].view(torch.uint8)[pages].view(F8).to(F64) * torch.exp2(sc[0][pages].to(F64) - 127)[..., None, None]
                kv.append(x.transpose(0, 1).reshape(case["Hkv"], -1, hd))
            at = lo * bs + torch.arange(kv[0].shape[1], device=out.device)
            t0 = g["token_offset"] + b * g["S"]
            for a in range(0, g["S"], 512):
                m = min(512, g["S"] - a)
                pos = p0 + a + torch.arange(m, device=out.device)[:, None]
                ok = (at <= pos) & (at > pos - W) if W else at <= pos
                for h in range(case["Hq"]):
                    q = s["q"][t0 + a:t0 + a + m, h].to(F64)
                    w = (q @ kv[0][h // G].t()) / math.sqrt(hd)
                    w = torch.softmax(w.masked_fill(~ok, -math.inf), -1)
                    out[t0 + a:t0 + a + m, h] = w @ kv[1][h // G]
    return out


def exact(case, seed):
    if case["kind"] not in ("rope", "write", "attend"):
        return None  # pages are moved, nothing is computed
    s = prepare(case, seed)
    if case["kind"] == "rope":
        return _exact_rope(s)
    return _exact_write(s) if case["kind"] == "write" else _exact_attend(s)
