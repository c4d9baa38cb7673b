"""The measured calls of rotary positions with several axes and of the 4-bit paged key/value cache with them: rows rotated,
rotated rows appended to the cache, the pages' digests, the pages that each row selects, and attention over those alone.

`listed()` names the cases and `draw(rng)` gives others of the same ranges; `prepare(case, seed)` makes what a caller has
in hand, `run(state)` makes one pass: with `own` false in elementary torch operations, with `own` true through libjepa.so.
`work(case)` counts the bytes and operations that a pass cannot do without, `exact(case, seed)` computes it in 64 bits.

Rotation. Element j of a rotated section has an angle A_j = pos[axis] * scale[axis] * theta^(-2 f / width) and a partner p:
out_j = x_j cos A_j -+ x_p sin A_j (minus for the first of a pair). form 0: pairs (2i, 2i + 1) with f = j % (width / 2), so
that a pair has two angles; 1: pairs (2i, 2i + 1), f = i; 2: pairs (i, i + width / 2), f = i; 3: pairs (i, i + W / 2) of all W rotated
elements, f = i and W for the width, the axis that whose half-width i falls into. Cosines and sines are f32, products and sums rounded to f32 each.

The cache is a byte tensor [n_pages][n_kv_head][page_size / 16][18 * head_dim]. A strip of 16 tokens of one head holds, with
NB = head_dim / 32 blocks of 32 values:
  K codes   [4 g][16 tokens][NB b][4 bytes]: dims 32 b + 8 g + (0, 2, 4, 6, 1, 3, 5, 7), from the low nibble up
  V codes   [16 tokens][head_dim / 2 bytes]: dims in order, from the low nibble up
  K scales  f16 [4 tokens / 4][NB][4 tokens % 4], then the V scales in the same order
A value is (code - 8) * scale, ggml's q4_0.

A page's digest, [n_pages][n_kv_head][2 * head_dim + 16] bytes: the largest value of each dimension of K over the page's tokens as
signed 8-bit codes, then the smallest, then their f32 scale (the largest magnitude / 127). A page's score for a row is the sum over the heads that share a K/V
head of the largest product that a key within these bounds could have with the head's query.
"""
import ctypes
import math
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30)}
NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]      # element of a K word's nibble, from the low one up
F16_MAX = 65504.0
TINY = 2.0 ** -100                       # queries and pages whose largest magnitude is below count as zeros


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the query and key heads of one step of 64 requests at far positions, three position axes through one set of frequencies
        dict(name="rotate 64 tokens f16", op="rope", n_rows=64, heads=40, hd=128, form=3, dims="32 48 48", theta=1e6, type="f16", grid="", far=100000, back=False),
        # the gradient of a long clip's queries: 32 frames of 16 x 16 patches, heads of 88
        dict(name="rotate clip gradient bf16", op="rope", n_rows=8192, heads=16, hd=88, form=1, dims="28 28 28", theta=1e4, type="bf16", grid="16 16", far=0, back=True),
        # one frame of 256 patches and two more tokens for each of 16 candidate rollouts, f32 rows as the library's projections write them
        dict(name="append frames f32", op="append", n_rows=4128, heads=16, kv_heads=16, hd=64, page=32, type="f32", form=0, dims="20 20 20", theta=1e4, grid="16 16",
             far=0),
        # a batch of prompts
        dict(name="append prompts bf16", op="append", n_rows=32768, heads=32, kv_heads=8, hd=128, page=16, type="bf16", form=3, dims="32 48 48", theta=1e6, grid="",
             far=0),
        # the pages that one token of each of 64 requests went to
        dict(name="digest 64 tokens", op="digest", n_seq=64, lo=200, hi=8000, new_lo=1, new_hi=1, kv_heads=8, hd=128, page=64, ragged=1),
        # all pages of a batch of prompts
        dict(name="digest prompts", op="digest", n_seq=6, lo=0, hi=0, new_lo=700, new_hi=12000, kv_heads=8, hd=128, page=16, ragged=2),
        # one token of each of 64 requests of very different lengths: at most 1024 tokens each
        dict(name="select 64 requests f16", op="select", n_seq=64, lo=200, hi=8000, new_lo=1, new_hi=1, heads=32, kv_heads=8, hd=128, page=16, type="f16", block=1,
             first=1, last=4, take=64, ragged=3),
        # two long documents, one token each
        dict(name="select long context bf16", op="select", n_seq=2, lo=90000, hi=131000, new_lo=1, new_hi=1, heads=64, kv_heads=8, hd=128, page=32, type="bf16", block=1,
             first=1, last=2, take=128, ragged=4),
        # a piece of a long prompt after the pieces before it
        dict(name="select prompt piece f16", op="select", n_seq=1, lo=14000, hi=14000, new_lo=2000, new_hi=2000, heads=32, kv_heads=4, hd=128, page=64, type="f16",
             block=1, first=1, last=2, take=16, ragged=5),
        # one token of one request: latency alone
        dict(name="attend one token f32", op="attend", n_seq=1, lo=5000, hi=5000, new_lo=1, new_hi=1, heads=16, kv_heads=16, hd=64, page=16, type="f32", block=1,
             first=1, last=2, take=32, ragged=6),
        # one token of each of 64 requests, grouped heads
        dict(name="attend 64 requests f16", op="attend", n_seq=64, lo=200, hi=8000, new_lo=1, new_hi=1, heads=32, kv_heads=8, hd=128, page=16, type="f16", block=1,
             first=1, last=4, take=64, ragged=7),
        # a piece of a long prompt, every row over its own pages
        dict(name="attend prompt piece bf16", op="attend", n_seq=1, lo=14000, hi=14000, new_lo=2000, new_hi=2000, heads=32, kv_heads=4, hd=128, page=64, type="bf16",
             block=1, first=1, last=2, take=16, ragged=8),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def _draw_axes(rng, hd):
    """A form and widths of its sections for heads of hd."""
    form = rng.randrange(4)
    if hd < 16:
        form = rng.randrange(2)
    unit = 16 if form == 2 else 2
    n = rng.randrange(1, min(4, hd // unit) + 1)
    left, widths = hd // unit, []
    for i in range(n):
        w = left // (n - i) if rng.random() < 0.5 else rng.randrange(1, left - (n - i - 1) + 1)
        widths.append(w * unit)
        left -= w
    if form == 3:
        short = sum(widths) % 16
        if short and widths[-1] > short:
            widths[-1] -= short
        elif short:
            widths = [16]
    return dict(form=form, dims=" ".join(map(str, widths)), theta=rng.choice([1e4, 1e6]), grid=rng.choice(["", "", "16 16", "9 14"]) if len(widths) == 3 else "",
                far=rng.choice([0, 1000, 1000000]))


def draw(rng):
    op = rng.choice(["rope", "append", "digest", "select", "select", "attend", "attend", "attend"])
    kind, ragged = rng.choice(list(TYPES)), rng.randrange(1 << 30)
    if op == "rope":
        hd, heads = 8 * rng.randrange(1, 33), rng.choice([1, 2, 3, 5, 12, 16, 40])
        return dict(op=op, n_rows=_log(rng, 1, min(32768, 50000000 // (hd * heads))), heads=heads, hd=hd, type=kind, back=rng.random() < 0.5, **_draw_axes(rng, hd))
    hd, kv_heads, page = rng.choice([32, 64, 96, 128]), rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([16, 32, 64, 128, 256])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    if op == "append":
        return dict(op=op, n_rows=_log(rng, 1, min(32768, 200000000 // (hd * (heads + 2 * kv_heads)))), heads=heads, kv_heads=kv_heads, hd=hd, page=page, type=kind,
                    **_draw_axes(rng, hd))
    how = rng.choice(["token", "token", "few", "prompt", "frames"])
    block = 1
    if how == "token":
        new, n_seq = 1, _log(rng, 1, 100)
        hi = _log(rng, 1, min(100000, 1500000 // n_seq // kv_heads + 1000))
    elif how == "few":
        new, n_seq = rng.randrange(2, 17), _log(rng, 1, 40)
        hi = _log(rng, 1, min(20000, 400000 // n_seq // kv_heads + 500))
    elif how == "prompt":
        n_seq = _log(rng, 1, 8)
        new = _log(rng, 2, 1000 // n_seq + 100)
        hi = rng.choice([0, _log(rng, 1, 8000)])
    else:
        n_seq, new = _log(rng, 1, 8), _log(rng, 2, 200)
        hi = new * rng.randrange(0, 8)
        block = rng.choice([0, new])
    take = _log(rng, 2, 256)
    first, last = rng.choice([0, 1, 2]), rng.choice([1, 2, 5])
    take = max(take, first + last)
    while op == "attend" and n_seq * new * kv_heads * take * page * hd > 5e8 and take > first + last:
        take = max(first + last, take // 2)
    while op == "attend" and n_seq * new * kv_heads * take * page * hd > 5e8:
        new = -(-new // 2)
    if op == "select":      # more pages than are taken: else there is nothing to select
        hi = max(hi, 60 * page)
        take = min(take, max(first + last + 4, (hi - hi // 2) // page // 2))
    case = dict(op=op, n_seq=n_seq, lo=hi if how == "frames" else hi - hi // 2, hi=hi, new_lo=max(1, new // 3) if how == "prompt" else new, new_hi=new, kv_heads=kv_heads, hd=hd,
                page=page, ragged=ragged)
    if op != "digest":
        case.update(heads=heads, type=kind, block=min(block, new) if how == "frames" else block, first=first, last=last, take=take)
    return case


def _lengths(case):
    """(tokens in the cache before, tokens that come) of each sequence."""
    rng = random.Random(case["ragged"])
    have = [rng.randint(case["lo"], case["hi"]) for _ in range(case["n_seq"])]
    return have, [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["n_seq"])]


def _pages(n, page):
    return -(-n // page)


def _visible(pos, total, block):
    return total if block == 0 else min(total, (pos // block + 1) * block)


def _rows_seen(case):
    """(sequence, tokens that it sees) of every row."""
    have, new = _lengths(case)
    return [(i, _visible(h + j, h + n, case["block"])) for i, (h, n) in enumerate(zip(have, new)) for j in range(n)]


def _touched(case):
    """(sequence, page of its table, tokens in it) of the pages that the step's tokens went to."""
    have, new = _lengths(case)
    page = case["page"]
    return [(i, p, min(page, h + n - p * page)) for i, (h, n) in enumerate(zip(have, new)) for p in range(h // page, _pages(h + n, page))]


def work(case):
    hd = case["hd"]
    size = torch.empty(0, dtype=TYPES[case["type"]][0]).element_size() if "type" in case else 0
    if case["op"] == "rope":
        n = case["n_rows"] * case["heads"] * hd
        return {"bytes": 2 * n * size + 4 * case["n_rows"] * len(case["dims"].split()), "flops": 3 * n}
    cell, digest = 2 * (hd // 2 + hd // 16), 2 * hd + 4      # bytes of one token of one head in the cache; of one page and head of the digests
    if case["op"] == "append":
        rows, kvh, heads = case["n_rows"], case["kv_heads"], case["heads"]
        return {"bytes": rows * (2 * heads * hd * size + kvh * (4 * hd * size + 2 * cell) + 8 + 4 * len(case["dims"].split())),
                "flops": rows * hd * (3 * heads + 9 * kvh)}
    if case["op"] == "digest":
        pages = _touched(case)
        return {"bytes": case["kv_heads"] * (sum(n for _, _, n in pages) * cell // 2 + len(pages) * (digest + 8 * hd)), "flops": 3 * case["kv_heads"] * hd * sum(n for _, _, n in pages)}
    have, new = _lengths(case)
    seen, page, take = _rows_seen(case), case["page"], case["take"]
    q = len(seen) * case["heads"] * hd * size
    lists = 4 * len(seen) * case["kv_heads"] * take
    if case["op"] == "select":
        return {"bytes": q + lists + case["kv_heads"] * digest * sum(_pages(h + n, page) for h, n in zip(have, new)),
                "flops": 4 * hd * case["kv_heads"] * sum(_pages(e, page) for _, e in seen)}
    tokens = [min(e, take * page) for _, e in seen]
    most = [0] * len(new)
    for (i, _), t in zip(seen, tokens):
        most[i] += t
    read = sum(min(h + n, m) for h, n, m in zip(have, new, most))
    return {"bytes": 2 * q + lists + read * case["kv_heads"] * cell, "flops": 4 * hd * case["heads"] * sum(tokens)}


# ------------------------------------------------------------------------------------------------ the rotation's and the cache's formats
def _axes(case):
    """(axis, frequency, partner, sign) of every element of a head; elements that are not rotated have axis -1."""
    widths, form, theta, hd = [int(w) for w in case["dims"].split()], case["form"], case["theta"], case["hd"]
    axis, freq, partner, sign = [-1] * hd, [0.0] * hd, list(range(hd)), [0.0] * hd
    at, total = 0, sum(widths)
    for a, w in enumerate(widths):
        for i in range(w // 2):
            if form == 3:
                x, y, fx, fy, of = at // 2 + i, at // 2 + i + total // 2, at // 2 + i, at // 2 + i, total
            elif form == 2:
                x, y, fx, fy, of = at + i, at + i + w // 2, i, i, w
            else:
                x, y, of = at + 2 * i, at + 2 * i + 1, w
                fx, fy = (2 * i % (w // 2), (2 * i + 1) % (w // 2)) if form == 0 else (i, i)
            for e, f, p, s in ((x, fx, y, -1.0), (y, fy, x, 1.0)):
                axis[e], freq[e], partner[e], sign[e] = a, theta ** (-2.0 * f / of), p, s
        at += w
    return axis, freq, partner, sign


def _quantize(x):
    """f32 values [..., head_dim] -> q4_0 codes (whole numbers) and f16 scales [..., head_dim / 32]. Values outside f16's range are held at its ends."""
    x = x.clamp(-F16_MAX, F16_MAX).reshape(*x.shape[:-1], -1, 32)
    m = x.gather(-1, x.abs().argmax(-1, keepdim=True))
    d = m / -8.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return (x * inv + 8.5).to(torch.int32).clamp(max=15).flatten(-2), d[..., 0].half()


def _bytes(codes):
    return (codes[..., 0::2] | (codes[..., 1::2] << 4)).to(torch.uint8)


def _nibbles(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def _pack(k, v):
    """f32 rows K and V [..., head_dim] -> the bytes of their token [..., 18 * head_dim / 16]: K codes, V codes, K scales, V scales."""
    lead, nb = k.shape[:-1], k.shape[-1] // 32
    (kc, kd), (vc, vd) = _quantize(k), _quantize(v)
    kc = kc.reshape(*lead, nb, 4, 8)[..., NIBBLES].transpose(-3, -2)
    return torch.cat([_bytes(kc).reshape(*lead, -1), _bytes(vc), kd.contiguous().view(torch.uint8), vd.contiguous().view(torch.uint8)], -1)


def _unpack(token, hd):
    """The bytes of tokens [..., 18 * head_dim / 16] -> f32 K and V [..., head_dim]."""
    lead, nb = token.shape[:-1], hd // 32
    kb, vb, kd, vd = token.split([hd // 2, hd // 2, 2 * nb, 2 * nb], -1)
    back = torch.tensor(NIBBLES, device=token.device).argsort()
    k = _nibbles(kb.reshape(*lead, 4, nb, 4))[..., back].transpose(-3, -2).reshape(*lead, nb, 32)
    v = _nibbles(vb).reshape(*lead, nb, 32)
    return [((codes.to(torch.int16) - 8).float() * d.contiguous().view(torch.float16).float()[..., None]).reshape(*lead, hd) for codes, d in ((k, kd), (v, vd))]


def _places(hd, device):
    """Where the bytes of each of a strip's 16 tokens lie in it: [16][18 * head_dim / 16]."""
    t, nb, a = torch.arange(16, device=device)[:, None], hd // 32, torch.arange(hd // 2, device=device)
    k = (a // (4 * nb) * 16 + t) * 4 * nb + a % (4 * nb)
    v = 8 * hd + t * (hd // 2) + a
    d = torch.arange(2 * nb, device=device)
    d = 16 * hd + 2 * ((t // 4 * nb + d // 2) * 4 + t % 4) + d % 2
    return torch.cat([k, v, d, d + hd], 1)


# ------------------------------------------------------------------------------------------------ inputs
def _rows(gen, shape, dtype, spread=1.0):
    x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    # a few channels are several times larger than the others, as keys and values of trained models are
    c = 1 + 3 * (torch.rand(shape[-1], generator=gen, device="cuda") < 0.05)
    return (x * c * spread).to(dtype)


def _filled(gen, n_pages, kv_heads, page, hd):
    """A cache whose every token holds a quantized row."""
    cache = torch.empty(n_pages, kv_heads, page // 16, 18 * hd, dtype=torch.uint8, device="cuda")
    places = _places(hd, "cuda").flatten()
    step = max(1, (1 << 25) // (kv_heads * page * hd))
    for a in range(0, n_pages, step):
        n = min(step, n_pages - a)
        k, v = (_rows(gen, (n, kv_heads, page // 16, 16, hd), torch.float32) for _ in range(2))
        cache[a:a + n, :, :, places] = _pack(k, v).flatten(-2)
    return cache


def _positions(gen, case):
    """[n_rows][axes]: tokens of frames by (frame, row, column), or of text, every axis the same, from somewhere up to `far` on."""
    n, axes = case["n_rows"], len(case["dims"].split())
    r = torch.arange(n, device="cuda")
    start = torch.randint(0, case["far"] + 1, (1,), generator=gen, device="cuda")
    if case["grid"]:
        h, w = (int(x) for x in case["grid"].split())
        return (torch.stack([r // (h * w), r // w % h, r % w], 1) + torch.stack([start[0], 0 * start[0], 0 * start[0]])).int().contiguous()
    at = r + start if n > 256 else torch.randint(0, case["far"] + 1, (n,), generator=gen, device="cuda")
    return at[:, None].expand(n, axes).int().contiguous()


def _rope_state(gen, case, st):
    axis, freq, partner, sign = _axes(case)
    dev = dict(device="cuda")
    widths = [int(w) for w in case["dims"].split()]
    st.update(widths=widths, scales=[1.0, 15 / 23, 15 / 23][:len(widths)] if case["grid"] else [1.0] * len(widths), pos=_positions(gen, case))
    st.update(axis=torch.tensor(axis, **dev), freq=torch.tensor(freq, dtype=torch.float64, **dev), partner=torch.tensor(partner, **dev),
              sign=torch.tensor(sign, **dev), axis_scale=torch.tensor(st["scales"] + [0.0], dtype=torch.float64, **dev))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    st = dict(case)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    hd = case["hd"]
    dtype = TYPES[case["type"]][0] if "type" in case else None
    if case["op"] == "rope":
        _rope_state(gen, case, st)
        # queries and keys lie in front of the values in one row, as a fused projection leaves them
        st["x"] = _rows(gen, (case["n_rows"], (case["heads"] + case["heads"] // 5) * hd), dtype)[:, :case["heads"] * hd]
        return st
    page, kvh = case["page"], case["kv_heads"]
    if case["op"] == "append":
        rows, heads = case["n_rows"], case["heads"]
        _rope_state(gen, case, st)
        n_pages = _pages(rows, page) * 2 + 1
        pages = torch.randperm(n_pages, generator=gen, device="cuda")[:_pages(rows, page)]
        slots = (pages[:, None] * page + torch.arange(page, device="cuda")).flatten()[:rows].contiguous()
        qkv = _rows(gen, (rows, (heads + 2 * kvh) * hd), dtype)
        st.update(n_pages=n_pages, slots=slots, q=qkv[:, :heads * hd], k=qkv[:, heads * hd:(heads + kvh) * hd], v=qkv[:, (heads + kvh) * hd:],
                  cache=torch.zeros(n_pages, kvh, page // 16, 18 * hd, dtype=torch.uint8, device="cuda"))
        return st
    have, new = _lengths(case)
    total = [h + n for h, n in zip(have, new)]
    used = [_pages(t, page) for t in total]
    n_pages, width = sum(used) + 3, max(used)
    order = torch.randperm(n_pages, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.full((len(total), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st.update(n_pages=n_pages, width=width, rows=starts[-1], longest=max(total), most=max(new), table=table, kv_len=ints(total), row_start=ints(starts))
    if case["op"] == "digest":
        touched = _touched(case)
        page_of = table.flatten()[torch.tensor([i * width + p for i, p, _ in touched], device="cuda")].contiguous()
        st.update(page_of=page_of, tokens=ints([n for _, _, n in touched]), cache=_filled(gen, n_pages, kvh, page, hd),
                  digest=torch.zeros(n_pages, kvh, 2 * hd + 16, dtype=torch.uint8, device="cuda"))
        return st
    st["q"] = _rows(gen, (starts[-1], case["heads"], hd), dtype, 0.7)
    if case["op"] == "select":
        # bounds around the page's mean, as the largest and smallest of its keys are
        mid, out = _rows(gen, (n_pages, kvh, hd), torch.float32, 0.5), _rows(gen, (n_pages, kvh, 2 * hd), torch.float32, 0.3).abs() + 1.0
        bounds = torch.cat([mid + out[..., :hd], mid - out[..., hd:]], -1)
        top = bounds.abs().amax(-1, keepdim=True)
        st["digest"] = torch.cat([torch.round(bounds * (127 / top)).to(torch.int8).view(torch.uint8), (top / 127).view(torch.uint8),
                                  torch.zeros(n_pages, kvh, 12, dtype=torch.uint8, device="cuda")], -1).contiguous()
        return st
    # pages as a selection gives them: the first and the last ones and others here and there, ascending, -1 behind the last
    take, seen = case["take"], [_pages(e, page) for _, e in _rows_seen(case)]
    see = torch.tensor(seen, device="cuda")[:, None, None]
    p = torch.arange(width, device="cuda")
    key = torch.rand(starts[-1], kvh, width, generator=gen, device="cuda")
    key = torch.where((p < case["first"]) | (p >= see - case["last"]), 2.0, key).masked_fill(p >= see, -1.0)
    best = key.topk(min(take, width), -1)
    chosen = torch.where(best.values < 0, width, best.indices).sort(-1).values
    chosen = torch.nn.functional.pad(torch.where(chosen == width, -1, chosen), (0, take - chosen.shape[-1]), value=-1)
    st.update(selected=chosen.int().contiguous(), scale=hd ** -0.5, cache=_filled(gen, n_pages, kvh, page, hd))
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_rotate(s, x, back=False):
    """Rows [n_rows][heads][head_dim] in f32, rotated (or their gradient turned back)."""
    angle = s["pos"].double() * s["axis_scale"][:len(s["widths"])]
    angle = torch.cat([angle, torch.zeros_like(angle[:, :1])], 1)[:, s["axis"]] * s["freq"]
    c, t = torch.cos(angle).float()[:, None], (torch.sin(angle).float() * s["sign"])[:, None]
    if back:
        t = t[..., s["partner"]]
    return x * c + x[..., s["partner"]] * t


def _plain_rope(s):
    x = s["x"].float().reshape(s["n_rows"], s["heads"], s["hd"])
    return _plain_rotate(s, x, s["back"]).reshape(s["n_rows"], -1).to(s["x"].dtype)


def _plain_append(s):
    hd, kvh, page, rows = s["hd"], s["kv_heads"], s["page"], s["n_rows"]
    page_of, strip, token = s["slots"] // page, s["slots"] % page // 16, s["slots"] % 16
    q, k, v = (s[x].float().reshape(rows, -1, hd) for x in "qkv")
    at = (page_of[:, None, None], torch.arange(kvh, device=k.device)[:, None], strip[:, None, None], _places(hd, k.device)[token][:, None])
    s["cache"][at] = _pack(_plain_rotate(s, k), v)
    k, v = _unpack(s["cache"][at], hd)
    return dict(q=_plain_rotate(s, q).reshape(rows, -1).to(s["q"].dtype), k=k.reshape(rows, -1).to(s["k"].dtype), v=v.reshape(rows, -1).to(s["v"].dtype))


def _plain_digest(s):
    hd, kvh, page = s["hd"], s["kv_heads"], s["page"]
    k, _ = _unpack(s["cache"][s["page_of"].long()][..., _places(hd, s["cache"].device)], hd)
    k = k.reshape(-1, kvh, page, hd)
    out = (torch.arange(page, device=k.device) >= s["tokens"][:, None])[:, None, :, None] | k.isnan()
    bounds = torch.cat([k.masked_fill(out, float("-inf")).amax(2), k.masked_fill(out, float("inf")).amin(2)], -1)
    bounds = torch.where(bounds.isinf(), 0.0, bounds)
    top = bounds.abs().amax(-1, keepdim=True)
    some = top >= TINY
    codes = torch.round(bounds * torch.where(some, torch.full_like(top, 127.0) / top, 0.0))
    scale = torch.where(some, top / 127, 0.0)
    s["digest"][s["page_of"].long()] = torch.cat([codes.to(torch.int8).view(torch.uint8), scale.view(torch.uint8), torch.zeros_like(s["digest"][:len(codes), :, :12])], -1)
    return (codes * scale).reshape(-1, kvh, 2, hd)


def _places_of_rows(s):
    """The sequence of each row, and its place there."""
    start, r = s["row_start"].long(), torch.arange(s["rows"], device=s["row_start"].device)
    i = torch.searchsorted(start[1:], r, right=True)
    return i, r - start[i]


def _of_sequences(s, x):
    """Rows [rows][...] -> [n_seq][most][...] (some other row behind a sequence's last)."""
    return x[(s["row_start"][:-1, None].long() + torch.arange(s["most"], device=x.device)).clamp(max=s["rows"] - 1)]


def _plain_end(s):
    """The tokens that each row [n_seq][most] sees."""
    start, total = s["row_start"].long(), s["kv_len"].long()
    pos = (total - (start[1:] - start[:-1]))[:, None] + torch.arange(s["most"], device=total.device)
    return total[:, None].expand_as(pos) if s["block"] == 0 else torch.minimum(total[:, None], (pos // s["block"] + 1) * s["block"])


def _plain_select(s):
    hd, kvh, page, take = s["hd"], s["kv_heads"], s["page"], s["take"]
    q = s["q"].float().reshape(s["rows"], kvh, -1, hd).double()
    q = torch.cat([q.clamp(min=0).sum(2), q.clamp(max=0).sum(2)], -1).float()                    # sums over the heads of one K/V head
    top = q.abs().amax(-1, keepdim=True)
    codes = torch.where(top.isfinite() & (top >= TINY), torch.round(q * (torch.full_like(top, 127.0) / top)), 0.0)
    codes = _of_sequences(s, codes)
    digest = s["digest"][s["table"].long().clamp(min=0)].transpose(1, 2)                          # [n][kvh][pages][bytes]
    dots = torch.matmul(codes.transpose(1, 2), digest[..., :2 * hd].contiguous().view(torch.int8).float().transpose(-1, -2))      # whole numbers below 2^24: exact
    score = dots * digest[..., 2 * hd:2 * hd + 4].contiguous().view(torch.float32).transpose(-1, -2)                              # [n][kvh][most][pages]
    see = (-(-_plain_end(s) // page))[:, None, :, None]
    p = torch.arange(s["width"], device=q.device)
    score = torch.where((p < s["first"]) | (p >= see - s["last"]), float("inf"), score).masked_fill(p >= see, float("-inf"))
    best = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :take]
    best = torch.where(best < see, best, s["width"]).sort(-1).values
    best = torch.nn.functional.pad(torch.where(best == s["width"], -1, best), (0, take - best.shape[-1]), value=-1)
    return best.transpose(1, 2)[_places_of_rows(s)].int()


def _plain_attend(s):
    hd, kvh, page, take, rows = s["hd"], s["kv_heads"], s["page"], s["take"], s["rows"]
    i, j = _places_of_rows(s)
    chosen = s["selected"].long()
    end = _plain_end(s)[i, j]
    phys = s["table"].long()[i[:, None, None], chosen.clamp(min=0)].clamp(min=0)
    strips = s["cache"][phys, torch.arange(kvh, device=phys.device)[:, None]]                     # [rows][kvh][take][strips][bytes]
    k, v = (x.reshape(rows, kvh, take * page, hd) for x in _unpack(strips[..., _places(hd, phys.device)], hd))
    pos = (chosen[..., None] * page + torch.arange(page, device=phys.device)).flatten(-2)
    seen = ((chosen >= 0)[..., None].expand(-1, -1, -1, page).flatten(-2) & (pos < end[:, None, None]))[:, :, None]
    logits = torch.matmul(s["q"].float().reshape(rows, kvh, -1, hd), k.transpose(-1, -2)) * s["scale"]
    logits = logits.masked_fill(~seen, float("-inf"))
    top = logits.amax(-1, keepdim=True)
    p = torch.exp(logits - torch.where(top.isinf(), 0.0, top))
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v.masked_fill(~seen.transpose(-1, -2), 0.0)) / torch.where(total == 0, 1.0, total)
    return out.reshape(rows, s["heads"], hd).to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------ the library's calls
def _lib():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jepa.cpp_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from jepa_amd import _lib as lib
    return lib


def _shape(s, lib):
    if "shape" not in s:
        s["shape"] = lib.CacheShape(s.get("heads", s["kv_heads"]), s["kv_heads"], s["hd"], s["page"], s["n_pages"])
    return ctypes.byref(s["shape"])


def _rotary(s, lib):
    if "rotary" not in s:
        s["rotary"] = lib.RopeAxes.of(s["hd"], s["form"], s["widths"], s["theta"], s["scales"])
    return ctypes.byref(s["rotary"])


def _own_rope(s):
    lib = _lib()
    x = s["x"]
    out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    lib.check(lib.lib().jepa_amd_rope_rows(x.device.index, _rotary(s, lib), TYPES[s["type"]][1], x.data_ptr(), x.stride(0), s["n_rows"], s["heads"], s["pos"].data_ptr(),
                                           int(s["back"]), out.data_ptr(), out.stride(0), torch.cuda.current_stream().cuda_stream), "jepa_amd_rope_rows")
    return out


def _own_append(s):
    lib = _lib()
    L, kind, rows, dev = lib.lib(), TYPES[s["type"]][1], s["n_rows"], s["cache"].device
    width, stream = s["kv_heads"] * s["hd"], torch.cuda.current_stream().cuda_stream
    q = torch.empty(s["q"].shape, dtype=s["q"].dtype, device=dev)
    k, v = (torch.empty(rows, width, dtype=s["k"].dtype, device=dev) for _ in range(2))
    lib.check(L.jepa_amd_cache_append(dev.index, _shape(s, lib), _rotary(s, lib), s["cache"].data_ptr(), kind, s["q"].data_ptr(), s["q"].stride(0), s["k"].data_ptr(),
                                      s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0), rows, s["pos"].data_ptr(), s["slots"].data_ptr(), q.data_ptr(), q.stride(0),
                                      stream), "jepa_amd_cache_append")
    lib.check(L.jepa_amd_cache_read(dev.index, _shape(s, lib), s["cache"].data_ptr(), s["slots"].data_ptr(), rows, kind, k.data_ptr(), width, v.data_ptr(), width,
                                    stream), "jepa_amd_cache_read")
    return dict(q=q, k=k, v=v)


def _own_digest(s):
    lib = _lib()
    L, dev, stream, n = lib.lib(), s["cache"].device, torch.cuda.current_stream().cuda_stream, s["page_of"].numel()
    bounds = torch.empty(n, s["kv_heads"], 2, s["hd"], device=dev)
    lib.check(L.jepa_amd_cache_digest(dev.index, _shape(s, lib), s["cache"].data_ptr(), s["n_seq"], s["rows"], s["row_start"].data_ptr(), s["kv_len"].data_ptr(),
                                      s["table"].data_ptr(), s["width"], s["digest"].data_ptr(), stream), "jepa_amd_cache_digest")
    lib.check(L.jepa_amd_cache_digest_read(dev.index, _shape(s, lib), s["digest"].data_ptr(), s["page_of"].data_ptr(), n, bounds.data_ptr(), stream), "jepa_amd_cache_digest_read")
    return bounds


def _own_select(s):
    lib = _lib()
    L, dev = lib.lib(), s["q"].device
    shape = _shape(s, lib)
    if "work" not in s:
        s["work"] = torch.empty(L.jepa_amd_cache_select_work_bytes(shape, s["n_seq"], s["rows"], s["width"], s["take"]), dtype=torch.uint8, device=dev)
    out = torch.empty(s["rows"], s["kv_heads"], s["take"], dtype=torch.int32, device=dev)
    lib.check(L.jepa_amd_cache_select(dev.index, shape, s["digest"].data_ptr(), TYPES[s["type"]][1], s["q"].data_ptr(), s["heads"] * s["hd"], s["n_seq"], s["rows"],
                                      s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["width"], s["block"], s["first"], s["last"], s["take"],
                                      out.data_ptr(), s["work"].data_ptr(), s["work"].numel(), torch.cuda.current_stream().cuda_stream), "jepa_amd_cache_select")
    return out


def _own_attend(s):
    lib = _lib()
    L, dev, row = lib.lib(), s["q"].device, s["heads"] * s["hd"]
    shape = _shape(s, lib)
    if "work" not in s:
        s["work"] = torch.empty(L.jepa_amd_cache_selected_work_bytes(shape, s["rows"], s["take"]), dtype=torch.uint8, device=dev)
    out = torch.empty_like(s["q"])
    lib.check(L.jepa_amd_cache_attention_selected(dev.index, shape, s["cache"].data_ptr(), TYPES[s["type"]][1], s["q"].data_ptr(), row, s["n_seq"], s["rows"],
                                                  s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["width"], s["selected"].data_ptr(), s["take"],
                                                  s["scale"], s["block"], out.data_ptr(), row, s["work"].data_ptr(), s["work"].numel(),
                                                  torch.cuda.current_stream().cuda_stream), "jepa_amd_cache_attention_selected")
    return out


def run(state):
    if own:
        return {"rope": _own_rope, "append": _own_append, "digest": _own_digest, "select": _own_select, "attend": _own_attend}[state["op"]](state)
    return {"rope": _plain_rope, "append": _plain_append, "digest": _plain_digest, "select": _plain_select, "attend": _plain_attend}[state["op"]](state)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _value(cache, page, head, token, dims, hd, which):
    """Values of `dims` of tokens (page, token) of one head, straight from the layout: f64 [tokens][dims]."""
    strip = cache[page, head, token // 16]
    t, nb = (token % 16)[:, None], hd // 32
    if which == "k":
        e = dims % 8
        nibble = (e % 2) * 4 + e // 2
        byte = ((dims % 32 // 8 * 16 + t) * nb + dims // 32) * 4 + nibble // 2
        base = 16 * hd
    else:
        nibble = dims % 2 + 0 * t
        byte = 8 * hd + t * (hd // 2) + dims // 2
        base = 17 * hd
    code = strip.gather(1, byte).long() >> (4 * (nibble % 2)) & 15
    at = base + 2 * ((t // 4 * nb + dims // 32) * 4 + t % 4)
    bits = strip.gather(1, at).to(torch.int16) | (strip.gather(1, at + 1).to(torch.int16) << 8)
    return (code.double() - 8) * bits.view(torch.float16).double()


def _rotations(case, s):
    """Of every pair of a head: its elements, and the cosines and sines of both their angles [n_rows], in 64 bits."""
    pos, at, total = s["pos"].cpu().numpy().astype(np.float64), 0, sum(s["widths"])
    for a, w in enumerate(s["widths"]):
        p = pos[:, a] * s["scales"][a]
        for i in range(w // 2):
            e = {0: (at + 2 * i, at + 2 * i + 1), 1: (at + 2 * i, at + 2 * i + 1), 2: (at + i, at + w // 2 + i), 3: (at // 2 + i, (at + total) // 2 + i)}[case["form"]]
            f = [(x - at) % (w // 2) if case["form"] == 0 else i + at // 2 if case["form"] == 3 else i for x in e]
            yield e, [p * math.exp(-2.0 * g / (total if case["form"] == 3 else w) * math.log(case["theta"])) for g in f]
        at += w


def _turned(case, s, x, back, ty):
    """Rows rotated pair by pair, in 64 bits or as the definition rounds in 32."""
    x = x.astype(ty).reshape(case["n_rows"], -1, case["hd"])
    out = x.copy()
    for (a, b), (ta, tb) in _rotations(case, s):
        ca, sa, cb, sb = (f(t).astype(ty)[:, None] for t in (ta, tb) for f in (np.cos, np.sin))
        out[..., a], out[..., b] = (x[..., a] * ca + x[..., b] * sb, x[..., b] * cb - x[..., a] * sa) if back else (x[..., a] * ca - x[..., b] * sa, x[..., b] * cb + x[..., a] * sb)
    return out.reshape(case["n_rows"], -1)


def exact(case, seed):
    if case["op"] == "select":
        return None
    s = prepare(case, seed)
    hd, page = case["hd"], case["page"] if "page" in case else 0
    if case["op"] == "rope":
        return _turned(case, s, s["x"].float().cpu().numpy(), case["back"], np.float64)
    if case["op"] == "append":
        out = {"q": _turned(case, s, s["q"].float().cpu().numpy(), False, np.float64)}
        for name in ("k", "v"):
            # the format's own definition of the codes is in 32 bits, as the rotated key's is; the values they stand for are exact in 64
            x = s[name].float().cpu().numpy()
            x = _turned(case, s, x, False, np.float32) if name == "k" else x
            x = np.clip(x, np.float32(-F16_MAX), np.float32(F16_MAX)).reshape(-1, 32)
            m = x[np.arange(len(x)), np.abs(x).argmax(1)][:, None]
            d = (m / np.float32(-8)).astype(np.float32)
            with np.errstate(divide="ignore"):
                inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
            code = np.minimum(15, np.trunc((x * inv).astype(np.float32) + np.float32(8.5)))
            out[name] = ((code.astype(np.float64) - 8) * d.astype(np.float16).astype(np.float64)).reshape(case["n_rows"], -1)
        return out
    kvh, dims = case["kv_heads"], torch.arange(hd, device="cuda")
    if case["op"] == "digest":
        if len(s["page_of"]) * kvh > 40000:
            return None
        out = np.zeros((len(s["page_of"]), kvh, 2, hd))
        pages, tokens = s["page_of"].tolist(), s["tokens"].tolist()
        for h in range(kvh):
            t = torch.cat([torch.arange(n) for n in tokens]).cuda()
            k = _value(s["cache"], torch.tensor(pages).repeat_interleave(torch.tensor(tokens)).cuda(), h, t, dims, hd, "k").cpu().numpy()
            at = np.concatenate([[0], np.cumsum(tokens)[:-1]])
            out[:, h, 0], out[:, h, 1] = np.maximum.reduceat(k, at), np.minimum.reduceat(k, at)
        top = np.abs(out).max((2, 3), keepdims=True).astype(np.float32)
        # codes and scale are 32-bit by definition
        with np.errstate(divide="ignore", invalid="ignore"):
            codes = np.where(top >= TINY, np.rint(out.astype(np.float32) * (np.float32(127) / top)), 0)
        return codes.astype(np.float64) * (top / np.float32(127)).astype(np.float64)
    if s["rows"] * kvh > 20000:
        return None
    group, end, chosen = case["heads"] // kvh, _rows_seen(case), s["selected"].tolist()
    out = torch.zeros(s["rows"], case["heads"], hd, dtype=torch.float64, device="cuda")
    for r, (i, e) in enumerate(end):
        for h in range(kvh):
            pages = [p for p in chosen[r][h] if p >= 0]
            if not pages:
                continue
            pos = (torch.tensor(pages, device="cuda")[:, None] * page + torch.arange(page, device="cuda")).flatten()
            if pages[-1] * page + page > e:
                pos = pos[pos < e]
            phys = s["table"][i].long()[pos // page]
            k, v = (_value(s["cache"], phys, h, pos % page, dims, hd, w) for w in ("k", "v"))
            out[r, h * group:(h + 1) * group] = torch.softmax(s["q"][r, h * group:(h + 1) * group].double() @ k.T * s["scale"], -1) @ v
    return out
