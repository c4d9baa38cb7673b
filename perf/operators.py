"""The measured calls of the 4-bit paged key/value cache: the block tables and slot maps of a step, rows written into
the cache and read back, and attention over it.

`listed()` names the cases and `draw(rng)` gives others of the same ranges; `prepare(case, seed)` makes what a caller has
in hand, `run(state)` makes one pass: with `own` false in elementary torch operations, with `own` true through libjepa.so.
`work(case)` counts the bytes and operations that a pass cannot do without, `exact(case, seed)` computes it in 64 bits.

The cache is a byte tensor [n_pages][n_kv_head][page_size / 16][18 * head_dim]. A strip of 16 tokens of one head holds, with
NB = head_dim / 32 blocks of 32 values:
  K codes   [4 g][16 tokens][NB b][4 bytes]: dims 32 b + 8 g + (0, 2, 4, 6, 1, 3, 5, 7), from the low nibble up
  V codes   [16 tokens][head_dim / 2 bytes]: dims in order, from the low nibble up
  K scales  f16 [4 tokens / 4][NB][4 tokens % 4], then the V scales in the same order
A value is (code - 8) * scale, ggml's q4_0.
"""
import ctypes
import os
import random
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30)}
NIBBLES = [0, 2, 4, 6, 1, 3, 5, 7]      # element of a K word's nibble, from the low one up
F16_MAX = 65504.0


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one token for each of many running requests, some of which end: what a server does before every step
        dict(name="plan one token each", op="plan", n_seq=256, lo=100, hi=8000, new_lo=1, new_hi=1, ended=16, page=64, spare=1.5, ragged=1),
        # prompts of all lengths admitted at once, small pages, the pool too small for the last ones
        dict(name="plan prompts", op="plan", n_seq=48, lo=0, hi=0, new_lo=1, new_hi=8000, ended=0, page=16, spare=0.9, ragged=2),
        # the rows of one step of 64 requests
        dict(name="store 64 tokens f16", op="store", n_rows=64, kv_heads=8, hd=128, page=64, type="f16", ragged=3),
        # one frame of 258 tokens for each of 16 candidate rollouts, f32 rows as the library's projections write them
        dict(name="store frames f32", op="store", n_rows=4128, kv_heads=16, hd=64, page=32, type="f32", ragged=4),
        # a batch of prompts
        dict(name="store prompts bf16", op="store", n_rows=32768, kv_heads=8, hd=128, page=16, type="bf16", ragged=5),
        # one token of one request: latency alone
        dict(name="attend one token f16", op="attend", n_seq=1, lo=1000, hi=1000, new_lo=1, new_hi=1, heads=16, kv_heads=16, hd=64, page=16, type="f16", block=1, ragged=6),
        # one token for each of 64 requests of very different lengths, grouped heads
        dict(name="attend 64 requests f16", op="attend", n_seq=64, lo=200, hi=8000, new_lo=1, new_hi=1, heads=32, kv_heads=8, hd=128, page=64, type="f16", block=1, ragged=7),
        # two long documents, one token each
        dict(name="attend long context bf16", op="attend", n_seq=2, lo=90000, hi=131000, new_lo=1, new_hi=1, heads=64, kv_heads=8, hd=128, page=64, type="bf16", block=1, ragged=8),
        # a few drafted tokens of each request, an odd head width
        dict(name="attend 5 drafted tokens f16", op="attend", n_seq=24, lo=500, hi=6000, new_lo=5, new_hi=5, heads=40, kv_heads=8, hd=96, page=32, type="f16", block=1, ragged=9),
        # a frame of 258 tokens for each of 8 candidate rollouts over the frames before it, f32
        dict(name="attend frames f32", op="attend", n_seq=8, lo=1032, hi=2064, new_lo=258, new_hi=258, heads=16, kv_heads=16, hd=64, page=32, type="f32", block=258, ragged=10),
        # prompts from an empty cache, causal
        dict(name="attend prompts bf16", op="attend", n_seq=4, lo=0, hi=0, new_lo=700, new_hi=6000, heads=32, kv_heads=8, hd=128, page=64, type="bf16", block=1, ragged=11),
        # a piece of a long prompt after the pieces before it
        dict(name="attend prompt piece f16", op="attend", n_seq=1, lo=14000, hi=14000, new_lo=2000, new_hi=2000, heads=32, kv_heads=4, hd=128, page=128, type="f16", block=1, ragged=12),
    ]


def _log(rng, lo, hi):
    """A whole number of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    page, ragged, kind = rng.choice([16, 32, 64, 128, 256]), rng.randrange(1 << 30), rng.choice(list(TYPES))
    op = rng.choice(["plan", "store", "attend", "attend", "attend"])
    if op == "plan":
        n_seq = _log(rng, 1, 400)
        hi = _log(rng, 1, 8000)
        return dict(op=op, n_seq=n_seq, lo=0 if rng.random() < 0.3 else _log(rng, 1, hi), hi=hi, new_lo=0, new_hi=_log(rng, 1, max(1, 200000 // n_seq)),
                    ended=rng.choice([0, 3, 8]), page=page, spare=rng.choice([0.5, 1.0, 1.5]), ragged=ragged)
    hd, kv_heads = rng.choice([32, 64, 96, 128]), rng.choice([1, 2, 3, 4, 8, 16])
    if op == "store":
        return dict(op=op, n_rows=_log(rng, 1, 32768 * 8 // max(8, kv_heads)), kv_heads=kv_heads, hd=hd, page=page, type=kind, ragged=ragged)
    heads = kv_heads * rng.choice([1, 2, 3, 4, 5, 8])
    how = rng.choice(["token", "token", "few", "prompt", "frames"])
    if how == "token":
        new, n_seq = 1, _log(rng, 1, 100)
        hi = _log(rng, 1, min(100000, 1500000 // n_seq // kv_heads + 1000))
        block = 1
    elif how == "few":
        new, n_seq = rng.randrange(2, 17), _log(rng, 1, 40)
        hi = _log(rng, 1, min(20000, 400000 // n_seq // kv_heads + 500))
        block = 1
    elif how == "prompt":
        n_seq = _log(rng, 1, 8)
        new = _log(rng, 2, 4000 // n_seq + 200)
        hi = rng.choice([0, _log(rng, 1, 4000)])
        block = 1
    else:
        n_seq, new = _log(rng, 1, 16), _log(rng, 2, 300)
        hi = new * rng.randrange(0, 8)
        block = rng.choice([0, new])
    while True:
        case = dict(op=op, n_seq=n_seq, lo=hi if how == "frames" else hi - hi // 2, hi=hi, new_lo=max(1, new // 3) if how == "prompt" else new, new_hi=new,
                    heads=heads, kv_heads=kv_heads, hd=hd, page=page, type=kind, block=block, ragged=ragged)
        if work(case)["flops"] < 5e11:
            return case
        new, hi, block = -(-new // 2), hi // 2, min(block, -(-new // 2))      # no more work than the largest listed case has


def _lengths(case):
    """(tokens in the cache before, tokens that come) of each sequence; a negative number of tokens ends one."""
    rng = random.Random(case["ragged"])
    have = [rng.randint(case["lo"], case["hi"]) for _ in range(case["n_seq"])]
    new = [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["n_seq"])]
    if case.get("ended"):
        new = [-h if i % case["ended"] == case["ended"] - 1 else n for i, (h, n) in enumerate(zip(have, new))]
    return have, new


def _pages(n, page):
    return -(-n // page)


def work(case):
    if case["op"] == "plan":
        have, new = _lengths(case)
        keep = [max(0, h + n) for h, n in zip(have, new)]
        moved = sum(abs(_pages(k, case["page"]) - _pages(h, case["page"])) for h, k in zip(have, keep))
        rows = sum(max(0, n) for n in new)
        return {"bytes": 20 * case["n_seq"] + 8 * moved + 8 * rows, "flops": 0}
    cell = 2 * (case["hd"] // 2 + case["hd"] // 16)      # bytes of one token of one head in the cache
    size = torch.empty(0, dtype=TYPES[case["type"]][0]).element_size()
    if case["op"] == "store":
        cells = case["n_rows"] * case["kv_heads"]
        return {"bytes": cells * (4 * case["hd"] * size + 2 * cell) + 16 * case["n_rows"], "flops": 6 * cells * case["hd"]}
    have, new = _lengths(case)
    pairs = sum(sum(_visible(h + j, h + n, case["block"]) for j in range(n)) for h, n in zip(have, new))
    rows = sum(new)
    read = sum(h + n for h, n in zip(have, new))
    return {"bytes": read * case["kv_heads"] * cell + 2 * rows * case["heads"] * case["hd"] * size, "flops": 4 * case["hd"] * case["heads"] * pairs}


def _visible(pos, total, block):
    return total if block == 0 else min(total, (pos // block + 1) * block)


# ------------------------------------------------------------------------------------------------ the cache's format
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


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    host = random.Random(seed)
    page = case["page"]
    st = dict(case)
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    if case["op"] == "plan":
        have, new = _lengths(case)
        keep = [max(0, h + n) for h, n in zip(have, new)]
        used = [_pages(h, page) for h in have]
        want = sum(max(0, _pages(k, page) - u) for k, u in zip(keep, used))
        free = int(want * case["spare"])
        n_pages = sum(used) + free + 7
        order = torch.randperm(n_pages, generator=gen, device="cuda", dtype=torch.int32)
        head = host.randrange(n_pages)
        ring = order.roll(head)
        width = max([_pages(max(h, k), page) for h, k in zip(have, keep)] + [1])
        table = torch.full((case["n_seq"], width), -1, dtype=torch.int32, device="cuda")
        taken = order[free + 7:]        # the pages that the sequences hold; seven pages belong to nobody
        at = 0
        for i, u in enumerate(used):
            table[i, :u] = taken[at:at + u]
            at += u
        rows = sum(max(0, n) for n in new)
        st.update(n_pages=n_pages, width=width, rows=rows, len=ints(have), new=ints(new), table=table, ring=ring, free=ints([head, free]))
        return st
    dtype, hd, kvh = TYPES[case["type"]][0], case["hd"], case["kv_heads"]
    if case["op"] == "store":
        rows = case["n_rows"]
        n_pages = _pages(rows, page) * 2 + 1
        pages = torch.randperm(n_pages, generator=gen, device="cuda")[:_pages(rows, page)]
        slots = (pages[:, None] * page + torch.arange(page, device="cuda")).flatten()[:rows].contiguous()
        # q, k and v lie side by side in one row, as a fused projection leaves them, with four query heads to each of k and v
        qkv = _rows(gen, (rows, 6 * kvh * hd), dtype)
        st.update(n_pages=n_pages, slots=slots, k=qkv[:, 4 * kvh * hd:5 * kvh * hd], v=qkv[:, 5 * kvh * hd:], heads=4 * kvh,
                  cache=torch.zeros(n_pages, kvh, page // 16, 18 * hd, dtype=torch.uint8, device="cuda"))
        return st
    have, new = _lengths(case)
    total = [h + n for h, n in zip(have, new)]
    used = [_pages(t, page) for t in total]
    n_pages = sum(used) + 3
    order = torch.randperm(n_pages, generator=gen, device="cuda", dtype=torch.int32)
    table = torch.full((len(total), max(used)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = _rows(gen, (starts[-1], case["heads"], hd), dtype, 0.7)
    st.update(n_pages=n_pages, width=max(used), rows=starts[-1], longest=max(total), most=max(new), q=q, scale=hd ** -0.5, table=table,
              kv_len=ints(total), row_start=ints(starts), cache=_filled(gen, n_pages, kvh, page, hd))
    return st


# ------------------------------------------------------------------------------------------------ plain forms
def _plain_plan(s):
    page, n_pages, rows = s["page"], s["n_pages"], s["rows"]
    have, new, table, ring = s["len"].long(), s["new"].long(), s["table"], s["ring"]
    width = table.shape[1]
    keep = (have + new).clamp(min=0)
    come = new.clamp(min=0)
    end = come.cumsum(0)
    row_start = torch.cat([end.new_zeros(1), end]).clamp(max=rows)
    bad = (have < 0) | (have > width * page) | (keep > width * page) | ((end > rows) & (come > 0))
    held, kept = -(-have // page), -(-keep // page)
    need = torch.where(bad, 0, (kept - held).clamp(min=0))
    head, count = s["free"].long().unbind()
    refused = bad | ((need > 0) & (need.cumsum(0) > count))
    need = torch.where(refused, 0, need)
    give = torch.where(refused, 0, (held - kept).clamp(min=0))
    kv_len = torch.where(refused, have.clamp(0, width * page), keep)
    j = torch.arange(width, device=table.device)
    take = (j >= held[:, None]) & (j < (held + need)[:, None])
    drop = (j >= kept[:, None]) & (j < (kept + give)[:, None])
    first, back = need.cumsum(0) - need, give.cumsum(0) - give
    from_ring = ring[(head + first[:, None] + j - held[:, None]) % n_pages]
    to_ring = torch.where(drop, (head + count + back[:, None] + j - kept[:, None]) % n_pages, n_pages)
    ring_out = torch.cat([ring, ring.new_zeros(1)]).scatter(0, to_ring.flatten(), table.flatten())[:n_pages]
    table_out = torch.where(take, from_ring, torch.where(drop, -1, table))
    r = torch.arange(rows, device=table.device)
    i = torch.searchsorted(end, r, right=True).clamp(max=len(have) - 1)
    pos = kv_len[i] - come[i] + r - row_start[i]
    slot = torch.where(refused[i] | (r >= end[-1]), -1, table_out[i, (pos // page).clamp(0, width - 1)].long() * page + pos % page)
    free = torch.stack([(head + need.sum()) % n_pages, count - need.sum() + give.sum()])
    return dict(table=table_out, ring=ring_out, free=free.int(), kv_len=kv_len.int(), row_start=row_start.int(), slot=slot, refused=refused.int())


def _plain_store(s):
    hd, kvh, page, rows = s["hd"], s["kv_heads"], s["page"], s["n_rows"]
    page_of, strip, token = s["slots"] // page, s["slots"] % page // 16, s["slots"] % 16
    k, v = (x.float().reshape(rows, kvh, hd) for x in (s["k"], s["v"]))
    at = (page_of[:, None, None], torch.arange(kvh, device=k.device)[:, None], strip[:, None, None], _places(hd, k.device)[token][:, None])
    s["cache"][at] = _pack(k, v)
    k, v = _unpack(s["cache"][at], hd)
    return dict(k=k.reshape(rows, -1).to(s["k"].dtype), v=v.reshape(rows, -1).to(s["v"].dtype))


def _plain_attend(s):
    hd, kvh, page, block = s["hd"], s["kv_heads"], s["page"], s["block"]
    group, n, longest, most = s["heads"] // kvh, s["n_seq"], s["longest"], s["most"]
    device = s["q"].device
    strips = s["cache"][s["table"].long().clamp(min=0)].movedim(2, 1)                  # [n][kvh][pages][strips][bytes]
    k, v = (x.reshape(n, kvh, -1, hd)[:, :, :longest] for x in _unpack(strips[..., _places(hd, device)], hd))
    start, total = s["row_start"].long(), s["kv_len"].long()
    r = torch.arange(most, device=device)
    come = start[1:] - start[:-1]
    at = (start[:-1, None] + r).clamp(max=s["rows"] - 1)
    q = s["q"].float()[at].reshape(n, most, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(n, kvh, group * most, hd)
    pos = (total - come)[:, None] + r
    end = total[:, None].expand(-1, most) if block == 0 else torch.minimum(total[:, None], (pos // block + 1) * block)
    seen = torch.arange(longest, device=device) < end[..., None]                       # [n][most][longest]
    logits = (torch.matmul(q, k.transpose(-1, -2)) * s["scale"]).reshape(n, kvh, group, most, longest)
    logits = logits.masked_fill(~seen[:, None, None], float("-inf"))
    p = torch.exp(logits - logits.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(n, kvh, group * most, longest), v).reshape(n, kvh, group, most, hd)
    out = out.permute(0, 3, 1, 2, 4).reshape(n, most, kvh * group, hd)
    i = torch.searchsorted(start[1:], torch.arange(s["rows"], device=device), right=True)
    return out[i, torch.arange(s["rows"], device=device) - start[i]].to(s["q"].dtype)


# ------------------------------------------------------------------------------------------------ the library's calls
def _lib():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "jepa.cpp_amd", "python")
    if path not in sys.path:
        sys.path.insert(0, path)
    from jepa_amd import _lib as lib
    return lib


def _shape(s, lib):
    if "shape" not in s:
        heads = s.get("heads", 1)
        s["shape"] = lib.CacheShape(heads, s.get("kv_heads", heads), s.get("hd", 64), s["page"], s["n_pages"])
    return ctypes.byref(s["shape"])


def _own_plan(s):
    lib = _lib()
    n, rows, dev = s["n_seq"], s["rows"], s["table"].device
    # the call works in place: on copies, so that a pass can be made again
    both = torch.cat((s["table"].flatten(), s["ring"]))
    table, ring = both[:s["table"].numel()].view_as(s["table"]), both[s["table"].numel():]
    kv_len, row_start, free = (torch.empty(m, dtype=torch.int32, device=dev) for m in (n, n + 1, 2))
    slot, refused = torch.empty(rows, dtype=torch.int64, device=dev), torch.empty(n, dtype=torch.int32, device=dev)
    lib.check(lib.lib().jepa_amd_cache_plan(dev.index, _shape(s, lib), n, rows, s["len"].data_ptr(), s["new"].data_ptr(), table.data_ptr(), s["width"],
                                            ring.data_ptr(), s["free"].data_ptr(), free.data_ptr(), kv_len.data_ptr(), row_start.data_ptr(), slot.data_ptr(),
                                            refused.data_ptr(), torch.cuda.current_stream().cuda_stream), "jepa_amd_cache_plan")
    return dict(table=table, ring=ring, free=free, kv_len=kv_len, row_start=row_start, slot=slot, refused=refused)


def _own_store(s):
    lib = _lib()
    L, kind, rows, dev = lib.lib(), TYPES[s["type"]][1], s["n_rows"], s["cache"].device
    width, stream = s["kv_heads"] * s["hd"], torch.cuda.current_stream().cuda_stream
    k, v = (torch.empty(rows, width, dtype=s["k"].dtype, device=dev) for _ in range(2))
    lib.check(L.jepa_amd_cache_store(dev.index, _shape(s, lib), s["cache"].data_ptr(), kind, s["k"].data_ptr(), s["k"].stride(0), s["v"].data_ptr(), s["v"].stride(0),
                                     rows, s["slots"].data_ptr(), stream), "jepa_amd_cache_store")
    lib.check(L.jepa_amd_cache_read(dev.index, _shape(s, lib), s["cache"].data_ptr(), s["slots"].data_ptr(), rows, kind, k.data_ptr(), width, v.data_ptr(), width,
                                    stream), "jepa_amd_cache_read")
    return dict(k=k, v=v)


def _own_attend(s):
    lib = _lib()
    L, dev, row = lib.lib(), s["q"].device, s["heads"] * s["hd"]
    shape = _shape(s, lib)
    if "work" not in s:
        s["work"] = torch.empty(L.jepa_amd_cache_work_bytes(shape, s["n_seq"], s["rows"], s["width"]), dtype=torch.uint8, device=dev)
    out = torch.empty_like(s["q"])
    lib.check(L.jepa_amd_cache_attention(dev.index, shape, s["cache"].data_ptr(), TYPES[s["type"]][1], s["q"].data_ptr(), row, s["n_seq"], s["rows"],
                                         s["row_start"].data_ptr(), s["kv_len"].data_ptr(), s["table"].data_ptr(), s["width"], s["scale"], s["block"], out.data_ptr(), row,
                                         s["work"].data_ptr(), s["work"].numel(), torch.cuda.current_stream().cuda_stream), "jepa_amd_cache_attention")
    return out


def run(state):
    if own:
        return {"plan": _own_plan, "store": _own_store, "attend": _own_attend}[state["op"]](state)
    return {"plan": _plain_plan, "store": _plain_store, "attend": _plain_attend}[state["op"]](state)


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


def exact(case, seed):
    if case["op"] == "plan":
        return None
    s = prepare(case, seed)
    hd, kvh, page = case["hd"], case["kv_heads"], case["page"]
    if case["op"] == "store":
        out = {}
        for name in ("k", "v"):
            # the format's own definition of the codes is in 32 bits; the values they stand for are exact in 64
            x = np.clip(s[name].float().cpu().numpy(), np.float32(-F16_MAX), np.float32(F16_MAX)).reshape(-1, 32)
            m = x[np.arange(len(x)), np.abs(x).argmax(1)][:, None]
            d = (m / np.float32(-8)).astype(np.float32)
            with np.errstate(divide="ignore"):
                inv = np.where(d != 0, np.float32(1) / d, np.float32(0)).astype(np.float32)
            code = np.minimum(15, np.trunc((x * inv).astype(np.float32) + np.float32(8.5)))
            out[name] = ((code.astype(np.float64) - 8) * d.astype(np.float16).astype(np.float64)).reshape(s["n_rows"], kvh * hd)
        return out
    if work(case)["flops"] > 6e12:
        return None
    group, dims = case["heads"] // kvh, torch.arange(hd, device="cuda")
    out = torch.empty(s["rows"], case["heads"], hd, dtype=torch.float64, device="cuda")
    starts = s["row_start"].tolist()
    for i, total in enumerate(s["kv_len"].tolist()):
        a, b = starts[i], starts[i + 1]
        token = torch.arange(total, device="cuda")
        pages = s["table"][i].long()[token // page]
        pos = total - (b - a) + torch.arange(b - a, device="cuda")
        end = torch.full_like(pos, total) if case["block"] == 0 else ((pos // case["block"] + 1) * case["block"]).clamp(max=total)
        hidden = (token >= end[:, None]).repeat_interleave(group, 0)
        for h in range(kvh):
            k, v = (_value(s["cache"], pages, h, token % page, dims, hd, w) for w in ("k", "v"))
            q = s["q"][a:b, h * group:(h + 1) * group].double().reshape(-1, hd)
            logits = (q @ k.T * s["scale"]).masked_fill(hidden, float("-inf"))
            out[a:b, h * group:(h + 1) * group] = (torch.softmax(logits, -1) @ v).reshape(b - a, group, hd)
    return out
