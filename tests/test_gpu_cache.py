"""The 4-bit paged key/value cache on the GPU (no counterpart in the reference): the planner against a sequential model of
it, stored rows against ggml's q4_0 bit for bit, attention against the definition in 64 bits on the values that the
cache holds, and the calls together as a step-by-step program makes them, eager and captured.

Attention's tolerance, for one row and head with out = sum_j p_j v_j and A = sum_j p_j |v_j| (both in 64 bits):
  the output's own rounding      eps_T / 2 |out| (half a step of its type), and half its smallest step
  16-bit types, weights in f16   2^-11 A (half a step of f16, eps / 2, relative to each weight)
  the 32-bit arithmetic          every score is a sum of head_dim products of a query held to 2^-22 of its row's largest
                                 value and an exact key, times a scale: off by at most (head_dim / 8 + 8) 2^-22 S,
                                 S = max_j scale |q|max |k_j|_1; the weights follow by the factor e^x ~ 1 + x on both sides
                                 of the fraction (twice), and their own 2^-21 and the sums' sqrt(n) 2^-24 come on top.
  bf16 rows, keys and values     where many rows share them the cached values are rounded to f16, 2^-11 relative: a score is off by at
                                 most 2^-11 S1, S1 = max_j scale sum_n |q_n| |k_jn|, on both sides of the fraction, and the sum over
                                 V by 2^-11 A
  small weights                  a weight enters the product with V as p_j d_j in f16 (the scale d_j of its block of V, the value
                                 at most 8 d_j), moved by a power of two that brings the largest p_j max d to 2^6 or more: f16's
                                 smallest step, half of it 2^-25, is 2^-31 of that largest one. Divided by the sum of the p_j, which
                                 is no less than the largest p_j, and times a code of at most 8 that is an error of at most
                                 2^-31 * 2 max|v| (the power of two above max d is under 2 max d) for each of the n keys.
"""
import ctypes as C

import numpy as np
import pytest

from jepa_amd import gguf

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30)}


def shape(jlib, n_head=4, n_kv_head=2, hd=64, page=16, n_pages=8):
    return jlib.CacheShape(n_head, n_kv_head, hd, page, n_pages)


def ok(jlib, rc):
    assert rc == 0, jlib.error_text()


def ints(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


# ------------------------------------------------------------------------------------------------ plan
def model_plan(ln, new, table, ring, free, n_rows, page):
    """The documented step, sequence by sequence."""
    n_pages, width = len(ring), table.shape[1]
    table, ring = table.copy(), ring.copy()
    head, count = free
    kv, start, slot, refused = [], [0], [-1] * n_rows, []
    taken = [0] * len(ln)
    at, front, back, short = 0, 0, 0, False
    drops = []
    for i, (h, c) in enumerate(zip(ln, new)):
        keep, cap = max(0, h + c), width * page
        rows = max(0, c)
        end = at + rows
        bad = h < 0 or h > cap or keep > cap or (rows > 0 and end > n_rows)
        need = 0 if bad else max(0, -(-keep // page) - -(-h // page))
        if need and (short or front + need > count):
            bad = short = True
        if not bad:
            held = -(-h // page)
            for k in range(need):
                table[i, held + k] = ring[(head + front + k) % n_pages]
            front += need
            if c < 0:
                drops.append((i, -(-keep // page), held))
            if rows:
                pos = np.arange(keep - rows, keep)
                slot[at:end] = [int(table[i, p // page]) * page + p % page for p in pos]
        kv.append(min(max(h, 0), cap) if bad else keep)
        refused.append(int(bad))
        at = end
        start.append(min(at, n_rows))
    for i, a, b in drops:
        for j in range(a, b):
            ring[(head + count + back) % n_pages] = table[i, j]
            table[i, j] = -1
            back += 1
    return dict(table=table, ring=ring, free=[(head + front) % n_pages, count - front + back], kv_len=kv, row_start=start, slot=slot, refused=refused)


def run_plan(jlib, ln, new, table, ring, free, n_rows, page, alias=False):
    n = len(ln)
    d = dict(len=ints(ln), new=ints(new), table=ints(table), ring=ints(ring), free=ints(free))
    out = d["free"] if alias else ints([-9, -9])
    kv = d["len"] if alias else torch.full((max(n, 1),), -9, dtype=torch.int32, device="cuda")
    start = torch.full((n + 1,), -9, dtype=torch.int32, device="cuda")
    slot = torch.full((n_rows + 1,), -9, dtype=torch.int64, device="cuda")
    refused = torch.full((max(n, 1),), -9, dtype=torch.int32, device="cuda")
    s = shape(jlib, page=page, n_pages=len(ring))
    torch.cuda.synchronize()
    ok(jlib, jlib.lib().jepa_amd_cache_plan(0, C.byref(s), n, n_rows, d["len"].data_ptr(), d["new"].data_ptr(), d["table"].data_ptr(), table.shape[1],
                                            d["ring"].data_ptr(), d["free"].data_ptr(), out.data_ptr(), kv.data_ptr(), start.data_ptr(), slot.data_ptr(),
                                            refused.data_ptr(), None))
    torch.cuda.synchronize()
    assert slot[n_rows] == -9
    got = dict(table=d["table"], ring=d["ring"], free=out, kv_len=kv[:n], row_start=start, slot=slot[:n_rows], refused=refused[:n])
    return {k: v.cpu().numpy() for k, v in got.items()}


def pool(rng, lens, page, width, spare, extra=0):
    """Tables of sequences of these lengths, and the ring of the other pages."""
    used = [-(-max(0, h) // page) for h in lens]
    n_pages = sum(used) + spare + extra
    order = rng.permutation(max(n_pages, 1)).astype(np.int32)
    table = np.full((len(lens), width), -1, np.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    ring = np.full(len(order), -1, np.int32)
    head = int(rng.integers(len(order)))
    ring[(head + np.arange(spare)) % len(order)] = order[at:at + spare]
    return table, ring, [head, spare]


@pytest.mark.parametrize("alias", [False, True])
@pytest.mark.parametrize("n,hi,most,page,spare,slack", [
    (1, 0, 1, 16, 1, 0), (1, 5, 40, 16, 3, 0), (3, 100, 20, 32, 9, 7), (64, 300, 1, 64, 64, 0), (65, 50, 33, 16, 60, 0), (200, 40, 100, 16, 500, -300),
    (1025, 30, 3, 16, 300, 5), (4096, 20, 2, 256, 2000, 0), (7, 400, 9000, 256, 200, 0), (5, 0, 20000, 16, 4000, -1), (2, 17, 0, 16, 0, 4),
    (2500, 40, 9, 16, 1500, 0), (4096, 100, 40, 32, 5000, 9), (1, 0, 4, 16, 1, 0), (1, 15, 4097, 128, 40, 0), (300, 200, 4, 128, 100, -9),
])
def test_plan(jlib, n, hi, most, page, spare, slack, alias):
    rng = np.random.default_rng(n * 7 + page)
    ln = rng.integers(0, hi + 1, n)
    new = rng.integers(0, most + 1, n)
    drop = rng.random(n) < 0.25 if n > 1 else np.zeros(n, bool)
    new = np.where(drop, -rng.integers(0, hi + 3, n), new)
    width = max(1, int(-(-max(1, (ln + np.maximum(new, 0)).max()) // page)) - (1 if n > 60 else 0))
    ln = np.minimum(ln, width * page)
    table, ring, free = pool(rng, ln, page, width, spare, 3)
    n_rows = max(0, int(np.maximum(new, 0).sum()) + slack)
    want = model_plan(ln.tolist(), new.tolist(), table, ring, free, n_rows, page)
    got = run_plan(jlib, ln, new, table, ring, free, n_rows, page, alias)
    for k in want:
        np.testing.assert_array_equal(got[k], np.asarray(want[k]), err_msg=k)


def test_plan_refusals_and_strange_lengths(jlib):
    """Negative lengths, lengths past the table, the largest ints, rows past n_rows and a ring that is none: refused, and
    the other sequences served."""
    page, width = 16, 4
    ln = [-1, 65, 64, 10, 2147483647, 0, 16, 0, 3]
    new = [5, 0, -2147483648, 3, 2147483647, 2147483647, 16, 1, 0]
    rng = np.random.default_rng(0)
    table, ring, free = pool(rng, [0, 0, 64, 10, 0, 0, 16, 0, 3], page, width, 6, 1)
    for n_rows in (0, 8, 9, 40):
        want = model_plan(ln, new, table, ring, free, n_rows, page)
        got = run_plan(jlib, ln, new, table, ring, free, n_rows, page)
        for k in want:
            np.testing.assert_array_equal(got[k], np.asarray(want[k]), err_msg=k)
    for free in ([-1, 3], [len(ring), 3], [0, len(ring) + 1], [0, -1]):
        got = run_plan(jlib, [0, 0], [1, 0], table[:2], ring, free, 1, page)
        assert got["refused"].tolist() == [1, 0] and got["free"].tolist() == [0, 0] and got["slot"].tolist() == [-1]
    got = run_plan(jlib, [], [], table[:0], ring, [2, 3], 5, page)      # no sequence: no row has a slot
    assert got["row_start"].tolist() == [0] and got["free"].tolist() == [2, 3] and got["slot"].tolist() == [-1] * 5
    bad = ring.copy()
    bad[:] = len(ring) + 5                                               # page numbers that the cache does not have
    got = run_plan(jlib, [0], [20], np.full((1, 4), -1, np.int32), bad, [0, 2], 20, page)
    assert got["slot"].tolist() == [-1] * 20 and got["kv_len"].tolist() == [20]


# ------------------------------------------------------------------------------------------------ store and read
def q4_0(x):
    """ggml's q4_0 values of f32 rows, from the block format."""
    if not x.size:
        return x
    raw = gguf.quantize(gguf.GGML_Q4_0, x).reshape(-1, 18)
    d = raw[:, :2].copy().view(np.float16).astype(np.float32)
    codes = np.concatenate([raw[:, 2:] & 15, raw[:, 2:] >> 4], 1).astype(np.float32)
    return ((codes - 8) * d).reshape(x.shape)


class Pool:
    """A cache with rows stored in it."""

    def __init__(self, jlib, n_head, n_kv_head, hd, page, n_pages, fill=0xff):
        self.jlib, self.s = jlib, shape(jlib, n_head, n_kv_head, hd, page, n_pages)
        self.page_bytes = jlib.lib().jepa_amd_cache_page_bytes(C.byref(self.s))
        self.cache = torch.full((n_pages * self.page_bytes,), fill, dtype=torch.uint8, device="cuda")      # 0xff: every scale NaN
        self.width = n_kv_head * hd

    def store(self, k, v, slot, kind, stream=None):
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_store(0, C.byref(self.s), self.cache.data_ptr(), TYPES[kind][1], k.data_ptr(), k.stride(0), v.data_ptr(),
                                                           v.stride(0), k.shape[0], slot.data_ptr(), stream))

    def read(self, slot, kind="f32", stream=None):
        k, v = (torch.full((slot.numel(), self.width), float("nan"), dtype=TYPES[kind][0], device="cuda") for _ in range(2))
        torch.cuda.synchronize()
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_read(0, C.byref(self.s), self.cache.data_ptr(), slot.data_ptr(), slot.numel(), TYPES[kind][1], k.data_ptr(),
                                                          k.stride(0), v.data_ptr(), v.stride(0), stream))
        return k, v

    def attend(self, q, start, kv_len, table, kind, block=1, scale=None, out=None, stream=None, work=None):
        L, n, rows = self.jlib.lib(), kv_len.numel(), q.shape[0]
        need = L.jepa_amd_cache_work_bytes(C.byref(self.s), n, rows, table.shape[1])
        work = torch.full((need,), 0xff, dtype=torch.uint8, device="cuda") if work is None else work
        out = torch.full((rows, q.shape[1]), float("nan"), dtype=q.dtype, device="cuda") if out is None else out
        if stream is None:
            torch.cuda.synchronize()
        ok(self.jlib, L.jepa_amd_cache_attention(0, C.byref(self.s), self.cache.data_ptr(), TYPES[kind][1], q.data_ptr(), q.stride(0), n, rows, start.data_ptr(),
                                                 kv_len.data_ptr(), table.data_ptr(), table.shape[1], self.s.head_dim ** -0.5 if scale is None else scale, block,
                                                 out.data_ptr(), out.stride(0), work.data_ptr(), need, stream))
        return out


def special_rows(rng, n, width):
    x = rng.standard_normal((n, width)).astype(np.float32)
    x[0] = 0.0
    if n > 6:
        x[1] = 1e-30                                     # a scale that f16 does not hold
        x[2, 0::2], x[2, 1::2] = 3.0, -3.0               # equal magnitudes: the first one's sign decides
        x[3] = np.round(x[3] * 4) / 4
        x[4, 5] = 1000.0
        x[5] = 2.0 ** -24                                # the smallest f16
        x[6, 0::2], x[6, 1::2] = -0.5, 0.5
    return x


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("hd,kvh,page", [(32, 1, 16), (32, 5, 64), (64, 2, 32), (96, 3, 16), (96, 1, 256), (128, 8, 64), (128, 1, 128), (64, 16, 16)])
def test_store_is_q4_0_bit_for_bit(jlib, hd, kvh, page, kind):
    rng = np.random.default_rng(hd + kvh)
    n, n_pages = 77, 9 + 77 // page * 2
    dtype = TYPES[kind][0]
    rows = [torch.from_numpy(special_rows(rng, n, kvh * hd)).to(dtype).cuda() for _ in range(2)]
    wide = torch.zeros(n, 4 * kvh * hd, dtype=dtype, device="cuda")      # rows inside wider ones, in another order
    wide[:, 2 * kvh * hd:3 * kvh * hd], wide[:, kvh * hd:2 * kvh * hd] = rows
    p = Pool(jlib, kvh, kvh, hd, page, n_pages)
    where = rng.permutation(n_pages * page)[:n]
    slot = ints(where, torch.int64)
    slot[[9, 30]] = torch.tensor([-1, n_pages * page], device="cuda")   # none, and one past the cache
    torch.cuda.synchronize()
    p.store(wide[:, 2 * kvh * hd:3 * kvh * hd], wide[:, kvh * hd:2 * kvh * hd], slot, kind)
    for name, got, x in zip("kv", p.read(slot), rows):
        want = q4_0(x.float().cpu().numpy())
        want[[9, 30]] = 0
        np.testing.assert_array_equal(got.cpu().numpy(), want, err_msg=name)
    for other in ("f16", "bf16"):
        for got, exact in zip(p.read(slot, other), p.read(slot)):
            assert torch.equal(got, exact.to(got.dtype))
    # every other slot is as it was: all bytes 0xff, so NaN
    rest = ints(np.setdiff1d(np.arange(n_pages * page), np.delete(where, [9, 30])), torch.int64)
    for x in p.read(rest):
        assert torch.isnan(x).all()


def test_store_outside_f16_and_not_finite(jlib):
    p = Pool(jlib, 2, 2, 64, 16, 2)
    k, v = torch.ones(6, 128, device="cuda"), torch.full((6, 128), 2.0, device="cuda")
    k[0, 3], v[1, 70] = 1e9, -3e38          # held at the ends
    k[2, 5], k[3, 64], v[4, 127] = float("nan"), float("inf"), float("-inf")
    slot = ints(np.arange(6) + 9, torch.int64)
    torch.cuda.synchronize()
    p.store(k, v, slot, "f32")
    gk, gv = (x.cpu().numpy() for x in p.read(slot))
    ck, cv = (x.clamp(-65504, 65504).cpu().numpy() for x in (k, v))
    for r, head in ((0, None), (1, None), (2, 0), (3, 1), (4, 1), (5, None)):
        for h in range(2):
            at = slice(64 * h, 64 * h + 64)
            if h == head:
                assert np.isnan(gk[r, at]).all() and (gv[r, at] == 0).all()
            else:
                np.testing.assert_array_equal(gk[r, at], q4_0(ck[r:r + 1, at])[0])
                np.testing.assert_array_equal(gv[r, at], q4_0(cv[r:r + 1, at])[0])


def test_no_rows(jlib):
    p = Pool(jlib, 2, 2, 64, 16, 2)
    e = torch.empty(0, 128, device="cuda")
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    p.store(e, e, none, "f32")
    p.read(none)
    p.attend(e, ints([0]), torch.empty(0, dtype=torch.int32, device="cuda"), ints(np.zeros((0, 1))), "f32")
    torch.cuda.synchronize()
    assert (p.cache == 0xff).all()


# ------------------------------------------------------------------------------------------------ attention
def reference(p, q, start, total, table, block, scale, kind):
    """(out, tolerance) in 64 bits from the values that the cache holds; NaN where the definition says so, and 0 where a row
    reads nothing."""
    s = p.s
    hd, kvh, group, page = s.head_dim, s.n_kv_head, s.n_head // s.n_kv_head, s.page_size
    out = torch.full((q.shape[0], s.n_head, hd), float("nan"), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    eps = torch.finfo(TYPES[kind][0]).eps / 2
    tiny = 2.0 ** -25 if kind == "f16" else 1e-38
    for i, n in enumerate(total):
        a, b = start[i], start[i + 1]
        if a == b:
            continue
        t = torch.arange(n, device="cuda")
        pages = torch.as_tensor(table[i], device="cuda").long()[t // page]
        there = (pages >= 0) & (pages < s.n_pages)
        slot = torch.where(there, pages * page + t % page, -1)
        k, v = (x.double().reshape(n, kvh, hd) for x in p.read(slot)) if n else (torch.zeros(0, kvh, hd, dtype=torch.float64, device="cuda"),) * 2
        pos = n - (b - a) + torch.arange(b - a, device="cuda")
        end = torch.full_like(pos, n) if block == 0 else torch.where(pos < 0, 0, ((pos // block + 1) * block).clamp(max=n))
        hidden = (t >= end[:, None]) | ~there
        for h in range(s.n_head):
            x = q[a:b, h * hd:(h + 1) * hd].double()
            z = x @ torch.nan_to_num(k[:, h // group]).T * scale
            z = torch.where(torch.isnan(k[:, h // group, 0]), float("nan"), z).masked_fill(hidden, float("-inf"))
            top = z.amax(-1, keepdim=True) if n else torch.zeros(b - a, 1, device="cuda")
            w = torch.where(hidden, 0.0, torch.exp(z - torch.where(torch.isneginf(top), 0.0, top)))
            l = w.sum(-1, keepdim=True)
            w = torch.where(l == 0, 0.0, w / l)
            y = w @ v[:, h // group]
            A = w @ v[:, h // group].abs()
            k1 = torch.nan_to_num(k[:, h // group]).abs().sum(-1)
            S = abs(scale) * x.abs().amax(-1, keepdim=True) * (k1.max() if n else 0.0)
            low = 0.0
            if kind == "bf16" and n:
                low = 2.0 ** -11 * (1 + 2 * abs(scale) * (x.abs() @ torch.nan_to_num(k[:, h // group]).abs().T).amax(-1, keepdim=True))
            f32 = low + 2 * (hd / 8 + 8) * 2.0 ** -22 * S + 2.0 ** -20 + (n ** 0.5) * 2.0 ** -24
            out[a:b, h] = y
            tol[a:b, h] = eps * y.abs() + tiny + n * 2.0 ** -30 * (v[:, h // group].abs().max() if n else 0.0) + (f32 + (2.0 ** -11 if kind != "f32" else 0.0)) * A * (1 + eps)
    return out.reshape(q.shape), tol.reshape(q.shape)


def filled(jlib, rng, heads, kvh, hd, page, lens, kind="f32", k_scale=1.0, v_scale=1.0, extra=2):
    """A cache with sequences of these lengths in shuffled pages; what no token holds is NaN."""
    used = [-(-n // page) for n in lens]
    n_pages = sum(used) + extra
    p = Pool(jlib, heads, kvh, hd, page, n_pages)
    order = rng.permutation(n_pages)
    table = np.full((len(lens), max(used + [1]) + 1), -1, np.int32)
    at = 0
    for i, u in enumerate(used):
        table[i, :u] = order[at:at + u]
        at += u
    slot = [int(table[i, t // page]) * page + t % page for i, n in enumerate(lens) for t in range(n)]
    gen = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    k, v = (torch.randn(len(slot), kvh * hd, generator=gen, device="cuda") * m for m in (k_scale, v_scale))
    if slot:
        s = ints(slot, torch.int64)
        torch.cuda.synchronize()
        p.store(k.to(TYPES[kind][0]), v.to(TYPES[kind][0]), s, kind)
        torch.cuda.synchronize()
    return p, table


def check(p, q, start, lens, table, kind, block=1, scale=None, rows=None):
    scale = p.s.head_dim ** -0.5 if scale is None else scale
    got = p.attend(q, ints(start), ints(lens), ints(table), kind, block, scale)
    torch.cuda.synchronize()
    want, tol = reference(p, q, start, lens, table, block, scale, kind)
    last = start[-1]
    assert torch.isnan(got[last:]).all()      # rows behind the last sequence: left as they were
    got, want, tol = got[:last].double(), want[:last], tol[:last]
    assert torch.equal(torch.isnan(got), torch.isnan(want)), "NaN in other places"
    off = torch.nan_to_num((got - want).abs() - tol, nan=0.0)
    assert (off <= 0).all(), f"off by {((got - want).abs() / tol).nan_to_num().max().item():.3g} of the tolerance at {torch.argmax(off).item()}"
    return got


def queries(rng, n, width, kind, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(int(rng.integers(1 << 30)))
    return (torch.randn(n, width, generator=gen, device="cuda") * scale).to(TYPES[kind][0])


LENGTHS = [0, 1, 2, 15, 16, 17, 31, 33, 63, 64, 65, 127, 129, 255, 256, 257, 300, 511, 513, 1000]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("hd,kvh,group,page", [(32, 2, 1, 16), (64, 1, 4, 64), (64, 16, 1, 32), (96, 2, 5, 16), (128, 2, 8, 64), (128, 1, 32, 256), (32, 1, 17, 128),
                                               (128, 3, 3, 32), (96, 1, 1, 64)])
def test_attention_one_token(jlib, hd, kvh, group, page, kind):
    """One row for each of sequences of every length around the tiles' sizes, none and one token among them."""
    rng = np.random.default_rng(hd + group)
    p, table = filled(jlib, rng, kvh * group, kvh, hd, page, LENGTHS)
    n = len(LENGTHS)
    q = queries(rng, n + 3, kvh * group * hd, kind)
    check(p, q, list(range(n + 1)), LENGTHS, table, kind)


@pytest.mark.parametrize("block", [0, 1, 2, 7, 64, 100000])
@pytest.mark.parametrize("kind,hd,kvh,group,page", [("f16", 64, 2, 2, 16), ("f32", 128, 1, 3, 64), ("bf16", 96, 2, 1, 32), ("f32", 32, 3, 1, 16), ("f16", 128, 2, 4, 64)])
def test_attention_ragged_rows(jlib, kind, hd, kvh, group, page, block):
    """Sequences with none to many new rows each, more rows than cached tokens among them (they read nothing), every mask."""
    rng = np.random.default_rng(hd * 3 + block % 100)
    lens = [5, 0, 40, 40, 333, 64, 1, 130, 700]
    rows = [5, 3, 0, 40, 17, 1, 4, 129, 66]
    start = [0] + np.cumsum(rows).tolist()
    p, table = filled(jlib, rng, kvh * group, kvh, hd, page, lens)
    q = queries(rng, start[-1] + 2, kvh * group * hd, kind)
    check(p, q, start, lens, table, kind, block)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,length,kvh,group,hd", [(300, 300, 2, 4, 64), (513, 900, 1, 8, 128), (258, 1032, 4, 1, 64), (64, 64, 1, 1, 32), (1000, 1000, 1, 3, 96),
                                                        (200, 5000, 2, 4, 128), (130, 3000, 1, 8, 96), (300, 2500, 2, 1, 32), (257, 1900, 3, 2, 64)])
def test_attention_prompt(jlib, kind, rows, length, kvh, group, hd):
    rng = np.random.default_rng(rows)
    lens, start = [length, 20], [0, rows, rows + 20]
    p, table = filled(jlib, rng, kvh * group, kvh, hd, 32, lens)
    q = queries(rng, start[-1], kvh * group * hd, kind)
    check(p, q, start, lens, table, kind, 1)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows,length,kvh,group,hd,block", [(800, 5000, 1, 1, 64, 1), (790, 3100, 2, 1, 96, 0), (400, 7000, 1, 2, 32, 1), (270, 9000, 1, 3, 128, 90)])
def test_attention_prompt_in_pieces(jlib, kind, rows, length, kvh, group, hd, block):
    """Few tiles of a prompt's columns over many keys: its pieces are joined."""
    rng = np.random.default_rng(24)
    p, table = filled(jlib, rng, kvh * group, kvh, hd, 64, [length, 70])
    start = [0, rows, rows + 1]
    check(p, queries(rng, rows + 1, kvh * group * hd, kind), start, [length, 70], table, kind, block)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("kvh,group", [(16, 4), (4, 16)])
def test_attention_many_short_prompts(jlib, kind, kvh, group):
    """Sequences of few columns each that fill the chip together, some of one row or none."""
    rng = np.random.default_rng(25)
    lens = rng.integers(1, 260, 70).tolist()
    rows = [min(n, int(r)) for n, r in zip(lens, rng.integers(0, 30, 70))]
    start = [0] + np.cumsum(rows).tolist()
    p, table = filled(jlib, rng, kvh * group, kvh, 32, 32, lens)
    check(p, queries(rng, start[-1], kvh * group * 32, kind), start, lens, table, kind, 1)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_long(jlib, kind):
    """Long sequences beside short ones: the keys of one row are split over many workgroups and joined."""
    rng = np.random.default_rng(3)
    lens = [20011, 3, 0, 7000]
    p, table = filled(jlib, rng, 8, 2, 128, 64, lens)
    q = queries(rng, 9, 8 * 128, kind)
    check(p, q, [0, 2, 4, 5, 9], lens, table, kind)
    check(p, q, [0, 0, 0, 0, 1], lens, table, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("q_scale,k_scale,v_scale", [(30.0, 3.0, 1.0), (1e-4, 1e-3, 1e-4), (1.0, 1.0, 2e-5), (0.05, 300.0, 6000.0), (1e3, 1e-3, 1.0), (0.0, 1.0, 1.0)])
def test_attention_magnitudes(jlib, kind, q_scale, k_scale, v_scale):
    """Peaked and flat softmaxes, tiny and large values: the error is relative to what is summed."""
    rng = np.random.default_rng(5)
    lens = [500, 70]
    p, table = filled(jlib, rng, 4, 2, 64, 16, lens, k_scale=k_scale, v_scale=v_scale)
    q = queries(rng, 40, 4 * 64, kind, q_scale)
    check(p, q, [0, 30, 40], lens, table, kind)


@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_mixed_magnitudes_of_v(jlib, kind):
    """Values that grow and shrink by large factors along the sequence, and a jump of the scores late in it."""
    rng = np.random.default_rng(6)
    n = 1500
    p, table = filled(jlib, rng, 2, 1, 64, 16, [n])
    slot = ints([int(table[0, t // 16]) * 16 + t % 16 for t in range(n)], torch.int64)
    k, v = p.read(slot)
    grow = torch.exp(torch.linspace(-9, 9, n, device="cuda"))[:, None]
    k[n - 200] *= 40
    for f in (grow, grow.flip(0)):
        torch.cuda.synchronize()
        p.store(k, v * f, slot, "f32")
        q = queries(rng, 20, 128, kind, 0.5)
        check(p, q, [0, 20], [n], table, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("group", [1, 9])
def test_attention_not_finite(jlib, kind, group):
    """NaN and infinity in cached rows reach the rows and heads that read them and no others; in a query, its row alone."""
    rng = np.random.default_rng(7)
    n, rows = 200, 150
    p, table = filled(jlib, rng, 2 * group, 2, 64, 16, [n])
    slot = ints([int(table[0, t // 16]) * 16 + t % 16 for t in range(n)], torch.int64)
    k, v = p.read(slot)
    k[130, 3], v[171, 64 + 40] = float("nan"), float("inf")
    torch.cuda.synchronize()
    p.store(k, v, slot, "f32")
    q = queries(rng, rows, 2 * group * 64, kind)
    q[20, 5] = float("nan")
    got = check(p, q, [0, rows], [n], table, kind).reshape(rows, 2 * group, 64)
    bad = torch.isnan(got).all(-1)
    assert bad[80:, :group].all() and not bad[:20].any() and bad[20, 0] and bad[121:, group:].all() and not bad[21:80].any() and not bad[:121, group:].any()
    q[20, 5], q[40, 64] = float("inf"), float("-inf")
    got = p.attend(q, ints([0, rows]), ints([n]), ints(table), kind).reshape(rows, 2 * group, 64)
    torch.cuda.synchronize()
    assert torch.isnan(got[20, 0]).all() and torch.isnan(got[40, 1]).all() and not torch.isnan(got[:20]).any()


def test_attention_pages_that_are_none(jlib):
    """Table entries outside the cache hide their tokens; a sequence of such pages alone reads nothing."""
    rng = np.random.default_rng(8)
    lens = [100, 33, 300]
    for kind, kvh in (("f32", 1), ("f16", 2)):
        p, table = filled(jlib, rng, 4, kvh, 64, 16, lens)
        table[0, 2], table[0, 6], table[1, :] = -1, p.s.n_pages, -7
        table[2, [0, 1, 2, 3, 9]] = [2147483647, -2147483648, -1, p.s.n_pages, -1]
        rows = [3, 2, 40]
        start = [0] + np.cumsum(rows).tolist()
        got = check(p, queries(rng, start[-1], 256, kind), start, lens, table, kind)
        assert (got[3:5] == 0).all()


def test_attention_lengths_past_the_table(jlib):
    """kv_len above what a table row holds is taken as that; a negative one as none. row_start behind n_rows is cut off there."""
    rng = np.random.default_rng(9)
    p, table = filled(jlib, rng, 2, 2, 32, 16, [48, 48, 48])
    table = table[:, :3].copy()
    q = queries(rng, 5, 64, "f16")
    got = p.attend(q, ints([0, 2, 4, 9]), ints([1000, -5, 48]), ints(table), "f16", 0)
    want, tol = reference(p, q, [0, 2, 4, 5], [48, 0, 48], table, 0, 32 ** -0.5, "f16")
    assert ((got.double() - want).abs() <= tol).all()


def test_attention_strides_and_neighbours(jlib):
    """Query and output rows inside wider ones: nothing beside them is written."""
    rng = np.random.default_rng(10)
    lens, rows = [90, 700], 140
    for kind in TYPES:
        p, table = filled(jlib, rng, 4, 2, 64, 32, lens)
        wide = queries(rng, rows, 600 * 2, kind)
        q = wide[:, 8:8 + 256]
        out = torch.full((rows, 1024), 7.0, dtype=TYPES[kind][0], device="cuda")
        start = [0, 90, 140]
        p.attend(q, ints(start), ints(lens), ints(table), kind, 1, out=out[:, 512:768])
        torch.cuda.synchronize()
        want, tol = reference(p, q.contiguous(), start, lens, table, 1, 0.125, kind)
        assert ((out[:, 512:768].double() - want).abs() <= tol).all()
        assert (out[:, :512] == 7).all() and (out[:, 768:] == 7).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("rows", [1, 40])
def test_attention_many_sequences_and_a_long_one(jlib, kind, rows):
    """More sequences than a wave has lanes, some split into pieces."""
    rng = np.random.default_rng(14)
    lens = rng.integers(1, 200, 70).tolist()
    lens[3], lens[66], lens[69] = 9000, 2100, 700
    p, table = filled(jlib, rng, 8, 1, 64, 64, lens)
    n = [0 if i % 9 == 5 else min(rows, lens[i]) for i in range(70)]
    start = [0] + np.cumsum(n).tolist()
    check(p, queries(rng, start[-1] + 1, 512, kind), start, lens, table, kind)


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("scale", [0.0, -0.125, 1.0, 1e-30])
def test_attention_scales(jlib, kind, scale):
    rng = np.random.default_rng(15)
    lens, start = [300, 40], [0, 90, 130]
    p, table = filled(jlib, rng, 4, 1, 64, 16, lens, k_scale=0.3)
    q = queries(rng, 130, 256, kind)
    check(p, q, start, lens, table, kind, 1, scale)
    check(p, q, [0, 2, 5], lens, table, kind, 7, scale)


def test_attention_row_starts_that_overlap(jlib):
    """row_start that runs backwards: sequences claim the same rows. Which one a row comes from is not said, but every row is written by
    one of them or left, and nothing beside the rows is touched."""
    rng = np.random.default_rng(16)
    lens = [3000, 2900, 2800, 2700]
    p, table = filled(jlib, rng, 4, 2, 64, 64, lens)
    for kind in TYPES:
        out = torch.full((40, 256), 7.0, dtype=TYPES[kind][0], device="cuda")
        for start in ([0, 12, 3, 12, 2], [12, 0, 12, 0, 12], [-5, 40, -40, 12, 12], [2147483647, -2147483648, 12, 1, 9]):
            p.attend(queries(rng, 12, 256, kind), ints(start), ints(lens), ints(table), kind, 1, out=out[:12])
            torch.cuda.synchronize()
            assert (out[12:] == 7).all() and not torch.isnan(out).any()


@pytest.mark.parametrize("n_seq,kind", [(8, "f16"), (8, "f32"), (70, "f16"), (70, "bf16")])
def test_row_starts_that_overlap_leave_the_work_space_usable(jlib, n_seq, kind):
    """Overlapping rows ask for more pieces than the call launches; the next call in the same work space comes out as in a new one."""
    rng = np.random.default_rng(23)
    lens = rng.integers(1500, 2500, n_seq).tolist()
    p, table = filled(jlib, rng, 2, 1, 64, 64, lens)
    rows = 2 * n_seq
    q = queries(rng, rows, 128, kind)
    work = torch.zeros(jlib.lib().jepa_amd_cache_work_bytes(C.byref(p.s), n_seq, rows, table.shape[1]), dtype=torch.uint8, device="cuda")
    start = list(range(0, rows + 1, 2))
    want = check(p, q, start, lens, table, kind)
    out = torch.empty_like(q)
    for bad in ([rows * (i % 2) for i in range(n_seq + 1)], [max(rows - 3 * i, 0) if i % 2 else 0 for i in range(n_seq + 1)]):
        p.attend(q, ints(bad), ints(lens), ints(table), kind, 1, out=out, work=work)
        torch.cuda.synchronize()
        out.fill_(float("nan"))
        p.attend(q, ints(start), ints(lens), ints(table), kind, 1, out=out, work=work)
        torch.cuda.synchronize()
        assert torch.equal(out.double(), want)


def test_attention_many_sequences(jlib):
    rng = np.random.default_rng(11)
    lens = rng.integers(0, 60, 1500).tolist()
    rows = rng.integers(0, 3, 1500)
    start = [0] + np.cumsum(rows).tolist()
    p, table = filled(jlib, rng, 2, 1, 32, 16, lens)
    q = queries(rng, start[-1], 64, "bf16")
    check(p, q, start, lens, table, "bf16", 1)


def test_offsets_past_32_bits(jlib):
    """A cache of 5 GiB whose last pages are used: byte offsets past 2^32."""
    hd, kvh, page = 128, 8, 256
    n_pages = 5 * 2 ** 30 // (kvh * page // 16 * 18 * hd)
    p = Pool(jlib, 16, kvh, hd, page, n_pages)
    rng = np.random.default_rng(12)
    n = 700
    table = np.array([[n_pages - 1, 3, n_pages - 2]], np.int32)
    slot = ints([int(table[0, t // page]) * page + t % page for t in range(n)], torch.int64)
    k, v = (queries(rng, n, kvh * hd, "f16") for _ in range(2))
    torch.cuda.synchronize()
    p.store(k, v, slot, "f16")
    for got, x in zip(p.read(slot), (k, v)):
        np.testing.assert_array_equal(got.cpu().numpy(), q4_0(x.float().cpu().numpy()))
    check(p, queries(rng, 3, 16 * hd, "f16"), [0, 3], [n], table, "f16")


def test_same_pages_in_two_sequences(jlib):
    """A prefix that sequences share is read by each; equal rows give equal bits, and so do repeated calls."""
    rng = np.random.default_rng(13)
    p, table = filled(jlib, rng, 8, 2, 64, 16, [4000])
    table = np.repeat(table, 3, 0)
    one = queries(rng, 1, 512, "f32")
    q = one.expand(3, -1).contiguous()
    a = check(p, q, [0, 1, 2, 3], [4000] * 3, table, "f32")
    assert torch.equal(a[0], a[1]) and torch.equal(a[0], a[2])
    for _ in range(3):
        assert torch.equal(a, check(p, q, [0, 1, 2, 3], [4000] * 3, table, "f32"))


def test_one_work_space_for_calls_of_many_shapes(jlib):
    """One work space, used by one call after another and for other things between: nothing in it matters to the next call."""
    rng = np.random.default_rng(17)
    calls, first = [], []
    for kind, kvh, group, hd, lens, rows in (("f16", 2, 4, 128, [5000, 40, 1300], 1), ("f32", 4, 1, 64, [2500, 900], 200), ("bf16", 1, 8, 96, [3000, 3000], 40),
                                             ("bf16", 1, 1, 32, [20000], 3), ("f16", 8, 1, 64, rng.integers(1, 3000, 70).tolist(), 2)):
        p, table = filled(jlib, rng, kvh * group, kvh, hd, 64, lens)
        start = (np.arange(len(lens) + 1) * rows).tolist()
        calls.append((p, queries(rng, start[-1], kvh * group * hd, kind), start, lens, table, kind))
    size = max(jlib.lib().jepa_amd_cache_work_bytes(C.byref(p.s), len(lens), q.shape[0], table.shape[1]) for p, q, _s, lens, table, _k in calls)
    work = torch.zeros(size, dtype=torch.uint8, device="cuda")
    for again in range(4):
        for i, (p, q, start, lens, table, kind) in enumerate(calls):
            if again == 1:
                work.random_(0, 256)
            if again == 2:
                work.view(torch.int32)[:16384].random_(-2 ** 31, 2 ** 31 - 1)
                work[7::8] = 0
            out = torch.full_like(q, float("nan"))
            torch.cuda.synchronize()
            p.attend(q, ints(start), ints(lens), ints(table), kind, 1, out=out, work=work)
            torch.cuda.synchronize()
            if again == 0:
                check(p, q, start, lens, table, kind)
                first.append(out)
            assert torch.equal(out, first[i]), (again, i)


# ------------------------------------------------------------------------------------------------ together
class Program:
    """The calls as a step-by-step program makes them, on one stream, its lengths and tables on the device throughout."""

    def __init__(self, jlib, n_seq, heads, kvh, hd, page, n_pages, width, n_rows, kind):
        self.p = Pool(jlib, heads, kvh, hd, page, n_pages)
        self.jlib, self.kind, self.n_rows, self.n_seq = jlib, kind, n_rows, n_seq
        i32 = lambda *n, v=0: torch.full(n, v, dtype=torch.int32, device="cuda")  # noqa: E731
        self.len, self.new, self.table, self.free = i32(n_seq), i32(n_seq), i32(n_seq, width, v=-1), ints([0, n_pages])
        self.ring = torch.arange(n_pages, dtype=torch.int32, device="cuda")
        self.start, self.refused, self.slot = i32(n_seq + 1), i32(n_seq), torch.zeros(n_rows, dtype=torch.int64, device="cuda")
        dtype = TYPES[kind][0]
        self.q, self.out = (torch.zeros(n_rows, heads * hd, dtype=dtype, device="cuda") for _ in range(2))
        self.k, self.v = (torch.zeros(n_rows, kvh * hd, dtype=dtype, device="cuda") for _ in range(2))
        self.work = torch.empty(jlib.lib().jepa_amd_cache_work_bytes(C.byref(self.p.s), n_seq, n_rows, width), dtype=torch.uint8, device="cuda")

    def step(self, stream, block=1):
        p, L = self.p, self.jlib.lib()
        ok(self.jlib, L.jepa_amd_cache_plan(0, C.byref(p.s), self.n_seq, self.n_rows, self.len.data_ptr(), self.new.data_ptr(), self.table.data_ptr(),
                                            self.table.shape[1], self.ring.data_ptr(), self.free.data_ptr(), self.free.data_ptr(), self.len.data_ptr(),
                                            self.start.data_ptr(), self.slot.data_ptr(), self.refused.data_ptr(), stream))
        p.store(self.k, self.v, self.slot, self.kind, stream)
        p.attend(self.q, self.start, self.len, self.table, self.kind, block, out=self.out, stream=stream, work=self.work)


def fresh(rng, prog, new):
    prog.new.copy_(ints(new))
    for t in (prog.q, prog.k, prog.v):
        t.copy_(queries(rng, t.shape[0], t.shape[1], prog.kind))
    prog.out.fill_(float("nan"))


def verify(prog, held, new, block=1):
    """The step's output against the definition on q4_0 values of every row that the sequences were given."""
    rows, start = np.maximum(new, 0), [0] + np.cumsum(np.maximum(new, 0)).tolist()
    for i, n in enumerate(new):
        if n < 0:
            held[i] = held[i][:max(0, len(held[i]) + n)]
        else:
            kv = [q4_0(x[start[i]:start[i + 1]].float().cpu().numpy()) for x in (prog.k, prog.v)]
            held[i] = held[i] + list(zip(*kv))
    assert prog.refused.sum().item() == 0
    lens = [len(h) for h in held]
    assert prog.len.tolist() == lens and prog.start.tolist() == start
    table = prog.table.cpu().numpy()
    s = prog.p.s
    for i, h in enumerate(held):
        if h:
            slot = ints([int(table[i, t // s.page_size]) * s.page_size + t % s.page_size for t in range(len(h))], torch.int64)
            for got, want in zip(prog.p.read(slot), zip(*h)):
                np.testing.assert_array_equal(got.cpu().numpy(), np.stack(want))
    want, tol = reference(prog.p, prog.q, start, lens, table, block, s.head_dim ** -0.5, prog.kind)
    a = start[-1]
    assert ((prog.out[:a].double() - want[:a]).abs() <= tol[:a]).all()
    assert torch.isnan(prog.out[a:]).all()
    assert rows.sum() == a


@pytest.mark.parametrize("kind,heads,kvh,hd,page", [("f32", 4, 4, 64, 16), ("f16", 8, 2, 128, 32), ("bf16", 3, 1, 96, 16)])
def test_steps_together(jlib, kind, heads, kvh, hd, page):
    """Prompts, single tokens, drops, ends and new requests, step after step on a stream of the caller's."""
    rng = np.random.default_rng(hd)
    prog = Program(jlib, 4, heads, kvh, hd, page, 60, 20, 80, kind)
    side = torch.cuda.Stream()
    held = [[] for _ in range(4)]
    for new in ([40, 17, 0, 1], [1, 1, 1, 1], [5, -3, 20, 1], [-46, 1, 1, 1], [33, 1, -1000, 30], [1, 1, 7, 0], [0, 0, 0, 0], [1, -16, 1, 1]):
        fresh(rng, prog, new)
        torch.cuda.synchronize()
        prog.step(side.cuda_stream)
        side.synchronize()
        verify(prog, held, np.array(new))


def test_step_captured_and_replayed(jlib):
    """The whole step in a HIP graph, replayed with new lengths and rows while the program runs its own eager work between."""
    rng = np.random.default_rng(21)
    side = torch.cuda.Stream()
    prog = Program(jlib, 3, 8, 2, 64, 16, 400, 200, 24, "f16")
    held = [[] for _ in range(3)]
    fresh(rng, prog, [9, 0, 4])
    torch.cuda.synchronize()
    prog.step(side.cuda_stream)
    side.synchronize()
    verify(prog, held, np.array([9, 0, 4]))
    prog.new.zero_()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        prog.step(side.cuda_stream)
    other = Program(jlib, 3, 8, 2, 64, 16, 40, 20, 24, "f16")
    for new in ([8, 8, 8], [1, 1, 1], [20, -3, 2], [1, 1, 1], [-4, 5, 1], [1, 1, 1]):
        fresh(rng, prog, new)
        fresh(rng, other, [1, 2, 3])
        torch.cuda.synchronize()
        g.replay()
        other.step(None)
        torch.cuda.synchronize()
        verify(prog, held, np.array(new))
    del g


def test_two_graphs_at_once(jlib):
    """Two captured steps with caches and work spaces of their own, replayed on two streams together, against eager runs."""
    rng = np.random.default_rng(22)
    progs, graphs, streams = [], [], [torch.cuda.Stream() for _ in range(2)]
    lens = [[3000, 10, 500], [2500, 900, 0]]
    for n, side in zip(lens, streams):
        prog = Program(jlib, 3, 4, 1, 128, 16, 500, 300, 3, "f32")
        filler, table = filled(jlib, rng, 4, 1, 128, 16, n, extra=500 - sum(-(-x // 16) for x in n))
        prog.p = filler
        prog.table[:, :table.shape[1]] = ints(table)
        used = sum(-(-x // 16) for x in n)
        left = np.setdiff1d(np.arange(500), table[table >= 0])
        prog.ring[:len(left)] = ints(left)
        prog.free.copy_(ints([0, 500 - used]))
        prog.start.copy_(ints([0, 1, 2, 3]))
        prog.len.copy_(ints(n))
        fresh(rng, prog, [0, 0, 0])
        torch.cuda.synchronize()

        def attend(prog=prog, side=side):
            prog.p.attend(prog.q, prog.start, prog.len, prog.table, "f32", 1, out=prog.out, stream=side.cuda_stream, work=prog.work)
        attend()
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            attend()
        progs.append((prog, attend))
        graphs.append(g)
    for _ in range(4):
        for prog, _a in progs:
            fresh(rng, prog, [0, 0, 0])
        torch.cuda.synchronize()
        for _k in range(3):
            for g, side in zip(graphs, streams):
                with torch.cuda.stream(side):
                    g.replay()
        torch.cuda.synchronize()
        got = [prog.out.clone() for prog, _a in progs]
        for (prog, attend), side, x in zip(progs, streams, got):
            prog.out.fill_(float("nan"))
            torch.cuda.synchronize()
            attend()
            torch.cuda.synchronize()
            assert torch.equal(prog.out, x) and not torch.isnan(x).any()
    graphs.clear()
