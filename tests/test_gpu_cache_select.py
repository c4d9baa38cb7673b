"""Digests of the 4-bit cache's pages, the pages that rows select by them, and attention over those on the GPU (no counterpart in the reference): digests and selections
against the definition with whole numbers, bit for bit; attention against the definition in 64 bits on the values that the cache holds; the calls
together as a program makes them step by step, eager and captured.

Attention's tolerance for one row, head and dimension n, out_n = sum_j p_j v_jn, A_n = sum_j p_j |v_jn| and N_n = sum_j |v_jn| over the tokens that the row reads:
  the output's own rounding   eps_T / 2 |out_n|, and half its smallest step
  a value                     enters exactly; for bf16 rows rounded to f16, 2^-11 A_n
  a weight                    16-bit rows: 2^-11 relative (half a step of f16); f32 rows 2^-20 with the exponential and the sums. The sum that divides is of the same
                              rounded weights, so that it counts with |v_jn - out_n|: at most A_n + |out_n|. Weights far below the largest (brought to 2^10 or
                              more) lose half of f16's smallest step: 2^-35 N_n
  scores                      head_dim products of a query held to 2^-22 and an exact key in 32 bits, times a scale: off by (head_dim / 8 + 8) 2^-22 S at most,
                              S = max_j scale |q|max |k_j|_1, on both sides of the fraction: twice that, times A_n
"""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
np = pytest.importorskip("numpy")

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30)}
TINY = np.float32(2.0 ** -100)


def ok(jlib, rc):
    assert rc == 0, jlib.error_text()


def ints(a, dtype=torch.int32):
    return torch.tensor(np.asarray(a), dtype=dtype, device="cuda")


class Cache:
    """A cache of random rows with sequences' pages here and there."""

    def __init__(self, jlib, heads, kvh, hd, page, lens, rng, extra=3, scale=1.0, fill=True, width=None):
        self.jlib, self.hd, self.kvh, self.heads, self.page = jlib, hd, kvh, heads, page
        used = [-(-n // page) for n in lens]
        self.n_pages, self.width = sum(used) + extra, max(used + [1]) if width is None else width
        self.s = jlib.CacheShape(heads, kvh, hd, page, self.n_pages)
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), self.width), -1, np.int32)
        at = 0
        for i, u in enumerate(used):
            self.table[i, :u] = order[at:at + u]
            at += u
        L = jlib.lib()
        self.mem = torch.zeros(self.n_pages * L.jepa_amd_cache_page_bytes(C.byref(self.s)), dtype=torch.uint8, device="cuda")
        self.digest = torch.zeros(self.n_pages, kvh, 2 * hd + 16, dtype=torch.uint8, device="cuda")
        if fill:
            n = self.n_pages * page
            k, v = (torch.tensor(rng.standard_normal((n, kvh * hd)).astype(np.float32) * scale, device="cuda") for _ in range(2))
            self.store(k, v, torch.arange(n, device="cuda"))

    def store(self, k, v, slot):
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_store(0, C.byref(self.s), self.mem.data_ptr(), 0, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), k.shape[0],
                                                           slot.data_ptr(), None))

    def read(self):
        """All keys and values, [page][token][kvh][hd]."""
        n = self.n_pages * self.page
        k, v = (torch.empty(n, self.kvh * self.hd, device="cuda") for _ in range(2))
        slot = torch.arange(n, device="cuda")
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_read(0, C.byref(self.s), self.mem.data_ptr(), slot.data_ptr(), n, 0, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                                          None))
        return (x.reshape(self.n_pages, self.page, self.kvh, self.hd) for x in (k, v))

    def make_digest(self, start, lens, rows, stream=None):
        self.given = ints(start), ints(lens), ints(self.table)
        start, lens, table = self.given
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_digest(0, C.byref(self.s), self.mem.data_ptr(), lens.numel(), rows, start.data_ptr(), lens.data_ptr(), table.data_ptr(),
                                                            self.width, self.digest.data_ptr(), stream))

    def select(self, q, kind, start, lens, block, first, last, take, rows=None, out=None, table=None, stream=None, work=None, ld=None):
        rows = q.shape[0] if rows is None else rows
        t = [ints(start), ints(lens), ints(self.table if table is None else table)]
        out = torch.full((rows, self.kvh, take), -7, dtype=torch.int32, device="cuda") if out is None else out
        need = self.jlib.lib().jepa_amd_cache_select_work_bytes(C.byref(self.s), len(lens), rows, self.width, take)
        work = torch.full((max(need, 16),), 0xa5, dtype=torch.uint8, device="cuda") if work is None else work
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_select(0, C.byref(self.s), self.digest.data_ptr(), TYPES[kind][1], q.data_ptr(), q.stride(0) if ld is None else ld, len(lens),
                                                            rows, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), self.width, block, first, last, take, out.data_ptr(),
                                                            work.data_ptr() if need else None, need, stream))
        torch.cuda.synchronize()
        return out

    def attend(self, q, kind, start, lens, chosen, block, scale, out=None, work=None, table=None, stream=None):
        rows, take = chosen.shape[0], chosen.shape[2]
        t = [ints(start), ints(lens), ints(self.table if table is None else table)]
        out = torch.full_like(q, float("nan")) if out is None else out
        need = self.jlib.lib().jepa_amd_cache_selected_work_bytes(C.byref(self.s), rows, take)
        work = torch.full((max(need, 16),), 0x5a, dtype=torch.uint8, device="cuda") if work is None else work
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_attention_selected(0, C.byref(self.s), self.mem.data_ptr(), TYPES[kind][1], q.data_ptr(), q.stride(0), len(lens), rows,
                                                                        t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), self.width, chosen.data_ptr(), take, scale, block,
                                                                        out.data_ptr(), out.stride(0), work.data_ptr() if need else None, need, stream))
        torch.cuda.synchronize()
        return out


def queries(rng, n, width, kind, scale=1.0):
    return torch.tensor(rng.standard_normal((n, width)).astype(np.float32) * scale, device="cuda").to(TYPES[kind][0])


def rows_of(lens, new):
    """row_start, and (sequence, position) of each row."""
    start = [0] + np.cumsum(new).tolist()
    return start, [(i, n - c + j) for i, (n, c) in enumerate(zip(lens, new)) for j in range(c)]


def visible(pos, n, block):
    return n if block == 0 else 0 if pos < 0 else min(n, (pos // block + 1) * block)


# ------------------------------------------------------------------------------------------------ digests
def box(k):
    """Keys [tokens][hd] f32 (NaN ones do not count) -> codes [2 hd], scale, as the definition makes them in f32."""
    k = k[~np.isnan(k).any(1)]
    b = np.concatenate([k.max(0), k.min(0)]) if len(k) else np.zeros(2 * k.shape[1], np.float32)
    top = np.abs(b).max()
    if top < TINY:
        return np.zeros(len(b), np.int8), np.float32(0)
    return np.rint(b * (np.float32(127) / top)).astype(np.int8), top / np.float32(127)


def digests(c, pages):
    d = c.digest.cpu().numpy()[pages]
    return d[..., :2 * c.hd].view(np.int8), d[..., 2 * c.hd:2 * c.hd + 4].copy().view(np.float32)[..., 0], d[..., 2 * c.hd + 4:]


@pytest.mark.parametrize("hd,kvh,page,lens,new", [
    (128, 2, 64, [100, 1, 64, 65], [1, 1, 1, 1]), (64, 3, 16, [40, 200, 0, 17, 33], [40, 3, 0, 17, 16]), (96, 1, 32, [700], [650]), (32, 5, 256, [300, 1000], [2, 1000]),
    (128, 8, 16, [3000, 50], [2990, 7]), (64, 1, 128, [129, 128, 127] * 30, [5, 128, 1] * 30), (32, 1, 16, list(range(1, 200)), [1] * 199), (96, 2, 16, [16] * 300, [16] * 300),
])
def test_digest(jlib, hd, kvh, page, lens, new):
    rng = np.random.default_rng(hd + page)
    c = Cache(jlib, kvh, kvh, hd, page, lens, rng)
    # some keys NaN, a page of zeros, a page of one tiny value
    n = c.n_pages * page
    k, v = (torch.tensor(rng.standard_normal((n, kvh * hd)).astype(np.float32) * np.exp(2 * rng.standard_normal((n, 1))).astype(np.float32), device="cuda") for _ in range(2))
    k[rng.random(n) < 0.05] = float("nan")
    k[c.table[0, 0] * page:(c.table[0, 0] + 1) * page] = 0
    c.store(k, v, torch.arange(n, device="cuda"))
    start, _ = rows_of(lens, new)
    rows = start[-1] + 5
    c.digest.fill_(0x77)
    c.make_digest(start, lens, rows)
    keys = next(c.read()).cpu().numpy()
    touched = [(i, p) for i, (m, r) in enumerate(zip(lens, new)) for p in range((m - r) // page, -(-m // page)) if r]
    pages = [c.table[i, p] for i, p in touched]
    codes, scales, rest = digests(c, pages)
    assert not rest.any()
    for at, (i, p) in enumerate(touched):
        for h in range(kvh):
            want, s = box(keys[pages[at], :min(page, lens[i] - p * page), h])
            np.testing.assert_array_equal(codes[at, h], want)
            assert scales[at, h] == s
    others = [p for p in range(c.n_pages) if p not in set(pages)]
    assert (c.digest[others] == 0x77).all()
    # the values that they stand for, and pages that are none
    at = ints(pages + [-1, c.n_pages, 2 ** 31 - 1])
    bounds = torch.full((len(at), kvh, 2, hd), float("nan"), device="cuda")
    ok(jlib, jlib.lib().jepa_amd_cache_digest_read(0, C.byref(c.s), c.digest.data_ptr(), at.data_ptr(), len(at), bounds.data_ptr(), None))
    got = bounds.cpu().numpy()
    np.testing.assert_array_equal(got[:len(pages)].reshape(len(pages), kvh, -1), codes.astype(np.float32) * scales[..., None])
    assert not got[len(pages):].any()


def test_digest_magnitudes(jlib):
    """The largest and smallest values that a page holds, a page below 2^-100 (f16 scales end before: by bytes), scales of both signs."""
    rng = np.random.default_rng(1)
    c = Cache(jlib, 1, 1, 32, 16, [80], rng, fill=False)
    n = c.n_pages * 16
    k = torch.tensor(rng.standard_normal((n, 32)).astype(np.float32), device="cuda")
    for i, f in enumerate((65000.0, 1e-6, 6e-7, -1.0, 1e-9)):
        k[c.table[0, i] * 16:(c.table[0, i] + 1) * 16] *= f
    c.store(k, k, torch.arange(n, device="cuda"))
    c.make_digest([0, 80], [80], 80)
    keys = next(c.read()).cpu().numpy()
    codes, scales, _ = digests(c, c.table[0])
    for p in range(5):
        want, s = box(keys[c.table[0, p], :, 0])
        np.testing.assert_array_equal(codes[p, 0], want)
        assert scales[p, 0] == s


def test_digest_pages_that_are_none_and_no_rows(jlib):
    rng = np.random.default_rng(2)
    c = Cache(jlib, 2, 2, 64, 16, [64, 40], rng)
    c.table[0, 1], c.table[0, 2], c.table[1, 0] = -5, c.n_pages, 2 ** 31 - 1
    c.digest.fill_(0x33)
    c.make_digest([0, 64, 104], [64, 40], 104)
    want = {c.table[0, 0], c.table[0, 3], c.table[1, 1], c.table[1, 2]}
    assert {p for p in range(c.n_pages) if (c.digest[p] != 0x33).any()} == want
    before = c.digest.clone()
    for start, lens, rows in (([0, 0, 0], [64, 40], 104), ([0, 64, 104], [64, 40], 0), ([50, 50, 50], [64, 40], 60), ([0, 3, 3], [0, 0], 9)):
        c.make_digest(start, lens, rows)
        torch.cuda.synchronize()
        assert torch.equal(c.digest, before)


# ------------------------------------------------------------------------------------------------ selection
def choose(c, q, lens, where, block, first, last, take, table=None):
    """The documented selection with whole numbers: [rows][kvh][take]."""
    table = c.table if table is None else table
    hd, kvh, group = c.hd, c.kvh, c.heads // c.kvh
    d = c.digest.cpu().numpy()
    codes, scales = d[..., :2 * hd].view(np.int8).astype(np.int64), d[..., 2 * hd:2 * hd + 4].copy().view(np.float32)[..., 0]
    x = q.float().cpu().numpy().reshape(q.shape[0], kvh, group, hd)
    out = np.full((len(where), kvh, take), -1, np.int32)
    for r, (i, pos) in enumerate(where):
        see = -(-visible(pos, lens[i], block) // c.page)
        for h in range(kvh):
            if see <= take:
                out[r, h, :see] = np.arange(see)
                continue
            v = x[r, h].astype(np.float64)
            f = np.concatenate([np.maximum(v, 0).sum(0), np.minimum(v, 0).sum(0)]).astype(np.float32)
            top = np.abs(f).max() if np.isfinite(v).all() else np.float32(np.inf)
            y = np.rint(f * (np.float32(127) / top)).astype(np.int64) if TINY <= top < np.inf else np.zeros(2 * hd, np.int64)
            free = np.arange(first, see - last)
            page = table[i, free].astype(np.int64)
            bad = (page < 0) | (page >= c.n_pages)
            page[bad] = 0
            score = (codes[page, h] @ y).astype(np.float32) * scales[page, h]
            score[bad] = -np.inf
            best = free[np.argsort(-score, kind="stable")[:take - first - last]]
            n = np.concatenate([np.arange(first), np.sort(best), np.arange(see - last, see)])
            out[r, h] = n
    return out


def random_digests(rng, c, levels=0):
    """Digests of boxes around random means; of a few whole levels, so that many pages score alike."""
    mid = rng.standard_normal((c.n_pages, c.kvh, c.hd)).astype(np.float32) * 0.5
    out = 1 + 0.3 * np.abs(rng.standard_normal((c.n_pages, c.kvh, 2 * c.hd))).astype(np.float32)
    b = np.concatenate([mid + out[..., :c.hd], mid - out[..., c.hd:]], -1)
    if levels:
        b = np.repeat(rng.integers(-levels, levels + 1, (c.n_pages, c.kvh, 1)), 2 * c.hd, -1).astype(np.float32)
        b[..., 0] = levels
    top = np.abs(b).max(-1, keepdims=True)
    codes = np.rint(b * (np.float32(127) / top)).astype(np.int8)
    d = np.concatenate([codes.view(np.uint8), (top / np.float32(127)).astype(np.float32).view(np.uint8), np.zeros((c.n_pages, c.kvh, 12), np.uint8)], -1)
    c.digest.copy_(torch.tensor(d, device="cuda"))


SELECT = [
    # kind, kvh, group, hd, page, lens, rows of each, block, first, last, take
    ("f16", 2, 4, 128, 16, [1000, 30, 5000], [1, 1, 1], 1, 1, 2, 16), ("bf16", 3, 1, 64, 32, [4000], [1], 1, 0, 1, 5), ("f32", 1, 8, 96, 16, [3000, 2999], [3, 1], 1, 2, 3, 64),
    ("f32", 4, 2, 32, 64, [70000], [1], 0, 0, 1, 256), ("f16", 8, 1, 128, 16, [40000, 17000], [1, 2], 1, 1, 1, 200), ("bf16", 2, 5, 128, 16, [20000], [1], 1, 4, 9, 14),
    ("f16", 1, 1, 64, 16, [9000], [2], 1, 0, 1, 1), ("f32", 16, 2, 64, 16, [900, 1200, 16], [300, 258, 16], 1, 1, 2, 12), ("f16", 4, 8, 128, 64, [16000], [1100], 1, 1, 2, 16),
    ("bf16", 8, 4, 96, 16, [5000, 0, 2100], [600, 0, 400], 7, 0, 1, 256), ("f16", 16, 1, 32, 32, [3000] * 4, [129] * 4, 129, 1, 1, 31), ("f32", 8, 3, 128, 256, [30000], [700], 0, 0, 2, 30),
    ("f16", 2, 2, 64, 16, [600] * 100, [1] * 100, 1, 1, 1, 8), ("bf16", 64, 1, 32, 16, [2500, 900], [50, 30], 1, 3, 3, 7), ("f32", 2, 1, 64, 16, [50000], [1], 1, 0, 1, 255), ("f16", 4, 2, 64, 16, [20000, 4500], [300, 90], 1, 1, 2, 200), ("f32", 8, 1, 32, 16, [9000], [200], 50, 0, 1, 2),
]


@pytest.mark.parametrize("kind,kvh,group,hd,page,lens,new,block,first,last,take", SELECT)
def test_select(jlib, kind, kvh, group, hd, page, lens, new, block, first, last, take):
    rng = np.random.default_rng(take * 7 + hd)
    c = Cache(jlib, kvh * group, kvh, hd, page, lens, rng, fill=False)
    start, where = rows_of(lens, new)
    q = queries(rng, start[-1], kvh * group * hd, kind, 0.7)
    for levels in (0, 2):
        random_digests(rng, c, levels)
        got = c.select(q, kind, start, lens, block, first, last, take).cpu().numpy()
        np.testing.assert_array_equal(got, choose(c, q, lens, where, block, first, last, take))


@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("kind", list(TYPES))
def test_select_queries_that_are_odd(jlib, rows, kind):
    """NaN, infinities, zeros, the smallest and largest values of the type among a K/V head's queries; negative scores; heads on either side of zero."""
    rng = np.random.default_rng(rows)
    kvh, group, hd, page, take = 8, 2, 64, 16, 10
    lens, new = [4000], [rows]
    c = Cache(jlib, kvh * group, kvh, hd, page, lens, rng, fill=False)
    random_digests(rng, c)
    start, where = rows_of(lens, new)
    q = queries(rng, rows, kvh * group * hd, kind).reshape(rows, kvh, group, hd)
    f = torch.finfo(TYPES[kind][0])
    q[0, 0, 0, 0], q[0, 1, 1, 5], q[-1, 2, 0, 3] = float("nan"), float("inf"), float("-inf")
    q[0, 3], q[-1, 4] = 0, f.max
    q[0, 5] = f.tiny
    q[-1, 6] *= 1e-30
    q = q.reshape(rows, -1)
    got = c.select(q, kind, start, lens, 1, 1, 1, take).cpu().numpy()
    np.testing.assert_array_equal(got, choose(c, q, lens, where, 1, 1, 1, take))
    # boxes wholly on one side: every score below zero for some, above for others
    c.digest[..., :2 * hd] = torch.where(c.digest[..., :2 * hd] == 0, 1, c.digest[..., :2 * hd].view(torch.int8).abs().view(torch.uint8))
    got = c.select(-q.abs(), kind, start, lens, 1, 0, 1, take).cpu().numpy()
    np.testing.assert_array_equal(got, choose(c, -q.abs(), lens, where, 1, 0, 1, take))


@pytest.mark.parametrize("rows", [1, 700])
def test_select_pages_that_are_none(jlib, rows):
    """Entries of the table that are no pages come last, in their order; rows of no sequence are left as they are; a padded table does not matter."""
    rng = np.random.default_rng(8)
    kvh, hd, page, take, lens = 8, 64, 16, 20, [1500, 2500]
    c = Cache(jlib, kvh, kvh, hd, page, lens, rng, fill=False, width=1300)
    random_digests(rng, c)
    table = c.table.copy()
    table[0, rng.permutation(90)[:80]] = -1
    table[1, rng.permutation(150)[:100]] = c.n_pages
    start, where = rows_of(lens, [rows, rows])
    q = queries(rng, 2 * rows + 3, kvh * hd, "f16")
    got = c.select(q, "f16", start, lens, 1, 1, 2, take, table=table).cpu().numpy()
    np.testing.assert_array_equal(got[:2 * rows], choose(c, q[:2 * rows], lens, where, 1, 1, 2, take, table))
    assert (got[2 * rows:] == -7).all()
    # rows before the first sequence
    got = c.select(q, "f16", [3, 3 + rows, 3 + 2 * rows], lens, 1, 1, 2, take, table=table).cpu().numpy()
    np.testing.assert_array_equal(got[3:], choose(c, q[3:], lens, where, 1, 1, 2, take, table))
    assert (got[:3] == -7).all()


def test_select_row_starts_and_lengths_out_of_range(jlib):
    """Nothing is read or written out of range whatever row_start and kv_len hold: rows that no sequence has are left."""
    rng = np.random.default_rng(9)
    c = Cache(jlib, 4, 4, 32, 16, [3000, 500], rng, fill=False)
    random_digests(rng, c)
    q = queries(rng, 9, 128, "f32")
    for start, lens in (([0, 4, 9], [2 ** 31 - 1, -5]), ([-9, 3, 2 ** 31 - 1], [3000, 500]), ([9, 9, 9], [3000, 500]), ([5, 2, 9], [3000, 500]), ([0, 9, 9], [3, 500])):
        got = c.select(q, "f32", start, lens, 1, 1, 2, 8).cpu().numpy()
        assert ((got >= -1) & (got < c.width) | (got == -7)).all()
        out = c.attend(q, "f32", start, lens, ints(np.where(got == -7, 0, got)), 1, 0.1)
        assert out.shape == q.shape
        c.make_digest(start, lens, 9)
    torch.cuda.synchronize()


def test_select_long_tables_of_many_rows(jlib):
    """More rows than are split into pieces, over more pages than a workgroup takes at once; the sequences name the same pages."""
    rng = np.random.default_rng(23)
    c = Cache(jlib, 2, 1, 32, 16, [32000], rng, fill=False)
    c.table = np.repeat(c.table, 1100, 0)
    lens = rng.integers(25000, 32001, 1100).tolist()
    start, where = rows_of(lens, [1] * 1100)
    q = queries(rng, 1100, 64, "bf16")
    for levels in (0, 3):
        random_digests(rng, c, levels)
        for first, take in ((1, 256), (0, 3)):
            got = c.select(q, "bf16", start, lens, 1, first, 1, take).cpu().numpy()
            np.testing.assert_array_equal(got, choose(c, q, lens, where, 1, first, 1, take))


def test_select_many_sequences(jlib):
    rng = np.random.default_rng(10)
    lens = rng.integers(0, 400, 4096).tolist()
    new = [min(n, int(r)) for n, r in zip(lens, rng.integers(0, 3, 4096))]
    c = Cache(jlib, 2, 1, 32, 16, lens, rng, fill=False)
    random_digests(rng, c)
    start, where = rows_of(lens, new)
    q = queries(rng, start[-1], 64, "f16")
    got = c.select(q, "f16", start, lens, 1, 1, 1, 6).cpu().numpy()
    np.testing.assert_array_equal(got, choose(c, q, lens, where, 1, 1, 1, 6))


def test_select_one_work_space(jlib):
    """Calls of many shapes one after the other in one work space, which holds anything at first."""
    rng = np.random.default_rng(11)
    work = None
    for kvh, lens, take in ((1, [70000], 40), (4, [40000], 256), (2, [20000, 33000], 9), (1, [70000], 40)):
        c = Cache(jlib, kvh, kvh, 32, 16, lens, rng, fill=False)
        random_digests(rng, c)
        start, where = rows_of(lens, [1] * len(lens))
        q = queries(rng, len(lens), kvh * 32, "bf16")
        if work is None:
            work = torch.full((jlib.lib().jepa_amd_cache_select_work_bytes(C.byref(c.s), 8, 64, 1 << 20, 256),), 0xff, dtype=torch.uint8, device="cuda")
        for _ in range(3):
            got = c.select(q, "bf16", start, lens, 1, 1, 1, take, work=work).cpu().numpy()
            np.testing.assert_array_equal(got, choose(c, q, lens, where, 1, 1, 1, take))


# ------------------------------------------------------------------------------------------------ attention
def definition(c, q, lens, where, chosen, block, scale, kind, table=None):
    """(out, tolerance) [rows][heads][hd] in 64 bits, on the values that the cache holds."""
    table = c.table if table is None else table
    hd, kvh, group, page = c.hd, c.kvh, c.heads // c.kvh, c.page
    k, v = (x.double() for x in c.read())
    out, tol = (torch.zeros(q.shape[0], c.heads, hd, dtype=torch.float64, device="cuda") for _ in range(2))
    eps = torch.finfo(TYPES[kind][0]).eps / 2
    for r, (i, pos) in enumerate(where):
        end = visible(pos, lens[i], block)
        for h in range(kvh):
            tokens = [(table[i, p], t) for p in chosen[r][h] if 0 <= p < -(-end // page) and 0 <= table[i, p] < c.n_pages for t in range(min(page, end - p * page))]
            if not tokens:
                continue
            pg, t = torch.tensor(np.array(tokens), device="cuda").T
            kh, vh = k[pg, t, h], v[pg, t, h]
            x = q[r].double().reshape(c.heads, hd)[h * group:(h + 1) * group]
            w = torch.softmax(x @ kh.T.contiguous() * scale, -1)
            y, A, N = w @ vh, w @ vh.abs(), vh.abs().sum(0)
            S = abs(scale) * x.abs().amax(-1, keepdim=True) * kh.abs().sum(-1).max()
            f = 2.0 ** -20 + 2 * (hd / 8 + 8) * 2.0 ** -22 * S + (0 if kind == "f32" else 2.0 ** -11)
            sl = slice(h * group, (h + 1) * group)
            out[r, sl] = y
            tol[r, sl] = eps * y.abs() * (1 + f) + f * (A + y.abs()) + (2.0 ** -11 * A if kind == "bf16" else 0) + 2.0 ** -35 * N + (2.0 ** -25 if kind == "f16" else 1e-38)
    return out, tol


def lists(rng, c, lens, where, block, take):
    """Pages here and there in any order, with entries that are none among them."""
    out = np.full((len(where), c.kvh, take), -1, np.int32)
    for r, (i, pos) in enumerate(where):
        see = -(-visible(pos, lens[i], block) // c.page)
        for h in range(c.kvh):
            p = rng.permutation(see)[:take] if see else np.zeros(0, int)
            out[r, h, rng.permutation(take)[:len(p)]] = p
    return out


def near(got, want, tol):
    bad = ~((got.double().reshape(want.shape) - want).abs() <= tol)
    assert not bad.any(), (bad.nonzero()[:5], got.reshape(want.shape)[bad][:5], want[bad][:5], tol[bad][:5])


ATTEND = [
    # kvh, group, hd, page, lens, rows of each, block, take
    (2, 1, 32, 16, [100], [1], 1, 3), (1, 4, 64, 64, [1000, 64, 1], [1, 1, 1], 1, 8), (2, 8, 128, 16, [3000, 200], [1, 2], 1, 64), (1, 17, 96, 32, [500], [3], 1, 9),
    (3, 5, 64, 16, [900], [1], 0, 200), (1, 1, 128, 256, [5000], [1], 1, 12), (1, 33, 32, 128, [700, 128], [1, 2], 1, 4), (16, 1, 64, 16, [5000], [1], 1, 32),
    (8, 2, 96, 16, [300, 0, 40], [5, 0, 40], 7, 10), (4, 3, 128, 64, [2000], [40], 40, 16), (2, 16, 64, 32, [20000], [2], 1, 256), (4, 1, 32, 16, [33] * 70, [1] * 70, 1, 2),
    # more units than the chip holds waves
    (16, 2, 32, 16, [600], [300], 1, 8), (8, 4, 64, 16, [700, 300], [400, 210], 1, 5), (4, 20, 128, 32, [900], [450], 0, 3), (8, 1, 96, 64, [500], [450], 9, 6),
    (64, 1, 128, 16, [200], [64], 1, 7),
]


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("kvh,group,hd,page,lens,new,block,take", ATTEND)
def test_attention(jlib, kind, kvh, group, hd, page, lens, new, block, take):
    rng = np.random.default_rng(hd + take)
    c = Cache(jlib, kvh * group, kvh, hd, page, lens, rng)
    start, where = rows_of(lens, new)
    q = queries(rng, start[-1] + 2, kvh * group * hd, kind)
    chosen = np.concatenate([lists(rng, c, lens, where, block, take), np.zeros((2, kvh, take), np.int32)])
    got = c.attend(q, kind, start, lens, ints(chosen), block, hd ** -0.5)
    want, tol = definition(c, q[:-2], lens, where, chosen, block, hd ** -0.5, kind)
    near(got[:-2], want, tol)
    assert torch.isnan(got[-2:]).all()      # rows behind the last
    again = c.attend(q, kind, start, lens, ints(chosen), block, hd ** -0.5)
    assert torch.equal(again[:-2], got[:-2])


@pytest.mark.parametrize("rows", [1, 500])
@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_entries_that_are_none(jlib, kind, rows):
    """Negative entries, pages past what the row sees or past the table, table entries that are no page, pages named twice, rows that read nothing."""
    rng = np.random.default_rng(12)
    kvh, hd, page, lens = 8, 64, 16, [rows + 300, rows]
    c = Cache(jlib, kvh, kvh, hd, page, lens, rng)
    table = c.table.copy()
    table[0, 3], table[0, 5] = -1, c.n_pages
    start, where = rows_of(lens, [rows, rows])
    q = queries(rng, 2 * rows, kvh * hd, kind)
    chosen = rng.integers(-3, c.width + 3, (2 * rows, kvh, 9)).astype(np.int32)
    chosen[0, 0], chosen[-1, 1] = -1, 2 ** 31 - 1
    chosen[0, 2], chosen[0, 3] = 3, 5
    chosen[-1, 0, :2] = 0
    got = c.attend(q, kind, start, lens, ints(chosen), 1, 0.125, table=table)
    want, tol = definition(c, q, lens, where, chosen, 1, 0.125, kind, table)
    near(got, want, tol)
    out = got.reshape(2 * rows, kvh, hd)
    assert (out[0, 0] == 0).all() and (out[-1, 1] == 0).all() and (out[0, 2] == 0).all() and (out[0, 3] == 0).all()


@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_what_must_not_be_read(jlib, kind, rows):
    """NaN keys and the largest values in pages that are not selected and in tokens that the row does not see do not change it; in a token that it reads they do."""
    rng = np.random.default_rng(13)
    kvh, hd, page, n = 16, 64, 16, 400
    c = Cache(jlib, kvh, kvh, hd, page, [n], rng)
    start, where = rows_of([n], [rows])
    q = queries(rng, rows, kvh * hd, kind)
    chosen = lists(rng, c, [n], where, 1, 6)
    chosen[chosen == 2] = 3      # page 2 is never read
    chosen[:, 0, 0] = [pos // page for _, pos in where]
    want = c.attend(q, kind, start, [n], ints(chosen), 1, 0.125)
    k, v = (x.reshape(-1, kvh * hd).clone() for x in c.read())
    slot = torch.arange(c.n_pages * page, device="cuda")
    dirty = (slot // page == int(c.table[0, 2])) | (slot // page == int(c.table[0, -1])) & (slot % page >= (n - 1) % page + 1)
    k[dirty], v[dirty] = float("nan"), 60000.0
    c.store(k, v, slot)
    got = c.attend(q, kind, start, [n], ints(chosen), 1, 0.125)
    assert torch.equal(got, want)
    last = torch.tensor([int(c.table[0, (n - 1) // page]) * page + (n - 1) % page], device="cuda")
    c.store(torch.full((1, kvh * hd), float("nan"), device="cuda"), torch.ones(1, kvh * hd, device="cuda"), last)
    got = c.attend(q, kind, start, [n], ints(chosen), 1, 0.125).reshape(rows, kvh, hd)
    assert torch.isnan(got[-1, 0]).all()
    if rows > 1:
        assert not torch.isnan(got[:-1]).any()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("q_scale,k_scale", [(30.0, 3.0), (1e-4, 1e-3), (0.0, 1.0), (1e3, 1e-3)])
def test_attention_magnitudes_and_scales(jlib, kind, q_scale, k_scale):
    rng = np.random.default_rng(14)
    c = Cache(jlib, 6, 2, 64, 32, [900], rng, scale=k_scale)
    start, where = rows_of([900], [4])
    q = queries(rng, 4, 384, kind, q_scale)
    chosen = lists(rng, c, [900], where, 1, 20)
    for scale in (0.125, -0.125, 0.0):
        want, tol = definition(c, q, [900], where, chosen, 1, scale, kind)
        near(c.attend(q, kind, start, [900], ints(chosen), 1, scale), want, tol)


@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("kind", list(TYPES))
def test_attention_of_the_largest_queries_and_values(jlib, kind, rows):
    """Queries up to the type's end put all weight on the largest scores, without a NaN; a mean of f16's largest values stays finite."""
    rng = np.random.default_rng(22)
    kvh, group, hd, page, n = 2, 2, 64, 16, 640
    c = Cache(jlib, kvh * group, kvh, hd, page, [n], rng)
    start, where = rows_of([n], [rows])
    chosen = lists(rng, c, [n], where, 1, 12)
    chosen[:, :, 0] = 0
    for top in (1.0, 0.25, 2.0 ** -9):
        q = queries(rng, rows, kvh * group * hd, "f32")
        q = (q / q.abs().max() * (torch.finfo(TYPES[kind][0]).max * top)).to(TYPES[kind][0])
        want, tol = definition(c, q, [n], where, chosen, 1, hd ** -0.5, kind)
        got = c.attend(q, kind, [0, rows], [n], ints(chosen), 1, hd ** -0.5)
        near(got, want, tol)
        # the tolerance says little here: but where one score is well ahead of the others the output is its value, rounded. Ahead by the scores' own rounding and
        # by 40 after the scale, so that the others weigh less than 640 e^-40 < 2^-48 together
        k, v = (x.double() for x in c.read())
        for r in (0, rows - 1):
            pg, t = torch.tensor([(c.table[0, p], t) for p in chosen[r][1] if 0 <= p for t in range(min(page, visible(where[r][1], n, 1) - p * page))], device="cuda").T
            s = k[pg, t, 1] @ q[r, -hd:].double()
            if len(s) > 1 and s.topk(2).values.diff().abs() < max(s.abs().max().item() * 2.0 ** -9, 40 * hd ** 0.5):
                continue
            best = v[pg, t, 1][s.argmax()]
            assert ((got[r, -hd:].double() - best).abs() <= torch.finfo(TYPES[kind][0]).eps * best.abs() + 1e-7).all()
    big = torch.full((c.n_pages * page, kvh * hd), 65504.0, device="cuda")
    k = next(c.read()).reshape(-1, kvh * hd).clone()
    c.store(k, big, torch.arange(c.n_pages * page, device="cuda"))
    got = c.attend(queries(rng, rows, kvh * group * hd, kind), kind, [0, rows], [n], ints(chosen), 1, hd ** -0.5).double()
    assert ((got - 65504).abs() <= 65504 * (torch.finfo(TYPES[kind][0]).eps / 2 + 2.0 ** -20)).all()


@pytest.mark.parametrize("kind", list(TYPES))
def test_all_pages_selected_is_attention(jlib, kind):
    """Every page of a short context, against the call that reads all: both are within their tolerance of the definition."""
    rng = np.random.default_rng(15)
    lens, new = [500, 37, 240], [3, 37, 1]
    c = Cache(jlib, 8, 2, 128, 16, lens, rng)
    start, where = rows_of(lens, new)
    q = queries(rng, start[-1], 1024, kind)
    c.make_digest([0, 500, 537, 777], lens, 777)
    chosen = c.select(q, kind, start, lens, 1, 1, 1, 32)
    got = c.attend(q, kind, start, lens, chosen, 1, 128 ** -0.5)
    want, tol = definition(c, q, lens, where, chosen.tolist(), 1, 128 ** -0.5, kind)
    near(got, want, tol)
    dense, L = torch.empty_like(q), jlib.lib()
    work = torch.empty(L.jepa_amd_cache_work_bytes(C.byref(c.s), 3, start[-1], c.width), dtype=torch.uint8, device="cuda")
    t = [ints(start), ints(lens), ints(c.table)]
    ok(jlib, L.jepa_amd_cache_attention(0, C.byref(c.s), c.mem.data_ptr(), TYPES[kind][1], q.data_ptr(), 1024, 3, start[-1], t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(),
                                        c.width, 128 ** -0.5, 1, dense.data_ptr(), 1024, work.data_ptr(), work.numel(), None))
    near(dense, want, tol + (2.0 ** -11 * 40 * want.abs().max() if kind == "bf16" else 0))


def test_attention_strides(jlib):
    rng = np.random.default_rng(16)
    c = Cache(jlib, 4, 2, 32, 16, [300], rng)
    start, where = rows_of([300], [5])
    wide = queries(rng, 5, 128 + 24, "f16")
    q = wide[:, 8:136]
    chosen = ints(lists(rng, c, [300], where, 1, 4))
    want = c.attend(q.contiguous(), "f16", start, [300], chosen, 1, 0.2)
    out = torch.full((5, 160), 5.0, dtype=torch.float16, device="cuda")
    got = c.attend(q, "f16", start, [300], chosen, 1, 0.2, out=out[:, 16:144])
    assert torch.equal(got, want) and (out[:, :16] == 5).all() and (out[:, 144:] == 5).all()
    random_digests(rng, c)
    assert torch.equal(c.select(q, "f16", start, [300], 1, 0, 1, 3), c.select(q.contiguous(), "f16", start, [300], 1, 0, 1, 3))


def test_one_work_space_for_all_calls(jlib):
    """Selection in pieces, attention over selected pages in pieces and attention over all take turns in one work space, which holds anything at first."""
    rng = np.random.default_rng(24)
    L, work = jlib.lib(), None
    for kvh, n, take in ((1, 40000, 60), (2, 9000, 200), (1, 40000, 60)):
        c = Cache(jlib, 2 * kvh, kvh, 32, 16, [n], rng)
        start, where = rows_of([n], [2])
        q = queries(rng, 2, 64 * kvh, "f16")
        random_digests(rng, c)
        if work is None:
            need = [L.jepa_amd_cache_select_work_bytes(C.byref(c.s), 1, 8, 1 << 16, 256), L.jepa_amd_cache_selected_work_bytes(C.byref(c.s), 8, 256),
                    L.jepa_amd_cache_work_bytes(C.byref(c.s), 8, 64, 1 << 16)]
            work = torch.randint(0, 256, (max(need),), dtype=torch.uint8, device="cuda")
        want_list, outs, dense = choose(c, q, [n], where, 1, 1, 2, take), [], []
        for _ in range(3):
            chosen = c.select(q, "f16", start, [n], 1, 1, 2, take, work=work)
            np.testing.assert_array_equal(chosen.cpu().numpy(), want_list)
            outs.append(c.attend(q, "f16", start, [n], chosen, 1, 0.2, work=work))
            t, out = [ints(start), ints([n]), ints(c.table)], torch.empty_like(q)
            ok(jlib, L.jepa_amd_cache_attention(0, C.byref(c.s), c.mem.data_ptr(), 1, q.data_ptr(), q.stride(0), 1, 2, t[0].data_ptr(), t[1].data_ptr(), t[2].data_ptr(), c.width, 0.2, 1,
                                                out.data_ptr(), out.stride(0), work.data_ptr(), work.numel(), None))
            dense.append(out)
        want, tol = definition(c, q, [n], where, want_list, 1, 0.2, "f16")
        near(outs[0], want, tol)
        want, tol = definition(c, q, [n], where, np.tile(np.arange(c.width), (2, kvh, 1)), 1, 0.2, "f16")
        near(dense[0], want, tol)
        torch.cuda.synchronize()
        assert all(torch.equal(x, outs[0]) for x in outs) and all(torch.equal(x, dense[0]) for x in dense)


def test_offsets_past_32_bits(jlib):
    """A cache and digests whose far pages lie past 2^32 bytes."""
    hd, kvh, page, n_pages = 128, 8, 256, 16000
    s = jlib.CacheShape(8, kvh, hd, page, n_pages)
    L = jlib.lib()
    per = L.jepa_amd_cache_page_bytes(C.byref(s))
    assert per * n_pages > 1 << 32
    small = jlib.CacheShape(8, kvh, hd, page, 4)
    rng = np.random.default_rng(17)
    c = Cache(jlib, 8, kvh, hd, page, [900], rng, extra=0)
    far = Cache.__new__(Cache)
    far.__dict__.update(c.__dict__)
    far.s, far.n_pages = s, n_pages
    far.mem = torch.empty(n_pages * per, dtype=torch.uint8, device="cuda")
    far.digest = torch.empty(n_pages, kvh, 2 * hd + 16, dtype=torch.uint8, device="cuda")
    far.table = c.table + (n_pages - 4)
    far.mem[(n_pages - 4) * per:] = c.mem
    del small
    q = queries(rng, 1, 1024, "f16")
    for x in (c, far):
        x.make_digest([0, 900], [900], 900)
    assert torch.equal(far.digest[n_pages - 4:], c.digest)
    a, b = (x.select(q, "f16", [0, 1], [900], 1, 0, 1, 3) for x in (c, far))
    assert torch.equal(a, b)
    assert torch.equal(c.attend(q, "f16", [0, 1], [900], a, 1, 0.1), far.attend(q, "f16", [0, 1], [900], b, 1, 0.1))


# ------------------------------------------------------------------------------------------------ together
class Program:
    """A program's buffers and its step: plan, append, digest, select, attention, all on one stream."""

    def __init__(self, jlib, n_seq, heads, kvh, hd, page, n_pages, width, rows, kind, take, first=1, last=2):
        self.jlib, self.kind, self.take, self.first, self.last, self.rows, self.width, self.n_seq = jlib, kind, take, first, last, rows, width, n_seq
        self.s = jlib.CacheShape(heads, kvh, hd, page, n_pages)
        self.axes = jlib.RopeAxes.of(hd, 3, (hd // 2, hd // 4, hd // 4), 1e4)
        L, dt = jlib.lib(), TYPES[kind][0]
        z = lambda *n, dtype=torch.int32: torch.zeros(*n, dtype=dtype, device="cuda")  # noqa: E731
        self.mem = z(n_pages * L.jepa_amd_cache_page_bytes(C.byref(self.s)), dtype=torch.uint8)
        self.digest = z(n_pages * L.jepa_amd_cache_digest_bytes(C.byref(self.s)), dtype=torch.uint8)
        self.len, self.new, self.start, self.refused = z(n_seq), z(n_seq), z(n_seq + 1), z(n_seq)
        self.table, self.ring, self.free = torch.full((n_seq, width), -1, dtype=torch.int32, device="cuda"), torch.arange(n_pages, dtype=torch.int32, device="cuda"), ints([0, n_pages])
        self.slot, self.pos = z(rows, dtype=torch.int64), z(rows, 3)
        self.q, self.k, self.v, self.out = z(rows, heads * hd, dtype=dt), z(rows, kvh * hd, dtype=dt), z(rows, kvh * hd, dtype=dt), z(rows, heads * hd, dtype=dt)
        self.turned, self.chosen = z(rows, heads * hd, dtype=dt), z(rows, kvh, take)
        self.work = z(max(16, L.jepa_amd_cache_select_work_bytes(C.byref(self.s), n_seq, rows, width, take)), dtype=torch.uint8)
        self.work2 = z(max(16, L.jepa_amd_cache_selected_work_bytes(C.byref(self.s), rows, take)), dtype=torch.uint8)

    def step(self, stream):
        L, s, kind, p = self.jlib.lib(), C.byref(self.s), TYPES[self.kind][1], lambda t: t.data_ptr()
        ok(self.jlib, L.jepa_amd_cache_plan(0, s, self.n_seq, self.rows, p(self.len), p(self.new), p(self.table), self.width, p(self.ring), p(self.free), p(self.free), p(self.len),
                                            p(self.start), p(self.slot), p(self.refused), stream))
        ok(self.jlib, L.jepa_amd_cache_append(0, s, C.byref(self.axes), p(self.mem), kind, p(self.q), self.q.stride(0), p(self.k), self.k.stride(0), p(self.v), self.v.stride(0),
                                              self.rows, p(self.pos), p(self.slot), p(self.turned), self.turned.stride(0), stream))
        ok(self.jlib, L.jepa_amd_cache_digest(0, s, p(self.mem), self.n_seq, self.rows, p(self.start), p(self.len), p(self.table), self.width, p(self.digest), stream))
        ok(self.jlib, L.jepa_amd_cache_select(0, s, p(self.digest), kind, p(self.turned), self.turned.stride(0), self.n_seq, self.rows, p(self.start), p(self.len), p(self.table),
                                              self.width, 1, self.first, self.last, self.take, p(self.chosen), p(self.work), self.work.numel(), stream))
        ok(self.jlib, L.jepa_amd_cache_attention_selected(0, s, p(self.mem), kind, p(self.turned), self.turned.stride(0), self.n_seq, self.rows, p(self.start), p(self.len),
                                                          p(self.table), self.width, p(self.chosen), self.take, self.s.head_dim ** -0.5, 1, p(self.out), self.out.stride(0),
                                                          p(self.work2), self.work2.numel(), stream))

    def fresh(self, rng, new):
        self.new.copy_(ints(new))
        for t in (self.q, self.k, self.v):
            t.copy_(queries(rng, t.shape[0], t.shape[1], self.kind))
        self.pos.copy_(ints(rng.integers(0, 5000, tuple(self.pos.shape))))
        self.out.fill_(float("nan"))
        self.chosen.fill_(-9)

    def verify(self, new):
        """The step against the definitions, on what the cache and the digests hold."""
        assert self.refused.sum().item() == 0
        lens, start = self.len.tolist(), self.start.tolist()
        c = Cache.__new__(Cache)
        s = self.s
        c.__dict__.update(jlib=self.jlib, hd=s.head_dim, kvh=s.n_kv_head, heads=s.n_head, page=s.page_size, n_pages=s.n_pages, width=self.width, s=s, table=self.table.cpu().numpy(),
                          mem=self.mem, digest=self.digest.reshape(s.n_pages, s.n_kv_head, -1))
        where = [(i, lens[i] - (start[i + 1] - start[i]) + j) for i in range(self.n_seq) for j in range(start[i + 1] - start[i])]
        n, turned = start[-1], torch.full_like(self.q, float("nan"))
        ok(self.jlib, self.jlib.lib().jepa_amd_rope_rows(0, C.byref(self.axes), TYPES[self.kind][1], self.q.data_ptr(), self.q.stride(0), self.rows, s.n_head, self.pos.data_ptr(), 0,
                                                         turned.data_ptr(), turned.stride(0), None))
        assert torch.equal(turned, self.turned)
        # the keys and values that came
        k, v = (torch.empty(n, s.n_kv_head * s.head_dim, device="cuda") for _ in range(2))
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_read(0, C.byref(s), self.mem.data_ptr(), self.slot.data_ptr(), n, 0, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), None))
        # half a step of q4_0 is a sixteenth of the block's largest value (7 / 8 of it on the far side: an eighth there), f16's scale 2^-11 of it
        err = (v - self.v[:n].float()).abs().unflatten(1, (-1, 32)).amax(-1)
        assert (err <= self.v[:n].float().abs().unflatten(1, (-1, 32)).amax(-1) * (0.125 + 2.0 ** -10)).all()
        keys = next(c.read()).cpu().numpy()
        for i, m in enumerate(new):
            for p in range(max(0, lens[i] - max(m, 0)) // c.page, -(-lens[i] // c.page)) if m > 0 else ():
                codes, scales, _ = digests(c, [c.table[i, p]])
                for h in range(c.kvh):
                    want, sc = box(keys[c.table[i, p], :min(c.page, lens[i] - p * c.page), h])
                    np.testing.assert_array_equal(codes[0, h], want)
                    assert scales[0, h] == sc
        chosen = self.chosen.cpu().numpy()
        np.testing.assert_array_equal(chosen[:n], choose(c, self.turned[:n], lens, where, 1, self.first, self.last, self.take))
        want, tol = definition(c, self.turned[:n], lens, where, chosen[:n], 1, s.head_dim ** -0.5, self.kind)
        near(self.out[:n], want, tol)
        assert torch.isnan(self.out[n:]).all() and (chosen[n:] == -9).all()


@pytest.mark.parametrize("kind,heads,kvh,hd,page,take", [("f32", 4, 4, 64, 16, 5), ("f16", 8, 2, 128, 32, 4), ("bf16", 3, 1, 32, 16, 6)])
def test_steps_together(jlib, kind, heads, kvh, hd, page, take):
    """Prompts, single tokens, drops, ends and new requests, step after step on a stream of the caller's."""
    rng = np.random.default_rng(hd)
    prog = Program(jlib, 4, heads, kvh, hd, page, 120, 30, 300, kind, take)
    side = torch.cuda.Stream()
    for new in ([140, 47, 0, 100], [1, 1, 1, 1], [5, -3, 90, 1], [-100, 1, 1, 1], [120, 1, -1000, 30], [1, 1, 70, 0], [0, 0, 0, 0], [1, -16, 1, 1]):
        prog.fresh(rng, new)
        torch.cuda.synchronize()
        prog.step(side.cuda_stream)
        side.synchronize()
        prog.verify(new)


def test_step_captured_and_replayed(jlib):
    """The whole step in a HIP graph, replayed with new lengths and rows while the program runs its own eager work between; two graphs at once."""
    rng = np.random.default_rng(21)
    progs, graphs, sides = [], [], [torch.cuda.Stream() for _ in range(2)]
    for side in sides:
        prog = Program(jlib, 3, 8, 2, 64, 16, 3000, 1100, 24, "f16", 7)
        prog.fresh(rng, [9, 0, 4])
        torch.cuda.synchronize()
        prog.step(side.cuda_stream)
        side.synchronize()
        prog.verify([9, 0, 4])
        prog.new.zero_()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            prog.step(side.cuda_stream)
        progs.append(prog)
        graphs.append(g)
    other = Program(jlib, 3, 8, 2, 64, 16, 200, 20, 24, "f16", 7)
    for new in ([8, 8, 8], [20, 2, 2], [1, 1, 1], [24, -3, 0], [22, 1, 1], [24, 0, 0], [-4, 5, 1], [24, 0, 0], [1, 1, 1]):
        for prog in progs:
            prog.fresh(rng, new)
        other.fresh(rng, [1, 2, 3])
        torch.cuda.synchronize()
        for g, side in zip(graphs, sides):
            with torch.cuda.stream(side):
                g.replay()
        other.step(None)
        torch.cuda.synchronize()
        for prog in progs:
            prog.verify(new)
    graphs.clear()


@pytest.mark.parametrize("hd,page,take", [(64, 16, 4), (128, 64, 1), (96, 32, 9), (32, 16, 200)])
def test_attention_of_few_bf16_rows_takes_values_as_they_are(jlib, hd, page, take):
    """Keys of zeros, so that all weights are the same power of two, and values that nearly cancel in pairs. What is left off: the output's rounding, half a step of
    bf16 (2^-8 relative), and the sum of `tokens` exact products in 32 bits with the weights' sum, its reciprocal and the product, (tokens + 4) 2^-24 of the sum of magnitudes."""
    rng = np.random.default_rng(33)
    n = take * page
    c = Cache(jlib, 2, 1, hd, page, [n], rng, fill=False)
    v = torch.tensor(rng.standard_normal((n // 2, 1, hd)).astype(np.float32), device="cuda")
    v = torch.cat([v, -v * (1 + 2.0 ** -9)], 1).reshape(n, hd)      # (a scale some steps of f16 further)
    slot = torch.tensor(c.table[0].astype(np.int64)[:, None] * page + np.arange(page), device="cuda").flatten()
    c.store(torch.zeros(n, hd, device="cuda"), v, slot)
    q = queries(rng, 1, 2 * hd, "bf16")
    got = c.attend(q, "bf16", [0, 1], [n], ints(np.arange(take)[None, None]), 1, hd ** -0.5).double().reshape(2, hd)
    held = list(c.read())[1].double()[torch.tensor(c.table[0].astype(np.int64), device="cuda"), :, 0].reshape(n, hd)
    want, A = held.mean(0), held.abs().mean(0)
    tol = want.abs() * 2.0 ** -8 + (n + 4) * 2.0 ** -24 * A * (1 + 2.0 ** -8) + 1e-38
    assert ((got - want).abs() <= tol).all(), ((got - want).abs() / tol).max()


@pytest.mark.parametrize("rows", [1, 600])
@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_select_sums_past_the_ends_of_f32(jlib, kind, rows):
    """Finite queries whose sum over the heads passes f32's largest value, and ones whose sums are all below 2^-100, score zero everywhere: the lowest pages. At
    either end, just inside, they are ranked as any others."""
    rng = np.random.default_rng(32)
    kvh, group, hd, page, take, n = 8, 2, 64, 16, 10, 3000
    c = Cache(jlib, kvh * group, kvh, hd, page, [n], rng, fill=False)
    random_digests(rng, c)
    start, where = rows_of([n], [rows])
    base = (rng.integers(-64, 65, (rows, kvh, group, hd)) / 64.0).astype(np.float32)
    base[..., 3] = 1.0      # its sum over the heads: 2
    zero = [*range(take - 1)]
    for power, ranked in ((126, True), (127, False), (-101, True), (-102, False)):
        q = torch.tensor(base * np.float32(2.0) ** power, device="cuda").reshape(rows, -1).to(TYPES[kind][0])
        assert torch.isfinite(q).all()
        got = c.select(q, kind, start, [n], 1, 0, 1, take).cpu().numpy()
        last = np.array([-(-visible(p, n, 1) // page) - 1 for _, p in where])
        if ranked:
            plain = torch.tensor(base, device="cuda").reshape(rows, -1).to(TYPES[kind][0])
            np.testing.assert_array_equal(got, choose(c, plain, [n], where, 1, 0, 1, take))
        else:
            assert (got[..., :-1] == zero).all() and (got[..., -1] == last[:, None]).all()


# ------------------------------------------------------------------------------------------------ steps of one prompt and many single tokens
@pytest.mark.parametrize("kind,hd,page,at", [("f16", 64, 16, 0), ("bf16", 128, 64, 30), ("f32", 32, 16, 63)])
def test_a_prompt_among_single_tokens(jlib, kind, hd, page, at):
    """A piece of a prompt and 63 single tokens in one call, a few sequences that get none among them: tiles of 16 rows that are 16 sequences', and of both kinds."""
    rng = np.random.default_rng(hd + at)
    kvh, group, take = 8, 2, 9
    lens = rng.integers(12 * page, 40 * page, 68).tolist()
    new = [1] * 68
    lens[at], new[at] = 60 * page + 5, 300
    for i in (5, 40, 41, 66):
        new[i] = 0
    c = Cache(jlib, kvh * group, kvh, hd, page, lens, rng)
    start, where = rows_of(lens, new)
    c.make_digest(start, [0] * 68, start[-1])
    assert not c.digest.any()
    random_digests(rng, c)
    others = c.digest.clone()
    c.make_digest(start, lens, start[-1])
    keys = next(c.read()).cpu().numpy()
    touched = [(i, p) for i, (m, r) in enumerate(zip(lens, new)) for p in range((m - r) // page, -(-m // page)) if r]
    pages = [c.table[i, p] for i, p in touched]
    codes, scales, _ = digests(c, pages)
    for n, (i, p) in enumerate(touched):
        for h in range(kvh):
            want, s = box(keys[pages[n], :min(page, lens[i] - p * page), h])
            np.testing.assert_array_equal(codes[n, h], want)
            assert scales[n, h] == s
    others[pages] = c.digest[pages]
    assert torch.equal(c.digest, others)
    q = queries(rng, start[-1], kvh * group * hd, kind)
    got = c.select(q, kind, start, lens, 1, 1, 2, take)
    np.testing.assert_array_equal(got.cpu().numpy(), choose(c, q, lens, where, 1, 1, 2, take))
    out = c.attend(q, kind, start, lens, got, 1, hd ** -0.5)
    some = [r for r, (i, _) in enumerate(where) if i != at] + list(range(start[at], start[at + 1], 50))
    want, tol = definition(c, q[some], lens, [where[r] for r in some], got[some].tolist(), 1, hd ** -0.5, kind)
    near(out[some], want, tol)


@pytest.mark.parametrize("kvh,group,rows", [(2, 5, 1), (8, 3, 400)])
@pytest.mark.parametrize("kind", list(TYPES))
def test_select_against_the_sum_over_heads(jlib, kind, kvh, group, rows):
    """The score as it is defined, head by head and dimension by dimension: the sum of max(q hi, q lo). Queries of small whole numbers whose positive and
    negative sums over the heads reach 127 are their own codes, so that both are the same whole number times the page's scale, rounded once."""
    rng = np.random.default_rng(31)
    hd, page, take, n = 96, 16, 12, 3000
    c = Cache(jlib, kvh * group, kvh, hd, page, [n], rng, fill=False)
    random_digests(rng, c)
    start, where = rows_of([n], [rows])
    x = rng.integers(-20, 21, (rows, kvh, group, hd))
    sums = np.where(x[:, :, 1:, 7] > 0, x[:, :, 1:, 7], 0).sum(-1)
    x[:, :, 0, 7] = 127 - sums      # dimension 7's positive sum: 127, which no other one's of `group` values passes
    x[:, :, 1:, 7] = np.maximum(x[:, :, 1:, 7], 0)
    assert np.abs(x).max() <= 127 and np.maximum(x, 0).sum(2).max() == 127 and np.minimum(x, 0).sum(2).min() >= -127
    q = torch.tensor(x.reshape(rows, -1).astype(np.float32), device="cuda").to(TYPES[kind][0])
    got = c.select(q, kind, start, [n], 1, 1, 1, take).cpu().numpy()
    d = c.digest.cpu().numpy()[c.table[0]]
    codes, scale = d[..., :2 * hd].view(np.int8).astype(np.int64), d[..., 2 * hd:2 * hd + 4].copy().view(np.float32)[..., 0]
    for r in range(0, rows, 13):
        see = -(-visible(where[r][1], n, 1) // page)
        for h in range(kvh):
            hi, lo = codes[1:see - 1, h, :hd], codes[1:see - 1, h, hd:]
            whole = sum(np.maximum(x[r, h, j] * hi, x[r, h, j] * lo).sum(-1) for j in range(group))
            score = (whole.astype(np.float64) * scale[1:see - 1, h].astype(np.float64)).astype(np.float32)      # (24 by 24 bits: exact in 64, rounded once)
            best = 1 + np.sort(np.argsort(-score, kind="stable")[:take - 2])
            np.testing.assert_array_equal(got[r, h], np.concatenate([[0], best, [see - 1]]))
