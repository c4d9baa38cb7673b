"""Rotary positions of several axes on the GPU (no counterpart in the reference but its tables): rows rotated and their gradients against the definition in
more than 64 bits, against differences, and against the library's own host tables; rows appended to the 4-bit cache against the same rows
rotated and stored by two calls, bit for bit.

Tolerance of an element x_a cos A -+ x_b sin A: with u = 2^-24, the cosine, the sine, both products and their sum are rounded to f32, so that x_a cos A is off by
2 u |x_a| (u of a cosine of 1 at most, u of the product), x_b sin A by 2 u |x_b|, the sum by u |out|; the angle, pos * rev with rev rounded to 64 bits
and the product rounded, is off by 2 * 2^-53 |A| and moves the element by that times |x_a| + |x_b|; the Taylor series by 2^-40 times the same. On top comes the output's own
rounding, eps_T / 2 |out|, and half its smallest step.
"""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
np = pytest.importorskip("numpy")

pytestmark = pytest.mark.gpu

TYPES = {"f32": (torch.float32, 0), "f16": (torch.float16, 1), "bf16": (torch.bfloat16, 30)}
SMALLEST = {"f32": 2.0 ** -149, "f16": 2.0 ** -24, "bf16": 2.0 ** -133}


def ok(jlib, rc):
    assert rc == 0, jlib.error_text()


def rotate(jlib, axes, x, pos, kind, back=False, out=None, heads=None, stream=None):
    """x [rows][heads * hd] (any row stride) -> rotated; out may be x."""
    out = torch.full((x.shape[0], x.shape[1]), float("nan"), dtype=x.dtype, device="cuda") if out is None else out
    heads = x.shape[1] // axes.head_dim if heads is None else heads
    ok(jlib, jlib.lib().jepa_amd_rope_rows(0, C.byref(axes), TYPES[kind][1], x.data_ptr(), x.stride(0), x.shape[0], heads, pos.data_ptr(), int(back), out.data_ptr(),
                                           out.stride(0), stream))
    return out


def pairs(form, dims):
    """(a, b, axis, frequency index of a, of b, width) of every pair."""
    at, total = 0, sum(dims)
    for axis, w in enumerate(dims):
        for i in range(w // 2):
            if form == 0:
                yield at + 2 * i, at + 2 * i + 1, axis, 2 * i % (w // 2), (2 * i + 1) % (w // 2), w
            elif form == 1:
                yield at + 2 * i, at + 2 * i + 1, axis, i, i, w
            elif form == 2:
                yield at + i, at + i + w // 2, axis, i, i, w
            else:
                yield at // 2 + i, at // 2 + i + total // 2, axis, at // 2 + i, at // 2 + i, total
        at += w


def definition(x, pos, form, dims, theta, scale, back, kind):
    """x [rows][heads][hd] f64, pos [rows][axes] -> (out, tolerance)."""
    out, u = x.copy(), 2.0 ** -24
    eps = torch.finfo(TYPES[kind][0]).eps / 2
    tol = np.zeros_like(x)
    for a, b, axis, fa, fb, w in pairs(form, dims):
        ang = [pos[:, axis].astype(np.longdouble) * np.longdouble(scale[axis]) * np.longdouble(theta) ** (np.longdouble(-2 * f) / w) for f in (fa, fb)]
        ca, cb, sa, sb = (f(t).astype(np.float64)[:, None] for f in (np.cos, np.sin) for t in ang)
        xa, xb = x[..., a], x[..., b]
        out[..., a], out[..., b] = (xa * ca + xb * sb, xb * cb - xa * sa) if back else (xa * ca - xb * sa, xb * cb + xa * sb)
        off = 2 * u + 2.0 ** -40 + 2.0 ** -52 * np.maximum(np.abs(ang[0]), np.abs(ang[1])).astype(np.float64)[:, None]
        for e in (a, b):
            tol[..., e] = off * (np.abs(xa) + np.abs(xb)) + (u + eps) * np.abs(out[..., e]) + SMALLEST[kind]
    return out, tol


def given(rng, rows, heads, hd, kind):
    return torch.tensor(rng.standard_normal((rows, heads * hd)), dtype=TYPES[kind][0], device="cuda")


def check(got, x, pos, form, dims, theta, scale, back, kind, hd):
    want, tol = definition(x.double().cpu().numpy().reshape(x.shape[0], -1, hd), pos.cpu().numpy(), form, dims, theta, scale, back, kind)
    got = got.double().cpu().numpy().reshape(want.shape)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (np.argwhere(bad)[:5], got[bad][:5], want[bad][:5], tol[bad][:5])


# form, head width, dims: the repository's own 3-axis sections (20 of 64, 28 of 88), sections that end inside 8 elements, one pair, whole heads
LAYOUTS = [(0, 64, (20, 20, 20)), (0, 88, (28, 28, 28)), (0, 8, (2, 2, 2)), (0, 32, (10, 6)), (1, 64, (20, 20, 20)), (1, 80, (26, 26, 26)), (1, 128, (128,)), (1, 16, (2,)),
           (1, 256, (64, 64, 64, 64)), (1, 24, (6, 10, 4, 2)), (2, 128, (32, 48, 48)), (2, 64, (16, 16)), (2, 256, (16, 112, 32, 96)), (2, 16, (16,)), (3, 128, (32, 48, 48)),
           (3, 64, (64,)), (3, 96, (2, 6, 8)), (3, 256, (100, 60, 80)), (3, 32, (10, 14, 6, 2))]


@pytest.mark.parametrize("back", [False, True])
@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("form,hd,dims", LAYOUTS)
def test_rotation(jlib, form, hd, dims, kind, back):
    rng = np.random.default_rng(hd * 4 + form)
    for rows, heads, far in ((1, 1, 3), (7, 5, 1000), (37, 3, 1 << 20), (300, 17, 70000)):
        scale = [1.0, 15 / 23, -0.5, 2.0][:len(dims)]
        axes = jlib.RopeAxes.of(hd, form, dims, 10000.0, scale)
        x = given(rng, rows, heads, hd, kind)
        pos = torch.tensor(rng.integers(-far, far + 1, (rows, len(dims))), dtype=torch.int32, device="cuda")
        check(rotate(jlib, axes, x, pos, kind, back), x, pos, form, dims, 10000.0, scale, back, kind, hd)


@pytest.mark.parametrize("theta", [1e4, 1e6, 0.01])
def test_far_positions(jlib, theta):
    """Positions at the ends of int32, and angles that are whole quarters but for their rounding (position 710 is 113 turns and 6e-5)."""
    rng = np.random.default_rng(3)
    pos = torch.tensor([[2 ** 31 - 1, -2 ** 31], [-2 ** 31, 0], [0, 2 ** 31 - 1], [710, -710], [355, 44], [1, -1], [1 << 30, 12345678]], dtype=torch.int32, device="cuda")
    x = given(rng, 7, 2, 64, "f32")
    dims, scale = (40, 24), (1.0, 1.0)
    if theta < 1:
        scale = (2.0 ** -20, 2.0 ** -20)      # (frequencies rise with the index here)
    check(rotate(jlib, jlib.RopeAxes.of(64, 1, dims, theta, scale), x, pos, "f32"), x, pos, 1, dims, theta, scale, False, "f32", 64)


@pytest.mark.parametrize("form,hd,dims", [(0, 64, (20, 20, 20)), (1, 24, (6, 10)), (2, 64, (32, 16)), (3, 64, (20, 12))])
def test_gradient_against_differences(jlib, form, hd, dims):
    """The rotation is linear in x: d(sum_j y_j x'_j) / dx_e by a step of one is what the gradient of y gives, to both sides' rounding."""
    rng = np.random.default_rng(form)
    axes = jlib.RopeAxes.of(hd, form, dims)
    pos = torch.tensor(np.tile(rng.integers(0, 500, (1, len(dims))), (hd + 1, 1)), dtype=torch.int32, device="cuda")
    x = given(rng, 1, 1, hd, "f32")
    steps = torch.cat([x, x + torch.eye(hd, device="cuda")])
    step = (steps[1:] - x).double().diagonal()      # as they came out in f32
    y = given(rng, 1, 1, hd, "f32")
    z = rotate(jlib, axes, steps, pos, "f32").double() @ y.double()[0]
    got = rotate(jlib, axes, y, pos[:1].contiguous(), "f32", back=True).double()[0]
    # each side's elements are off by 6 u of the pair's values (above): hd of them by |y|, and one
    tol = 6 * 2.0 ** -24 * 2 * (y.abs().max() * (steps.abs().max() + 1)) * hd
    assert ((z[1:] - z[0]) / step - got).abs().max() <= tol


@pytest.mark.parametrize("form", [0, 1, 2, 3])
@pytest.mark.parametrize("kind", list(TYPES))
def test_in_place_strided_and_neighbours(jlib, form, kind):
    """Rows inside wider ones, in place and into others: the same bits, and nothing beside the heads is touched."""
    rng = np.random.default_rng(form)
    hd, heads, dims = 64, 5, (16, 32)
    axes = jlib.RopeAxes.of(hd, form, dims)
    wide = given(rng, 33, heads + 3, hd, kind)
    pos = torch.tensor(rng.integers(0, 900, (33, 2)), dtype=torch.int32, device="cuda")
    x = wide[:, hd:(1 + heads) * hd]
    want = rotate(jlib, axes, x.contiguous(), pos, kind)
    other = torch.full((33, (heads + 1) * hd), 7.0, dtype=wide.dtype, device="cuda")
    rotate(jlib, axes, x, pos, kind, out=other[:, :heads * hd])
    assert torch.equal(other[:, :heads * hd], want) and (other[:, heads * hd:] == 7).all()
    before = wide.clone()
    rotate(jlib, axes, x, pos, kind, out=x)
    assert torch.equal(wide[:, hd:(1 + heads) * hd], want)
    assert torch.equal(wide[:, :hd], before[:, :hd]) and torch.equal(wide[:, (1 + heads) * hd:], before[:, (1 + heads) * hd:])


@pytest.mark.parametrize("form,dims", [(0, (6, 14)), (1, (6, 14)), (2, (16,)), (3, (10, 6))])
def test_elements_that_do_not_turn_and_not_finite_ones(jlib, form, dims):
    """The rest of a head comes out bit for bit, whatever is in it; a NaN stays in its pair."""
    hd = 32
    axes = jlib.RopeAxes.of(hd, form, dims)
    x = torch.linspace(-1, 1, 3 * hd, device="cuda").reshape(3, hd)
    rest = sum(dims)
    x[0, rest], x[1, rest + 1], x[2, rest + 2], x[2, rest + 3] = float("nan"), float("inf"), -0.0, 1e-42
    a, b = next(iter(pairs(form, dims)))[:2]
    x[1, a] = float("nan")
    pos = torch.full((3, len(dims)), 5, dtype=torch.int32, device="cuda")
    got = rotate(jlib, axes, x, pos, "f32")
    assert torch.equal(got[:, rest:].view(torch.int32), x[:, rest:].view(torch.int32))
    nan = torch.isnan(got[:, :rest])
    assert nan[1, a] and nan[1, b] and nan.sum() == 2


@pytest.mark.parametrize("variant", [0, 1])
def test_the_encoder_tables_rotation(jlib, variant):
    """Forms 0 and 1 are the rotations of the library's host tables (reference src/rope3d.cpp:9-134), with the 2.1 interpolation as the axes' scales. The
    tables' angles are f32 products of an f32 frequency: off by 3 * 2^-24 of an angle below 24, which is up to 24 * 3 u of a pair's values."""
    hd, grid, train = 64, (3, 24, 23), (16, 16)
    n = grid[0] * grid[1] * grid[2]
    c, s = (np.empty((n, hd), np.float32) for _ in range(2))
    L = jlib.lib()
    L.jepa_amd_rope_tables.argtypes = [C.c_int] * 8 + [C.c_float, C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_void_p]
    ok(jlib, L.jepa_amd_rope_tables(hd, *grid, variant, 1, *train, 10000.0, None, n, 1, c.ctypes.data, s.ctypes.data))
    rng = np.random.default_rng(0)
    x = given(rng, n, 1, hd, "f32")
    t = np.arange(n)
    pos = torch.tensor(np.stack([t // (24 * 23), t // 23 % 24, t % 23], 1), dtype=torch.int32, device="cuda")
    got = rotate(jlib, jlib.RopeAxes.of(hd, variant, (20, 20, 20), 10000.0, (1.0, 15 / 23, 15 / 22)), x, pos, "f32").cpu().double().numpy()
    v = x.cpu().double().numpy()
    swapped = v.reshape(n, -1, 2)[..., ::-1].reshape(n, hd)
    want = v * c + swapped * s
    assert np.abs(got - want).max() <= (24 * 3 + 6) * 2.0 ** -24 * (np.abs(v) + np.abs(swapped)).max()


def test_no_rows_other_streams_and_replays(jlib):
    rng = np.random.default_rng(5)
    axes = jlib.RopeAxes.of(64, 3, (32, 16, 16))
    x, pos = given(rng, 40, 6, 64, "bf16"), torch.tensor(rng.integers(0, 5000, (40, 3)), dtype=torch.int32, device="cuda")
    ok(jlib, jlib.lib().jepa_amd_rope_rows(0, C.byref(axes), 30, None, 64, 0, 1, None, 0, None, 64, None))
    want = rotate(jlib, axes, x, pos, "bf16")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    rotate(jlib, axes, x, pos, "bf16", out=out, stream=side.cuda_stream)
    side.synchronize()
    assert torch.equal(out, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        rotate(jlib, axes, x, pos, "bf16", out=out, stream=side.cuda_stream)
    for i in range(3):
        x.copy_(given(rng, 40, 6, 64, "bf16"))
        pos.copy_(torch.tensor(rng.integers(0, 5000, (40, 3)), dtype=torch.int32, device="cuda"))
        want = rotate(jlib, axes, x, pos, "bf16")
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    del g


# ------------------------------------------------------------------------------------------------ append
class Cache:
    def __init__(self, jlib, heads, kvh, hd, page, n_pages):
        self.jlib, self.s = jlib, jlib.CacheShape(heads, kvh, hd, page, n_pages)
        self.mem = torch.full((n_pages * jlib.lib().jepa_amd_cache_page_bytes(C.byref(self.s)),), 0x5a, dtype=torch.uint8, device="cuda")

    def store(self, k, v, slot, kind):
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_store(0, C.byref(self.s), self.mem.data_ptr(), TYPES[kind][1], k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0),
                                                           k.shape[0], slot.data_ptr(), None))

    def append(self, axes, q, k, v, pos, slot, kind, out=None, stream=None):
        ok(self.jlib, self.jlib.lib().jepa_amd_cache_append(0, C.byref(self.s), C.byref(axes), self.mem.data_ptr(), TYPES[kind][1], q.data_ptr() if q is not None else None,
                                                            q.stride(0) if q is not None else 0, k.data_ptr(), k.stride(0), v.data_ptr(), v.stride(0), k.shape[0],
                                                            pos.data_ptr(), slot.data_ptr(), out.data_ptr() if q is not None else None,
                                                            out.stride(0) if q is not None else 0, stream))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("form,hd,dims", [(0, 64, (20, 20, 20)), (1, 96, (30, 34, 32)), (2, 128, (32, 48, 48)), (3, 128, (32, 48, 48)), (3, 32, (6, 10)), (0, 32, (10, 6)),
                                          (2, 96, (16, 64)), (1, 64, (64,)), (3, 96, (90, 6)), (2, 32, (16,))])
def test_append_is_rotate_and_store(jlib, form, hd, dims, kind):
    rng = np.random.default_rng(hd + form)
    axes = jlib.RopeAxes.of(hd, form, dims, 1e6, [1.0, 0.5, 2.0][:len(dims)])
    for rows, kvh, group, page in ((1, 1, 1, 16), (5, 3, 2, 32), (70, 2, 4, 16), (600, 8, 1, 64), (3000, 5, 3, 16)):
        n_pages = -(-rows // page) * 2 + 1
        a, b = (Cache(jlib, kvh * group, kvh, hd, page, n_pages) for _ in range(2))
        x = given(rng, rows, kvh * (group + 2), hd, kind)
        q, k, v = x[:, :kvh * group * hd], x[:, kvh * group * hd:kvh * (group + 1) * hd], x[:, kvh * (group + 1) * hd:]
        pos = torch.tensor(rng.integers(0, 100000, (rows, len(dims))), dtype=torch.int32, device="cuda")
        slot = torch.tensor(rng.permutation(n_pages * page)[:rows], device="cuda")
        slot[rng.random(rows) < 0.1] = -1
        if rows > 4:
            slot[3] = n_pages * page
            k[2, hd // 2], v[4, 1] = float("nan"), float("inf")
        out = torch.full((rows, kvh * group * hd + 64), 3.0, dtype=x.dtype, device="cuda")
        a.append(axes, q, k, v, pos, slot, kind, out)
        # the definition rounds nothing between the rotation and the quantizer: both in f32
        b.store(rotate(jlib, axes, k.float(), pos, "f32"), v.float(), slot, "f32")
        assert torch.equal(a.mem, b.mem)
        assert torch.equal(out[:, :kvh * group * hd], rotate(jlib, axes, q, pos, kind)) and (out[:, kvh * group * hd:] == 3).all()
        # keys and values alone, and queries in place
        a.mem.fill_(0x5a)
        a.append(axes, None, k, v, pos, slot, kind)
        assert torch.equal(a.mem, b.mem)
        want = rotate(jlib, axes, q, pos, kind)
        a.append(axes, q, k, v, pos, slot, kind, q)
        assert torch.equal(a.mem, b.mem) and torch.equal(q, want)


def test_append_no_rows(jlib):
    c = Cache(jlib, 2, 1, 32, 16, 2)
    ok(jlib, jlib.lib().jepa_amd_cache_append(0, C.byref(c.s), C.byref(jlib.RopeAxes.of(32, 1, (32,))), c.mem.data_ptr(), 0, None, 0, None, 32, None, 32, 0, None, None,
                                              None, 0, None))
    torch.cuda.synchronize()
    assert (c.mem == 0x5a).all()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("form,hd,dims,partner", [(0, 96, (30, 34, 32), 1), (1, 96, (30, 34, 32), 1), (2, 96, (16, 64), 8), (3, 96, (90, 6), 48), (2, 64, (16, 32), 8), (3, 32, (10, 6), 8)])
def test_append_rows_do_not_touch_each_other(jlib, form, hd, dims, partner, kind):
    """A NaN or an infinity in the first row's first elements, in the partners they turn with or in its values, stored or not: its own head is stored as none, every
    other row as if it stood alone (heads of 96 leave lanes of a row without work)."""
    rng = np.random.default_rng(hd * 4 + form)
    axes = jlib.RopeAxes.of(hd, form, dims, 1e4)
    rows, kvh, page = 37, 3, 16
    given_k, given_v = given(rng, rows, kvh, hd, kind), given(rng, rows, kvh, hd, kind)
    pos = torch.tensor(rng.integers(0, 1000, (rows, len(dims))), dtype=torch.int32, device="cuda")
    for of_v, at, bad in ((False, 0, "nan"), (False, partner, "inf"), (True, 5, "-inf"), (True, 0, "nan")):
        for stored in (True, False):
            k, v = given_k.clone(), given_v.clone()
            (v if of_v else k)[0, hd + at] = float(bad)      # of head 1
            slot = torch.arange(rows, device="cuda")
            if not stored:
                slot[0] = -1
            a, b = (Cache(jlib, kvh, kvh, hd, page, 3) for _ in range(2))
            a.append(axes, None, k, v, pos, slot, kind)
            b.store(rotate(jlib, axes, k.float(), pos, "f32"), v.float(), slot, "f32")
            got_k, got_v = (torch.zeros(rows, kvh * hd, device="cuda") for _ in range(2))
            ok(jlib, jlib.lib().jepa_amd_cache_read(0, C.byref(a.s), a.mem.data_ptr(), slot.data_ptr(), rows, 0, got_k.data_ptr(), got_k.stride(0), got_v.data_ptr(),
                                                    got_v.stride(0), None))
            odd = torch.isnan(got_k).reshape(rows, kvh, hd)
            assert not odd[1:].any(), f"{int(odd[1:].any(-1).sum())} heads of other rows, {at} of {'v' if of_v else 'k'} {bad}, stored {stored}"
            assert odd[0, 1].all() == stored and not odd[0, ::2].any()
            assert torch.equal(a.mem, b.mem)
