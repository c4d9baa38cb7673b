"""The 4-bit paged cache's rows on the GPU, beside test_gpu_cache: the bytes that a store leaves, against the quantizer whose blocks they are
said to be, and rows at the least alignment that the calls take. No counterpart in the reference."""
import pytest

import test_gpu_cache as base

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
np = pytest.importorskip("numpy")


def blocks_in(p, slots, hd, kvh, page):
    """(scales' bits [rows][kvh][blocks], codes [rows][kvh][hd]) of K and of V, read from the layout's bytes."""
    raw, nb = p.cache.cpu().numpy().reshape(-1, kvh, page // 16, 18 * hd), hd // 32
    out = []
    for which in "kv":
        d, c = np.zeros((len(slots), kvh, nb), np.uint16), np.zeros((len(slots), kvh, hd), np.uint8)
        for r, slot in enumerate(slots):
            t = slot % 16
            strips = raw[slot // page, :, slot % page // 16]
            for b in range(nb):
                at = 16 * hd + 2 * ((t // 4 * nb + b) * 4 + t % 4) + (hd if which == "v" else 0)
                d[r, :, b] = strips[:, at] | (strips[:, at + 1].astype(np.uint16) << 8)
            for w in range(hd // 8):
                b, g = w // 4, w % 4
                at = ((g * 16 + t) * nb + b) * 4 if which == "k" else 8 * hd + t * (hd // 2) + 4 * w
                for n in range(8):
                    e = (n % 4) * 2 + n // 4 if which == "k" else n
                    c[r, :, 8 * w + e] = strips[:, at + n // 2] >> (4 * (n % 2)) & 15
        out.append((d, c))
    return out


@pytest.mark.parametrize("kind", list(base.TYPES))
@pytest.mark.parametrize("hd,kvh,page", [(32, 3, 16), (64, 2, 32), (96, 1, 16), (128, 2, 64)])
def test_bytes_are_the_quantizers(jlib, hd, kvh, page, kind):
    """Scales and codes bit for bit as jepa_amd_quantize_rows makes them, zeros of both signs and the least magnitudes among them."""
    rng = np.random.default_rng(hd)
    n = 40
    dtype, code = base.TYPES[kind]
    rows = []
    for _ in range(2):
        x = base.special_rows(rng, n, kvh * hd)
        x[7], x[8, 0::2], x[9, 1::2], x[9, 0::2] = -0.0, -0.0, -0.0, 0.0      # all, then the first, then the second of a zero block
        x[8, 1::2] = 0.0
        x[10] = rng.choice([-0.0, 0.0], kvh * hd)
        x[11, 0], x[11, 1:] = -0.0, np.float32(1e-30)
        x[12] *= 2.0 ** -22
        x[13] *= 1e-7
        rows.append(torch.from_numpy(x).to(dtype).cuda())
    p = base.Pool(jlib, kvh, kvh, hd, page, 6)
    slots = rng.permutation(6 * page)[:n]
    torch.cuda.synchronize()
    p.store(rows[0], rows[1], base.ints(slots, torch.int64), kind)
    torch.cuda.synchronize()
    for name, x, (d, c) in zip("kv", rows, blocks_in(p, slots, hd, kvh, page)):
        x, raw = x.float(), torch.empty(n * kvh * hd // 32, 18, dtype=torch.uint8, device="cuda")
        torch.cuda.synchronize()
        base.ok(jlib, jlib.lib().jepa_amd_quantize_rows(0, 2, x.data_ptr(), x.numel(), raw.data_ptr()))
        torch.cuda.synchronize()
        raw = raw.cpu().numpy()
        np.testing.assert_array_equal(d.reshape(-1), raw[:, 0] | (raw[:, 1].astype(np.uint16) << 8), err_msg=name + " scales")
        np.testing.assert_array_equal(c.reshape(-1, 32), np.concatenate([raw[:, 2:] & 15, raw[:, 2:] >> 4], 1), err_msg=name + " codes")


@pytest.mark.parametrize("kind", list(base.TYPES))
@pytest.mark.parametrize("rows", [3, 400])
@pytest.mark.parametrize("hd,kvh,group", [(64, 2, 2), (96, 1, 3), (128, 1, 1), (32, 3, 1)])
def test_rows_at_odd_multiples_of_16_bytes(jlib, hd, kvh, group, rows, kind):
    """Start and stride of every row array 16 bytes past a multiple of 32: the same as from rows side by side."""
    dtype, code = base.TYPES[kind]
    step = 16 // torch.empty(0, dtype=dtype).element_size()      # elements of 16 bytes
    rng = np.random.default_rng(rows + hd)

    def apart(x):
        wide = torch.full((x.shape[0], (x.shape[1] // (2 * step) + 1) * 2 * step + 3 * step), 7.0, dtype=dtype, device="cuda")
        out = wide[:, step:step + x.shape[1]]
        assert out.data_ptr() % 32 == 16 and out.stride(0) * out.element_size() % 32 == 16
        out.copy_(x)
        return out, wide

    p = base.Pool(jlib, kvh * group, kvh, hd, 16, rows // 16 + 1)
    k, v = (base.queries(rng, rows, kvh * hd, kind) for _ in range(2))
    slot = torch.arange(rows, device="cuda")
    p.store(k, v, slot, kind)
    want = p.read(slot, kind)
    p.cache.fill_(0xff)
    (ka, _), (va, _) = apart(k), apart(v)
    torch.cuda.synchronize()
    p.store(ka, va, slot, kind)
    (kr, kw), (vr, vw) = apart(torch.zeros_like(k)), apart(torch.zeros_like(v))
    torch.cuda.synchronize()
    base.ok(jlib, jlib.lib().jepa_amd_cache_read(0, base.C.byref(p.s), p.cache.data_ptr(), slot.data_ptr(), rows, code, kr.data_ptr(), kr.stride(0), vr.data_ptr(),
                                                 vr.stride(0), None))
    torch.cuda.synchronize()
    q = base.queries(rng, rows, kvh * group * hd, kind)
    (qa, _), (oa, ow) = apart(q), apart(torch.zeros_like(q))
    table = base.ints(np.arange(rows // 16 + 1)[None])
    out = p.attend(q, base.ints([0, rows]), base.ints([rows]), table, kind)
    p.attend(qa, base.ints([0, rows]), base.ints([rows]), table, kind, out=oa)
    torch.cuda.synchronize()
    for got, wide, exact in ((kr, kw, want[0]), (vr, vw, want[1]), (oa, ow, out)):
        assert torch.equal(got, exact) and not torch.isnan(got).any()
        assert (wide[:, :step] == 7).all() and (wide[:, step + got.shape[1]:] == 7).all()
