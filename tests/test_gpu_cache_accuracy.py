"""Accuracy of attention over the 4-bit paged cache (no counterpart in the reference) where values differ by large factors: among the
tokens that a row reads, from one block of the head to another, and in tokens that it must not read. Against the definition in 64 bits
on the values that the cache holds, with the calls of test_gpu_cache.

Tolerance for one row, head and dimension n, out_n = sum_j p_j v_jn over the keys j that the row reads, A_n = sum_j p_j |v_jn| and
N_n = sum_j |v_jn|:
  the output's own rounding   eps_T / 2 |out_n| (half a step of its type), and half its smallest step
  a value                     enters exactly: a code (4 bits) times its f16 scale (11) is the sum of two f16
  a weight                    16-bit rows: one f16, half a step 2^-11 relative. f32 rows: two f16, 2^-22, and the product of both low terms
                              that is left out, 2^-11 2^-11; with the 32-bit exponential and sums 2^-20 in all.
                              The largest is brought to 2^10 or more, so half of f16's smallest step, 2^-25, is 2^-35 of the largest, which is at
                              most their sum: 2^-35 N_n for both. (The sum that divides is of the same rounded weights, so a weight's error
                              counts with v_jn - out_n instead of v_jn: at most A_n + |out_n| in all, and about A_n where the errors of many
                              keys have no common sign. A_n is asked for.)
  scores                      head_dim products of a query held to 2^-22 and an exact key in 32 bits, times a scale: off by at most
                              (head_dim / 8 + 8) 2^-22 S, S = max_j scale |q|max |k_j|_1, on both sides of the fraction (e^x ~ 1 + x): twice that,
                              times A_n. The queries here are small, so that this is not what decides.
  bf16 rows, where many share the keys: keys and values rounded to f16, 2^-11 relative: 2^-11 A_n for the values, 2^-11 S1 on both
                              sides for the scores, S1 = max_j scale sum_n |q_n| |k_jn|; and a value below f16's normal range, 2^-14, is
                              off by 2^-25 at most (an exact multiple of 2^-24 there, so by nothing).
"""
import pytest

import test_gpu_cache as base

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")
np = pytest.importorskip("numpy")

KINDS = list(base.TYPES)
# (rows of a sequence as long as they are, K/V heads, heads of each, head width): the first three have few columns a sequence, the others many
SHAPES = [(150, 2, 1, 64), (90, 1, 3, 128), (130, 1, 1, 96), (1000, 2, 1, 64), (500, 1, 4, 128), (300, 1, 3, 96), (420, 1, 2, 32)]


def definition(p, q, n, table, scale, kind):
    """(out, tolerance) [rows][heads][head_dim] of the last rows of one causal sequence of n tokens."""
    hd, kvh, heads = p.s.head_dim, p.s.n_kv_head, p.s.n_head
    rows, group = q.shape[0], heads // kvh
    t = torch.arange(n, device="cuda")
    k, v = (x.double().reshape(n, kvh, hd) for x in p.read(torch.as_tensor(table[0], device="cuda").long()[t // p.s.page_size] * p.s.page_size + t % p.s.page_size))
    hidden = t > (n - rows + torch.arange(rows, device="cuda"))[:, None]
    out, tol = (torch.empty(rows, heads, hd, dtype=torch.float64, device="cuda") for _ in range(2))
    for h in range(heads):
        x, kh, vh = q[:, h * hd:(h + 1) * hd].double(), k[:, h // group], v[:, h // group]
        w = torch.softmax((x @ kh.T.contiguous() * scale).masked_fill(hidden, float("-inf")), -1)
        seen = (~hidden).double()
        y, A, N = w @ vh, w @ vh.abs(), seen @ vh.abs()
        S = scale * x.abs().amax(-1, keepdim=True) * kh.abs().sum(-1).max()
        f = 2.0 ** -20 + 2 * (hd / 8 + 8) * 2.0 ** -22 * S
        if kind != "f32":
            f = f + 2.0 ** -11
        if kind == "bf16":
            f = f + 2.0 ** -11 * (1 + 2 * scale * (x.abs() @ kh.abs().T.contiguous()).amax(-1, keepdim=True))
        out[:, h] = y
        tol[:, h] = torch.finfo(base.TYPES[kind][0]).eps / 2 * y.abs() * (1 + f) + f * A + 2.0 ** -35 * N + (2.0 ** -25 if kind == "f16" else 1e-38)
    return out, tol


class Sequence:
    """One sequence of n tokens, its values as a test wants them."""

    def __init__(self, jlib, seed, n, kvh, group, hd):
        rng = np.random.default_rng(seed)
        self.p, self.table = base.filled(jlib, rng, kvh * group, kvh, hd, 32, [n])
        self.slot = base.ints([int(self.table[0, t // 32]) * 32 + t % 32 for t in range(n)], torch.int64)
        self.k, self.v = self.p.read(self.slot)
        self.n, self.rng, self.width, self.scale = n, rng, kvh * group * hd, hd ** -0.5

    def set(self, k, v):
        torch.cuda.synchronize()
        self.p.store(k, v, self.slot, "f32")
        torch.cuda.synchronize()

    def run(self, q, kind):
        got = self.p.attend(q, base.ints([0, q.shape[0]]), base.ints([self.n]), base.ints(self.table), kind, 1, self.scale)
        torch.cuda.synchronize()
        return got.reshape(q.shape[0], -1, self.p.s.head_dim)

    def check(self, q, kind):
        got = self.run(q, kind)
        want, tol = definition(self.p, q, self.n, self.table, self.scale, kind)
        off = (got.double() - want).abs()
        assert not torch.isnan(got).any() and (off <= tol).all(), f"off by {(off / tol).max().item():.3g} of the tolerance at {torch.argmax(off / tol).item()}"
        return got


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,kvh,group,hd", SHAPES)
def test_a_later_token_changes_nothing(jlib, rows, kvh, group, hd, kind):
    """Whatever lies in a token that a row must not read, its output has the same bits, and the accuracy of one without it."""
    s = Sequence(jlib, rows + hd, rows, kvh, group, hd)
    q = base.queries(s.rng, rows, s.width, kind, 0.02)
    for size in (1e-3, 1e-2, 1.0):
        for at in (40, rows - 5):
            s.set(s.k, s.v * size)
            before = s.check(q, kind)
            for k, v in ((1.0, 6e4), (300.0, 1e3), (1.0, 0.0), (1.0, float("nan"))):
                kk, vv = s.k.clone(), s.v * size
                kk[at] *= k
                vv[at] *= v
                s.set(kk, vv)
                got = s.run(q, kind)
                assert torch.equal(got[:at], before[:at]), (size, at, k, v)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,kvh,group,hd", SHAPES)
def test_blocks_of_very_different_size(jlib, rows, kvh, group, hd, kind):
    """Values of one block of 32 dimensions many times larger than the next one's."""
    s = Sequence(jlib, rows + hd + 1, rows, kvh, group, hd)
    q = base.queries(s.rng, rows, s.width, kind, 0.02)
    for sizes in ((1.0, 1e4, 1e-1, 1e3), (1e4, 1e-2, 1.0, 1e-1), (1e-2, 1.0, 1e4, 1e-2)):
        f = torch.tensor([sizes[b % 4] for b in range(kvh * hd // 32)], device="cuda").repeat_interleave(32)
        s.set(s.k, s.v * f)
        s.check(q, kind)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,kvh,group,hd", SHAPES)
def test_values_that_grow_along_the_sequence(jlib, rows, kvh, group, hd, kind):
    """Rows at every place of a sequence whose values grow, shrink, or stand out at a few tokens by factors of up to 10^6."""
    s = Sequence(jlib, rows + hd + 2, rows, kvh, group, hd)
    q = base.queries(s.rng, rows, s.width, kind, 0.02)
    grow = torch.exp(torch.linspace(-7, 7, rows, device="cuda"))[:, None]
    some = torch.where(torch.arange(rows, device="cuda") % 61 == 37, 3e4, 0.03)[:, None]
    for f in (grow, grow.flip(0), some):
        s.set(s.k, s.v * f)
        s.check(q, kind)


@pytest.mark.parametrize("rows", [1, 1000])
def test_means_of_the_largest_f16_stay_finite(jlib, rows):
    """Every value +-65504: a mean of them is that, whatever the weights round to. One token of 64 has the largest weight,
    and the others' common one takes 64 places between two powers of two."""
    n = 1000
    s = Sequence(jlib, 5, n, 1, 1, 64)
    k, v = torch.zeros(n, 64, device="cuda"), torch.full((n, 64), 1e6, device="cuda")
    k[7::64, 0] = -8.0      # a q4_0 block of its largest value and zeros: exact
    v[:, 32:] = -1e6      # (a q4_0 block reaches its largest magnitude on one side only)
    s.set(k, v)
    q = torch.zeros(rows, 64, dtype=torch.float16, device="cuda")
    q[:, 0] = -1.0
    want = torch.tensor([65504.0] * 32 + [-65504.0] * 32, device="cuda")
    for i in range(64):
        got = s.p.attend(q, base.ints([0, rows]), base.ints([n]), base.ints(s.table), "f16", 0, np.log(2.0) / 8 * (1 + i / 64))
        torch.cuda.synchronize()
        assert ((got.float() - want).abs() <= 32).all(), i      # (a step of f16 there)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,kvh,group,hd", SHAPES)
def test_queries_with_one_large_element(jlib, rows, kvh, group, hd, kind):
    """An element of the query 2^13 to 2^19 times the others' size, which meets keys that are 0 there: the others decide the scores, and
    count with their own bits.

    Tolerance: one score is a sum of products of exact keys and a query held to 2^-22 of each element (16-bit rows: exactly) or half of
    f16's smallest step where the row's largest element is 2^14, 2^-39 of that: off by Q = scale sum_n |k_n| (2^-22 |q_n| + 2^-39 |q|max) and the 32-bit
    sums' (head_dim / 8 + 8) 2^-22 of S1 = max_j scale sum_n |q_n| |k_jn|, on both sides of the fraction; the rest as above."""
    s = Sequence(jlib, rows + hd + 3, rows, kvh, group, hd)
    s.k[:, ::hd] = 0.0
    s.set(s.k, s.v)
    s.k, s.v = s.p.read(s.slot)
    assert (s.k[:, ::hd] == 0).all()
    for large in (2.0 ** 9, 2.0 ** 13, 2.0 ** 15 - 16):
        q = base.queries(s.rng, rows, s.width, kind, 0.06)
        q[:, ::hd] = large
        got = s.run(q, kind).double()
        hidden = torch.triu(torch.ones(rows, rows, dtype=torch.bool, device="cuda"), 1)
        for h in range(kvh * group):
            at = slice(h // group * hd, (h // group + 1) * hd)
            x, k, v = q[:, h * hd:(h + 1) * hd].double(), s.k[:, at].double(), s.v[:, at].double()
            w = torch.softmax((x @ k.T.contiguous() * s.scale).masked_fill(hidden, float("-inf")), -1)
            y, A, N = w @ v, w @ v.abs(), (~hidden).double() @ v.abs()
            S1 = s.scale * (x.abs() @ k.abs().T.contiguous()).amax(-1, keepdim=True)
            Q = 2.0 ** -22 * S1 + 2.0 ** -39 * large * s.scale * k.abs().sum(-1).max()
            f = 2.0 ** -20 + 2 * (Q + (hd / 8 + 8) * 2.0 ** -22 * S1) + (2.0 ** -11 if kind != "f32" else 0.0) + (2.0 ** -11 * (1 + 2 * S1) if kind == "bf16" else 0.0)
            tol = torch.finfo(base.TYPES[kind][0]).eps / 2 * y.abs() * (1 + f) + f * A + 2.0 ** -35 * N + (2.0 ** -25 if kind == "f16" else 1e-38)
            off = (got[:, h] - y).abs()
            assert (off <= tol).all(), f"{large}: off by {(off / tol).max().item():.3g} of the tolerance"
