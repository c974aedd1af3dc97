"""Sampling's exact promises: whole-number weights, so ids and kept numbers equal a plain form's, whatever the split.

The plain form takes the fp32 quotient and exponential of torch and does the rest in whole numbers. ids and kept have
to be equal; log probabilities come from the same whole numbers, at most the two sums and their quotient rounded to
fp32 (3 x 2^-24) and a logarithm good to 2^-23 of its size: below 2^-21 of the larger of that size and of 1."""
import numpy as np
import pytest

import test_paged_gpu as paged
from test_paged_gpu import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

ONE = 1 << 24


def share(fraction, total, up):
    return fraction * (total >> 24) + ((fraction * (total & (ONE - 1)) + (ONE - 1 if up else 0)) >> 24)


def plain(torch, x, t, k, p, mp):  # noqa: F811
    """The kept weights of one row [vocab] as whole numbers."""
    x = torch.where(x.isnan(), -np.inf, x.float())
    top = x.max()
    e = torch.exp((x - top) / torch.tensor(t, dtype=torch.float32, device="cuda"))
    e = torch.where(x == top, 1.0, e)
    w = torch.where(x == -np.inf, 0.0, e.double() * 2.0 ** 40).floor().long()
    order = torch.sort(x, descending=True, stable=True).indices
    s = w[order]
    if 0 < k < len(s):
        s[k:] = 0
    if p < 1.0:
        upto = s.cumsum(0)
        need = max(share(round(float(np.float32(p)) * ONE), int(upto[-1]), True), 1)
        s = torch.where(upto - s < need, s, 0)
    least = int(np.ceil(float(np.float32(mp)) * 2.0 ** 40))
    s = torch.where(s >= least, s, 0)
    return torch.zeros_like(w).scatter_(0, order, s)


SETTINGS = [(1.0, 0, 1.0, 0.0), (0.7, 7, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05), (0.8, 50, 0.95, 0.01), (1.1, 200, 0.9, 0.0),
            (0.9, 1500, 0.97, 0.0), (1.0, 0, 0.999, 0.002), (3.0, 3000, 1.0, 0.0)]


def logits(rng, shape, rows, vocab):
    x = 2.5 * rng.standard_normal((rows, vocab))
    if shape == "words":  # an unlikely background and a likely head
        for r in range(rows):
            n = min(300, vocab)
            x[r, rng.permutation(vocab)[:n]] = 18.0 - 1.6 * np.log(1 + np.arange(n)) + rng.standard_normal(n)
    if shape == "steps":
        x = np.floor(2.0 * x) / 2.0
    if shape == "holes":
        x[:, rng.permutation(vocab)[:vocab // 3]] = -np.inf
        x[:, rng.permutation(vocab)[:vocab // 5]] = np.nan
    return x


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab,shape", [(2, "normal"), (37, "steps"), (1000, "normal"), (1025, "words"), (5003, "holes"), (32001, "words"),
                                         (107520, "words"), (107520, "normal"), (80001, "steps"), (600001, "words")])
def test_ids_equal_the_plain_form(torch, pkg, dtype, vocab, shape):  # noqa: F811
    """u at and one step below the points where the id changes, and anywhere."""
    rng = np.random.default_rng(vocab)
    for n, (t, k, p, mp) in enumerate(SETTINGS):
        row = logits(rng, shape, 1, vocab)
        x = torch.tensor(row).to(paged.dt(torch, dtype)).cuda()
        w = plain(torch, x[0], t, k, p, mp)
        upto, total = w.cumsum(0), int(w.sum())
        at = [int(i) for i in rng.permutation(torch.nonzero(w).view(-1).cpu().numpy())[:6]]
        points = {int(m) for m in rng.integers(0, ONE, 4)} | {0, ONE - 1}
        for i in at:  # the least m whose share reaches the running sum
            lo, hi, c = 0, ONE, int(upto[i])
            while lo < hi:
                mid = (lo + hi) // 2
                lo, hi = (lo, mid) if share(mid, total, False) >= c else (mid + 1, hi)
            points |= {min(lo, ONE - 1), max(lo - 1, 0)}
        points = sorted(points)
        u = (np.array(points) / ONE).astype(np.float32)
        ids, lp, kept, _ = paged.run_sample(torch, pkg.runtime, np.repeat(row, len(u), 0), dtype, t, k, p, mp, u)
        want = [int((upto <= share(m, total, False)).sum()) for m in points]
        assert ids.tolist() == want, (t, k, p, mp)
        assert (kept == int((w > 0).sum())).all(), (t, k, p, mp)
        exact = np.array([np.log(float(w[i])) - np.log(float(total)) for i in want])
        assert (np.abs(lp - exact) <= 2.0 ** -21 * np.maximum(1.0, np.abs(exact))).all()


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("vocab", [900, 3001, 30000, 107520])
def test_rows_do_not_depend_on_the_batch(torch, pkg, dtype, vocab):  # noqa: F811
    """The same rows alone, in batches of 9, 32 and 100 (other numbers of blocks a row), from other offsets, again."""
    rng, rt = np.random.default_rng(vocab), pkg.runtime
    x = logits(rng, "words", 100, vocab)
    t = rng.choice([0.0, 0.7, 1.0, 1.4], 100)
    k = rng.choice([0, 1, 40, 300, 2500], 100)
    p, mp = rng.choice([1.0, 0.95, 0.5], 100), rng.choice([0.0, 0.0, 0.03], 100)
    u = rng.random(100).astype(np.float32)
    whole = paged.run_sample(torch, rt, x, dtype, t, k, p, mp, u)[:3]

    def part(a, b, stride=None, offset=0):
        got = paged.run_sample(torch, rt, x[a:b], dtype, t[a:b], k[a:b], p[a:b], mp[a:b], u[a:b], stride, offset)[:3]
        for g, w in zip(got, whole):
            assert (g == w[a:b]).all(), (a, b, stride, offset)
    for r in range(0, 100, 7):
        part(r, r + 1)
    for n in (9, 32):
        for a in range(0, 100 - n, 2 * n):
            part(a, a + n)
    part(0, 100)
    part(3, 35, vocab + 3, 1)
    part(3, 12, vocab + 1, 5)


def test_quotients_are_the_ieee_ones(torch, pkg):  # noqa: F811
    """Two logits a row, the second kept exactly when min_p is at most its exponential: 4 million quotients, each
    below and at the threshold. (The exponential of the quotient one ulp off differs in most places here: the
    quotients lie between -11 and -0.5, and a weight keeps all of its exponential's bits.)"""
    rt, rows = pkg.runtime, 65535
    gen = torch.Generator(device="cuda").manual_seed(11)
    rand = lambda: torch.rand(rows, generator=gen, device="cuda")  # noqa: E731
    zero = torch.full((rows,), 0.5, device="cuda")
    ids, kept = (torch.zeros(rows, dtype=torch.int32, device="cuda") for _ in range(2))
    for turn in range(64):
        T = (0.05 + 4.0 * rand()) if turn % 4 else 10.0 ** (12.0 * rand() - 6.0)
        top = 30.0 * (rand() - 0.5) * (turn % 2)
        x = torch.stack([top, top - (0.5 + 10.4 * rand()) * T], 1).contiguous()
        q = (x[:, 1] - x[:, 0]) / T
        e = torch.exp(q)
        usable = (q < -0.4) & (e >= 2.0 ** -16)
        assert int(usable.sum()) > 0.9 * rows
        for min_p, number in ((e, 2), (torch.nextafter(e, torch.ones_like(e)), 1)):
            rt.k_sample(x.data_ptr(), 2, rows, 2, 2, T.data_ptr(), 0, 0, min_p.data_ptr(), zero.data_ptr(), ids.data_ptr(), 0, kept.data_ptr())
            torch.cuda.synchronize()
            assert bool((kept[usable] == number).all()), (turn, int((kept[usable] != number).sum()))
