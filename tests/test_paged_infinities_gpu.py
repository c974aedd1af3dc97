"""Infinite values in the paged serving step: what the formulas make of them, and nothing else, comes out.

A visible key of finite score has a probability above zero, however small, so an infinite value of it makes its
output infinite, as long as the probability itself does not vanish in fp32 (below 2^-126 of the largest). Finite
columns keep the tolerances of the attention's other tests: half an ulp of the stored type, and 2^-15 of the
largest visible value."""
import numpy as np
import pytest

import test_paged_gpu as paged
from test_paged_gpu import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

INF = float("inf")


@pytest.mark.parametrize("dtype,powers", [
    ("f16", [13, 20, 23, 24.5, 26, 28, 30, 34, 36, 38.5, 40, 45, 60, 100, 123]), ("bf16", [13, 20, 40, 100, *np.linspace(117.0, 125.0, 41)])])
@pytest.mark.parametrize("n,strong,infinite", [(50, 0, 3), (50, 0, 40), (50, 49, 3), (700, 0, 3), (700, 699, 5), (9000, 0, 8998), (9000, 8999, 1)])
def test_infinite_values_of_unlikely_keys(torch, pkg, dtype, powers, n, strong, infinite):  # noqa: F811
    """Request i has one likely key; all others are 2^-powers[i] as likely or (heads from the second on) up to 2^(powers[i] / 8) likelier,
    one of them with infinite values."""
    c = paged.Case(torch, pkg.runtime, [n] * len(powers), 16, 1, 64, 16, dtype, poison=False, seed=n)
    c.k.zero_()
    c.q.zero_()
    c.q[..., 0] = 16.0 - 0.125 * torch.arange(16, device="cuda")
    c.q[..., 1] = 1.0
    at = lambda r, p: (int(c.table[r, p // 16]), p % 16)  # noqa: E731
    for r, power in enumerate(powers):
        for page in c.table[r]:
            c.k[int(page), :, 0, 0] = -power * float(np.log(2.0)) * 8.0 / 16.0  # scale 1/8
            c.k[int(page), :, 0, 1] = -0.02 * r  # probabilities of any mantissa
        c.k[at(r, strong)] = 0.0
        v = c.v[at(r, infinite)][0]
        v[3], v[5], v[60] = INF, -INF, INF
    out, lse = c.run()
    for r, power in enumerate(powers):
        assert np.isposinf(out[r][:, [3, 60]]).all() and np.isneginf(out[r][:, 5]).all(), (power, out[r][0, [3, 5, 60]])
        c.v[at(r, infinite)][0][[3, 5, 60]] = 0.0
    finite = [i for i in range(64) if i not in (3, 5, 60)]
    c.k64, c.v64, c.q64 = (x.double().cpu().numpy() for x in (c.k, c.v, c.q))
    for r in range(len(powers)):
        o, l, big = paged.attention_reference(c.q64[r].reshape(1, 16, 64), c.k64, c.v64, c.table[r], n, 0, c.scale, 16, c.pages)
        tol = paged.half_ulp(dtype) * np.abs(o) + 2.0 ** -15 * big[:, None] + (2.0 ** -25 if dtype == "f16" else 0.0)
        assert (np.abs(out[r] - o) <= tol)[:, finite].all()
        assert (np.abs(lse[r] - l) <= 2.0 ** -16 + 2.0 ** -22 * np.abs(l)).all()
