"""Requests whose visible scores are all -inf get zeros and a log-sum-exp of -inf, whatever their values hold."""
import numpy as np
import pytest

import test_paged_gpu as paged
from test_paged_gpu import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("lens", [[50, 1, 30], [700, 900, 20], [9000, 5000, 3], [300] * 200])
def test_no_score_and_infinite_values(torch, pkg, dtype, lens):  # noqa: F811
    c = paged.Case(torch, pkg.runtime, lens, 16, 1, 64, 16, dtype, poison=False, sharp=1.0)
    c.q[..., 0] = 1.0
    for r in range(0, len(lens), 2):  # every other request: q.k = -inf for every key
        for page in c.table[r][:-(-lens[r] // 16)]:
            c.k[int(page), :, :, 0] = float("-inf")
            c.v[int(page), 3, :, 5] = float("inf")
            c.v[int(page), 0, :, 6] = float("nan")
            c.v[int(page), 0, :, 7] = float("-inf")
    out, lse = c.run()
    assert (out[::2] == 0).all() and np.isneginf(lse[::2]).all()
    c.q64 = c.q.double().cpu().numpy()
    c.check(out, lse, rows=range(1, len(lens), 2))
