"""The append without a rotation or a norm: every value is kept to itself, infinities and NaN among them."""
import numpy as np
import pytest

import test_paged_gpu as paged
from test_paged_gpu import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,heads,kv,dim", [(3, 4, 2, 128), (5, 3, 1, 64), (1000, 16, 4, 128)])
def test_values_pass_unchanged(torch, pkg, dtype, tokens, heads, kv, dim):  # noqa: F811
    rt, ty, page = pkg.runtime, paged.dt(torch, dtype), 16
    rng = np.random.default_rng(tokens)
    x = rng.standard_normal((tokens, heads + 2 * kv, dim))
    for value in (np.inf, -np.inf, np.nan, -0.0):
        x[rng.random(x.shape) < 0.02] = value
    qkv = torch.tensor(x).to(ty).cuda()
    pages = -(-tokens // page)
    keys, values = (torch.zeros(pages, page, kv, dim, dtype=ty, device="cuda") for _ in range(2))
    q = torch.zeros(tokens, heads, dim, dtype=ty, device="cuda")
    cache = rt.PagedCache(keys.data_ptr(), values.data_ptr(), paged.CODE[dtype], pages, page, kv, dim, page * kv * dim, kv * dim, dim)
    slots = paged.ints(torch, rng.permutation(pages * page)[:tokens])
    rt.k_paged_qkv(cache, qkv.data_ptr(), (heads + 2 * kv) * dim, tokens, heads, 0, 0, 1e-6, 0, 0, 0, slots.data_ptr(), q.data_ptr(), heads * dim)
    torch.cuda.synchronize()
    at = slots.long()
    for got, want in ((q, qkv[:, :heads]), (keys.view(-1, kv, dim)[at], qkv[:, heads:heads + kv]), (values.view(-1, kv, dim)[at], qkv[:, heads + kv:])):
        assert torch.equal(got.isnan(), want.isnan())
        assert torch.equal(torch.where(got.isnan(), 0, got).view(torch.int16), torch.where(want.isnan(), 0, want).view(torch.int16))
