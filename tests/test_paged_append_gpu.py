"""The append at the lengths of prompts, where a warp takes a whole token (from 148 x 32 steps of 256 / head_dim heads
on), just below and above the change, with heads that do not fill the last step or batch of steps."""
import pytest

import test_paged_gpu as paged
from test_paged_gpu import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,heads,kv,dim,page,norm,rope,layout", [
    (473, 16, 1, 128, 16, True, True, "token"), (474, 16, 1, 128, 16, True, True, "token"), (1000, 17, 1, 128, 16, True, True, "head"),
    (1500, 15, 3, 64, 24, True, True, "token"), (789, 20, 2, 128, 5, True, True, "token"), (700, 33, 11, 64, 8, True, True, "head"),
    (2001, 4, 4, 128, 1, False, True, "token"), (1200, 40, 10, 128, 16, True, False, "head"), (5000, 1, 1, 64, 3, False, False, "token")])
def test_append_of_prompts(torch, pkg, dtype, tokens, heads, kv, dim, page, norm, rope, layout):  # noqa: F811
    paged.test_qkv_append(torch, pkg, dtype, tokens, heads, kv, dim, page, norm, rope, layout)
