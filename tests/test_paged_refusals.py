"""The paged serving step's entry points refuse arguments that no kernel could take, before any device is
touched: every call here fails on the host, so no GPU is needed and the pointers are never followed."""
import math

import pytest

P = 1 << 20  # a 16-byte aligned address nothing reads


def cache(rt, **change):
    v = dict(keys=P, values=P, dtype=0, pages=8, page_size=16, kv_heads=2, head_dim=128, page_stride=4096, token_stride=256,
             head_stride=128)
    v.update(change)
    return rt.PagedCache(*v.values())


BAD_CACHES = [dict(keys=None), dict(values=None), dict(dtype=2), dict(dtype=-1), dict(pages=0), dict(page_size=0), dict(kv_heads=0),
              dict(kv_heads=257), dict(head_dim=96), dict(head_dim=0), dict(page_stride=4097), dict(token_stride=4),
              dict(head_stride=-8), dict(keys=P + 8), dict(values=P + 2), dict(pages=1 << 20, page_size=1 << 12)]


def refused(pkg, call, *args):
    with pytest.raises(pkg.PlamoError) as e:
        call(*args)
    assert "CUDA" not in str(e.value)


def each(good, bad):
    for name, values in bad.items():
        for v in values:
            yield {**good, name: v}


def test_plan_refusals(pkg):
    good = dict(lens=P, append=P + 64, rows=4, page_size=16, pages=100, table=P, table_stride=8, free_list=P, free_count=P,
                new_lens=P + 128, row_start=P, slots=P, positions=P, tokens=64, counts=P + 256)
    bad = dict(lens=[None], append=[None], rows=[0, -1, 8193], page_size=[0, -16], pages=[0, 1 << 30], table=[None], table_stride=[0, 1 << 30],
               free_list=[None], free_count=[None, P + 256], new_lens=[None, P, P + 64], row_start=[None], slots=[None], positions=[None],
               tokens=[0, -1, 2 ** 31 - 1], counts=[None])
    for args in each(good, bad):
        refused(pkg, pkg.runtime.k_paged_plan, *args.values())


def test_qkv_refusals(pkg):
    rt = pkg.runtime
    good = dict(cache=cache(rt), qkv=P, qkv_stride=2560, tokens=4, heads=16, q_norm=P, k_norm=P, eps=1e-6, rope=P, rope_rows=100,
                positions=P, slots=P, q=P, q_stride=2048)
    bad = dict(cache=[cache(rt, **c) for c in BAD_CACHES], qkv=[None, P + 2], qkv_stride=[2552, 2561], tokens=[0, -3], heads=[0, 257],
               q_norm=[P + 4], k_norm=[P + 8], eps=[-1.0, math.nan], rope=[P + 4], rope_rows=[0], positions=[None], slots=[None],
               q=[None, P + 6], q_stride=[2040, 2049])
    for args in each(good, bad):
        refused(pkg, rt.k_paged_qkv, *args.values())


def test_attention_refusals(pkg):
    rt = pkg.runtime
    size = rt.paged_attention_workspace()
    good = dict(cache=cache(rt), q=P, q_stride=2048, q_rows=4, heads=16, table=P, table_stride=8, lens=P, rows=4, row_start=0, max_len=128,
                window=0, scale=0.1, out=P, out_stride=2048, lse=P, workspace=P, workspace_bytes=size)
    bad = dict(cache=[cache(rt, **c) for c in BAD_CACHES], q=[None, P + 2], q_stride=[2040, 2050], q_rows=[0, 3], heads=[0, 15, 258],
               table=[None], table_stride=[0, 7], lens=[None], rows=[0, 8193], max_len=[0, 129], window=[-1],
               scale=[math.nan, math.inf, 0.0, -0.1], out=[None, P + 4], out_stride=[2040, 2052], workspace=[None, P + 8],
               workspace_bytes=[0, size - 1])
    for args in each(good, bad):
        refused(pkg, rt.k_paged_attention, *args.values())
    with pytest.raises(pkg.PlamoError, match=f"{size} bytes needed"):
        rt.k_paged_attention(*{**good, "workspace_bytes": 16}.values())


def test_sample_refusals(pkg):
    good = dict(logits=P, dtype=0, rows=4, vocab=1000, row_stride=1000, temperature=P, top_k=P, top_p=P, min_p=P, u=P, ids=P)
    bad = dict(logits=[None, P + 1], dtype=[-1, 3], rows=[0, 65536], vocab=[0, (1 << 22) + 1], row_stride=[999], u=[None], ids=[None])
    for args in each(good, bad):
        refused(pkg, pkg.runtime.k_sample, *args.values())
    refused(pkg, pkg.runtime.k_sample, *{**good, "dtype": 2, "logits": P + 2}.values())
