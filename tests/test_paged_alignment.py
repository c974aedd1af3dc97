"""The paged serving step's entry points refuse arrays of 32-bit values off a 4-byte boundary, which no kernel could read.
Every call here fails on the host, so no GPU is needed and the pointers are never followed."""
import pytest

from test_paged_refusals import P, cache

AT = [P + (1 << 12) * i for i in range(16)]


def check(pkg, call, good, names):
    for name in names:
        for off in (1, 2, 3):
            with pytest.raises(pkg.PlamoError) as e:
                call(*{**good, name: good[name] + off}.values())
            assert "aligned" in str(e.value), name


def test_plan(pkg):
    good = dict(lens=AT[0], append=AT[1], rows=4, page_size=16, pages=100, table=AT[2], table_stride=8, free_list=AT[3], free_count=AT[4],
                new_lens=AT[5], row_start=AT[6], slots=AT[7], positions=AT[8], tokens=64, counts=AT[9])
    check(pkg, pkg.runtime.k_paged_plan, good, ["lens", "append", "table", "free_list", "free_count", "new_lens", "row_start", "slots",
                                                "positions", "counts"])


def test_qkv(pkg):
    good = dict(cache=cache(pkg.runtime), qkv=P, qkv_stride=2560, tokens=4, heads=16, q_norm=P, k_norm=P, eps=1e-6, rope=P, rope_rows=100,
                positions=P, slots=P, q=P, q_stride=2048)
    check(pkg, pkg.runtime.k_paged_qkv, good, ["positions", "slots"])


def test_attention(pkg):
    rt = pkg.runtime
    good = dict(cache=cache(rt), q=P, q_stride=2048, q_rows=4, heads=16, table=P, table_stride=8, lens=P, rows=4, row_start=P, max_len=128,
                window=0, scale=0.1, out=P, out_stride=2048, lse=P, workspace=P, workspace_bytes=rt.paged_attention_workspace())
    check(pkg, rt.k_paged_attention, good, ["table", "lens", "row_start", "lse"])


def test_sample(pkg):
    good = dict(logits=P, dtype=0, rows=4, vocab=1000, row_stride=1000, temperature=P, top_k=P, top_p=P, min_p=P, u=P, ids=P, logprobs=P, kept=P)
    check(pkg, pkg.runtime.k_sample, good, ["temperature", "top_k", "top_p", "min_p", "u", "ids", "logprobs", "kept"])
