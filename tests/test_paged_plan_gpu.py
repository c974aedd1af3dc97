"""The page plan beyond what test_paged_gpu.py asks of it: requests that end with pages given up, and calls of more
pieces of work than threads. Everything is a whole number, so results have to be equal."""
import numpy as np
import pytest

import test_paged_gpu as paged
from test_paged_gpu import torch  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu


def plan_reference(lens, append, page, pages, table, free_list, free_count, tokens):
    """The plan request by request; an ended request frees those of its entries that are pages."""
    table, free, width = [list(r) for r in table], list(free_list[:free_count]), len(table[0])
    for r, a in enumerate(append):
        if a < 0:
            free += [e for e in table[r][:min(-(-max(lens[r], 0) // page), width)] if 0 <= e < pages]
    # the rest as where every ended request has given up all its pages before
    before = [0 if a < 0 else n for n, a in zip(lens, append)]
    out = paged.plan_reference(before, append, page, pages, table, free, len(free), tokens)
    out["free_list"] = (free + [None] * pages)[:pages]
    return out


def same(torch, pkg, args):  # noqa: F811
    got, want = paged.run_plan(torch, pkg.runtime, *args), plan_reference(*args)
    for k, w in want.items():
        assert len(w) == len(got[k]) and all(x is None or x == y for x, y in zip(w, got[k])), k
    count, free = got["counts"][0], got["free_list"]
    assert all(0 <= e < args[3] for e in free[:count])
    return got


def test_a_given_up_page_is_not_free(torch, pkg):  # noqa: F811
    # request 0 ends with its first page given up: one page comes back, and two would be needed
    got = same(torch, pkg, ([20, 0], [-1, 32], 16, 8, [[-1, 5], [-1, -1]], [], 0, 40))
    assert got["counts"] == [1, 32, 0, 1] and got["new_lens"] == [0, 0] and got["free_list"][0] == 5
    # with a second free page both are granted, the last freed one first
    got = same(torch, pkg, ([20, 0], [-1, 32], 16, 8, [[-1, 5], [-1, -1]], [2], 1, 40))
    assert got["counts"] == [0, 32, 2, 0] and got["table"][1] == [5, 2] and min(got["slots"][:32]) >= 0


@pytest.mark.parametrize("kind", ["behind a window", "anywhere", "past the cache", "all"])
@pytest.mark.parametrize("rows,page,width,most,ended,spare", [(2, 16, 8, 20, 1, 3), (33, 8, 70, 9, 12, 10), (300, 4, 9, 30, 100, 50),
                                                              (1000, 16, 40, 5, 999, 7), (8192, 2, 3, 2, 4000, 900)])
def test_ended_requests_with_pages_given_up(torch, pkg, kind, rows, page, width, most, ended, spare):  # noqa: F811
    for seed in range(2):
        rng = np.random.default_rng(rows + seed)
        lens, append, page, pages, table, free, count, tokens = paged.make_plan(seed, rows, page, width, most, ended, spare, full=seed == 1)
        for r, a in enumerate(append):
            held = -(-lens[r] // page)
            if a >= 0 or not held or r % 5 == 4:
                continue
            gone = {"behind a window": range(int(rng.integers(0, held + 1))), "anywhere": rng.permutation(held)[:int(rng.integers(0, held + 1))],
                    "past the cache": rng.permutation(held)[:held // 2], "all": range(held)}[kind]
            for j in gone:
                table[r][j] = int(rng.choice([pages, 2 ** 31 - 1, -(2 ** 31)])) if kind == "past the cache" else -1
        same(torch, pkg, (lens, append, page, pages, table, free, count, tokens))


def test_a_request_whose_page_was_given_up_ends_and_its_pages_serve_others(torch, pkg):  # noqa: F811
    """Requests that slide and end for many steps: every page is held by one request or free, at every step."""
    rng, rows, page, width, pages, window = np.random.default_rng(1), 12, 4, 30, 90, 20
    lens, table, free, count = [0] * rows, [[-1] * width for _ in range(rows)], list(range(pages)), pages
    for _ in range(60):
        append = [int(rng.integers(1, 9)) if n + 8 <= width * page and rng.random() < 0.9 else -1 for n in lens]
        got = same(torch, pkg, (lens, append, page, pages, table, free, count, 200))
        lens, table, count = got["new_lens"], got["table"], got["counts"][0]
        width_rows = np.array(table).reshape(rows, width)
        free = got["free_list"][:count]
        for r, a in enumerate(append):  # the server's part: an ended row is empty, pages behind the window are given up
            if a < 0:
                width_rows[r] = -1
            for j in range(max(0, lens[r] - window) // page):
                if width_rows[r, j] >= 0:
                    free.append(int(width_rows[r, j]))
                    count += 1
                    width_rows[r, j] = -1
        table = width_rows.tolist()
        held = [e for r in range(rows) for e in table[r][:-(-lens[r] // page)] if e >= 0]
        assert sorted(held + free) == list(range(pages))


@pytest.mark.parametrize("rows,page,width,most,ended,spare", [(700, 16, 60, 512, 20, 9000), (2, 1, 200000, 90000, 0, 190000)])
def test_more_tokens_than_threads(torch, pkg, rows, page, width, most, ended, spare):  # noqa: F811
    args = paged.make_plan(5, rows, page, width, most, ended, spare)
    if rows == 2:
        args = ([7, 3], [80001, 79995], *args[2:7], 160000)
    assert args[-1] > 148 * 1024
    same(torch, pkg, args)
