"""The page plan refuses arrays that overlap: every block reads the inputs while others already write. Every call here
fails on the host, so no GPU is needed and the pointers are never followed."""
import itertools

import pytest

WRITTEN = ["table", "free_list", "new_lens", "row_start", "slots", "positions", "counts"]
READ = ["lens", "append", "free_count"]


def arguments():
    """Arrays side by side, none of them overlapping."""
    at, good = 1 << 20, dict(rows=4, page_size=16, pages=100, table_stride=8, tokens=64)
    sizes = dict(lens=4, append=4, table=32, free_list=100, free_count=1, new_lens=4, row_start=5, slots=64, positions=64, counts=4)
    for name, n in sizes.items():
        good[name] = at
        at += 4 * n
    return good, sizes


def call(pkg, a):
    pkg.runtime.k_paged_plan(a["lens"], a["append"], a["rows"], a["page_size"], a["pages"], a["table"], a["table_stride"], a["free_list"],
                             a["free_count"], a["new_lens"], a["row_start"], a["slots"], a["positions"], a["tokens"], a["counts"])


@pytest.mark.parametrize("written,other", [(w, o) for w, o in itertools.product(WRITTEN, WRITTEN + READ) if w != o])
def test_an_overlap_is_refused(pkg, written, other):
    good, sizes = arguments()
    # its first value on the other's last, its last on the other's first, and on the same place
    for at in (good[other] + 4 * (sizes[other] - 1), good[other] - 4 * (sizes[written] - 1), good[other]):
        with pytest.raises(pkg.PlamoError, match="must not overlap"):
            call(pkg, {**good, written: at})
