"""The paged serving step's kernels (plamo_k_paged_plan, _qkv, _attention, plamo_k_sample) against plain
restatements in 64 bits, at the sizes, masks and layouts where they can go wrong.

Tolerances, from the arithmetic (half an ulp of the stored type is h = 2^-8 of the value for bf16, 2^-11 for
fp16):
- append: h |y| for the one rounding, and 2^-20 of the two products' sizes for the fp32 operations before it
  (a mean of up to 128 squares, a square root, a reciprocal and four products: below 16 roundings of 2^-24).
- attention: h |o|, and 2^-15 of the largest visible |v|: the probabilities' pairs carry 16 bits (2^-17),
  scores up to 64 powers of two are good to four roundings (64 * 4 * 2^-24 = 2^-16), sums to 2^-20.
  lse: 2^-16 absolute for the scores, and 2^-22 of its size.
- sampling: the id's interval of the running probability, widened by d = 2^-17, holds u: an fp32 logit
  difference of at most 28 temperatures is good to 2^-24 of itself, so a weight to 28 * 2^-23 < 2^-18.
  The kept number lies between those of limits moved by d; without top-p and min-p it is exact.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

D17 = 2.0 ** -17


@pytest.fixture(scope="module")
def torch():
    t = pytest.importorskip("torch")
    if not t.cuda.is_available():
        pytest.skip("CUDA device required")
    return t


def half_ulp(dtype):
    return 2.0 ** -8 if dtype == "bf16" else 2.0 ** -11


def dt(torch, name):
    return {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}[name]


CODE = {"bf16": 0, "f16": 1, "f32": 2}


def ints(torch, v):
    return torch.tensor(np.asarray(v, dtype=np.int32), device="cuda")


# ------------------------------------------------------------------------------------------ plan

def plan_reference(lens, append, page, pages, table, free_list, free_count, tokens):
    """The plan request by request. `free_list` is a list with room for `pages` entries."""
    table, free = [list(r) for r in table], list(free_list[:free_count])
    width = len(table[0])
    for r, a in enumerate(append):
        if a < 0:
            free += table[r][:min(-(-max(lens[r], 0) // page), width)]
    listed = list(free)
    new_lens, starts, slots, positions = [], [0], [], []
    refused, dry, granted, at = 0, 0, 0, 0
    for r, a in enumerate(append):
        n, add = max(lens[r], 0), max(a, 0)
        held = min(-(-n // page), width)
        if a < 0:
            new_lens.append(0)
        else:
            need = -(-(n + add) // page) - held
            fits = n + add <= width * page and at + add <= tokens
            dry += need if fits else 0
            ok = fits and (need == 0 or dry <= len(listed))
            if ok:
                for j in range(need):
                    table[r][held + j] = free.pop()
                granted += need
            else:
                refused += 1
            new_lens.append(n + add if ok else n)
            for i in range(add):
                p = n + i
                slots.append(table[r][p // page] * page + p % page if ok else -1)
                positions.append(p if ok else -1)
        at += add
        starts.append(at)
    pad = lambda v: (v + [-1] * tokens)[:tokens]  # noqa: E731
    out_list = (listed + [None] * pages)[:pages]
    return dict(table=table, free_list=out_list, new_lens=new_lens, row_start=starts, slots=pad(slots), positions=pad(positions),
                counts=[len(listed) - granted, at, granted, refused])


def run_plan(torch, rt, lens, append, page, pages, table, free_list, free_count, tokens, stream=0):
    rows = len(lens)
    t = dict(lens=ints(torch, lens), append=ints(torch, append), table=ints(torch, table),
             free_list=ints(torch, list(free_list) + [-7] * (pages - len(free_list))), free_count=ints(torch, [free_count]),
             new_lens=ints(torch, [-9] * rows), row_start=ints(torch, [-9] * (rows + 1)), slots=ints(torch, [-9] * tokens),
             positions=ints(torch, [-9] * tokens), counts=ints(torch, [-9] * 4))
    torch.cuda.synchronize()
    rt.k_paged_plan(t["lens"].data_ptr(), t["append"].data_ptr(), rows, page, pages, t["table"].data_ptr(), len(table[0]),
                    t["free_list"].data_ptr(), t["free_count"].data_ptr(), t["new_lens"].data_ptr(), t["row_start"].data_ptr(),
                    t["slots"].data_ptr(), t["positions"].data_ptr(), tokens, t["counts"].data_ptr(), stream)
    torch.cuda.synchronize()
    return {k: v.cpu().tolist() for k, v in t.items()}


def make_plan(seed, rows, page, width, most, ended, spare, full=False):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, width * page - (0 if full else most) + 1, rows).tolist()
    append = rng.integers(0, most + 1, rows).tolist()
    for r in rng.choice(rows, size=min(rows, ended), replace=False):
        append[r] = -1
    held = [-(-n // page) for n in lens]
    pages = sum(held) + spare + 1
    order = rng.permutation(pages).tolist()
    table, at = [], 0
    for h in held:
        table.append(order[at:at + h] + [-1] * (width - h))
        at += h
    return lens, append, page, pages, table, order[at:at + spare], spare, max(1, sum(a for a in append if a > 0)) + 3


@pytest.mark.parametrize("rows,page,width,most,ended,spare", [
    (1, 16, 8, 5, 0, 4), (1, 1, 3, 1, 1, 0), (3, 16, 4, 33, 1, 40), (32, 16, 20, 1, 2, 40), (33, 24, 7, 40, 5, 20),
    (255, 8, 12, 9, 30, 100), (257, 1, 40, 7, 3, 500), (1000, 16, 9, 50, 100, 700), (8192, 2, 3, 2, 900, 3000)])
def test_plan(torch, pkg, rows, page, width, most, ended, spare):
    for seed in range(3):
        args = make_plan(seed, rows, page, width, most, ended, spare, full=seed == 2)
        got, want = run_plan(torch, pkg.runtime, *args), plan_reference(*args)
        for k, w in want.items():
            assert all(x is None or x == y for x, y in zip(w, got[k])) and len(w) == len(got[k]), (seed, k)


def test_plan_tokens_past_capacity_refused(torch, pkg):
    args = ([3, 0, 5], [4, 6, 2], 4, 30, [[1, -1, -1], [-1] * 3, [2, 3, -1]], [9, 10, 11, 12, 13], 5, 9)
    got, want = run_plan(torch, pkg.runtime, *args), plan_reference(*args)
    assert want["counts"][3] == 2 and got["counts"] == want["counts"]
    for k in ("slots", "positions", "new_lens", "row_start", "table"):
        assert got[k] == want[k]


def test_plan_entries_outside_the_cache_give_no_slot(torch, pkg):
    # request 0 appends into a held page whose entry is no page; request 1 is granted an entry past the cache
    got = run_plan(torch, pkg.runtime, [2, 4], [2, 1], 4, 5, [[-3, -1], [1, -1]], [77], 1, 4)
    assert got["slots"] == [-1, -1, -1, -1] and got["positions"] == [2, 3, 4, -1]


# ------------------------------------------------------------------------------------------ append

def rope_bits(torch, rows, dim):
    freq = 1e4 ** (-np.arange(0, dim, 2) / dim)
    angle = torch.tensor(np.arange(rows)[:, None] * freq)
    bits = [x.to(torch.bfloat16).view(torch.int16).to(torch.int32) & 0xFFFF for x in (angle.cos(), angle.sin())]
    return (bits[0] | (bits[1] << 16)).cuda(), [x.to(torch.bfloat16).double().numpy() for x in (angle.cos(), angle.sin())]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("tokens,heads,kv,dim,page,norm,rope,layout", [
    (1, 16, 1, 128, 16, True, True, "token"), (33, 16, 4, 128, 16, True, True, "head"), (257, 3, 3, 64, 24, True, True, "token"),
    (7, 5, 1, 64, 1, False, True, "head"), (19, 8, 2, 128, 5, True, False, "token"), (2, 1, 1, 64, 3, False, False, "token")])
def test_qkv_append(torch, pkg, dtype, tokens, heads, kv, dim, page, norm, rope, layout):
    rng, rt, ty = np.random.default_rng(tokens + dim), pkg.runtime, dt(torch, dtype)
    pages, width, pad = -(-tokens // page) + 2, (heads + 2 * kv) * dim, 16
    qkv = torch.tensor(rng.standard_normal((tokens, width + pad)), dtype=ty).cuda()
    qkv[0, :dim] *= 100.0
    weights = [torch.tensor(0.2 * rng.standard_normal(dim), dtype=ty).cuda() for _ in range(2)]
    rows = 300
    table, (cos, sin) = rope_bits(torch, rows, dim)
    positions, slots = rng.integers(0, rows, tokens), rng.permutation(pages * page)[:tokens]
    if tokens > 6:  # tokens without a slot or with a position outside the table
        slots[1], slots[2] = -1, pages * page
        if rope:
            positions[3], positions[4] = -1, rows
    shape = (pages, page, kv, dim) if layout == "token" else (pages, kv, page, dim)
    caches = [torch.full(shape, 7.0 + i, dtype=ty, device="cuda") for i in range(2)]
    st = caches[0].stride() if layout == "token" else [caches[0].stride()[i] for i in (0, 2, 1, 3)]
    q = torch.full((tokens, heads * dim + pad), 5.0, dtype=ty, device="cuda")
    cache = rt.PagedCache(caches[0].data_ptr(), caches[1].data_ptr(), CODE[dtype], pages, page, kv, dim, st[0], st[1], st[2])
    pos_t, slot_t = ints(torch, positions), ints(torch, slots)
    rt.k_paged_qkv(cache, qkv.data_ptr(), width + pad, tokens, heads, weights[0].data_ptr() if norm else 0,
                   weights[1].data_ptr() if norm else 0, 1e-6, table.data_ptr() if rope else 0, rows, pos_t.data_ptr(),
                   slot_t.data_ptr(), q.data_ptr(), heads * dim + pad)
    torch.cuda.synchronize()
    x = qkv[:, :width].double().cpu().numpy().reshape(tokens, heads + 2 * kv, dim)
    y = x.copy()
    if norm:
        w = [1.0 + v.double().cpu().numpy() for v in weights]
        scale = 1.0 / np.sqrt((x ** 2).mean(-1, keepdims=True) + 1e-6)
        y[:, :heads] = (x * scale)[:, :heads] * w[0]
        y[:, heads:heads + kv] = (x * scale)[:, heads:heads + kv] * w[1]
    size = np.abs(y)
    if rope:
        at = np.clip(positions, 0, rows - 1)
        c, s = cos[at][:, None], sin[at][:, None]
        a, b = y[..., :dim // 2].copy(), y[..., dim // 2:].copy()
        turned = np.concatenate([a * c - b * s, b * c + a * s], -1)
        size = np.concatenate([abs(a * c) + abs(b * s), abs(b * c) + abs(a * s)], -1)
        y[:, :heads + kv] = turned[:, :heads + kv]
    tol = half_ulp(dtype) * np.abs(y) + 2.0 ** -20 * size + (2.0 ** -25 if dtype == "f16" else 0.0)
    live = (slots >= 0) & (slots < pages * page) & ((positions >= 0) & (positions < rows) if rope else True)
    got = q.double().cpu().numpy()
    assert (got[:, heads * dim:] == 5.0).all()
    got = got[:, :heads * dim].reshape(tokens, heads, dim)
    assert (np.abs(got - y[:, :heads]) <= tol[:, :heads])[live].all() and (got[~live] == 0).all()
    perm = (0, 1, 2, 3) if layout == "token" else (0, 2, 1, 3)
    k, v = (c.permute(*perm).reshape(pages * page, kv, dim).double().cpu().numpy() for c in caches)
    at = slots[live]
    assert (np.abs(k[at] - y[live, heads:heads + kv]) <= tol[live, heads:heads + kv]).all()
    assert (v[at] == x[live, heads + kv:]).all()
    rest = np.ones(pages * page, dtype=bool)
    rest[at] = False
    assert (k[rest] == 7.0).all() and (v[rest] == 8.0).all()


# ------------------------------------------------------------------------------------------ attention

def attention_reference(q, keys, values, table, n, window, scale, page, pages):
    """One request in 64 bits: q [kv, group, dim], keys / values [pages, page, kv, dim]."""
    kv, group, dim = q.shape
    at = np.arange(max(0, n - window) if window else 0, n)
    page_of = np.asarray(table)[at // page] if n else np.zeros(0, int)
    held = (page_of >= 0) & (page_of < pages)
    at, page_of = at[held], page_of[held]
    if not len(at):
        return np.zeros((kv * group, dim)), np.full(kv * group, -np.inf), np.zeros(kv * group)
    k, v = keys[page_of, at % page], values[page_of, at % page]
    s = np.einsum("hgd,thd->hgt", q, k) * scale
    top = s.max(-1, keepdims=True)
    p = np.exp(s - top)
    out = np.einsum("hgt,thd->hgd", p, v) / p.sum(-1)[..., None]
    lse = top[..., 0] + np.log(p.sum(-1))
    return out.reshape(-1, dim), lse.reshape(-1), np.repeat(np.abs(v).max((0, 2)), group)


class Case:
    """A paged cache on the device with `lens` requests, every slot that no request sees poisoned with NaN."""

    def __init__(self, torch, rt, lens, heads, kv, dim, page, dtype="bf16", window=0, layout="token", holes=(), seed=0, sharp=2.0,
                 width=None, poison=True):
        rng = np.random.default_rng(seed)
        self.torch, self.rt, self.lens, self.heads, self.kv, self.dim, self.page = torch, rt, list(lens), heads, kv, dim, page
        self.dtype, self.window, rows = dtype, window, len(lens)
        held = [-(-max(n, 0) // page) for n in lens]
        self.width = width or max(1, max(held))
        self.pages = sum(held) + 2
        order = rng.permutation(self.pages)
        self.table = np.full((rows, self.width), -1, dtype=np.int32)
        seen, at = np.zeros((self.pages, page), dtype=bool), 0
        for r, h in enumerate(held):
            self.table[r, :h] = order[at:at + h]
            at += h
        for r, j, entry in holes:
            self.table[r, j] = entry
        for r, n in enumerate(lens):
            for p in range(max(0, n - window) if window else 0, max(n, 0)):
                e = self.table[r, p // page]
                if 0 <= e < self.pages:
                    seen[e, p % page] = True
        ty = dt(torch, dtype)
        k, v = (rng.standard_normal((self.pages, page, kv, dim)) for _ in range(2))
        if poison:
            k[~seen], v[~seen] = np.nan, np.nan
        k, v, q = (torch.tensor(x).to(ty) for x in (k, v, sharp * rng.standard_normal((rows, heads, dim))))
        self.k64, self.v64, self.q64 = (x.double().numpy() for x in (k, v, q))
        if layout == "head":
            k, v = k.permute(0, 2, 1, 3), v.permute(0, 2, 1, 3)
        self.k, self.v, self.q = k.contiguous().cuda(), v.contiguous().cuda(), q.cuda()
        st = self.k.stride() if layout == "token" else [self.k.stride()[i] for i in (0, 2, 1, 3)]
        self.cache = rt.PagedCache(self.k.data_ptr(), self.v.data_ptr(), CODE[dtype], self.pages, page, kv, dim, st[0], st[1], st[2])
        self.scale = dim ** -0.5
        self.t_table, self.t_lens = ints(torch, self.table), ints(torch, lens)
        self.work = torch.full((rt.paged_attention_workspace(),), 255, dtype=torch.uint8, device="cuda")

    def run(self, q=None, rows=None, row_start=None, max_len=None, stream=0, lse=True, pad=0):
        torch, rows = self.torch, rows or len(self.lens)
        q = self.q if q is None else q
        n = q.shape[0]
        out = torch.full((n, self.heads * self.dim + pad), 3.0, dtype=q.dtype, device="cuda")
        l_out = torch.full((n, self.heads), 3.0, device="cuda")
        torch.cuda.synchronize()
        self.rt.k_paged_attention(self.cache, q.data_ptr(), q.stride(0), n, self.heads, self.t_table.data_ptr(), self.width,
                                  self.t_lens.data_ptr(), rows, row_start.data_ptr() if row_start is not None else 0,
                                  max_len or self.width * self.page, self.window, self.scale, out.data_ptr(), out.stride(0),
                                  l_out.data_ptr() if lse else 0, self.work.data_ptr(), self.work.numel(), stream)
        torch.cuda.synchronize()
        if pad:
            assert (out[:, self.heads * self.dim:] == 3.0).all()
        return out[:, :self.heads * self.dim].double().cpu().numpy().reshape(n, self.heads, self.dim), l_out.double().cpu().numpy()

    def check(self, out, lse, rows=None, max_len=None):
        for r in range(len(self.lens)) if rows is None else rows:
            n = min(max(self.lens[r], 0), max_len or 1 << 30)
            o, l, big = attention_reference(self.q64[r].reshape(self.kv, -1, self.dim), self.k64, self.v64, self.table[r], n,
                                            self.window, self.scale, self.page, self.pages)
            tol = half_ulp(self.dtype) * np.abs(o) + 2.0 ** -15 * big[:, None] + (2.0 ** -25 if self.dtype == "f16" else 0.0)
            assert (np.abs(out[r] - o) <= tol).all(), (r, n, np.nanmax(np.abs(out[r] - o) - tol))
            if lse is not None:
                inf = np.isneginf(l)
                assert (np.isneginf(lse[r]) == inf).all()
                assert (np.abs(lse[r] - l)[~inf] <= 2.0 ** -16 + 2.0 ** -22 * np.abs(l[~inf])).all(), r


SHAPES = [  # heads, kv heads, dim, page
    (16, 1, 128, 16), (16, 4, 128, 16), (1, 1, 64, 1), (14, 2, 64, 24), (8, 8, 128, 64), (20, 1, 128, 8), (32, 1, 64, 32),
    (33, 1, 128, 5), (64, 8, 64, 128)]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("heads,kv,dim,page", SHAPES)
def test_attention_short(torch, pkg, dtype, heads, kv, dim, page):
    c = Case(torch, pkg.runtime, [0, 1, 2, 15, 16, 17, 63, 64, 65, 130, 255, 257, 0, 400], heads, kv, dim, page, dtype)
    c.check(*c.run(pad=8))


@pytest.mark.parametrize("lens,window", [
    ([5000], 0), ([4097, 1, 0, 2300], 0), ([1500] * 20, 0), ([40] * 300, 0), ([0] * 7 + [3000] + [0] * 7, 0),
    ([5000, 100, 2048, 2049, 0, 1], 2048), ([700, 3], 1), ([700, 64, 65], 64), ([3001] * 9, 777)])
def test_attention_lengths(torch, pkg, lens, window):
    c = Case(torch, pkg.runtime, lens, 16, 1, 128, 16, window=window)
    c.check(*c.run())


@pytest.mark.parametrize("lens,heads,kv,dtype", [([32768], 16, 1, "bf16"), ([20001, 9], 16, 4, "f16"), ([12345] * 5, 32, 1, "bf16"),
                                                 ([9000, 30001, 2], 8, 2, "f16")])
def test_attention_long(torch, pkg, lens, heads, kv, dtype):
    c = Case(torch, pkg.runtime, lens, heads, kv, 128, 64, dtype)
    c.check(*c.run())


def test_attention_many_requests(torch, pkg):
    rng = np.random.default_rng(4)
    c = Case(torch, pkg.runtime, rng.integers(0, 60, 8192).tolist(), 2, 1, 64, 16)
    c.check(*c.run(), rows=range(0, 8192, 13))


@pytest.mark.parametrize("rows,top,heads,kv,page,window", [(400, 700, 16, 1, 16, 0), (300, 500, 8, 4, 24, 0), (350, 900, 4, 1, 16, 301),
                                                           (600, 300, 2, 2, 7, 290)])
def test_attention_many_cut_requests(torch, pkg, rows, top, heads, kv, page, window):
    """More requests and heads than blocks, some of them cut between two."""
    lens = np.random.default_rng(rows).integers(0, top + 1, rows)
    lens[::17] = 0
    lens[5] = top
    c = Case(torch, pkg.runtime, lens.tolist(), heads, kv, 64, page, window=window)
    out, lse = c.run()
    c.check(out, lse, rows=list(range(0, rows, 7)) + [5])
    assert (c.run()[0] == out).all()


@pytest.mark.parametrize("page,window", [(24, 0), (5, 0), (48, 0), (24, 4001), (16, 4001), (16, 3000)])
def test_attention_long_odd_pages(torch, pkg, page, window):
    c = Case(torch, pkg.runtime, [6001, 9, 4096, 0, 7777], 16, 1, 128, page, window=window, holes=[(0, 2, -1), (2, 3, -1)])
    c.check(*c.run())


def test_attention_packed_rows_long(torch, pkg):
    """As test_attention_packed_rows, where the requests are cut."""
    c = Case(torch, pkg.runtime, [9000, 70, 12001, 40, 5000], 16, 4, 128, 16)
    counts = [1, 0, 2, 1, 0]
    start = np.concatenate([[0], np.cumsum(counts)])
    q = torch.randn(int(start[-1]), 16, 128, device="cuda").bfloat16()
    rows = [r for r in range(5) if counts[r]]
    for r in rows:
        q[start[r + 1] - 1] = c.q[r]
    out, lse = c.run(q=q, row_start=ints(torch, start))
    full_out, full_lse = np.zeros((5, 16, 128)), np.zeros((5, 16))
    for r in rows:
        full_out[r], full_lse[r] = out[start[r + 1] - 1], lse[start[r + 1] - 1]
    c.check(full_out, full_lse, rows=rows)
    assert (out[1] == 3.0).all() and (lse[1] == 3.0).all()


def test_attention_all_requests_empty(torch, pkg):
    c = Case(torch, pkg.runtime, [0] * 40, 16, 1, 128, 16)
    out, lse = c.run()
    assert (out == 0).all() and np.isneginf(lse).all()
    c = Case(torch, pkg.runtime, [0, -5], 16, 1, 128, 16, width=300)
    out, lse = c.run()
    assert (out == 0).all() and np.isneginf(lse).all()


@pytest.mark.parametrize("layout", ["token", "head"])
def test_attention_layouts_and_holes(torch, pkg, layout):
    # pages given up (-1), an entry past the cache, a request without any page, one hole in the middle
    holes = [(0, 0, -1), (0, 1, -1), (1, 3, 10 ** 6), (2, 0, -1), (2, 1, -5), (3, 2, -1)]
    c = Case(torch, pkg.runtime, [100, 90, 30, 1000, 77], 16, 2, 128, 16, layout=layout, holes=holes)
    out, lse = c.run()
    c.check(out, lse)
    assert (out[2] == 0).all()


def test_attention_max_len_limits_lengths(torch, pkg):
    c = Case(torch, pkg.runtime, [500, 80, 100], 16, 1, 128, 16, poison=False)
    c.check(*c.run(max_len=100), max_len=100)


def test_attention_packed_rows(torch, pkg):
    """Queries of a packed step: the request's last token; requests without tokens are skipped."""
    c = Case(torch, pkg.runtime, [300, 7, 900, 64, 0], 16, 1, 128, 16)
    counts = [3, 0, 1, 2, 1]
    start = np.concatenate([[0], np.cumsum(counts)])
    q = torch.randn(int(start[-1]), 16, 128, device="cuda").bfloat16()
    for r in range(5):
        if counts[r]:
            q[start[r + 1] - 1] = c.q[r]
    out, lse = c.run(q=q, row_start=ints(torch, start))
    rows = [r for r in range(5) if counts[r]]
    last = {r: start[r + 1] - 1 for r in rows}
    full_out, full_lse = np.zeros((5, 16, 128)), np.zeros((5, 16))
    for r in rows:
        full_out[r], full_lse[r] = out[last[r]], lse[last[r]]
    c.check(full_out, full_lse, rows=rows)
    others = [i for i in range(int(start[-1])) if i not in last.values()]
    assert (out[others] == 3.0).all() and (lse[others] == 3.0).all()
    # rows that name no query are not touched
    bad = ints(torch, [0, 100, 100, 100, 100, 100])
    out, _ = c.run(q=q, row_start=bad)
    assert (out == 3.0).all()


def test_attention_infinities(torch, pkg):
    """Visible infinities go through the formula; scores that are all -inf give zeros."""
    c = Case(torch, pkg.runtime, [50, 50, 40], 16, 1, 128, 16, poison=False)
    with torch.no_grad():
        page = int(c.table[0, 0])
        c.v[page, 3, 0, 7] = float("inf")           # request 0: one output column infinite
        for p in range(50):                          # request 1: q.k = -inf for every key
            c.k[int(c.table[1, p // 16]), p % 16, 0, 0] = float("-inf")
        c.q[1, :, 0] = 1.0
        c.k[int(c.table[2, 0]), 5, 0, 0] = float("nan")  # request 2: a visible NaN
    out, lse = c.run()
    assert np.isposinf(out[0, :, 7]).all() and np.isfinite(np.delete(out[0], 7, -1)).all()
    assert (out[1] == 0).all() and np.isneginf(lse[1]).all()
    assert np.isnan(out[2]).all() and np.isnan(lse[2]).all()


def test_attention_tiny_probabilities_add_up(torch, pkg):
    """One strong key and thousands of keys 2^-20 as likely: their sum must not be lost."""
    for dtype in ("bf16", "f16"):
        c = Case(torch, pkg.runtime, [9000], 16, 1, 64, 16, dtype, poison=False)
        c.k.zero_()
        c.q.zero_()
        c.q[..., 0] = 16.0
        c.k[..., 0] = -6.9315
        c.k[int(c.table[0, 0]), 0, 0, 0] = 0.0
        c.v.fill_(1.0)
        c.v[int(c.table[0, 0]), 0] = 0.0
        c.k64, c.v64, c.q64 = (x.double().cpu().numpy() for x in (c.k, c.v, c.q))
        out, lse = c.run()
        o, l, _ = attention_reference(c.q64[0].reshape(1, 16, 64), c.k64, c.v64, c.table[0], 9000, 0, c.scale, 16, c.pages)
        assert (np.abs(out[0] - o) <= (half_ulp(dtype) + 2.0 ** -12) * o).all()
        assert (np.abs(lse[0] - l) <= 2.0 ** -16).all()


@pytest.mark.parametrize("dtype,head_dim", [("bf16", 128), ("f16", 64)])
@pytest.mark.parametrize("requests", [2, 10, 25, 50, 90])
def test_attention_cut_requests(torch, pkg, requests, dtype, head_dim):
    """Long requests beside none, one and a few keys: every number of pieces a head, every size of cluster."""
    rng = np.random.default_rng(requests)
    for longest in (700, 2500, 9000):
        lens = rng.integers(longest // 2, longest + 1, requests)
        lens[:requests // 5] = rng.integers(0, 40, requests // 5)
        lens[-1] = longest
        c = Case(torch, pkg.runtime, list(map(int, rng.permutation(lens))), 5, 1, head_dim, 16, dtype=dtype)
        c.check(*c.run())


def test_attention_offsets_past_32_bits(torch, pkg):
    """Three pages 2^30 + 8 elements apart: byte and element offsets pass 2^31 and 2^32."""
    rt, step = pkg.runtime, (1 << 30) + 8
    buf = torch.empty(3 * step + 4096, dtype=torch.bfloat16, device="cuda")
    c = Case(torch, rt, [40], 16, 1, 128, 16, poison=False)
    table = [[2, 0, 1]]
    base = buf.data_ptr()
    for i in range(3):
        for off, src in ((0, c.k), (2048, c.v)):
            buf[i * step + off:i * step + off + 2048] = src[int(c.table[0, [1, 2, 0][i]])].reshape(-1)
    c.cache = rt.PagedCache(base, base + 4096, 0, 3, 16, 1, 128, step, 128, 128)
    c.t_table = ints(torch, table)
    c.check(*c.run())
    # and the append reaches the same places
    qkv = torch.randn(3, 3 * 128, device="cuda").bfloat16()
    q = torch.empty(3, 128, dtype=torch.bfloat16, device="cuda")
    slots = ints(torch, [32, 5, 31])
    rt.k_paged_qkv(c.cache, qkv.data_ptr(), 384, 3, 1, 0, 0, 1e-6, 0, 0, 0, slots.data_ptr(), q.data_ptr(), 128)
    torch.cuda.synchronize()
    for t, (page, off) in enumerate([(2, 0), (0, 5), (1, 15)]):
        at = page * step + off * 128
        assert (buf[at:at + 128] == qkv[t, 128:256]).all() and (buf[at + 2048:at + 2176] == qkv[t, 256:]).all()


def test_same_bits_on_another_stream_and_again(torch, pkg):
    c = Case(torch, pkg.runtime, [3000, 17, 900, 32000], 16, 1, 128, 32)
    first = c.run()
    s = torch.cuda.Stream()
    for _ in range(3):
        again = c.run(stream=s.cuda_stream)
        assert (again[0] == first[0]).all() and (again[1] == first[1]).all()
    assert (c.run(lse=False)[0] == first[0]).all()


# ------------------------------------------------------------------------------------------ sampling

def run_sample(torch, rt, x, dtype, temperature=None, top_k=None, top_p=None, min_p=None, u=None, stride=None, offset=0):
    rows, vocab = x.shape
    stride = stride or vocab
    buf = torch.zeros(offset + rows * stride, dtype=dt(torch, dtype), device="cuda")
    view = torch.as_strided(buf, (rows, vocab), (stride, 1), offset)
    view.copy_(torch.as_tensor(x))
    f = lambda v, ty: None if v is None else torch.tensor(np.broadcast_to(v, rows).copy(), dtype=ty, device="cuda")  # noqa: E731
    args = [f(temperature, torch.float32), f(top_k, torch.int32), f(top_p, torch.float32), f(min_p, torch.float32),
            f(u, torch.float32)]
    ids, kept = ints(torch, [-9] * rows), ints(torch, [-9] * rows)
    lp = torch.full((rows,), 9.0, device="cuda")
    torch.cuda.synchronize()
    rt.k_sample(view.data_ptr(), CODE[dtype], rows, vocab, stride, *[0 if a is None else a.data_ptr() for a in args],
                ids.data_ptr(), lp.data_ptr(), kept.data_ptr())
    torch.cuda.synchronize()
    return ids.cpu().numpy(), lp.double().cpu().numpy(), kept.cpu().numpy(), view.double().cpu().numpy()


def sample_check(x, i, lp, kept, t, k, p, mp, u):
    """One row in 64 bits: the id is kept, its interval holds u, the kept number and the log probability fit."""
    x = np.where(np.isnan(x), -np.inf, x)
    w = np.exp((x - x.max()) / t)
    order = np.argsort(-x, kind="stable")
    ws = w[order]
    if k and k > 0:
        ws = np.where(np.arange(len(x)) < k, ws, 0.0)
    before = np.cumsum(ws) - ws
    total = ws.sum()

    def keep(slack):
        # weights below 2^-40 are whole zeros
        return (ws > 2.0 ** -40 * (1 - slack)) & (before < (p + slack) * total) & (ws >= mp * (1 - slack))
    least, most = keep(-D17), keep(D17)
    least[0] = most[0] = True
    assert least.sum() <= kept <= most.sum(), (least.sum(), kept, most.sum())
    run = np.zeros(len(x))
    run[order[:kept]] = ws[:kept]
    assert i in order[:kept]
    upto = run.cumsum()
    W = upto[-1]
    assert (upto[i] - run[i]) / W <= u + D17 and upto[i] / W >= u - D17
    assert abs(lp - np.log(run[i] / W)) <= 2.0 ** -16 + 2.0 ** -22 * abs(lp)


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,vocab,stride,offset", [(1, 1, None, 0), (3, 2, None, 0), (5, 33, 41, 3), (4, 1000, None, 0),
                                                      (3, 5003, 5004, 1), (9, 32001, None, 0), (2, 107520, None, 0),
                                                      (40, 4096, None, 0), (70, 777, None, 0)])
def test_sample_settings(torch, pkg, dtype, rows, vocab, stride, offset):
    rng = np.random.default_rng(vocab + rows)
    for n, (t, k, p, mp) in enumerate([(1.0, 0, 1.0, 0.0), (0.7, 7, 1.0, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 1.0, 0.05),
                                       (0.8, 50, 0.95, 0.01), (2.0, 1, 0.5, 0.0), (1.0, vocab, 0.999, 0.0), (1.0, 3, 1e-9, 1.0)]):
        x = 3.0 * rng.standard_normal((rows, vocab))
        if n % 2:
            x[:, rng.integers(0, vocab, min(vocab, 20))] += 6.0
        u = rng.random(rows).astype(np.float32)
        ids, lp, kept, seen = run_sample(torch, pkg.runtime, x, dtype, t, k, p, mp, u, stride, offset)
        for r in range(rows):
            sample_check(seen[r], ids[r], lp[r], kept[r], t, k, p, mp, u[r])
            if p == 1.0 and mp == 0.0 and 0 < k < vocab:
                assert kept[r] == k


@pytest.mark.parametrize("dtype,vocab,shape", [
    ("f32", 30011, "narrow"), ("bf16", 107520, "narrow"), ("f16", 50000, "sorted"), ("f32", 107520, "sorted"), ("bf16", 40000, "steps"),
    ("f32", 1300001, "normal"), ("bf16", 2100000, "normal"), ("f32", 20000, "zero"), ("bf16", 9000, "zero")])
def test_sample_unusual_distributions(torch, pkg, dtype, vocab, shape):
    """Kept sets of thousands, values next to each other or in each other's reach, rows past shared memory."""
    rng, rows = np.random.default_rng(vocab), 3
    x = {"narrow": lambda: 1e-3 * rng.standard_normal((rows, vocab)) + 7.0,
         "sorted": lambda: np.repeat(-np.arange(vocab)[None] * 1e-3, rows, 0),
         "steps": lambda: np.floor(4.0 * rng.standard_normal((rows, vocab))),
         "normal": lambda: 3.0 * rng.standard_normal((rows, vocab)),
         "zero": lambda: rng.standard_normal((rows, vocab)) * 10.0 ** rng.integers(-30, 1, (rows, vocab))}[shape]()
    for k, p, mp in ((0, 1.0, 0.0), (100, 1.0, 0.0), (300, 0.9, 0.0), (700, 1.0, 0.0), (5000, 0.5, 0.0), (0, 0.3, 0.0), (0, 0.97, 0.0),
                     (0, 0.97, 0.3), (vocab - 1, 0.999, 0.0)):
        u = rng.random(rows).astype(np.float32)
        ids, lp, kept, seen = run_sample(torch, pkg.runtime, x, dtype, 0.9, k, p, mp, u)
        for r in range(rows):
            sample_check(seen[r], ids[r], lp[r], kept[r], 0.9, k, p, mp, u[r])
            if p == 1.0 and k:
                assert kept[r] == k


@pytest.mark.parametrize("heads", [(1, 2, 63, 64), (65, 127, 128, 129), (1023, 1024, 1025, 1030), (4000, 500, 9000, 8191)])
@pytest.mark.parametrize("dtype,vocab", [("bf16", 9003), ("f32", 120001)])
def test_sample_few_and_many_within_reach(torch, pkg, dtype, vocab, heads):
    """All but a row's `heads` values are too unlikely to weigh anything; those lie next to each other or anywhere."""
    rng, rows = np.random.default_rng(sum(heads)), 2 * len(heads)
    x = np.full((rows, vocab), -60.0)
    for r in range(rows):
        n = heads[r // 2]
        at = rng.permutation(vocab)[:n] if r % 2 else (vocab - n) // 3 + np.arange(n)
        x[r, at] = 1.5 * rng.standard_normal(n)
    for k, p, mp in ((0, 1.0, 0.0), (0, 0.9, 0.0), (60, 1.0, 0.0), (100, 0.8, 0.0), (128, 0.95, 0.02), (200, 0.5, 0.1), (0, 0.999, 0.0)):
        u = rng.random(rows).astype(np.float32)
        ids, lp, kept, seen = run_sample(torch, pkg.runtime, x, dtype, 0.8, k, p, mp, u)
        for r in range(rows):
            sample_check(seen[r], ids[r], lp[r], kept[r], 0.8, k, p, mp, u[r])
            if p == 1.0 and mp == 0.0:
                assert kept[r] == min(k or vocab, heads[r // 2])


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_sample_extreme_temperatures(torch, pkg, dtype):
    x = np.random.default_rng(5).standard_normal((4, 3000))
    x[1], x[2, 7], x[3, [3, 2000]] = -np.inf, -np.inf, np.inf
    for t in (1e-30, 1e-18, 1e18, 1e30, np.inf):
        for k, p in ((0, 1.0), (10, 1.0), (0, 0.5)):
            ids, lp, kept, seen = run_sample(torch, pkg.runtime, x, dtype, t, k, p, None, 0.5)
            assert ids[1] == 0 and kept[1] == 0 and np.isneginf(lp[1])
            assert kept[3] == (1 if p == 0.5 else 2) and ids[3] == (3 if p == 0.5 else 2000)
            for r in (0, 2):
                full = 3000 - (r == 2)
                if t > 1:
                    assert kept[r] == (10 if k else full if p == 1.0 else (full + 1) // 2)
                else:
                    assert kept[r] == 1 and ids[r] == seen[r].argmax() and lp[r] == 0


def test_sample_ties_go_to_the_lowest_index(torch, pkg):
    rt = pkg.runtime
    x = np.zeros((1, 3000))
    x[0, 100::100] = 4.0  # 29 equal best
    u = lambda i, n: (i + 0.5) / n  # noqa: E731
    for k in (1, 5, 29):
        for i in range(k):
            ids, lp, kept, _ = run_sample(torch, rt, x, "bf16", 1.0, k, None, None, u(i, k))
            assert ids[0] == 100 * (i + 1) and kept[0] == k and abs(lp[0] + np.log(k)) < 1e-6
    ids, _, kept, _ = run_sample(torch, rt, x, "f32", 0.05, None, 0.5, None, 0.999)  # 14.5 of 29: 15 ids
    assert kept[0] == 15 and ids[0] == 1500
    flat = np.full((2, 70001), -2.5)
    ids, _, kept, _ = run_sample(torch, rt, flat, "f16", 1.0, [0, 40000], [0.25, 0.5], None, [0.0, 0.99999994])
    assert list(kept) == [17501, 20000] and list(ids) == [0, 19999]
    # -0 and 0 are equal
    z = np.full((1, 40), -50.0)
    z[0, 7], z[0, 9], z[0, 30] = -0.0, 0.0, -0.0
    ids, _, kept, _ = run_sample(torch, rt, z, "f32", 1.0, 2, None, None, 0.9)
    assert ids[0] == 9 and kept[0] == 2


def test_sample_greedy_and_odd_controls(torch, pkg):
    rt, rng = pkg.runtime, np.random.default_rng(8)
    x = rng.standard_normal((6, 5000))
    x[:, 77] = x[:, 4444] = 9.0
    t = np.array([0.0, -1.0, np.nan, 0.0, 1e-6, 0.0])
    ids, lp, kept, _ = run_sample(torch, rt, x, "f32", t, None, None, None, [0.0, 0.9, 0.5, 1.0, 0.2, np.nan])
    assert list(ids) == [77] * 6 and list(kept) == [1, 1, 1, 1, 2, 1] and (lp[[0, 1, 2, 3, 5]] == 0).all()
    # u outside [0, 1): the first and the last kept id
    ids, _, _, _ = run_sample(torch, rt, x, "f32", 1e-6, None, None, None, [-3.0, 1.0, 7.0, np.nan, 0.0, 0.6])
    assert list(ids) == [77, 4444, 4444, 77, 77, 4444]
    # controls out of range: k < 0 and > vocab off, p <= 0 keeps one, p NaN off, min_p above 1 keeps the best
    y = np.array([[0.0, 1.0, 3.0, 2.0]] * 6)
    _, _, kept, _ = run_sample(torch, rt, y, "f32", 1.0, [-1, 9, 0, 0, 0, 2], [1, 1, -1, np.nan, 0, 2], [0, -1, 0, 0, 0, 0], 0.5)
    assert list(kept) == [4, 4, 1, 4, 1, 2]
    _, _, kept, _ = run_sample(torch, rt, y, "f32", np.inf, None, None, [5.0, np.nan, 0, 0, 0, 1.0], 0.5)
    assert list(kept) == [4] * 6


def test_sample_infinities_and_nothing_to_choose(torch, pkg):
    rt, inf, nan = pkg.runtime, np.inf, np.nan
    x = np.full((5, 300), -inf)
    x[1] = nan
    x[2, 200] = -3.0e4
    x[3, [5, 250]] = inf
    x[3, 9] = 3.0
    x[4, 30:] = nan
    x[4, 10], x[4, 20] = 1.0, 1.0
    for dtype in ("bf16", "f16", "f32"):
        for t, k, p in ((1.0, 0, 1.0), (0.5, 3, 0.9), (2.0, 0, 0.5)):
            ids, lp, kept, _ = run_sample(torch, rt, x, dtype, t, k, p, None, 0.75)
            assert list(ids[:3]) == [0, 0, 200] and list(kept[:3]) == [0, 0, 1]
            assert np.isneginf(lp[:2]).all() and lp[2] == 0
            want = 1 if p == 0.5 else 2
            assert kept[3] == want and ids[3] == (5 if want == 1 else 250)
            assert kept[4] == want and ids[4] == (10 if want == 1 else 20)
        ids, _, kept, _ = run_sample(torch, rt, x, dtype, 0.0, None, None, None, 0.75)
        assert list(ids) == [0, 0, 200, 5, 10] and list(kept) == [0, 0, 1, 1, 1]


def test_sample_follows_the_distribution(torch, pkg):
    """A grid of u walks through the ids in proportion to their probabilities."""
    x = np.log(np.array([[0.5, 0.0625, 0.25, 0.1875]]))
    n = 4096
    ids, _, _, _ = run_sample(torch, pkg.runtime, np.repeat(x, n, 0), "f32", None, None, None, None, (np.arange(n) + 0.5) / n)
    assert (np.diff(ids) >= 0).all()
    assert np.abs(np.bincount(ids, minlength=4) / n - np.exp(x[0])).max() <= 1.5 / n


# ------------------------------------------------------------------------------------------ all four

def test_step_in_a_cuda_graph(torch, pkg):
    """Plan, append, attention and sampling captured as one graph give what they give one by one."""
    rt, rng = pkg.runtime, np.random.default_rng(12)
    lens, append, page, pages, table, free, count, tokens = make_plan(3, 20, 16, 80, 1, 2, 60)
    rows, heads, kv, dim, vocab = 20, 16, 1, 128, 5000
    i32 = lambda v: ints(torch, v)  # noqa: E731
    t = dict(lens=i32(lens), append=i32(append), table=i32(table), free_list=i32(free + [0] * (pages - len(free))), count=i32([count]),
             new=i32([0] * rows), start=i32([0] * (rows + 1)), slots=i32([0] * tokens), pos=i32([0] * tokens), counts=i32([0] * 4))
    caches = [torch.randn(pages, page, kv, dim, device="cuda").bfloat16() for _ in range(2)]
    cache = rt.PagedCache(caches[0].data_ptr(), caches[1].data_ptr(), 0, pages, page, kv, dim, page * dim, dim, dim)
    qkv = torch.randn(tokens, (heads + 2 * kv) * dim, device="cuda").bfloat16()
    norms = [torch.tensor(0.1 * rng.standard_normal(dim)).bfloat16().cuda() for _ in range(2)]
    rope, _ = rope_bits(torch, 80 * page + 1, dim)
    q, out = (torch.zeros(tokens, heads * dim, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    work = torch.empty(rt.paged_attention_workspace(), dtype=torch.uint8, device="cuda")
    logits = (3 * torch.randn(rows, vocab, device="cuda")).bfloat16()
    u, ids = torch.rand(rows, device="cuda"), i32([0] * rows)
    temperature, top_k, top_p = torch.full((rows,), 0.8, device="cuda"), i32([40] * rows), torch.full((rows,), 0.9, device="cuda")

    def step(stream):
        rt.k_paged_plan(t["lens"].data_ptr(), t["append"].data_ptr(), rows, page, pages, t["table"].data_ptr(), 80, t["free_list"].data_ptr(),
                        t["count"].data_ptr(), t["new"].data_ptr(), t["start"].data_ptr(), t["slots"].data_ptr(), t["pos"].data_ptr(),
                        tokens, t["counts"].data_ptr(), stream)
        rt.k_paged_qkv(cache, qkv.data_ptr(), qkv.shape[1], tokens, heads, norms[0].data_ptr(), norms[1].data_ptr(), 1e-6, rope.data_ptr(),
                       rope.shape[0], t["pos"].data_ptr(), t["slots"].data_ptr(), q.data_ptr(), heads * dim, stream)
        rt.k_paged_attention(cache, q.data_ptr(), heads * dim, tokens, heads, t["table"].data_ptr(), 80, t["new"].data_ptr(), rows,
                             t["start"].data_ptr(), 80 * page, 0, dim ** -0.5, out.data_ptr(), heads * dim, 0, work.data_ptr(),
                             work.numel(), stream)
        rt.k_sample(logits.data_ptr(), 0, rows, vocab, vocab, temperature.data_ptr(), top_k.data_ptr(), top_p.data_ptr(), 0, u.data_ptr(),
                    ids.data_ptr(), 0, 0, stream)

    torch.cuda.synchronize()
    step(0)
    torch.cuda.synchronize()
    results = [t["new"], t["slots"], t["counts"], t["table"], caches[0], caches[1], q, out, ids]
    want = [r.clone() for r in results]
    assert int((ids > 0).sum()) and float(out.float().abs().max()) > 0
    s, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.stream(s):
        g.capture_begin()
        step(s.cuda_stream)
        g.capture_end()
        for r in (t["new"], t["slots"], t["counts"], q, out, ids):
            r.zero_()
        for _ in range(3):
            g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(results, want))
