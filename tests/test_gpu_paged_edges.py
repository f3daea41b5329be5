"""Edges of the paged key / value cache's operators: what a row's company in the batch may change, numbers at the ends of
their formats, infinities and NaN in every place, long pieces, shared pages in odd places, tables of 2^31 entries."""
import math

import pytest
import torch

from tests import paged_reference as R
from tests.test_gpu_paged import DTYPES, check_attend, fill, make

pytestmark = pytest.mark.gpu
LN2 = 0.6931471824645996  # in fp32; times log2(e) in fp32 this is exactly 1, so scores are powers of two


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability(0)[0] != 10:
        pytest.fail("GPU tests need an sm_100 device")


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("tokens", [1, 16, 40])
def test_scores_of_2_to_the_29(tokens, dtype):
    """Scores near the end of what 16-bit queries and keys give, where fp32 counts in steps of 32: the best key is further
    from the next than those steps, so it takes everything."""
    past, dim, heads = 300, 128, 4
    c, g = make(1, 1, dim, dtype, 32, [past + tokens], seed=11)
    keys, values = fill(c, [past + tokens], g)
    keys = (torch.rand(past + tokens, dim, generator=g) * 4096 - 2048).to(dtype)
    pos = torch.arange(past + tokens)
    c.data[0, 0][c.table.cpu()[0].long()[pos // 32].cuda(), 0, (pos % 32).cuda()] = keys.cuda()
    q = (torch.rand(1, tokens, heads, dim, generator=g) * 4096 - 2048).to(dtype)
    s = torch.einsum("thd,jd->thj", q[0].double(), keys.double()) * 8
    s = s.masked_fill(pos[None, None] > past + torch.arange(tokens)[:, None, None], -math.inf)
    top = s.topk(2, dim=-1)
    out = c.attend(0, q.cuda(), torch.tensor([past], device="cuda"), scale=8.0)[0].cpu()
    # a product's 128 terms of up to 2^25 are summed with steps of at most 2^9 each (2^32 in fp32, cut off): 2^16 in all
    clear = top.values[..., 0] - top.values[..., 1] > 2.0 ** 17
    assert clear.double().mean() > 0.9
    assert torch.equal(out[clear], values[0][0][top.indices[..., 0]][clear])
    assert c.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("tokens", [1, 7, 16, 32, 40])
def test_a_row_alone_and_in_a_batch(tokens, dtype):
    """The weights' rounding to 16 bits does not depend on where the batch cuts a row's keys.

    Scores are multiples of 2^-6 (in powers of two), so they are exact whatever maximum is taken off, and values are +-1:
    weights of [2^-3, 1] in 8 or 11 bits add up exactly in fp32 (1024 of them: at most 10 + 3 + 11 bits).  What the cut
    may change is the fp32 order of the 1024 weights' sum, at most 1024 * 2^-24 = 2^-14 of it: a result moves by one step
    of its type at most, and only where it lies that near to the middle between two: 2^-14 / 2^-8 of the results in bf16,
    2^-14 / 2^-11 in fp16, twice that for the two sides."""
    keys_n, heads, dim, rows = 1024, 4, 64, 45
    c, g = make(1, 1, dim, dtype, 64, [keys_n], seed=tokens, extra=0)
    sign = lambda *s: (torch.randint(0, 2, s, generator=g) * 2 - 1).to(dtype)  # noqa: E731
    table = c.table.cpu()[0].long()
    c.data[0, 0, table[:16].cuda(), 0] = sign(keys_n, dim).view(16, 64, dim).cuda()
    c.data[0, 1, table[:16].cuda(), 0] = sign(keys_n, dim).view(16, 64, dim).cuda()
    q = 3 * sign(1, tokens, heads, dim).cuda()
    start = torch.tensor([keys_n - tokens], device="cuda")
    alone = c.attend(0, q, start, scale=LN2 / 64)

    from domino_b200 import PagedKVCache

    many = PagedKVCache(1, rows, 1, c.pages, dim, dtype, "cuda", page_size=64, row_pages=c.row_pages)
    many.data.copy_(c.data)
    many.table.copy_(c.table.expand(rows, -1))
    past = torch.randint(0, keys_n - tokens, (rows,), generator=g)  # the others are shorter, by every length
    past[::5] = keys_n - tokens
    out = many.attend(0, q.expand(rows, -1, -1, -1).contiguous(), past.cuda(), scale=LN2 / 64)
    eps = torch.finfo(dtype).eps / 2
    a, b = alone.double(), out[::5].double()
    step = 2 * eps * torch.maximum(a.abs(), b.abs())
    assert ((a - b).abs() <= 1.01 * step + 2.0 ** -24).all()
    share = (a != b).double().mean().item()
    assert share <= 2 * 2.0 ** -14 / eps, share
    assert many.status() == 0


@pytest.mark.parametrize("tokens,heads,window", [(300, 1, 0), (300, 1, 60000), (16, 4, 0), (33, 3, 50000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_non_finite_values_in_long_pieces(tokens, heads, window, dtype):
    """A NaN and infinities that only some queries see, at the end of 65 536 keys that one CTA walks: everything else is
    as without them, no wait gives up, and the next call on the cache is right."""
    from domino_b200 import PagedKVCache

    past, dim, page, rows = 65536, 64, 128, 148
    own = -(-tokens // page)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    c = PagedKVCache(1, rows, 1, past // page + rows * own, dim, dtype, "cuda", page_size=page, row_pages=past // page + own)
    c.table[:, : past // page] = torch.arange(past // page, dtype=torch.int32, device="cuda")
    c.table[:, past // page:] = past // page + torch.arange(rows * own, dtype=torch.int32, device="cuda").view(rows, own)
    c.data.copy_(torch.randn(c.data.shape, generator=g, device="cuda"))
    q = torch.randn(rows, tokens, heads, dim, generator=g, device="cuda").to(dtype)
    start = torch.full((rows,), past, device="cuda")
    clean = c.attend(0, q, start, window=window)
    assert c.status() == 0 and bool(torch.isfinite(clean).all())
    t = tokens // 2
    edge = past - window + 1 + t if window else None  # seen by tokens 0 .. t, left behind by those after them
    spots = []
    for b, value in ((0, float("nan")), (3, float("inf")), (rows - 1, float("-inf"))):
        spots.append((b, t, slice(t, None), value, (0, 1, past // page + b * own + t // page, 0, t % page, 9)))
    if window:
        spots.append((None, None, slice(0, t + 1), float("nan"), (0, 1, edge // page, 0, edge % page, 20)))
    want, kept = clean.clone(), {}
    for b, _, seen, value, at in spots:
        kept[at] = c.data[at].clone()
        c.data[at] = value
        rows_hit = slice(None) if b is None else slice(b, b + 1)
        want[rows_hit, seen, :, at[-1]] = value
    out = c.attend(0, q, start, window=window)
    assert c.status() == 0
    assert torch.equal(torch.isnan(out), torch.isnan(want))
    assert torch.equal(out.nan_to_num(nan=0.0), want.nan_to_num(nan=0.0))
    for *_, at in spots:
        c.data[at] = kept[at]
    again = c.attend(0, q, start, window=window)
    assert c.status() == 0 and torch.equal(again, clean)


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
@pytest.mark.parametrize("tokens,dim,past", [(1, 128, 40), (1, 64, 3000), (3, 128, 700), (16, 128, 1500), (16, 64, 9000),
                                             (30, 128, 900), (90, 64, 3000)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_an_infinite_value_that_is_seen(tokens, dim, past, dtype, value):
    """An infinity or a NaN among the values, old (every query sees it, in a tile that all see) and new (only the queries
    behind it do): the results that it is part of are that infinity or a NaN, all others are as without it.

    Queries and keys are of order one, so no weight is anywhere near the end of fp32."""
    c, g = make(1, 2, dim, dtype, 32, [past + tokens], seed=tokens + dim)
    fill(c, [past + tokens], g)
    q = torch.randn(1, tokens, 8, dim, generator=g).to(dtype).cuda()
    start = torch.tensor([past], device="cuda")
    clean = c.attend(0, q, start)
    spots = [0, 5, past // 2, past - 1, past + tokens // 2]
    for j in spots:
        at = (0, 1, int(c.table[0, j // 32]), 1, j % 32, 7)
        keep = c.data[at].clone()
        c.data[at] = value
        out = c.attend(0, q, start)
        c.data[at] = keep
        t0 = max(j - past, 0)
        want = torch.full_like(out[0, t0:, 4:, 7], value)  # key head 1 serves query heads 4 .. 7
        assert torch.allclose(out[0, t0:, 4:, 7], want, equal_nan=True), j
        out[0, t0:, 4:, 7] = clean[0, t0:, 4:, 7]
        assert torch.equal(out, clean), j
    # two infinities of one sign, far apart and side by side, then a NaN's worth: one of each sign
    for signs in ((1, 1), (1, -1)):
        for j0, j1 in ((0, past // 2), (5, 6), (past // 2, past + tokens // 2)):
            keep = []
            for j, s in zip((j0, j1), signs):
                at = (0, 1, int(c.table[0, j // 32]), 0, j % 32, 3)
                keep.append((at, c.data[at].clone()))
                c.data[at] = s * float("inf")
            out = c.attend(0, q, start)
            for at, x in keep:
                c.data[at] = x
            t0 = max(j1 - past, 0)
            got = out[0, t0:, :4, 3]
            assert bool((got == float("inf")).all() if signs[1] > 0 else torch.isnan(got).all()), (signs, j0, j1)
            assert bool((out[0, :t0, :4, 3] == float("inf")).all()) or t0 == 0
    assert c.status() == 0


def _one_key_above(n, tokens, below, dtype):
    """148 rows of `tokens` queries over n keys in one piece each: key 0 has score 0 and value -1, the others score -below
    (in powers of two) and value 1.  Returns the results and what they are in 64 bits."""
    from domino_b200 import PagedKVCache

    dim, rows = 64, 148
    c = PagedKVCache(1, rows, 1, n // 128, dim, dtype, "cuda", page_size=128, row_pages=n // 128)
    c.table.copy_(torch.arange(n // 128, dtype=torch.int32).expand(rows, -1))
    c.data[0, 0].zero_()
    c.data[0, 0, :, :, :, 0] = -below
    c.data[0, 0, 0, 0, 0, 0] = 0.0
    c.data[0, 1].fill_(1.0)
    c.data[0, 1, 0, 0, 0] = -1.0
    q = torch.zeros(rows, tokens, 1, dim, dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    out = c.attend(0, q, torch.full((rows,), n - tokens, device="cuda"), scale=LN2)
    assert c.status() == 0
    score = torch.tensor(below, dtype=torch.float64).to(dtype).double().item()
    others = torch.arange(n - tokens, n, dtype=torch.float64) * 2.0 ** -score
    return out.double().cpu(), ((others - 1) / (others + 1))[None, :, None, None]


@pytest.mark.parametrize("tokens,below", [(130, 25.046875), (130, 18.40625), (300, 24.59375), (100, 25.046875)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_key_far_above_very_many(tokens, below, dtype):
    """A key that takes nearly all the weight and 65535 others `below` powers of two under it: their sum is part of the
    result as it is part of the row's sum.

    One rounding of every weight and of the result; at most 1024 additions to the row's sum (2^-24 each).  The products'
    sum lies in (1/2, 1]: taken one product at a time and rounded to nearest in fp32, whose steps there are 2^-24, each of
    the 65535 moves it by 2^-25 from the exact one at most, 2^-9 in all, and equal products all to the same side (those
    below 2^-25 leave it where it is)."""
    out, ref = _one_key_above(65536, tokens, below, dtype)
    assert (out - ref).abs().max() <= 2 * torch.finfo(dtype).eps / 2 + 1024 * 2.0 ** -24 + 65535 * 2.0 ** -25


@pytest.mark.parametrize("tokens", [130, 300, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_below_fp16_normals_under_one_large_one(tokens, dtype):
    """The same with weights of 3.02 * 2^-25, whole steps of the products' sum but for 0.02 * 2^-25 each (2^-14.6 in all;
    3.08 and 2^-12.6 in bf16, whose scores are coarser): a weight that fp16 rounds to 2^-23 by itself would be 2^-9 off."""
    out, ref = _one_key_above(65536, tokens, 23.40625, dtype)
    assert (out - ref).abs().max() <= 2 * torch.finfo(dtype).eps / 2 + 1024 * 2.0 ** -24 + 2.0 ** -12.6


def test_compact_is_for_the_whole_table():
    """A view of the first rows does not know the other rows' tables: it may not move the pool's pages."""
    from domino_b200 import PagedKVCache

    c = PagedKVCache(1, 3, 1, 12, 8, torch.float32, "cuda", page_size=16, row_pages=2)
    c.table.copy_(torch.tensor([[9, -1], [3, 11], [7, -1]], dtype=torch.int32))
    c.refs[torch.tensor([9, 3, 11, 7], device="cuda")] = 1
    c.length.copy_(torch.tensor([10, 30, 16]))
    c.data.copy_(torch.arange(12.0).view(1, 1, 12, 1, 1, 1).expand_as(c.data))
    before = [x.clone() for x in (c.table, c.refs, c.data)]
    for view in (c.first_rows(1), c.first_rows(2), c.first_rows(2).first_rows(2)):
        with pytest.raises(ValueError, match="rows"):
            view.compact()
    assert all(torch.equal(a, b) for a, b in zip(before, (c.table, c.refs, c.data)))
    c.first_rows(3).compact()  # all of them
    assert c.table.tolist() == [[1, -1], [3, 2], [0, -1]]
    for b, stamps in enumerate(([9], [3, 11], [7])):
        assert [c.data[0, 0, p, 0, 0, 0].item() for p in c.table[b].tolist() if p >= 0] == stamps
    assert c.status() == 0


def test_compact_with_a_table_of_nearly_2_31_entries():
    """Entry numbers near 2^31 (a table of 8.6 GB, as much again in the scratch): the moved pages are followed in the
    last row as in the first."""
    from domino_b200 import PagedKVCache

    batch, row_pages = 1024, (1 << 21) - 1
    c = PagedKVCache(1, batch, 1, 10, 8, torch.bfloat16, "cuda", page_size=16, row_pages=row_pages)
    spots = [(0, 0), (0, row_pages - 1), (511, 77), (1023, row_pages - 300000), (1023, row_pages - 1)]
    for p, (b, i) in zip((9, 4, 7, 8, 2), spots):
        c.table[b, i] = p
        c.refs[p] = 1
    c.data.copy_(torch.arange(10.0).view(1, 1, 10, 1, 1, 1).expand_as(c.data))
    c.compact()
    assert c.status() == 0
    where = [int(c.table[b, i]) for b, i in spots]
    assert sorted(where) == [0, 1, 2, 3, 4]
    assert [c.data[0, 1, p, 0, 0, 0].item() for p in where] == [9, 4, 7, 8, 2]
    assert int((c.table >= 0).sum()) == 5
    del c
    torch.cuda.empty_cache()


@pytest.mark.parametrize("back", [0, 5, 16, 40])
def test_reserve_replaces_every_shared_page_it_reaches(back):
    """Rows that continue one row and are set back by hand (not by crop): all shared pages that the new positions reach
    are replaced, and the rows that are not asked for keep what they hold."""
    from domino_b200 import PagedKVCache

    page, n = 16, 70
    c = PagedKVCache(2, 4, 1, 40, 8, torch.float32, "cuda", page_size=page, row_pages=8)
    c.reserve(torch.tensor([n, 0, 0, 0], device="cuda"))
    k = torch.randn(4, n, 1, 8, device="cuda")
    start = torch.zeros(4, dtype=torch.long, device="cuda")
    lens = torch.tensor([n, 0, 0, 0], device="cuda")
    for layer in range(2):
        c.write(layer, None, k, k, None, start, lens)
    c.length.copy_(lens)
    c.fork(torch.zeros(4, dtype=torch.long, device="cuda"))
    old = c.table.clone()
    held = c.data.clone()
    c.length[:3] = back                       # rows 0 .. 2 go back; row 3 keeps all of it
    upto = torch.tensor([n, n, back + 20, 0], device="cuda")
    c.reserve(upto)
    assert c.status() == 0
    assert torch.equal(c.table[3], old[3])
    first, table = back // page, c.table.tolist()
    for b, up in ((0, n), (1, n), (2, back + 20)):
        own = table[b][first: -(-up // page)]
        assert all(c.refs[p] == 1 for p in own) and -1 not in own
        assert table[b][:first] == old[0, :first].tolist()
        for i in range(first, -(-up // page)):  # copies of what was there
            if i < 5:
                assert torch.equal(c.data[:, :, table[b][i]], held[:, :, int(old[0, i])])
    assert int(c.refs.sum()) == int((c.table >= 0).sum())
    new = torch.randn(4, n, 1, 8, device="cuda")
    m = torch.where(torch.arange(4, device="cuda") < 3, upto - back, 0)
    st = torch.where(torch.arange(4, device="cuda") < 3, back, 0)
    c.write(1, None, new, new, None, st, m)
    assert c.status() == 0
    for i in range(5):
        assert torch.equal(c.data[:, :, int(old[3, i])], held[:, :, int(old[3, i])])
    for b in range(3):
        pos = torch.arange(back, int(upto[b]))
        got = c.data[1, 0, c.table[b].cpu().long()[pos // page].cuda(), 0, (pos % page).cuda()]
        assert torch.equal(got, new[b, : len(pos), 0])


def test_reserve_lets_the_first_row_keep_pages_that_only_reaching_rows_hold():
    """Three rows share five pages, all are set back and all reach them: the first keeps the originals, the others copy;
    a pool that is too small leaves out the last requests and says so."""
    from domino_b200 import PagedKVCache, _lib

    for pages, ok in ((15, True), (12, False)):
        c = PagedKVCache(1, 3, 1, pages, 8, torch.float32, "cuda", page_size=16, row_pages=5)
        c.reserve(torch.tensor([80, 0, 0], device="cuda"))
        c.length.copy_(torch.tensor([80, 0, 0]))
        c.fork(torch.zeros(3, dtype=torch.long, device="cuda"))
        c.length.zero_()
        c.reserve(torch.full((3,), 80, device="cuda"))
        assert c.status() == (0 if ok else _lib.DD_STATUS_NO_PAGE)
        table = c.table.tolist()
        assert table[0] == [0, 1, 2, 3, 4] and table[1] == [5, 6, 7, 8, 9]
        assert table[2] == ([10, 11, 12, 13, 14] if ok else [10, 11, 2, 3, 4])
        assert c.refs.tolist() == ([1] * 15 if ok else [1, 1, 2, 2, 2] + [1] * 7)


class _AllSlots(R.HostPages):
    """The host model with the sharing rule for every slot that a row reaches."""

    def reserve(self, upto):
        cap = self.row_pages * self.page
        reach = [(b, i) for b, u in enumerate(upto) if min(u, cap) > self.length[b]
                 for i in range(self.length[b] // self.page, math.ceil(min(u, cap) / self.page))]
        by_page = {}
        for b, i in reach:
            by_page.setdefault(self.table[b][i], []).append(b)
        want = []
        for b, i in reach:
            p = self.table[b][i]
            if p < 0:
                want.append((b, i, -1))
            elif self.refs[p] > 1 and (self.refs[p] > len(by_page[p]) or by_page[p][0] < b):
                want.append((b, i, p))
        free = self._free()
        for (b, i, old), new in zip(want, free):
            if old >= 0:
                self.refs[old] -= 1
                self.content[new] = self.content[old]
            self.table[b][i] = new
            self.refs[new] = 1
        return len(want) <= len(free) and all(u <= cap for u in upto)


@pytest.mark.parametrize("seed,batch,pages,page,row_pages", [(0, 4, 60, 16, 6), (1, 33, 400, 32, 9), (3, 7, 30, 64, 8),
                                                             (4, 300, 3000, 16, 40)])
def test_random_sequences_with_lengths_set_back_by_hand(seed, batch, pages, page, row_pages):
    """Random reserve / advance / fork / crop / lengths set back: tables, counts and contents as the host model's."""
    import random

    from domino_b200 import PagedKVCache, _lib
    from tests.test_gpu_paged import _same, _stamp

    rng = random.Random(seed)
    c = PagedKVCache(2, batch, 2, pages, 8, torch.float32, "cuda", page_size=page, row_pages=row_pages)
    h = _AllSlots(batch, pages, page, row_pages)
    c.data.copy_(torch.arange(-pages, 0).view(1, 1, pages, 1, 1, 1).expand_as(c.data))
    for step in range(40):
        op = rng.choice(["grow", "grow", "back", "fork", "crop"])
        if op == "grow":
            upto = [max(0, n + rng.choice([0, 1, page, 3 * page + 1, -5])) for n in h.length]
            c.reserve(torch.tensor(upto, device="cuda"))
            ok = h.reserve(upto)
            assert c.status() == (0 if ok else _lib.DD_STATUS_NO_PAGE)
            _same(c, h, step)
            for b in range(batch):
                n = h.length[b]
                while n < upto[b] and n < row_pages * page and h.table[b][n // page] >= 0 and h.refs[h.table[b][n // page]] == 1:
                    n += 1
                h.length[b] = n
            c.length.copy_(torch.tensor(h.length))
            _stamp(c, h, range(min(batch, 40)))
        elif op == "back":
            h.length = [rng.choice([n, n, n // 2, max(0, n - page)]) for n in h.length]
            c.length.copy_(torch.tensor(h.length))
        elif op == "crop":
            to = [max(-1, n - rng.choice([0, 0, 1, page, -9])) for n in h.length]
            c.crop(torch.tensor(to, device="cuda"))
            h.crop(to)
        else:
            src = [rng.choice([b, b, b, -1, rng.randrange(batch), 0]) for b in range(batch)]
            c.fork(torch.tensor(src, device="cuda"))
            h.fork(src)
        _same(c, h, step)


def threads_with_caches_of_their_own():
    """The first calls of a process come from several threads at once, each on a cache and a stream of its own."""
    import threading

    from domino_b200 import PagedKVCache, Rope

    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(2, 20, h, 64, generator=g).to(torch.bfloat16).cuda() for h in (4, 2, 2))
    start = torch.zeros(2, dtype=torch.long, device="cuda")
    rope = Rope(64, device="cuda")
    gate, results, errors = threading.Barrier(8), [None] * 8, []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            c = PagedKVCache(1, 2, 2, 8, 64, torch.bfloat16, "cuda", page_size=16, row_pages=4)
            torch.cuda.synchronize()
            gate.wait()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    c.reserve(start + 20)
                    out = c.attend(0, c.write(0, q, k, v, rope, start), start)
                    c.crop(start)
            stream.synchronize()
            assert c.status() == 0
            results[i] = out
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(8)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors
    assert all(torch.equal(results[0], r) for r in results[1:])


def test_first_calls_of_several_threads():
    """In a process of its own, where nothing has been called before."""
    import subprocess
    import sys

    code = "from tests.test_gpu_paged_edges import threads_with_caches_of_their_own as go; go()"
    for _ in range(2):
        r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
        assert r.returncode == 0, r.stderr[-2000:]


def test_status_sees_calls_on_other_streams():
    """A call that is still waiting on a stream of its own when the status is read from another."""
    from domino_b200 import PagedKVCache, _lib

    c = PagedKVCache(1, 1, 1, 2, 8, torch.float32, "cuda", page_size=16)
    x = torch.ones(1, 1, 1, 8, device="cuda")
    start = torch.zeros(1, dtype=torch.long, device="cuda")
    side = torch.cuda.Stream()
    c.write(0, None, x, x, None, start)  # (a kernel's first launch may wait for the device)
    assert c.status() == _lib.DD_STATUS_NO_PAGE
    with torch.cuda.stream(side):
        torch.cuda._sleep(100_000_000)  # about 50 ms
        c.write(0, None, x, x, None, start)  # no page
    assert c.status() == _lib.DD_STATUS_NO_PAGE
    assert c.status() == 0


@pytest.mark.parametrize("tokens,heads,dim", [(1, 4, 128), (7, 4, 64), (16, 4, 128), (33, 3, 96), (50, 4, 128), (300, 1, 64)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_a_query_that_sees_one_key_gives_its_value(tokens, heads, dim, dtype):
    """Bit for bit: a weight's rounding is part of the row's sum too.  (P v is exact in fp32, 1 / P and the product are
    within 2^-22 of v, and v is the nearest number of its type; in fp32 itself the weight is 1.)"""
    past = 200
    c, g = make(1, 2, dim, dtype, 32, [past + tokens], seed=tokens)
    keys, values = fill(c, [past + tokens], g)
    q = torch.randn(1, tokens, 2 * heads, dim, generator=g).to(dtype).cuda()
    out = c.attend(0, q, torch.tensor([past], device="cuda"), window=1)
    want = values[0][:, past:].transpose(0, 1).repeat_interleave(heads, dim=1)
    assert torch.equal(out[0].cpu(), want)


@pytest.mark.parametrize("tokens,past", [(16, 0), (16, 130), (1, 90), (64, 0), (200, 0), (64, 500)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_errors_against_a_result_rounded_once(tokens, past, dtype):
    """The 2-norm of the error in 64 bits against that of rounding the exact result alone.

    A row's weights w_i (sum 1) carry independent roundings d_i, at most half a step u relative and u / sqrt(3) in the mean
    square, and the largest counts as it was rounded: the result moves by sum w_i d_i v_i less the largest's part along the
    result itself, at most u / sqrt(3) * sqrt(sum w_i^2) |v| in the mean square, while |o| is sqrt(sum w_i^2) |v| for
    independent values.  The result's own rounding is u / sqrt(3) to u / (2 sqrt(3)) of |o| between the ends of a binade,
    about u / sqrt(3) * 0.72 over all of one, and the weights' the same 0.72: together sqrt(2) of the rounding alone."""
    kv, heads, dim = 2, 8, 64
    total = [past + tokens] * 6
    c, g = make(6, kv, dim, dtype, 64, total, seed=past)
    keys, values = fill(c, total, g)
    q = 2 * torch.randn(6, tokens, heads, dim, generator=g).to(dtype)
    out = c.attend(0, q.cuda(), torch.full((6,), past, device="cuda")).double().cpu()
    ref = R.attend(q, keys, values, [torch.ones(n, dtype=torch.bool) for n in total], [past] * 6, [tokens] * 6, True, 0, 0,
                   dim ** -0.5)
    err, own = (out - ref).norm(), (ref.to(dtype).double() - ref).norm()
    assert err <= 2 ** 0.5 * own, (err / own).item()


@pytest.mark.parametrize("tokens", [1, 16, 50])
@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_of_minus_infinity(tokens, dtype):
    """Keys whose score is -infinity have no weight beside others, and give zeros where there is no other."""
    past = 150
    c, g = make(1, 1, 64, dtype, 16, [past + tokens], seed=3)
    keys, values = fill(c, [past + tokens], g)
    q = (1 + torch.rand(1, tokens, 4, 64, generator=g)).to(dtype).cuda()
    start = torch.tensor([past], device="cuda")
    pages = c.table[0, : -(-(past + tokens) // 16)].long()
    keep = c.data[0, 0].clone()
    c.data[0, 0, :, :, :, 0] = -math.inf
    assert (c.attend(0, q, start) == 0).all()
    c.data[0, 0] = keep
    c.data[0, 0, pages[3], 0, 5, 0] = -math.inf  # position 53 alone
    seen = torch.ones(past + tokens, dtype=torch.bool)
    seen[53] = False
    check_attend(c, c.attend(0, q, start), q, keys, values, [past], [tokens], seen=[seen])
