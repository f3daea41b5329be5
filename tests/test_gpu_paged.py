"""The paged key / value cache (domino_b200.paged) against plain 64-bit restatements of its definitions.

Tolerances.  eps = finfo(dtype).eps / 2 is one rounding to the cache's type.  ``write`` rounds once; its fp32 arithmetic
(two products and a sum of values below |x| factor, a norm, a sine and cosine right to a few 2^-24) adds at most 2^-20 of
the largest value in the pair, so |error| <= eps |y| + 2^-20 max|x|.  ``attend`` gives a weighted mean of values |v| <=
vmax: the weights of the 16-bit types are rounded (relative eps each, so at most eps vmax in the mean), the result once
more (eps |o| <= eps vmax), and fp32 scores of size s are off by at most 2^-20 (1 + |s|) after the exponential, which
moves the mean by at most twice that times vmax."""
import math

import pytest
import torch

from tests import paged_reference as R

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope="module", autouse=True)
def _require_gpu():
    if not torch.cuda.is_available() or torch.cuda.get_device_capability(0)[0] != 10:
        pytest.fail("GPU tests need an sm_100 device")


def make(batch, kv_heads, dim, dtype, page, total, layers=1, seed=0, extra=3, poison=float("nan")):
    """A cache whose rows hold `total[b]` positions in scattered pages; every entry no row holds is `poison`."""
    from domino_b200 import PagedKVCache

    g = torch.Generator().manual_seed(seed)
    count = [-(-int(t) // page) for t in total]
    pages = sum(count) + extra
    c = PagedKVCache(layers, batch, kv_heads, pages, dim, dtype, "cuda", page_size=page,
                     row_pages=max(max(count), 1) + 1)
    order = torch.randperm(pages, generator=g)
    c.data.fill_(poison)
    at = 0
    for b in range(batch):
        own = order[at: at + count[b]]
        at += count[b]
        c.table[b, : count[b]] = own.int().cuda()
        c.refs[own.cuda()] = 1
    return c, g


def fill(c, total, g, layer=0):
    """Random keys and values for positions below total[b]; returns them per row, [KV, n, D] of the cache's type."""
    keys, values = [], []
    table = c.table.cpu()
    for b, n in enumerate(total):
        k = torch.randn(c.kv_heads, int(n), c.head_dim, generator=g).to(c.dtype)
        v = torch.randn(c.kv_heads, int(n), c.head_dim, generator=g).to(c.dtype)
        pos = torch.arange(int(n))
        at, off = table[b].long()[pos // c.page_size].cuda(), (pos % c.page_size).cuda()
        c.data[layer, 0][at, :, off] = k.transpose(0, 1).cuda()
        c.data[layer, 1][at, :, off] = v.transpose(0, 1).cuda()
        keys.append(k)
        values.append(v)
    return keys, values


def check_attend(c, out, q, keys, values, start, lens, causal=True, window=0, sinks=0, scale=None, seen=None):
    scale = c.head_dim ** -0.5 if scale is None else scale
    seen = [torch.ones(k.shape[1], dtype=torch.bool) for k in keys] if seen is None else seen
    ref = R.attend(q.cpu(), keys, values, seen, start, lens, causal, window, sinks, scale)
    out = out.double().cpu()
    assert bool(torch.isfinite(out).all()), (~torch.isfinite(out)).nonzero()[:5].tolist()
    eps = torch.finfo(c.dtype).eps / 2
    for b in range(c.batch):
        vmax = values[b].abs().max().item() if values[b].numel() else 0.0
        smax = (q[b].float().norm(dim=-1).max().item()
                * (keys[b].float().norm(dim=-1).max().item() if keys[b].numel() else 0.0) * scale)
        tol = (2 * eps + 2 * 2.0 ** -20 * (1 + smax)) * vmax
        err = (out[b] - ref[b]).abs().max().item()
        assert err <= tol, (b, err, tol)
        n = min(int(lens[b]), q.shape[1])
        assert bool((out[b, n:] == 0).all())
    return ref


CASES = [
    # heads, kv_heads, dim, page, tokens, past of each row, lens of each row
    (4, 2, 128, 64, 1, [0], [1]),
    (4, 2, 128, 64, 1, [1, 62, 63, 64, 65, 200], [1, 1, 1, 1, 0, 1]),
    (32, 8, 128, 64, 16, [500, 130], [16, 11]),
    (8, 2, 64, 16, 16, [0, 15, 16, 127, 128, 129], [16, 16, 1, 2, 16, 0]),
    (3, 1, 96, 32, 37, [91, 0], [37, 36]),
    (5, 1, 80, 128, 130, [257], [130]),
    (7, 7, 64, 32, 3, [1000, 3], [3, 3]),
    (40, 4, 128, 16, 33, [300, 17], [33, 20]),
    (2, 1, 8, 16, 5, [20], [5]),
    (4, 2, 16, 64, 16, [40, 0, 100], [16, 16, 3]),
    (2, 1, 256, 64, 9, [150, 0], [9, 5]),
    (2, 2, 136, 32, 4, [70], [4]),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("case", CASES)
def test_attend_causal_and_whole_block(case, dtype):
    heads, kv, dim, page, T, past, lens = case
    total = [p + n for p, n in zip(past, lens)]
    c, g = make(len(past), kv, dim, dtype, page, total, seed=T)
    keys, values = fill(c, total, g)
    q = torch.randn(len(past), T, heads, dim, generator=g).to(dtype).cuda() * 2
    start, n = torch.tensor(past, device="cuda"), torch.tensor(lens, device="cuda")
    for causal in (True, False):
        check_attend(c, c.attend(0, q, start, n, causal=causal), q, keys, values, past, lens, causal)
    if all(x == T for x in lens):
        check_attend(c, c.attend(0, q, start), q, keys, values, past, lens)
    assert c.status() == 0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 1), (17, 3), (128, 64), (129, 200), (100000, 4)])
def test_attend_window_and_sinks(window, sinks, dtype):
    past, lens, T = [700, 0, 130, 256], [40, 40, 7, 1], 40
    total = [p + n for p, n in zip(past, lens)]
    c, g = make(4, 2, 64, dtype, 32, total, seed=window)
    keys, values = fill(c, total, g)
    q = torch.randn(4, T, 6, 64, generator=g).to(dtype).cuda()
    out = c.attend(0, q, torch.tensor(past, device="cuda"), torch.tensor(lens, device="cuda"), window=window, sinks=sinks)
    check_attend(c, out, q, keys, values, past, lens, window=window, sinks=sinks)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_long_chunk_many_tiles(dtype):
    """Chunks of several query tiles, rows of very different length in one call: sampled rows against the definition."""
    past, lens, T = [1500, 0, 77], [300, 300, 120], 300
    total = [p + n for p, n in zip(past, lens)]
    c, g = make(3, 1, 128, dtype, 64, total, seed=5)
    keys, values = fill(c, total, g)
    q = torch.randn(3, T, 3, 128, generator=g).to(dtype).cuda()
    out = c.attend(0, q, torch.tensor(past, device="cuda"), torch.tensor(lens, device="cuda"))
    check_attend(c, out, q, keys, values, past, lens)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_what_is_not_seen_has_no_effect(dtype):
    """Infinities and NaN in positions behind the chunk, in front of the window, in later tokens of the chunk itself,
    and pages that the table does not have."""
    past, lens, T = [300, 130], [20, 5], 20
    total = [p + n for p, n in zip(past, lens)]
    for poison in (float("nan"), float("inf"), float("-inf"), torch.finfo(dtype).min):
        c, g = make(2, 2, 64, dtype, 16, [t + 40 for t in total], seed=9, poison=poison)
        keys, values = fill(c, total, g)
        q = torch.randn(2, T, 4, 64, generator=g).to(dtype).cuda()
        start, n = torch.tensor(past, device="cuda"), torch.tensor(lens, device="cuda")
        check_attend(c, c.attend(0, q, start, n), q, keys, values, past, lens)
        # row 0: pages 3 and 4 (positions 48 .. 79) missing, one below and one above the valid numbers
        c.table[0, 3], c.table[0, 4] = -7, c.pages + 5
        seen = [torch.ones(t, dtype=torch.bool) for t in total]
        seen[0][48:80] = False
        check_attend(c, c.attend(0, q, start, n), q, keys, values, past, lens, seen=seen)
        check_attend(c, c.attend(0, q, start, n, causal=False), q, keys, values, past, lens, causal=False, seen=seen)


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_non_finite_values_of_later_tokens_and_old_keys(dtype):
    """A NaN that one query sees is that query's alone: later tokens of the chunk and keys the window has left behind."""
    past, lens, T = [200], [24], 24
    c, g = make(1, 1, 64, dtype, 32, [224], seed=2)
    keys, values = fill(c, [224], g)
    q = torch.randn(1, T, 4, 64, generator=g).to(dtype).cuda()
    table = c.table.cpu()[0]

    def put(pos, kv, value):
        c.data[0, kv, int(table[pos // 32]), 0, pos % 32, 5] = value

    start = torch.tensor(past, device="cuda")
    put(210, 1, float("nan"))                      # the value of token 10: only tokens 10 .. 23 see it
    out = c.attend(0, q, start)
    good = c.attend(0, q, start, torch.tensor([10], device="cuda"))
    assert torch.isnan(out[0, 10:, :, 5]).all() and torch.isfinite(out[0, :10]).all()
    assert torch.isfinite(out[..., :5]).all() and torch.isfinite(out[..., 6:]).all()
    check = R.attend(q.cpu()[:, :10], [keys[0][:, :210]], [values[0][:, :210]], [torch.ones(210, dtype=torch.bool)], past,
                     [10], True, 0, 0, 0.125)
    eps = torch.finfo(dtype).eps / 2
    tol = (2 * eps + 2.0 ** -15) * values[0].abs().max().item()
    assert (out[0, :10].double().cpu() - check[0]).abs().max() <= tol
    assert (good[0, :10].double().cpu() - check[0]).abs().max() <= tol
    put(210, 1, 0.0)
    put(195, 1, float("inf"))                      # behind the window of 8 for tokens 3 .. 23, inside for 0 .. 2
    out = c.attend(0, q, start, window=8)
    assert torch.isinf(out[0, :3, :, 5]).all() and torch.isfinite(out[0, 3:]).all()
    put(195, 1, 0.0)
    put(195, 0, float("nan"))                      # a key
    out = c.attend(0, q, start, window=8)
    assert torch.isnan(out[0, :3]).all() and torch.isfinite(out[0, 3:]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_strides_layers_and_scale(dtype):
    """q as a slice of a wider projection, transposed heads, an unaligned base; layer 2 of 3; a scale of its own."""
    past, lens, T = [90, 33], [6, 6], 6
    total = [p + n for p, n in zip(past, lens)]
    c, g = make(2, 2, 64, dtype, 32, total, layers=3, seed=1)
    keys, values = fill(c, total, g, layer=2)
    start = torch.tensor(past, device="cuda")
    wide = torch.randn(2, T, 4 * 64 + 2 * 2 * 64, generator=g).to(dtype).cuda()
    heads_first = torch.randn(2, 4, T, 64, generator=g).to(dtype).cuda()
    flat = torch.randn(2 * T * 4 * 64 + 1, generator=g).to(dtype).cuda()
    for q in (wide[..., : 4 * 64].unflatten(-1, (4, 64)), heads_first.transpose(1, 2), flat[1:].view(2, T, 4, 64),
              wide[:, :, 64:128].unsqueeze(2).expand(2, T, 4, 64),
              torch.randn(2, T, 64, 4, generator=g).to(dtype).cuda().transpose(2, 3)):
        check_attend(c, c.attend(2, q, start, scale=0.31), q, keys, values, past, lens, scale=0.31)


def test_attend_large_scores_and_equal_scores():
    """Scores around +-1000 (one key takes everything) and all equal (a plain mean)."""
    c, g = make(1, 1, 64, torch.bfloat16, 64, [400], seed=4)
    keys, values = fill(c, [400], g)
    start = torch.tensor([399], device="cuda")
    q = (keys[0][0, 37] * 32).view(1, 1, 1, 64).cuda()
    out = c.attend(0, q, start, scale=0.5)
    assert torch.equal(out[0, 0, 0].cpu(), values[0][0, 37])
    out = c.attend(0, torch.zeros(1, 1, 1, 64, dtype=torch.bfloat16, device="cuda"), start)
    ref = values[0][0].double().mean(0)
    assert (out[0, 0, 0].double().cpu() - ref).abs().max() <= 2.0 ** -9 * ref.abs().max() + 2.0 ** -16


WRITE_CASES = [
    # heads, kv, dim, page, tokens, start, lens, rotary, interleaved
    (32, 8, 128, 64, 16, [500, 63], [16, 9], 128, False),
    (4, 2, 64, 16, 1, [0, 15, 16], [1, 1, 0], 64, False),
    (3, 1, 80, 32, 33, [7], [33], 20, False),
    (3, 1, 96, 32, 5, [1000000], [5], 24, True),
    (2, 2, 256, 128, 3, [130], [3], 64, False),
    (2, 1, 8, 16, 40, [3, 0], [40, 13], 8, True),
    (2, 1, 40, 16, 4, [9], [4], 0, False),
    (6, 3, 128, 64, 700, [65, 0, 100, 3], [700, 650, 1, 0], 64, True),
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("norm", [True, False])
@pytest.mark.parametrize("case", WRITE_CASES)
def test_write(case, norm, dtype):
    from domino_b200 import PagedKVCache, Rope

    heads, kv, dim, page, T, start, lens, rotary, interleaved = case
    B = len(start)
    g = torch.Generator().manual_seed(T)
    first = [s // page for s in start]
    count = [-(-(s + n) // page) - f for s, n, f in zip(start, lens, first)]
    count = [max(x, 0) for x in count]
    c = PagedKVCache(2, B, kv, sum(count) + 2, dim, dtype, "cuda", page_size=page, row_pages=max(start) // page + T)
    order = torch.randperm(c.pages, generator=g).int().cuda()
    at = 0
    for b in range(B):
        c.table[b, first[b]: first[b] + count[b]] = order[at: at + count[b]]
        at += count[b]
    c.refs[order[:at].long()] = 1
    c.data.fill_(7)
    fused = torch.randn(B, T, (heads + 2 * kv) * dim, generator=g).to(dtype).cuda()
    q, k, v = (x.unflatten(-1, (-1, dim)) for x in fused.split([heads * dim, kv * dim, kv * dim], dim=-1))
    qn = (1 + torch.randn(dim, generator=g) * 0.2).to(dtype).cuda() if norm else None
    kn = (1 + torch.randn(dim, generator=g) * 0.2).to(dtype).cuda() if norm else None
    rope = Rope(dim, theta=1e4, rotary_dim=rotary, interleaved=interleaved, factor=1.3, device="cuda")
    st, n = torch.tensor(start, device="cuda"), torch.tensor(lens, device="cuda")
    out = c.write(1, q, k, v, rope, st, n, q_norm=qn, k_norm=kn, eps=1e-5)
    assert c.status() == 0
    want = torch.full(c.data.shape, 7.0, dtype=torch.float64)
    eps = torch.finfo(dtype).eps / 2
    table = c.table.cpu().long()
    for b in range(B):
        m = lens[b]
        pos = torch.arange(start[b], start[b] + m)
        ref = []
        for x, w in ((q, qn), (k, kn)):
            x = R.norm_rows(x[b, :m].double().cpu(), None if w is None else w.cpu(), 1e-5)
            ref.append((R.rope_rows(x, pos, rope.inv_freq.cpu(), 1.3, interleaved), x))
        y, x = ref[0]
        assert ((out[b, :m].double().cpu() - y).abs() <= eps * y.abs() + 2.0 ** -20 * 1.3 * x.abs().amax(-1, keepdim=True)
                + 1e-7).all() if m else True
        assert (out[b, m:] == 0).all()
        at, off = table[b][pos // page], pos % page
        got = c.data[1, 0].double().cpu()[at, :, off]
        y, x = ref[1]
        if m:
            assert ((got - y).abs() <= eps * y.abs() + 2.0 ** -20 * 1.3 * x.abs().amax(-1, keepdim=True) + 1e-7).all()
        assert torch.equal(c.data[1, 1].cpu()[at, :, off], v[b, :m].cpu())
        want[1, 0][at, :, off] = got
        want[1, 1][at, :, off] = v[b, :m].double().cpu()
    assert torch.equal(c.data.double().cpu(), want)  # nothing else was written
    # keys and values alone, without a turn
    c.data.fill_(7)
    assert c.write(0, None, k, v, None, st, n) is None
    for b in range(B):
        pos = torch.arange(start[b], start[b] + lens[b])
        assert torch.equal(c.data[0, 0].cpu()[table[b][pos // page], :, pos % page], k[b, : lens[b]].cpu())


def test_write_strides_and_unaligned():
    from domino_b200 import PagedKVCache, Rope

    g = torch.Generator().manual_seed(0)
    c = PagedKVCache(1, 2, 2, 4, 64, torch.bfloat16, "cuda", page_size=16, row_pages=2)
    c.table.copy_(torch.tensor([[0, 2], [3, 1]], dtype=torch.int32))
    c.refs.fill_(1)
    rope = Rope(64, device="cuda")
    start = torch.tensor([3, 12], device="cuda")
    k = torch.randn(2, 2, 5, 64, generator=g).to(torch.bfloat16).cuda()     # heads before tokens
    v = torch.randn(2 * 5 * 2 * 64 + 3, generator=g).to(torch.bfloat16).cuda()[3:].view(2, 5, 2, 64)
    q = torch.randn(2, 5, 4, 64, generator=g).to(torch.bfloat16).cuda()
    a = c.write(0, q, k.transpose(1, 2), v, rope, start)
    first = c.data.clone()
    c.data.zero_()
    b = c.write(0, q.clone(), k.transpose(1, 2).contiguous(), v.clone(), rope, start)
    assert torch.equal(a, b) and torch.equal(first, c.data)


def test_write_refuses_pages_it_does_not_own():
    """A position behind the table, a missing page and a shared page: nothing is written there, a status bit says so."""
    from domino_b200 import PagedKVCache, _lib

    c = PagedKVCache(1, 2, 1, 3, 8, torch.float32, "cuda", page_size=16, row_pages=2)
    c.table.copy_(torch.tensor([[0, 2], [-1, 9]], dtype=torch.int32))
    c.refs.copy_(torch.tensor([2, 0, 1], dtype=torch.int32))
    x = torch.ones(2, 4, 1, 8, device="cuda")

    def go(a, b):
        c.write(0, None, x, x, None, torch.tensor([a, b], device="cuda"), torch.tensor([4, 0 if b < 0 else 4], device="cuda"))
        return c.status()

    assert go(0, -1) == _lib.DD_STATUS_SHARED_PAGE
    assert go(20, 0) == _lib.DD_STATUS_NO_PAGE
    assert (c.data[0, 0, 2, 0, 4:8] == 1).all() and c.data.sum() == 2 * 4 * 8
    assert go(30, 20) == _lib.DD_STATUS_NO_PAGE   # tokens 2 and 3 lie behind the table; row 1's page number is invalid
    assert c.data.sum() == 2 * 6 * 8
    assert go(-2, -1) == _lib.DD_STATUS_NO_PAGE | _lib.DD_STATUS_SHARED_PAGE  # positions -2, -1, then page 0


def _same(c, h, ids):
    assert c.table.tolist() == h.table
    assert c.length.tolist() == h.length
    assert c.refs.tolist() == h.refs
    held = [p for p in range(h.pages) if h.refs[p] > 0]
    got = c.data[:, :, :, 0, 0, 0].cpu()
    for p in held:
        assert (got[:, :, p] == h.content[p]).all(), p
    assert (c.data == c.data[:, :, :, :1, :1, :1]).all()


def _stamp(c, h, rows):
    """Give every page that only one row holds a number of its own (as a write into it would)."""
    for b in rows:
        for p in h.table[b]:
            if p >= 0 and h.refs[p] == 1:
                h.counter = getattr(h, "counter", 0) + 1
                h.content[p] = h.counter
                c.data[:, :, p] = h.counter


@pytest.mark.parametrize("seed,batch,pages,page,row_pages", [(0, 4, 40, 16, 6), (1, 33, 300, 32, 9), (2, 1, 3, 128, 5),
                                                             (3, 7, 20, 64, 8), (4, 1000, 5000, 16, 4)])
def test_pages_random_sequences_match_the_host_model(seed, batch, pages, page, row_pages):
    """Random reserve / advance / crop / fork / compact: tables, counts, lengths and page contents after every call,
    with pools that run out of pages on the way."""
    import random

    from domino_b200 import PagedKVCache, _lib

    rng = random.Random(seed)
    c = PagedKVCache(2, batch, 2, pages, 8, torch.float32, "cuda", page_size=page, row_pages=row_pages)
    h = R.HostPages(batch, pages, page, row_pages)
    c.data.copy_(torch.arange(-pages, 0).view(1, 1, pages, 1, 1, 1).expand_as(c.data))
    for step in range(25 if batch < 500 else 6):
        op = rng.choice(["grow", "grow", "grow", "crop", "fork", "compact"])
        if op == "grow":
            upto = [max(0, n + rng.choice([0, 1, 1, page - 1, page, 2 * page + 1, -5])) for n in h.length]
            c.reserve(torch.tensor(upto, device="cuda"))
            ok = h.reserve(upto)
            s = c.status()
            assert s == (0 if ok else _lib.DD_STATUS_NO_PAGE)
            _same(c, h, step)
            for b in range(batch):  # advance over positions that have pages of their own
                n = h.length[b]
                while n < upto[b] and n < row_pages * page and h.table[b][n // page] >= 0 and h.refs[h.table[b][n // page]] == 1:
                    n += 1
                h.length[b] = n
            c.length.copy_(torch.tensor(h.length))
            _stamp(c, h, range(min(batch, 40)))
        elif op == "crop":
            to = [max(-1, n - rng.choice([0, 0, 1, page, 3 * page, -9])) for n in h.length]
            c.crop(torch.tensor(to, device="cuda"))
            h.crop(to)
        elif op == "fork":
            src = [rng.choice([b, b, -1, rng.randrange(batch), 0]) for b in range(batch)]
            c.fork(torch.tensor(src, device="cuda"))
            h.fork(src)
        else:
            c.compact()
            h.compact()
        assert c.status() == 0 or op == "grow"
        _same(c, h, step)


def test_fork_flags_rows_that_do_not_exist():
    from domino_b200 import PagedKVCache, _lib

    c = PagedKVCache(1, 3, 1, 4, 8, torch.float32, "cuda", page_size=16)
    c.reserve(torch.tensor([10, 20, 0], device="cuda"))
    c.length.copy_(torch.tensor([10, 20, 0]))
    before = c.table.clone()
    c.fork(torch.tensor([3, -2, 2 ** 40], device="cuda"))
    assert c.status() == _lib.DD_STATUS_BAD_ROW
    assert torch.equal(c.table, before) and c.length.tolist() == [10, 20, 0]


@pytest.mark.parametrize("dtype", DTYPES)
def test_operators_together_as_a_server_uses_them(dtype):
    """A prompt, three rows that continue it, blocks of new tokens with rejections, a row given back, compaction: after
    every step the attention equals the definition over each row's own history."""
    from domino_b200 import PagedKVCache, Rope

    heads, kv, D, page, B = 4, 2, 64, 16, 4
    g = torch.Generator().manual_seed(3)
    c = PagedKVCache(2, B, kv, 40, D, dtype, "cuda", page_size=page, row_pages=10)
    rope = Rope(D, theta=1e4, device="cuda")
    hist = [(torch.zeros(0, kv, D), torch.zeros(0, kv, D)) for _ in range(B)]

    def step(T, lens):
        start = c.length.clone()
        n = torch.tensor(lens, device="cuda")
        c.reserve(start + n)
        q, k, v = (torch.randn(B, T, x, D, generator=g).to(dtype).cuda() for x in (heads, kv, kv))
        out = None
        for layer in range(2):
            qr = c.write(layer, q, k, v, rope, start, n)
            out = c.attend(layer, qr, start, n)
        c.length.add_(n)
        st = start.tolist()
        for b in range(B):
            pos = torch.arange(st[b], st[b] + lens[b])
            kr = R.rope_rows(k[b, : lens[b]].double().cpu(), pos, rope.inv_freq.cpu(), 1.0, False).to(dtype).double()
            hist[b] = (torch.cat([hist[b][0].double(), kr]), torch.cat([hist[b][1].double(), v[b, : lens[b]].double().cpu()]))
        keys = [x[0].transpose(0, 1) for x in hist]
        values = [x[1].transpose(0, 1) for x in hist]
        ref = R.attend(qr.cpu(), keys, values, [torch.ones(k.shape[1], dtype=torch.bool) for k in keys], st, lens, True, 0,
                       0, D ** -0.5)
        eps = torch.finfo(dtype).eps / 2
        # the reference's keys may round the other way: one more rounding of a key, which moves a score by eps |q||k| scale
        slack = 2 * eps * 14 * 14 / 8
        assert (out.double().cpu() - ref).abs().max() <= (2 * eps + slack + 2.0 ** -15) * 5
        assert c.status() == 0

    step(37, [37, 0, 0, 0])
    c.fork(torch.tensor([0, 0, 0, -1], device="cuda"))
    hist[1] = hist[2] = hist[0]
    for block, keep in ((8, [3, 8, 1, 0]), (8, [8, 2, 5, 8]), (1, [1, 1, 1, 1])):
        before = c.length.tolist()
        lens = [block, block, block, block if before[3] or keep[3] else 0]
        step(block, lens)
        to = [p + min(x, n) for p, x, n in zip(before, keep, lens)]
        c.crop(torch.tensor(to, device="cuda"))
        hist[:] = [(a[:n], b[:n]) for (a, b), n in zip(hist, to)]
    c.fork(torch.tensor([0, -1, 2, 2], device="cuda"))
    hist[1] = (hist[1][0][:0], hist[1][1][:0])
    hist[3] = hist[2]
    c.compact()
    used = int((c.refs > 0).sum())
    assert (c.refs[used:] == 0).all()
    step(5, [5, 3, 0, 5])


def test_captured_calls_replay_on_new_lengths():
    """One captured step (reserve, write, attend, crop) replayed while lengths move, against the same eager calls."""
    from domino_b200 import PagedKVCache, Rope

    B, T, H, KV, D = 2, 4, 4, 2, 64
    g = torch.Generator().manual_seed(8)
    rope = Rope(D, device="cuda")
    caches = [PagedKVCache(1, B, KV, 30, D, torch.bfloat16, "cuda", page_size=16, row_pages=12) for _ in range(2)]
    q, k, v = (torch.zeros(B, T, x, D, dtype=torch.bfloat16, device="cuda") for x in (H, KV, KV))
    keep = torch.zeros(B, dtype=torch.long, device="cuda")

    def step(c):
        start = c.length.clone()
        c.reserve(start + T)
        out = c.attend(0, c.write(0, q, k, v, rope, start), start)
        c.length.add_(T)
        c.crop(start + keep)
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(caches[0])
        caches[0].crop(torch.zeros_like(keep))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(caches[0])
    for i in range(12):
        for x in (q, k, v):
            x.copy_(torch.randn(x.shape, generator=g))
        keep.copy_(torch.tensor([1 + i % T, T]))
        graph.replay()
        eager = step(caches[1])
        assert torch.equal(captured, eager), i
        assert torch.equal(caches[0].table, caches[1].table) and torch.equal(caches[0].length, caches[1].length)
    assert caches[0].status() == 0 and caches[1].status() == 0


@pytest.mark.parametrize("case", [
    (200, 1, 64, 32, 2, [70, 5], [2, 1]),                # more query heads per key head than a tile has rows
    (256, 2, 128, 16, 1, [300], [1]),
    (6, 2, 72, 128, 20, [250, 0], [20, 20]),             # pages of a whole key tile; 72 and 104 values
    (22, 2, 104, 128, 40, [129], [40]),
])
@pytest.mark.parametrize("dtype", DTYPES)
def test_attend_odd_head_layouts(case, dtype):
    heads, kv, dim, page, T, past, lens = case
    total = [p + n for p, n in zip(past, lens)]
    c, g = make(len(past), kv, dim, dtype, page, total, seed=heads)
    keys, values = fill(c, total, g)
    q = torch.randn(len(past), T, heads, dim, generator=g).to(dtype).cuda()
    start, n = torch.tensor(past, device="cuda"), torch.tensor(lens, device="cuda")
    for causal in (True, False):
        check_attend(c, c.attend(0, q, start, n, causal=causal), q, keys, values, past, lens, causal)
    assert c.status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("batch,tokens,alive", [(450, 1, 450), (450, 2, 5), (40, 1, 2), (40, 70, 3), (33, 1, 33)])
def test_attend_many_rows_some_empty(batch, tokens, alive, dtype):
    """Batches of more rows than a warp or a block has lanes, with rows that have no tokens this time."""
    g = torch.Generator().manual_seed(batch + tokens)
    past = [int(x) for x in torch.randint(0, 300, (batch,), generator=g)]
    lens = [0] * batch
    for i, b in enumerate(torch.randperm(batch, generator=g)[:alive].tolist()):
        lens[b] = 1 + i % tokens
    total = [p + n for p, n in zip(past, lens)]
    c, g = make(batch, 1, 64, dtype, 32, total, seed=batch)
    keys, values = fill(c, total, g)
    q = torch.randn(batch, tokens, 4, 64, generator=g).to(dtype).cuda()
    out = c.attend(0, q, torch.tensor(past, device="cuda"), torch.tensor(lens, device="cuda"))
    check_attend(c, out, q, keys, values, past, lens)
    again = c.attend(0, q, torch.tensor(past, device="cuda"), torch.tensor(lens, device="cuda"))
    assert torch.equal(out, again)  # the joins add in the order of the CTAs, whoever finishes last


def test_rows_that_see_nothing():
    """Positions before the row's first key, and chunks behind the table's end, give zeros or what the table holds."""
    c, g = make(3, 1, 64, torch.bfloat16, 16, [40, 40, 40], seed=3)
    keys, values = fill(c, [40, 40, 40], g)
    q = torch.randn(3, 4, 2, 64, generator=g).to(torch.bfloat16).cuda()
    start = torch.tensor([-10, -2, 2 ** 40], device="cuda")
    out = c.attend(0, q, start)
    assert (out[0] == 0).all()                       # no key at all
    assert (out[1, :2] == 0).all() and (out[1, 2:] != 0).any()
    see = torch.arange(c.capacity) < 40              # the table's last page is missing
    k = torch.cat([keys[2], torch.zeros(1, c.capacity - 40, 64, dtype=torch.bfloat16)], 1)
    v = torch.cat([values[2], torch.zeros(1, c.capacity - 40, 64, dtype=torch.bfloat16)], 1)
    held = (c.table[2].cpu() >= 0).repeat_interleave(16)
    c.data[0, :, :, :, 8:][:, c.table[2, 2].item()] = 0  # entries 40 .. 47 of row 2's last page
    out = c.attend(0, q, start)
    ref = R.attend(q.cpu()[2:], [k], [v], [held], [c.capacity - 4], [4], False, 0, 0, 0.125)
    assert see.any() and (out[2].double().cpu() - ref[0]).abs().max() <= 2.0 ** -7 * v.abs().max()


def test_pool_past_32_bit_offsets():
    """Pages behind 2^31 elements of one plane, written, attended, copied on write and moved."""
    from domino_b200 import PagedKVCache, Rope

    pages, page, kv, D = 40000, 64, 8, 128           # 2.6e9 elements a plane
    c = PagedKVCache(1, 2, kv, pages, D, torch.bfloat16, "cuda", page_size=page, row_pages=4)
    c.refs.fill_(1)
    c.refs[-6:] = 0                                  # only the last pages are free
    g = torch.Generator().manual_seed(0)
    rope = Rope(D, device="cuda")
    q, k, v = (torch.randn(2, 100, h, D, generator=g).to(torch.bfloat16).cuda() for h in (8, kv, kv))
    start = torch.zeros(2, dtype=torch.long, device="cuda")
    n = torch.tensor([100, 0], device="cuda")
    c.reserve(start + n)
    assert c.table[0, :2].tolist() == [pages - 6, pages - 5]
    qr = c.write(0, q, k, v, rope, start, n)
    small = PagedKVCache(1, 2, kv, 4, D, torch.bfloat16, "cuda", page_size=page, row_pages=4)
    small.reserve(start + n)
    assert torch.equal(small.write(0, q, k, v, rope, start, n), qr)
    out = c.attend(0, qr, start, n)
    assert torch.equal(out, small.attend(0, qr, start, n))
    for x in (c, small):
        x.length.copy_(n)
        x.fork(torch.zeros(2, dtype=torch.long, device="cuda"))
        x.reserve(x.length + 20)                     # row 1 gets a copy of the shared last page
    assert torch.equal(c.attend(0, qr[:, :1], c.length - 1), small.attend(0, qr[:, :1], small.length - 1))
    assert c.table[1, 1] != c.table[0, 1]
    c.refs[: pages - 6] = 0
    before = c.attend(0, qr[:, :1], c.length - 1)
    c.compact()
    assert int(c.table.max()) < 5 and torch.equal(c.attend(0, qr[:, :1], c.length - 1), before)
    assert c.status() == 0


def test_calls_on_another_stream():
    from domino_b200 import PagedKVCache, Rope

    g = torch.Generator().manual_seed(1)
    rope = Rope(64, device="cuda")
    q, k, v = (torch.randn(2, 30, h, 64, generator=g).to(torch.float16).cuda() for h in (4, 2, 2))
    start = torch.zeros(2, dtype=torch.long, device="cuda")
    results = []
    for stream in (torch.cuda.current_stream(), torch.cuda.Stream()):
        c = PagedKVCache(1, 2, 2, 8, 64, torch.float16, "cuda", page_size=16, row_pages=4)
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            c.reserve(start + 30)
            out = c.attend(0, c.write(0, q, k, v, rope, start), start)
            c.length.add_(30)
            c.crop(start + 17)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        results.append((out, c.table.clone(), c.length.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_first_rows_share_the_pool():
    from domino_b200 import PagedKVCache

    c = PagedKVCache(1, 3, 1, 8, 8, torch.float32, "cuda", page_size=16, row_pages=2)
    one = c.first_rows(1)
    one.reserve(torch.tensor([20], device="cuda"))
    one.length.fill_(20)
    assert c.table.tolist() == [[0, 1], [-1, -1], [-1, -1]] and c.length.tolist() == [20, 0, 0]
    c.fork(torch.zeros(3, dtype=torch.long, device="cuda"))
    assert c.refs.tolist()[:2] == [3, 3]
    one.reserve(torch.tensor([25], device="cuda"))   # the shared second page is replaced for this row alone
    assert c.table.tolist() == [[0, 2], [0, 1], [0, 1]] and c.refs.tolist()[:3] == [3, 2, 1]
    with pytest.raises(ValueError):
        c.first_rows(4)


@pytest.mark.parametrize("tokens,dim,past", [(3, 128, 40), (3, 64, 2000), (16, 128, 1500), (30, 128, 900), (90, 128, 60),
                                             (90, 64, 3000)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_non_finite_value_in_every_kind_of_tile(tokens, dim, past, dtype):
    """A NaN value of the chunk's middle token, in calls with copies of the rows, one tile, pairs of tiles, whole items and
    items split over CTAs: the tokens before it are untouched, the others have the NaN in its place alone."""
    c, g = make(1, 2, dim, dtype, 32, [past + tokens], seed=tokens)
    keys, values = fill(c, [past + tokens], g)
    q = torch.randn(1, tokens, 8, dim, generator=g).to(dtype).cuda()
    start = torch.tensor([past], device="cuda")
    clean = c.attend(0, q, start)
    check_attend(c, clean, q, keys, values, [past], [tokens])
    j = past + tokens // 2
    c.data[0, 1, int(c.table[0, j // 32]), 1, j % 32, 7] = float("nan")  # key head 1: query heads 4 .. 7
    out = c.attend(0, q, start)
    assert torch.equal(out[:, :, :4], clean[:, :, :4])
    bad = torch.zeros_like(out, dtype=torch.bool)
    bad[:, tokens // 2:, 4:, 7] = True
    assert bool(torch.isnan(out[bad]).all()) and bool(torch.isfinite(out[~bad]).all())
    tol = (2 * torch.finfo(dtype).eps / 2 + 2.0 ** -13) * 2 * values[0].abs().max().item()
    assert (out[~bad].float() - clean[~bad].float()).abs().max() <= tol
    assert c.status() == 0
