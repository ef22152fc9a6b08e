"""Paged attention on the GPU where hidden positions hold anything that a float
can be: every row stays within a bound that counts what the row sees alone."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import pages_ref as R  # noqa: E402
import pages_seen as V  # noqa: E402
from test_pages_gpu import (TYPES, agree, fill, ftc, gen, make_batch,  # noqa: E402,F401
                            make_pages)

Q8 = [("f32", "q8"), ("f16", "q8"), ("bf16", "q8")]


def attend(ftc, q, cache, nh, nkv, hd, page, seqs, window=0, sink=0, seed=0, gain=1.5, edit=None,
           spare=0):
    """One call on random keys and values after ``edit(pages, table)``, with its
    rows held to the bound; ``spare``: pages that belong to no sequence."""
    g = gen(seed)
    n_pages = sum(max(0, -(-length // page)) for _, length in seqs) + spare
    pages = make_pages(ftc, cache, max(n_pages, 1), nkv, page, hd, g)
    batch, start, lens, table = make_batch(ftc, seqs, page, max(n_pages, 1), g)
    fill(pages, table, lens, g, gain)
    if edit:
        edit(pages, table)
    x = torch.randn((batch.n_tokens, nh * hd), generator=g, device="cuda").to(TYPES[q])
    got = ftc.attention_pages(x, nh, pages, batch, window=window, n_sink=sink)
    torch.cuda.synchronize()
    assert ftc.device_status() == 0
    want, bound = V.attention(x, nh, pages, table, start, lens, window, sink)
    agree(got, want, bound, list(range(batch.n_tokens)))
    return got, want


# sequences whose packed rows (4 query heads a KV head) are 4, 12, 40 and 360
KINDS = {"decode": [(1, 500), (1, 131)], "verify": [(3, 500), (3, 131)],
         "few": [(10, 500), (10, 131)], "chunk": [(90, 700), (90, 190)]}


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("junk", [1e3, 2.0 ** 20, 2.0 ** 31, 2.0 ** 40, 1e30])
@pytest.mark.parametrize("q,cache", Q8)
def test_scales_before_the_window(ftc, q, cache, junk, kind, page):
    """8-bit codes of 127 with a large finite scale at every position between
    the sinks and the oldest window of a call, the pages there all one page
    that was never written."""
    window, sink, seqs = 100, 5, KINDS[kind]
    spare = []

    def edit(pages, table):
        junk_page = next(p for p in range(pages.k.shape[0])
                         if not (table == p).any())
        spare.append(junk_page)
        for name in ("k", "v"):
            getattr(pages, name)[junk_page] = 127
            getattr(pages, name + "_scale")[junk_page] = junk
        for s, (n, length) in enumerate(seqs):
            first = length - n - window + 1  # the oldest position that a row's window holds
            for j in range(sink, first):
                c = j // page
                if c * page >= sink and (c + 1) * page <= first:
                    table[s, c] = junk_page
                    continue
                for name in ("k", "v"):
                    getattr(pages, name)[int(table[s, c]), :, j % page] = 127
                    getattr(pages, name + "_scale")[int(table[s, c]), :, j % page] = junk
    attend(ftc, q, cache, 8, 2, 64, page, seqs, window=window, sink=sink, edit=edit, seed=71,
           spare=1)
    assert spare


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["verify", "few", "chunk"])
@pytest.mark.parametrize("junk", [2.0 ** 20, 2.0 ** 31, 2.0 ** 40, 1e30])
@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("bf16", "q8")])  # f16 cannot hold the results
def test_scales_of_later_tokens(ftc, q, cache, junk, kind, hd):
    """The values of a call's later tokens grow from one to the next: no row
    loses anything to the tokens after it in its tile."""
    seqs = KINDS[kind]

    def edit(pages, table):
        for s, (n, length) in enumerate(seqs):
            for i in range(n // 3, n):
                j = length - n + i
                gain = junk ** ((i - n // 3 + 1) / (n - n // 3))
                pages.v_scale[int(table[s, j // 16]), :, j % 16] *= gain
    attend(ftc, q, cache, 8, 2, hd, 16, seqs, edit=edit, seed=73 + hd)


@pytest.mark.parametrize("q", ["f32", "bf16"])
def test_two_tokens(ftc, q):
    """The first of two tokens has its own value back, whatever the second's is."""
    def edit(pages, table):
        pages.v_scale[int(table[0, 0]), :, 1] *= 2.0 ** 40
    got, want = attend(ftc, q, "q8", 4, 1, 128, 16, [(2, 2)], edit=edit, seed=79)
    assert (got[0].abs().amax() > 0.1) and math.isfinite(float(want.abs().max()))


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("kind", ["verify", "few", "chunk"])
@pytest.mark.parametrize("junk", [2.0 ** 20, 2.0 ** 31, 2.0 ** 40, 1e30])
@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("bf16", "q8")])
def test_scales_that_leave_the_window(ftc, q, cache, junk, kind, hd):
    """Large values at the oldest positions of a call's windows, so that its
    first rows see them and its last rows do not."""
    window, seqs = 80, KINDS[kind]

    def edit(pages, table):
        for s, (n, length) in enumerate(seqs):
            oldest = length - n - window + 1
            for i in range(n // 2):
                j = oldest + i
                gain = junk ** (1 - i / n)
                pages.v_scale[int(table[s, j // 16]), :, j % 16] *= gain
    attend(ftc, q, cache, 8, 2, hd, 16, seqs, window=window, edit=edit, seed=83 + hd)


@pytest.mark.parametrize("n", [1, 3, 10, 90])
@pytest.mark.parametrize("q,cache", Q8)
def test_visible_value_row_that_is_not_a_number(ftc, q, cache, n):
    """A row of V that was stored as NaN makes the rows that see it NaN, also where
    its weight is too small for fp32; the rows before it stay as they are."""
    length = 30 + n
    pos = length - n // 2 - 1

    g = gen(89)
    pages = make_pages(ftc, cache, 10, 1, 16, 64, g)
    batch, start, lens, table = make_batch(ftc, [(n, length)], 16, 10, g)
    fill(pages, table, lens, g, 1.0)
    p, slot = int(table[0, pos // 16]), pos % 16
    pages.k[p, 0, slot], pages.k_scale[p, 0, slot] = -127, 1.0
    pages.v_scale[p, 0, slot] = math.nan
    x = torch.ones((n, 4 * 64), device="cuda").to(TYPES[q])  # the position's score: -1016
    got = ftc.attention_pages(x, 4, pages, batch)
    want, bound = V.attention(x, 4, pages, table, start, lens)
    agree(got, want, bound, list(range(n)))
    sees = torch.arange(length - n, length, device="cuda") >= pos
    assert torch.isnan(got[sees]).all() and torch.isfinite(got[~sees]).all() and sees.any()


WIDE = [("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("bf16", "bf16")]


@pytest.mark.parametrize("n", [1, 3, 10, 90])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
@pytest.mark.parametrize("q,cache", WIDE)
def test_visible_key_infinity(ftc, q, cache, bad, n):
    """A key element that overflowed its type: a score of -inf has no weight, one of
    +inf makes its row NaN, in chunks that every row sees whole and in others."""
    if (q, cache, n) == ("f32", "bf16", 10):
        n = 20  # 80 packed rows
    length = 300 + n

    def edit(pages, table):
        for pos, d in ((70, 3), (length - n // 2 - 1, 5)):
            pages.k[int(table[0, pos // 16]), 0, pos % 16, d] = bad
    got, want = attend(ftc, q, cache, 4, 1, 64, 16, [(n, length)], edit=edit, seed=97)
    # (every score at position 70 is infinite)
    heads = got.view(n, 4, 64)
    assert torch.equal(torch.isnan(heads).all(-1), torch.isnan(heads).any(-1))
    assert n == 1 or (torch.isnan(heads).any() and torch.isfinite(heads).any())


@pytest.mark.parametrize("n", [1, 3, 10, 90])
@pytest.mark.parametrize("q,cache", WIDE)
def test_scores_of_minus_infinity_alone(ftc, q, cache, n):
    """A row whose visible scores are all -inf has no weights: NaN.  It is no row that
    sees nothing, which gives zeros."""
    if (q, cache, n) == ("f32", "bf16", 10):
        n = 20
    g = gen(101)
    pages = make_pages(ftc, cache, 30, 1, 16, 64, g)
    seqs = [(n, n + 130), (n, n // 2)]
    batch, start, lens, table = make_batch(ftc, seqs, 16, 30, g)
    fill(pages, table, lens, g)
    x = torch.randn((2 * n, 4 * 64), generator=g, device="cuda").to(TYPES[q])
    x.view(2 * n, 4, 64)[:, :, 7] = 1.0
    for j in range(lens[0] - n // 2):
        pages.k[int(table[0, j // 16]), 0, j % 16, 7] = -math.inf
    got = ftc.attention_pages(x, 4, pages, batch)
    want, bound = V.attention(x, 4, pages, table, start, lens)
    agree(got, want, bound, list(range(2 * n)))
    assert torch.isnan(got[:n - n // 2]).all() and torch.isfinite(got[n - n // 2:n]).all()
    assert (got[n:2 * n - n // 2] == 0).all() and torch.isfinite(got[n:]).all()


def device_ms(call):
    """Least of five times of a captured call."""
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    times = []
    for _ in range(5):
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        graph.replay()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b))
    return min(times)


@pytest.mark.parametrize("q,cache", [("bf16", "bf16"), ("f16", "f16")])
def test_one_request_with_nan_leaves_the_others(ftc, q, cache):
    """A NaN among one request's values changes no bit of the others' results, nor
    their time by more than that request's own tile."""
    g = gen(103)
    seqs = [(64, 64)] + [(64, 16384)] * 47
    page = 64
    n_pages = 1 + 47 * 256
    pages = make_pages(ftc, cache, n_pages, 2, page, 128, g)
    for x in (pages.k, pages.v):
        x.normal_(generator=g)
    batch, start, lens, table = make_batch(ftc, seqs, page, n_pages, g)
    x = torch.randn((batch.n_tokens, 8 * 128), generator=g, device="cuda").to(TYPES[q])
    out = torch.empty_like(x)

    def call():
        ftc.attention_pages(x, 8, pages, batch, out=out)
    quick = device_ms(call)
    plain = out.clone()
    pages.v[int(table[0, 0]), :, 30, 5] = math.nan
    slow = device_ms(call)
    assert ftc.device_status() == 0
    assert torch.equal(out[64:], plain[64:]) and torch.equal(out[:30], plain[:30])
    assert torch.isnan(out[30:64].view(34, 8, 128)[:, :, 5]).all()
    # its own tile: 64 positions that 256 threads read one by one
    assert slow < 3 * quick, (slow, quick)


COMBOS = Q8 + WIDE
# sequences whose packed rows (4 query heads a KV head) need tiles of 16 rows, and of 64
ROWS = {"16 rows": [(4, 300), (3, 70), (3, 3)], "64 rows": [(10, 300), (16, 70), (5, 5)],
        "64 rows beside decode": [(1, 200), (10, 300), (1, 17), (16, 16)]}


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("window,sink", [(0, 0), (50, 0), (40, 70)])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q,cache", COMBOS)
def test_a_few_tokens(ftc, q, cache, hd, rows, window, sink, page):
    attend(ftc, q, cache, 8, 2, hd, page, ROWS[rows], window, sink, seed=107 + hd)


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q,cache", COMBOS)
def test_a_few_tokens_with_pages_that_are_not_mapped(ftc, q, cache, hd, rows):
    def edit(pages, table):
        table[0, 3] = -1
        table[1, 0] = pages.k.shape[0]
        table[2, :] = -9
    got, want = attend(ftc, q, cache, 8, 2, hd, 16, ROWS[rows], seed=109 + hd, edit=edit)
    n = [n for n, _ in ROWS[rows]]
    assert (got[n[0] + n[1]:n[0] + n[1] + n[2]] == 0).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q,cache", COMBOS)
def test_a_few_tokens_with_values_that_are_not_finite(ftc, q, cache, hd, rows, bad):
    """In K and V before the window and behind a row's position, and in V where
    rows see it."""
    seqs, window = ROWS[rows], 60
    n0, len0 = max(seqs, key=lambda x: x[1] if x[0] > 1 else 0)
    s0 = seqs.index((n0, len0))

    def edit(pages, table):
        last = len0 - 1  # the last row alone sees this one
        hidden = [0, 100, len0 - n0 - window]  # no row does
        for j in hidden + [last, len0 - n0 - 20]:
            p, slot = int(table[s0, j // 16]), j % 16
            names = ("k", "v") if j in hidden else ("v",)
            for name in names:
                if cache == "q8":
                    getattr(pages, name + "_scale")[p, 0, slot] = math.nan
                else:
                    getattr(pages, name)[p, 0, slot, 11] = bad
    got, want = attend(ftc, q, cache, 8, 2, hd, 16, seqs, window=window, seed=113 + hd, edit=edit)
    assert not torch.isfinite(got).all()
    assert torch.isfinite(got.view(len(got), 2, -1)[:, 1]).all()  # the other KV head


@pytest.mark.parametrize("n", [1, 10, 90])
@pytest.mark.parametrize("sink", [0, 3, 40])
@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "q8")])
def test_windows_past_the_table(ftc, q, cache, sink, n):
    """Positions far past the table, up to the last that 31 bits hold: windows over
    nothing, sinks that are there."""
    g = gen(127)
    pages = make_pages(ftc, cache, 12, 2, 16, 64, g)
    batch, start, lens, table = make_batch(ftc, [(n, 64), (n, 64), (n, 64)], 16, 12, g)
    fill(pages, table, lens, g)
    far = [2 ** 31 - 1, 2 ** 31 - 120, 64 + n // 2 + 30]
    batch.kv_len.copy_(torch.tensor(far))
    x = torch.randn((3 * n, 8 * 64), generator=g, device="cuda").to(TYPES[q])
    got = ftc.attention_pages(x, 8, pages, batch, window=30, n_sink=sink)
    assert ftc.device_status() == 0
    # the far rows see the sinks alone: as rows at position 64 + 30 and later do
    near = [64 + 30 + n] * 2 + far[2:]
    want, bound = V.attention(x, 8, pages, table, start, near, 30, sink)
    agree(got, want, bound, list(range(3 * n)))
    assert sink or (got[:2 * n] == 0).all()


@pytest.mark.parametrize("q,cache", COMBOS)
def test_rows_before_the_first_sequence(ftc, q, cache):
    """Rows before start[0] and behind the last sequence are padding; sequences
    without rows lie between others."""
    g = gen(131)
    pages = make_pages(ftc, cache, 20, 2, 16, 64, g)
    batch, start, lens, table = make_batch(ftc, [(0, 5), (4, 40), (0, 9), (6, 6), (0, 0)], 16, 20, g,
                                           tail=9)
    fill(pages, table, lens, g)
    start = [a + 3 for a in start]
    batch.start.copy_(torch.tensor(start))
    T = batch.n_tokens
    inside = torch.arange(T, device="cuda")
    inside = (inside >= 3) & (inside < 13)
    x = torch.randn((T, 8 * 64), generator=g, device="cuda").to(TYPES[q])
    kn, vn = (torch.randn((T, 2 * 64), generator=g, device="cuda") for _ in range(2))
    kn[~inside], vn[~inside] = math.nan, math.nan
    ftc.kv_pages_write(pages, kn, vn, batch)
    out = torch.full_like(x, 7.0)
    ftc.attention_pages(x, 8, pages, batch, out=out)
    want, bound = V.attention(x, 8, pages, table, start, lens)
    agree(out, want, bound, list(range(3, 13)))
    assert (out[~inside] == 7.0).all()
    k, v = (torch.full((T, 128), 7.0, device="cuda") for _ in range(2))
    ftc.kv_pages_read(pages, batch, k, v)
    for got, new in ((k, kn), (v, vn)):
        y = new[inside].view(-1, 2, 64)
        if cache == "q8":
            c, d = R.quantise(y)
            y = c.float() * d[..., None]
        else:
            y = y.to(TYPES[cache]).float()
        assert torch.equal(got[inside], y.view(-1, 128)) and (got[~inside] == 7.0).all()
