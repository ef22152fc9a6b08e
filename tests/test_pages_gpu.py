"""The paged KV cache and its attention on the GPU against their definitions in
64 bits (tests/pages_ref.py): stored codes and scales exactly, read rows to one
rounding, attention within the bound its arithmetic allows."""
import math

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import pages_ref as R  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.int8}
NAN = math.nan


@pytest.fixture(scope="module")
def ftc():
    assert torch.cuda.is_available(), "GPU test needs CUDA"
    from xwfes_b200 import ftc as mod
    mod.lib()
    return mod


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def make_pages(ftc, cache, n_pages, nkv, page, hd, g, pad=0, junk=NAN):
    """A pool whose every slot holds junk (16 bits) or code 85 with a junk
    scale (8 bits); ``pad``: unused elements between pages."""
    elems = nkv * page * hd
    dt = TYPES[cache]

    def pool():
        buf = torch.full((n_pages * (elems + pad),), 85 if cache == "q8" else junk, dtype=dt,
                         device="cuda")
        return buf.as_strided((n_pages, nkv, page, hd), (elems + pad, page * hd, hd, 1))

    k, v = pool(), pool()
    if cache != "q8":
        return ftc.KvPages(k, v)
    sc = [torch.full((n_pages, nkv, page), junk, device="cuda") for _ in range(2)]
    return ftc.KvPages(k, v, *sc)


def make_batch(ftc, seqs, page, n_pages, g, tail=0, cols=0, n_tokens=None, max_new=None):
    """seqs: [(new rows, length)].  Pages are handed out in shuffled order."""
    start, lens = [0], []
    for n, length in seqs:
        start.append(start[-1] + n)
        lens.append(length)
    per = [max(0, -(-length // page)) for length in lens]
    assert sum(per) <= n_pages
    cols = max([cols, 1] + per)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((len(seqs), cols), -1, dtype=torch.int32, device="cuda")
    at = 0
    for s, c in enumerate(per):
        table[s, :c] = order[at:at + c]
        at += c
    i32 = dict(dtype=torch.int32, device="cuda")
    batch = ftc.PageBatch(torch.tensor(start, **i32), torch.tensor(lens, **i32), table,
                          n_tokens=start[-1] + tail if n_tokens is None else n_tokens,
                          max_new=max([n for n, _ in seqs] + [0]) if max_new is None else max_new)
    return batch, start, lens, table


def put(pages, table, s, pos, name, x):
    """Row x [n_kv, hd] at position pos, written from the definition."""
    page = pages.page_size
    p, slot = int(table[s, pos // page]), pos % page
    pool = getattr(pages, name)
    if pool.dtype == torch.int8:
        c, d = R.quantise(x)
        pool[p, :, slot] = c
        getattr(pages, name + "_scale")[p, :, slot] = d
    else:
        pool[p, :, slot] = x.to(pool.dtype)


def fill(pages, table, lens, g, gain=1.0):
    """Random K and V at every position of every sequence."""
    page, n_pages = pages.page_size, pages.k.shape[0]
    for s, length in enumerate(lens):
        ids = [R.page_of(table.cpu(), s, j, page, n_pages) for j in range(0, max(length, 0), page)]
        for c, p in enumerate(ids):
            if p < 0:
                continue
            m = min(page, length - c * page)
            for name in ("k", "v"):
                x = torch.randn((pages.n_head_kv, m, pages.head_dim), generator=g,
                                device="cuda") * (gain if name == "k" else 1.0)
                pool = getattr(pages, name)
                if pool.dtype == torch.int8:
                    cds, d = R.quantise(x)
                    pool[p, :, :m] = cds
                    getattr(pages, name + "_scale")[p, :, :m] = d
                else:
                    pool[p, :, :m] = x.to(pool.dtype)


def same(a, b):
    return torch.equal(torch.nan_to_num(a.double(), nan=12345.0),
                       torch.nan_to_num(b.double(), nan=12345.0))


def agree(got, want, bound, rows):
    """Every element of the rows within its bound; NaN and infinities equal."""
    got, want, bound = got[rows].double(), want[rows], bound[rows]
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    odd = ~fin & ~torch.isnan(want)
    assert torch.equal(got[odd], want[odd])
    over = (got - want).abs()[fin] / bound[fin]
    assert over.numel() == 0 or float(over.max()) <= 1.0, f"{float(over.max())} of the bound"


SEQS = [(1, 1), (3, 40), (0, 17), (17, 17), (5, 130)]


# ------------------------------------------------------------ storing and reading

@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("cache", ["q8", "f16", "bf16"])
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
def test_write_is_the_definition(ftc, x, cache, hd):
    g = gen(hd)
    nkv, page = 3, 16
    pages = make_pages(ftc, cache, 20, nkv, page, hd, g, pad=16)
    batch, start, lens, table = make_batch(ftc, SEQS, page, 20, g, tail=2)
    T = batch.n_tokens
    wide = torch.randn((T, 2 * nkv * hd + 8), generator=g, device="cuda").to(TYPES[x])
    kn, vn = wide[:, :nkv * hd], wide[:, nkv * hd:2 * nkv * hd]
    want = {n: getattr(pages, n).clone() for n in ("k", "v")}
    if cache == "q8":
        want.update({n: getattr(pages, n).clone() for n in ("k_scale", "v_scale")})

    class Copy:
        page_size = page
    for n, t in want.items():
        setattr(Copy, n, t)
    for row, s, pos in R.rows_of(start, lens):
        put(Copy, table, s, pos, "k", kn[row].view(nkv, hd))
        put(Copy, table, s, pos, "v", vn[row].view(nkv, hd))
    ftc.kv_pages_write(pages, kn, vn, batch)
    for n, t in want.items():
        assert same(getattr(pages, n), t), n


def test_write_8bit_rounds_exactly(ftc):
    """Ties, values next to them, tiny and huge rows, zeros, one NaN, one
    infinity: the code is the exactly rounded quotient."""
    nkv, page, hd = 1, 16, 64
    rows = []
    for top in (127.0, 1.0, 3.7e-3, 65504.0, 3e38, 1e-36, 2e-38, 1e-43, 1e-45):
        d = (torch.tensor(top, dtype=torch.float64) / 127).float()
        x = ((torch.arange(64, dtype=torch.float64) * 2 - 63) / 2 * d.double()).float()
        x[0] = top
        for step in (-1, 0, 1):
            y = x.clone()
            if step:
                y[1:] = torch.nextafter(x[1:], torch.full_like(x[1:], step * math.inf))
            rows.append(y)
    rows.append(torch.zeros(64))
    for bad in (NAN, math.inf, -math.inf):
        y = torch.ones(64)
        y[9] = bad
        rows.append(y)
    x = torch.stack(rows).cuda()
    n = len(rows)
    pages = make_pages(ftc, "q8", 8, nkv, page, hd, None)
    batch, start, lens, table = make_batch(ftc, [(n, n)], page, 8, gen(1))
    ftc.kv_pages_write(pages, x, x.flip(0).contiguous(), batch)
    codes, d = R.quantise(x)
    j = torch.arange(n, device="cuda")
    ids = table[0, j // page].long()
    assert torch.equal(pages.k[ids, 0, j % page], codes)
    assert same(pages.k_scale[ids, 0, j % page], d)
    assert torch.equal(pages.v[ids, 0, j % page], codes.flip(0))
    k, v = ftc.kv_pages_read(pages, batch)
    assert same(k, (codes.float() * d[:, None]))
    assert torch.isnan(k[-3:]).all() and (k[-4] == 0).all()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("cache", ["q8", "f16", "bf16"])
@pytest.mark.parametrize("out", ["f32", "f16", "bf16"])
def test_read_is_the_definition(ftc, out, cache, hd):
    g = gen(hd + 1)
    nkv, page = 2, 32
    pages = make_pages(ftc, cache, 16, nkv, page, hd, g, pad=64)
    batch, start, lens, table = make_batch(ftc, SEQS + [(3, 2)], page, 16, g, tail=3)
    fill(pages, table, lens, g)
    table[4, 0] = -1    # positions 0 .. 31 of the last long sequence: not mapped
    table[4, 4] = 16    # 128 .. 129: past the pool
    T = batch.n_tokens
    k0 = torch.full((T, nkv * hd + 8), 7.0, dtype=TYPES[out], device="cuda")[:, :nkv * hd]
    v0 = torch.full((T, nkv * hd + 8), 7.0, dtype=TYPES[out], device="cuda")[:, :nkv * hd]
    k, v = ftc.kv_pages_read(pages, batch, k0, v0)
    assert k is k0 and v is v0
    tab = table.cpu()
    for name, got in (("k", k), ("v", v)):
        want = torch.full((T, nkv * hd), 7.0, dtype=TYPES[out], device="cuda")
        for row, s, pos in R.rows_of(start, lens):
            p = R.page_of(tab, s, pos, page, 16)
            if p < 0:
                want[row] = 0
                continue
            x = getattr(pages, name)[p, :, pos % page].float()
            if cache == "q8":
                x = x * getattr(pages, name + "_scale")[p, :, pos % page][:, None]
            want[row] = x.to(TYPES[out]).view(-1)
        assert same(got, want), name


def test_write_drops_rows_without_a_slot(ftc):
    """Unmapped pages, ids outside the pool, positions past the table and
    before zero: nothing is stored anywhere else."""
    g = gen(5)
    nkv, page, hd = 2, 16, 128
    pages = make_pages(ftc, "f16", 6, nkv, page, hd, g)
    batch, start, lens, table = make_batch(ftc, [(20, 40), (4, 2), (3, 3)], page, 6, g)
    table[0, 1] = 6
    table[0, 2] = -7
    lens[2] = 50
    batch.kv_len[2] = 50  # 47 .. 49: past the table
    before = pages.k.clone()
    x = torch.randn((27, nkv * hd), generator=g, device="cuda")
    ftc.kv_pages_write(pages, x, x, batch)
    for row, s, pos in R.rows_of(start, lens):
        p = R.page_of(table.cpu(), s, pos, page, 6)
        if p >= 0:
            before[p, :, pos % page] = x[row].view(nkv, hd).half()
    assert same(pages.k, before)


# ------------------------------------------------------------ attention

COMBOS = [("f32", "q8"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "q8"),
          ("bf16", "bf16"), ("bf16", "q8")]


def attend(ftc, q, cache, nh, nkv, hd, page, seqs, window=0, sink=0, seed=0, tail=0, gain=1.5,
           edit=None, scale=None, max_new=None):
    g = gen(seed)
    n_pages = sum(max(0, -(-length // page)) for _, length in seqs) + 2
    pages = make_pages(ftc, cache, n_pages, nkv, page, hd, g, pad=16)
    batch, start, lens, table = make_batch(ftc, seqs, page, n_pages, g, tail=tail,
                                           max_new=max_new)
    fill(pages, table, lens, g, gain)
    if edit:
        edit(pages, table)
    T = batch.n_tokens
    wide = torch.randn((T, nh * hd + 16), generator=g, device="cuda").to(TYPES[q])
    qq = wide[:, :nh * hd]
    out = torch.full((T, nh * hd + 8), 7.0, dtype=TYPES[q], device="cuda")[:, :nh * hd]
    got = ftc.attention_pages(qq, nh, pages, batch, window=window, n_sink=sink, out=out,
                              scale=scale)
    assert got is out
    torch.cuda.synchronize()
    assert ftc.device_status() == 0
    want, bound = R.attention(qq, nh, pages, table, start, lens, window, sink, scale)
    rows = [r for r, _, _ in R.rows_of(start, lens)]
    agree(got, want, bound, rows)
    rest = [r for r in range(T) if r not in set(rows)]
    assert (got[rest] == 7.0).all(), "padding rows keep what they held"
    return got, want


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q,cache", COMBOS)
def test_attention_types(ftc, q, cache, hd):
    """Decode and chunk sequences of every type and head size in one batch."""
    attend(ftc, q, cache, 8, 2, hd, 16,
           [(1, 1), (1, 200), (0, 30), (7, 7), (70, 333), (1, 64), (2, 129)], seed=hd, tail=2)


@pytest.mark.parametrize("nh,nkv", [(1, 1), (3, 1), (5, 5), (8, 1), (12, 4), (16, 1), (20, 1),
                                    (7, 1), (64, 2)])
@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("bf16", "bf16"), ("f16", "q8")])
def test_attention_head_layouts(ftc, q, cache, nh, nkv):
    attend(ftc, q, cache, nh, nkv, 128, 32, [(1, 150), (1, 31), (9, 64), (33, 100)], seed=nh)


@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("q,cache", [("f32", "f16"), ("bf16", "bf16"), ("bf16", "q8")])
def test_attention_page_sizes(ftc, q, cache, page):
    """Lengths on, before and behind page and tile edges."""
    attend(ftc, q, cache, 8, 2, 128, page,
           [(1, n) for n in (15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 256, 257, 513)] +
           [(40, 300), (128, 128), (130, 641)], seed=page)


@pytest.mark.parametrize("window,sink", [(1, 0), (1, 1), (7, 3), (64, 0), (64, 64), (100, 130),
                                         (129, 4), (4096, 4), (33, 1000)])
@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("f16", "f16"), ("bf16", "q8")])
def test_attention_window_and_sinks(ftc, q, cache, window, sink):
    attend(ftc, q, cache, 8, 2, 64, 16,
           [(1, 500), (1, 40), (3, 3), (90, 700), (140, 140), (1, 129)], window=window, sink=sink,
           seed=window + sink)


@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("f32", "bf16"), ("bf16", "q8"),
                                     ("f16", "f16")])
def test_attention_long_contexts(ftc, q, cache):
    """Contexts long enough to be split, beside short ones."""
    attend(ftc, q, cache, 8, 2, 128, 64, [(1, 9001), (1, 5), (2, 6000), (40, 5000), (1, 4096)],
           seed=9)


@pytest.mark.parametrize("q,cache", [("bf16", "bf16"), ("f16", "q8"), ("f32", "f16")])
def test_attention_long_chunk(ftc, q, cache):
    attend(ftc, q, cache, 4, 1, 128, 64, [(700, 1500), (1, 800), (257, 257)], seed=10)


@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("bf16", "bf16")])
@pytest.mark.parametrize("window", [2**31 - 1, 2**31, 2**40])
def test_attention_widest_windows(ftc, q, cache, window):
    """A window of all 31 bits, with rows before position 0 in the tile."""
    attend(ftc, q, cache, 8, 2, 64, 16, [(40, 25), (3, 70), (1, 9)], window=window, sink=2**33,
           seed=15)


@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("q,cache", [("bf16", "bf16"), ("f16", "q8"), ("f16", "f16")])
def test_attention_many_short_tiles(ftc, q, cache, hd):
    """More tiles of a few chunks than the device has SMs: many short
    sequences, and one prompt under a window."""
    attend(ftc, q, cache, 32, 2, hd, 64,
           [(16 - s % 3, 16 + (s * 389) % 1380) for s in range(80)], seed=hd)
    attend(ftc, q, cache, 64, 4, hd, 16, [(641, 700)], window=200, sink=5, seed=hd + 1)


@pytest.mark.parametrize("max_new", [0, 1])
@pytest.mark.parametrize("q,cache", [("bf16", "q8"), ("f32", "f16")])
def test_attention_does_not_lean_on_max_new(ftc, q, cache, max_new):
    """The hint picks kernels; a wrong or missing one costs only time."""
    attend(ftc, q, cache, 8, 2, 128, 16, [(1, 77), (90, 200), (17, 17)], seed=4, max_new=max_new)


@pytest.mark.parametrize("q,cache", COMBOS)
def test_attention_peaked_scores(ftc, q, cache):
    """Scores of hundreds: all weight on a few positions; later maxima far
    above earlier ones."""
    attend(ftc, q, cache, 4, 2, 128, 16, [(1, 700), (50, 300), (1, 3)], gain=40.0, seed=12)


def test_attention_scale(ftc):
    attend(ftc, "f32", "f16", 4, 2, 64, 16, [(1, 90), (30, 60)], scale=0.7, seed=13)


@pytest.mark.parametrize("q,cache", COMBOS)
@pytest.mark.parametrize("bad", [NAN, math.inf])
def test_attention_hidden_positions_do_not_leak(ftc, q, cache, bad):
    """NaN and infinities behind a row's position, before its window, in
    unused slots and in pages of other sequences reach no row that does not
    see them; a row that sees one in V has it, and only it, in its output."""
    seqs = [(60, 200), (1, 90), (20, 20)]

    def edit(pages, table):
        for s, pos in ((0, 170), (0, 3), (2, 10)):
            p, slot = int(table[s, pos // 16]), pos % 16
            for name in ("k", "v"):
                if pages.k.dtype == torch.int8:
                    getattr(pages, name + "_scale")[p, 0, slot] = NAN
                else:
                    getattr(pages, name)[p, 0, slot, 5] = bad if name == "v" else NAN
    got, want = attend(ftc, q, cache, 4, 2, 128, 16, seqs, window=100, edit=edit, seed=3)
    # rows of positions 140 .. 169 see neither 3 nor 170
    assert torch.isfinite(got[:30]).all() and torch.isnan(got[30]).any()
    assert torch.isfinite(got[60]).all()


@pytest.mark.parametrize("q,cache", [("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
@pytest.mark.parametrize("bad", [NAN, math.inf, -math.inf])
def test_attention_visible_value_infinity(ftc, q, cache, bad):
    """One V element that is not finite: its dimension alone, in the rows that
    see it, in a whole tile and on a causal edge."""
    def edit(pages, table):
        for s, pos, d in ((0, 20, 7), (0, 190, 9), (1, 60, 3)):
            pages.v[int(table[s, pos // 16]), 0, pos % 16, d] = bad
    got, want = attend(ftc, q, cache, 2, 1, 64, 16, [(60, 200), (1, 90)], edit=edit, seed=6)
    view = got.view(-1, 2, 64)
    assert not torch.isfinite(view[:60, :, 7]).any() and torch.isfinite(view[:, :, 8]).all()
    assert torch.isfinite(view[:50, :, 9]).all() and not torch.isfinite(view[50:60, :, 9]).any()


@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("bf16", "bf16"), ("f16", "q8")])
def test_attention_unmapped_pages(ftc, q, cache):
    """Pages that are not mapped are not seen; a row that sees no position
    gives zeros; more rows than positions give rows before position 0."""
    def edit(pages, table):
        table[0, 1] = -1
        table[0, 4] = 1 << 30
        table[1, :] = -1
        table[2, 0] = -5
    seqs = [(70, 150), (3, 40), (1, 16), (40, 25), (5, 0)]
    got, want = attend(ftc, q, cache, 8, 2, 128, 16, seqs, edit=edit, seed=8)
    assert (got[70:73] == 0).all() and (got[73] == 0).all()
    assert (got[74:89] == 0).all() and (got[89:114] != 0).any(1).all() and (got[114:] == 0).all()


def test_attention_past_the_table(ftc):
    """kv_len past the table's columns: those positions are not seen."""
    g = gen(2)
    pages = make_pages(ftc, "f16", 8, 1, 16, 64, g)
    batch, start, lens, table = make_batch(ftc, [(1, 64), (30, 64)], 16, 8, g)
    fill(pages, table, lens, g)
    lens = [90, 75]
    batch.kv_len.copy_(torch.tensor(lens))
    q = torch.randn((31, 128), generator=g, device="cuda")
    got = ftc.attention_pages(q, 2, pages, batch)
    want, bound = R.attention(q, 2, pages, table, start, lens)
    agree(got, want, bound, list(range(31)))


def test_offsets_past_32_bits(ftc):
    """Pages 2^31 elements apart and more: every offset is 64 bits wide."""
    g = gen(21)
    nkv, page, hd, n = 1, 16, 64, 4
    stride = (1 << 31) + 64
    bufs = [torch.empty(stride * (n - 1) + page * hd, dtype=torch.int8, device="cuda")
            for _ in range(2)]
    k, v = (b.as_strided((n, nkv, page, hd), (stride, page * hd, hd, 1)) for b in bufs)
    sc = [torch.ones((n, nkv, page), device="cuda") for _ in range(2)]
    pages = ftc.KvPages(k, v, *sc)
    batch, start, lens, table = make_batch(ftc, [(33, 64)], page, n, g)
    x = torch.randn((64, hd), generator=g, device="cuda")
    full = ftc.PageBatch(torch.tensor([0, 64], dtype=torch.int32, device="cuda"), batch.kv_len,
                         table, n_tokens=64)
    ftc.kv_pages_write(pages, x, -x, full)
    back, _ = ftc.kv_pages_read(pages, full)
    codes, d = R.quantise(x)
    assert torch.equal(back, codes.float() * d[:, None])
    for dt in (torch.float32, torch.bfloat16):
        q = torch.randn((33, 2 * hd), generator=g, device="cuda").to(dt)
        got = ftc.attention_pages(q, 2, pages, batch)
        want, bound = R.attention(q, 2, pages, table, start, lens)
        agree(got, want, bound, list(range(33)))


# ------------------------------------------------------------ use

@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("bf16", "bf16")])
def test_a_generation_of_two_sequences(ftc, q, cache):
    """Prompt in chunks, then single tokens: store, attend and read together,
    each step against the definition over what was stored; and a snapshot of
    everything at the end."""
    g = gen(31)
    nh, nkv, hd, page = 8, 2, 64, 16
    n_pages = 20
    pages = make_pages(ftc, cache, n_pages, nkv, page, hd, g)
    order = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = order.view(2, 10).contiguous()
    lens = [0, 0]
    kept = [[], []]
    for new in ([50, 3], [21, 40], [1, 1], [1, 0], [1, 1]):
        start = [0, new[0], new[0] + new[1]]
        lens = [a + b for a, b in zip(lens, new)]
        T = start[-1]
        i32 = dict(dtype=torch.int32, device="cuda")
        batch = ftc.PageBatch(torch.tensor(start, **i32), torch.tensor(lens, **i32), table,
                              n_tokens=T, max_new=max(new))
        qkv = torch.randn((T, (nh + 2 * nkv) * hd), generator=g, device="cuda").to(TYPES[q])
        qq, kn, vn = qkv.split([nh * hd, nkv * hd, nkv * hd], dim=1)
        ftc.kv_pages_write(pages, kn, vn, batch)
        got = ftc.attention_pages(qq, nh, pages, batch)
        want, bound = R.attention(qq, nh, pages, table, start, lens)
        agree(got, want, bound, list(range(T)))
        for s in range(2):
            kept[s].append(kn[start[s]:start[s + 1]])
    i32 = dict(dtype=torch.int32, device="cuda")
    whole = ftc.PageBatch(torch.tensor([0, lens[0], sum(lens)], **i32),
                          torch.tensor(lens, **i32), table, n_tokens=sum(lens))
    k, _ = ftc.kv_pages_read(pages, whole)
    x = torch.cat(kept[0] + kept[1]).float().view(-1, nkv, hd)
    if cache == "q8":
        codes, d = R.quantise(x)
        x = codes.float() * d[..., None]
    assert torch.equal(k, x.view(-1, nkv * hd))


def _graph_setup(ftc, q, cache, seqs, g, n_tokens):
    pages = make_pages(ftc, cache, 64, 2, 16, 128, g)
    batch, start, lens, table = make_batch(ftc, seqs, 16, 64, g, cols=30, n_tokens=n_tokens)
    fill(pages, table, lens, g)
    qq = torch.randn((n_tokens, 8 * 128), generator=g, device="cuda").to(TYPES[q])
    return pages, batch, start, lens, table, qq


@pytest.mark.parametrize("q,cache", [("f32", "q8"), ("bf16", "bf16")])
def test_captured_call_follows_the_batch(ftc, q, cache):
    """One captured call, replayed on other lengths, row counts and pages."""
    g = gen(41)
    pages, batch, start, lens, table, qq = _graph_setup(ftc, q, cache, [(40, 300), (1, 200)], g,
                                                        n_tokens=64)
    out = torch.zeros_like(qq)
    ftc.attention_pages(qq, 8, pages, batch, out=out)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ftc.attention_pages(qq, 8, pages, batch, out=out)
    for st, ln in (([0, 40, 41], [300, 200]), ([0, 1, 64], [17, 150]), ([0, 0, 1], [0, 1]),
                   ([0, 30, 33], [290, 3])):
        batch.start.copy_(torch.tensor(st))
        batch.kv_len.copy_(torch.tensor(ln))
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want, bound = R.attention(qq, 8, pages, table, st, ln)
        agree(out, want, bound, list(range(st[-1])))
        assert (out[st[-1]:] == 7.0).all()
    del graph


def test_two_graphs_and_two_streams(ftc):
    """Calls on two streams at once, eager and captured: each has its own
    workspace and gives the bits it gives alone."""
    g = gen(43)
    sets = [_graph_setup(ftc, "bf16", "q8", [(40, 300), (1, 200)], g, 41),
            _graph_setup(ftc, "f32", "f16", [(1, 400), (3, 90)], g, 4)]
    alone = [ftc.attention_pages(s[5], 8, s[0], s[1]) for s in sets]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for s in sets:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ftc.attention_pages(s[5], 8, s[0], s[1]))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o, a in zip(outs, alone):
            assert torch.equal(o, a)
    eager = [ftc.attention_pages(s[5], 8, s[0], s[1], stream=st) for s, st in zip(sets, streams)]
    raw = ftc.attention_pages(sets[0][5], 8, sets[0][0], sets[0][1],
                              stream=streams[1].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(e, a) for e, a in zip(eager + [raw], alone + alone[:1]))


def test_results_repeat(ftc):
    g = gen(47)
    for q, cache in COMBOS:
        pages, batch, *_, qq = _graph_setup(ftc, q, cache, [(40, 300), (1, 450), (3, 200)], g, 44)
        a = ftc.attention_pages(qq, 8, pages, batch)
        for _ in range(3):
            assert torch.equal(ftc.attention_pages(qq, 8, pages, batch), a)


def test_empty_batches(ftc):
    g = gen(51)
    pages = make_pages(ftc, "q8", 4, 2, 16, 64, g)
    i32 = dict(dtype=torch.int32, device="cuda")
    none = ftc.PageBatch(torch.zeros(1, **i32), torch.zeros(0, **i32),
                         torch.zeros((0, 3), **i32), n_tokens=0)
    x = torch.empty((0, 128), device="cuda")
    ftc.kv_pages_write(pages, x, x, none)
    assert ftc.kv_pages_read(pages, none)[0].shape == (0, 128)
    assert ftc.attention_pages(torch.empty((0, 256), device="cuda"), 4, pages, none).shape == (0, 256)
    idle = ftc.PageBatch(torch.zeros(3, **i32), torch.zeros(2, **i32),
                         torch.zeros((2, 3), **i32), n_tokens=2)
    y = torch.full((2, 256), 7.0, device="cuda")
    assert (ftc.attention_pages(torch.ones_like(y), 4, pages, idle, out=y) == 7.0).all()


def test_many_sequences(ftc):
    """2048 single-token sequences, lengths 0 to 40."""
    g = gen(53)
    seqs = [(1 if i % 7 else 0, i % 41) for i in range(2048)]
    pages = make_pages(ftc, "q8", 4800, 1, 16, 64, g, junk=0.01)
    batch, start, lens, table = make_batch(ftc, seqs, 16, 4800, g)
    for dt in (torch.float32, torch.bfloat16):
        q = torch.randn((batch.n_tokens, 2 * 64), generator=g, device="cuda").to(dt)
        got = ftc.attention_pages(q, 2, pages, batch)
        want, bound = R.attention(q, 2, pages, table, start, lens)
        agree(got, want, bound, list(range(batch.n_tokens)))


# ------------------------------------------------------------ refusals

def test_python_refusals(ftc):
    g = gen(61)
    pages = make_pages(ftc, "f16", 8, 2, 16, 64, g)
    batch, *_ = make_batch(ftc, [(1, 20), (3, 30)], 16, 8, g)
    good = torch.zeros((4, 128), device="cuda")
    q = torch.zeros((4, 256), device="cuda")
    k = torch.zeros((4, 2, 16, 64), dtype=torch.float16, device="cuda")
    for call in (
            lambda: ftc.KvPages(k, k.bfloat16()), lambda: ftc.KvPages(k.float(), k.float()),
            lambda: ftc.KvPages(k.to(torch.int8), k.to(torch.int8)),
            lambda: ftc.KvPages(k, k, k[..., 0].float(), k[..., 0].float()),
            lambda: ftc.KvPages(k.cpu(), k.cpu()),
            lambda: ftc.KvPages(k.transpose(1, 2), k.transpose(1, 2)),
            lambda: ftc.KvPages.empty(4, 2, 16, 64, dtype="Q4_K"),
            lambda: ftc.PageBatch(batch.start.long(), batch.kv_len, batch.page_table, 4),
            lambda: ftc.PageBatch(batch.start[:-1], batch.kv_len, batch.page_table, 4),
            lambda: ftc.PageBatch(batch.start, batch.kv_len, batch.page_table[:, ::2], 4),
            lambda: ftc.kv_pages_write(pages, good[:3], good[:3], batch),
            lambda: ftc.kv_pages_write(pages, good, good.half(), batch),
            lambda: ftc.kv_pages_write(pages, good.double(), good.double(), batch),
            lambda: ftc.kv_pages_write(pages, good.cpu(), good.cpu(), batch),
            lambda: ftc.kv_pages_read(pages, batch, k_out=good),
            lambda: ftc.attention_pages(good, 4, pages, batch),
            lambda: ftc.attention_pages(q, 4, pages, batch, out=q.half())):
        with pytest.raises(ValueError):
            call()
    for call in (
            lambda: ftc.attention_pages(torch.zeros((4, 192), device="cuda"), 3, pages, batch),
            lambda: ftc.attention_pages(q.bfloat16(), 4, pages, batch),
            lambda: ftc.attention_pages(q, 4, pages, batch, window=-1),
            lambda: ftc.attention_pages(q, 4, pages, batch, scale=0.0),
            lambda: ftc.attention_pages(q, 4, pages, batch, scale=NAN),
            lambda: ftc.kv_pages_write(ftc.KvPages(k[:, :, :12].contiguous(),
                                                   k[:, :, :12].contiguous()), good, good, batch)):
        with pytest.raises(ftc.FtcError):
            call()
