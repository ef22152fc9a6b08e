"""The paged-cache entry points refuse bad arguments before touching CUDA, and
the 64-bit forms their GPU tests compare with hold on small cases by hand."""
import ctypes as C
import math
import os

import pytest

from xwfes_b200 import formats as F, ftc

P = 4096  # any aligned non-null address: refused calls do not follow it


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(ftc.LIB_PATH):
        from xwfes_b200 import build
        build.build()
    return ftc.lib()


def pages(**kw):
    d = dict(dtype=ftc.KV_Q8, n_pages=8, page_size=16, n_head_kv=2, head_dim=64, k=P, v=P,
             page_stride=2048, k_scale=P, v_scale=P, scale_stride=32)
    d.update(kw)
    return ftc.KvPagesDesc(**d)


def batch(**kw):
    d = dict(n_seqs=2, n_tokens=4, max_new=3, start=P, kv_len=P, page_table=P, table_cols=3,
             table_stride=3)
    d.update(kw)
    return ftc.PageBatchDesc(**d)


BAD_PAGES = [
    (dict(dtype=F.F32), -2, "dtype"), (dict(dtype=F.Q8_0), -2, "dtype"),
    (dict(head_dim=96), -2, "head_dim"), (dict(page_size=8), -2, "page_size"),
    (dict(page_size=48), -2, "page_size"), (dict(page_size=512), -2, "page_size"),
    (dict(n_head_kv=0), -1, "n_head_kv"), (dict(n_head_kv=1025), -1, "n_head_kv"),
    (dict(n_pages=0), -1, "n_pages"), (dict(n_pages=1 << 31), -1, "n_pages"),
    (dict(page_stride=2047), -1, "page_stride"), (dict(page_stride=2056), -1, "page_stride"),
    (dict(dtype=F.F16, page_stride=2052), -1, "page_stride"),
    (dict(k=None), -1, "null"), (dict(v=P + 8), -1, "aligned"), (dict(k_scale=None), -1, "null"),
    (dict(v_scale=P + 4), -1, "aligned"), (dict(scale_stride=31), -1, "scale_stride"),
    (dict(scale_stride=34), -1, "scale_stride"),
]
BAD_BATCH = [
    (dict(n_seqs=-1), -1, "negative"), (dict(n_tokens=-1), -1, "negative"),
    (dict(max_new=-1), -1, "negative"), (dict(n_seqs=2049), -2, "2048"),
    (dict(n_tokens=(1 << 24) + 1), -2, "2^24"), (dict(start=None), -1, "null"),
    (dict(kv_len=None), -1, "null"), (dict(page_table=None), -1, "null"),
    (dict(table_cols=0), -1, "table_cols"), (dict(table_cols=4), -1, "table_cols"),
    (dict(table_cols=1 << 27, table_stride=1 << 27), -1, "table_cols"),
]


def calls(lib, pg, bt, x=P, stride=128, dtype=F.F32):
    ref = lambda d: C.byref(d) if d is not None else None  # noqa: E731
    yield lib.ftc_kv_pages_write(ref(pg), ref(bt), x, x, dtype, stride, None)
    yield lib.ftc_kv_pages_read(ref(pg), ref(bt), x, x, dtype, stride, None)
    yield lib.ftc_attention_pages(ref(pg), ref(bt), x, dtype, stride, 2, 1.0, 0, 0, x, stride,
                                  None, 0, None)


@pytest.mark.parametrize("change,rc,word", BAD_PAGES)
def test_bad_caches_are_refused(lib, change, rc, word):
    for got in calls(lib, pages(**change), batch()):
        assert got == rc and word in ftc.last_error()
    assert lib.ftc_attention_pages_workspace_bytes(C.byref(pages(**change)), C.byref(batch()), 2,
                                                   F.F32) == 0


@pytest.mark.parametrize("change,rc,word", BAD_BATCH)
def test_bad_batches_are_refused(lib, change, rc, word):
    for got in calls(lib, pages(), batch(**change)):
        assert got == rc and word in ftc.last_error()


def test_bad_rows_are_refused(lib):
    for kw, rc in ((dict(x=None), -1), (dict(x=P + 8), -1), (dict(stride=127), -1),
                   (dict(stride=130), -1), (dict(dtype=F.Q8_0), -2),
                   (dict(dtype=F.F16, stride=132), -1)):
        for got in calls(lib, pages(), batch(), **kw):
            assert got == rc, (kw, ftc.last_error())
    for got in calls(lib, None, batch()):
        assert got == -1
    for got in calls(lib, pages(), None):
        assert got == -1


def test_bad_attention_arguments_are_refused(lib):
    def call(n_head=4, scale=1.0, window=0, sink=0, q=F.F32, stride=256, pg=None, out=P):
        return lib.ftc_attention_pages(C.byref(pg or pages()), C.byref(batch()), P, q, stride,
                                       n_head, scale, window, sink, out, stride, None, 0, None)
    assert call(n_head=3) == -1 and "n_head" in ftc.last_error()
    assert call(n_head=0) == -1 and call(n_head=16384, stride=1 << 20) == -1
    for s in (0.0, -1.0, math.inf, math.nan):
        assert call(scale=s) == -1 and "scale" in ftc.last_error()
    assert call(window=-1) == -1 and call(sink=-1) == -1
    assert call(out=None) == -1 and call(stride=252) == -1
    f16 = pages(dtype=F.F16)
    bf16 = pages(dtype=F.BF16)
    assert call(q=F.BF16, pg=f16) == -2 and call(q=F.F16, pg=bf16) == -2
    assert call(q=F.Q8_0) == -2


def test_empty_batches_need_nothing(lib):
    for bt in (batch(n_seqs=0, start=None, kv_len=None, page_table=None, table_cols=0),
               batch(n_tokens=0, table_cols=0)):
        for got in calls(lib, pages(), bt, x=None):
            assert got == 0, ftc.last_error()


def test_injected_failures(lib, monkeypatch):
    for i, name in enumerate(("ftc_kv_pages_write", "ftc_kv_pages_read", "ftc_attention_pages")):
        monkeypatch.setenv("FTC_INJECT_FAIL", name)
        assert list(calls(lib, pages(), batch(n_tokens=0)))[i] == -5
    monkeypatch.delenv("FTC_INJECT_FAIL")


def test_reference_forms_by_hand():
    torch = pytest.importorskip("torch")
    import pages_ref as R
    codes, d = R.quantise(torch.tensor([[127.0, 0.5, 1.5, -2.5], [0.0] * 4,
                                        [1.0, math.nan, 0, 0]]))
    assert codes.tolist() == [[127, 0, 2, -2], [0] * 4, [0] * 4]
    assert d[:2].tolist() == [1.0, 0.0] and torch.isnan(d[2])

    class Pages:
        head_dim, n_head_kv, page_size = 2, 1, 2
        k = torch.tensor([[[[1.0, 0.0], [0.0, 1.0]]], [[[2.0, 0.0], [9.0, 9.0]]]]).half()
        v = torch.tensor([[[[1.0, 2.0], [3.0, 4.0]]], [[[5.0, 6.0], [math.nan, 9.0]]]]).half()
        k_scale = v_scale = None
    q = torch.tensor([[1.0, 0.0], [0.0, 0.0], [1.0, 0.0]])
    table = torch.tensor([[0, 1], [1, 7]], dtype=torch.int32)
    # sequence 0: positions 1 and 2; sequence 1: position 0 of page 1
    out, bound = R.attention(q, 1, Pages, table, [0, 2, 3], [3, 1], scale=1.0)
    a, b = math.e / (math.e + 1), 1 / (math.e + 1)
    assert out[0].tolist() == pytest.approx([a + 3 * b, 2 * a + 4 * b], abs=1e-12)
    assert out[1].tolist() == pytest.approx([3.0, 4.0], abs=1e-12)
    assert out[2].tolist() == [5.0, 6.0] and (bound > 0).all()
    win, _ = R.attention(q, 1, Pages, table, [0, 2, 3], [3, 1], window=1, n_sink=1, scale=1.0)
    assert win[1].tolist() == pytest.approx([3.0, 4.0], abs=1e-12)
    assert win[0].tolist() == pytest.approx([a + 3 * b, 2 * a + 4 * b], abs=1e-12)
    assert R.attention(q, 1, Pages, table, [0, 0, 2], [0, 1], scale=1.0)[0][0].tolist() == [0, 0]
