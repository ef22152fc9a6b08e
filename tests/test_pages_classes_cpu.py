"""Which tile a call's sequences get, read from the size of the workspace: so that
a test that means to run a kernel runs it."""
import ctypes as C
import os

import pytest

from xwfes_b200 import formats as F, ftc

P = 4096  # any aligned non-null address: sizing a workspace does not follow it
Q = {"f32": F.F32, "f16": F.F16, "bf16": F.BF16}
KV = {"f16": F.F16, "bf16": F.BF16, "q8": ftc.KV_Q8}
COMBOS = [("f32", "q8"), ("f32", "f16"), ("f32", "bf16"), ("f16", "f16"), ("f16", "q8"),
          ("bf16", "bf16"), ("bf16", "q8")]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(ftc.LIB_PATH):
        from xwfes_b200 import build
        build.build()
    return ftc.lib()


def sms():
    try:
        import torch
        if torch.cuda.is_available():
            return torch.cuda.get_device_properties(0).multi_processor_count
    except ImportError:
        pass
    return 148


def workspace(lib, q, cache, hd, nh, nkv, n_seqs, n_tokens, max_new):
    elem = 1 if cache == "q8" else 2
    pages = ftc.KvPagesDesc(KV[cache], 8, 16, nkv, hd, P, P, nkv * 16 * hd * elem,
                            P if elem == 1 else None, P if elem == 1 else None, nkv * 16)
    batch = ftc.PageBatchDesc(n_seqs, n_tokens, max_new, P, P, P, 3, 3)
    n = lib.ftc_attention_pages_workspace_bytes(C.byref(pages), C.byref(batch), nh, Q[q])
    assert n > 0, ftc.last_error()
    return n


def up(n):
    return (n + 255) // 256 * 256


def set_bytes(ctas, rows, hd):
    """Workspace of one set of tiles: its cut tiles, statistics and sums."""
    return up(20 * ctas) + up(16 * ctas * rows) + up(8 * ctas * rows * hd)


def tile_rows(lib, q, cache, hd, nh, nkv, n_seqs, n_tokens, max_new):
    """Packed rows of the call's tiles, one number per set of sequences, ascending."""
    n, g = workspace(lib, q, cache, hd, nh, nkv, n_seqs, n_tokens, max_new), sms()
    sizes = {}
    for occ in (1, 2, 3):
        for rows in (8, 16, 64, 128, 256):
            sizes.setdefault(set_bytes(occ * g, rows, hd), (rows,))
    both = {a + b: tuple(sorted(r + s)) for a, r in sizes.items() for b, s in sizes.items()}
    assert n in sizes or n in both, n
    return sizes.get(n) or both[n]


def expected(q, cache, hd, rows):
    if rows <= 16:
        return 8 if rows <= 8 else 16
    if rows <= 64 and (q, cache, hd) != ("f32", "bf16", 64):
        return 64
    if hd == 256:
        return 64
    return 128 if q == "f32" else 256


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q,cache", COMBOS)
@pytest.mark.parametrize("new", [1, 2, 3, 4, 5, 10, 16, 17, 90])
def test_sequences_of_one_size(lib, q, cache, hd, new):
    assert tile_rows(lib, q, cache, hd, 8, 2, 3, 3 * new, new) == \
        (expected(q, cache, hd, 4 * new),)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("q,cache", COMBOS)
@pytest.mark.parametrize("new", [5, 10, 17, 90])
def test_single_tokens_beside_others(lib, q, cache, hd, new):
    assert tile_rows(lib, q, cache, hd, 8, 2, 2, new + 1, new) == \
        (8, expected(q, cache, hd, 4 * new))


def test_fp32_over_bf16_of_64_has_no_64_row_tile(lib):
    one = [workspace(lib, "f32", "bf16", 64, 8, 2, 1, n, n) for n in (5, 16, 90)]
    assert one[0] == one[1] == one[2]
