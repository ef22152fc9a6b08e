"""Plain 64-bit forms of the paged-cache operators, position by position from
their definitions, and the error bound that attention's arithmetic allows."""
import math

import torch

EPS_HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def rows_of(start, kv_len):
    """[(row, sequence, position)] of a batch (host lists)."""
    out = []
    for s in range(len(kv_len)):
        n = start[s + 1] - start[s]
        out += [(start[s] + i, s, kv_len[s] - n + i) for i in range(n)]
    return out


def page_of(table, s, pos, page_size, n_pages):
    if pos < 0 or pos // page_size >= table.shape[1]:
        return -1
    p = int(table[s, pos // page_size])
    return p if 0 <= p < n_pages else -1


def quantise(x):
    """(codes int8, scale fp32) of rows x [..., head_dim]."""
    x = x.double()
    top = x.abs().amax(-1)
    d = (top / 127).float()
    bad = ~torch.isfinite(x).all(-1)
    q = torch.where((d > 0)[..., None], x / d.double()[..., None], torch.zeros_like(x))
    codes = torch.nan_to_num(q.round().clamp(-127, 127))
    codes[bad] = 0
    d = torch.where(bad, torch.full_like(d, math.nan), d)
    return codes.to(torch.int8), d


def values(pool, scale, ids, slots):
    """Cached rows in 64 bits: [len, n_kv, head_dim]."""
    x = pool[ids, :, slots].double()
    if scale is not None:
        x = x * scale[ids, :, slots].double()[..., None]
    return x


def attention(q, n_head, pages, table, start, kv_len, window=0, n_sink=0, scale=None):
    """(out, bound) in 64 bits on q's device; rows outside the batch are NaN in
    ``out``.  ``bound``: what the kernels' arithmetic may be off by, with
    u = half a step of a type and everything relative to sum_j w_j |v_j|:
      * scores: q is split into 16-bit pieces that keep 2^-22 of a value,
        products are exact, each matrix instruction of 16 terms rounds its
        running sum at most twice (2 * 2^-23 of sum |q_i k_i|); the 8-bit
        scale, the score scale and the exponent's argument add 6 roundings.
        A score off by e moves every weight by at most 2 e;
      * weights: fp32 where q is fp32 (2^-22), else one rounding to the 16-bit
        operand type (f16, or bf16 over a bf16 cache);
      * the weighted sum and the sum of weights: the same two roundings per
        16 positions, plus one for each of up to 64 joined parts;
      * f16 weights (all but over a bf16 cache) lie on a grid that ends in steps
        of 2^-24.  The kernels hold them 2^up times the weight relative to the
        row's largest (14 for fp32 q, at least 6 for 16-bit q), times V's
        scale relative to at most twice the largest one: each is off by at
        most half a step, 2^-25, of 2^-up * 2 max|v| on top of its relative
        error, and the sum of weights is at least 1 in these units, so n
        positions add n * 2^-(24 + up) * max|v|;
      * one rounding of the result to q's type."""
    hd, nkv, page = pages.head_dim, pages.n_head_kv, pages.page_size
    n_pages = pages.k.shape[0]
    g = n_head // nkv
    scale = hd ** -0.5 if scale is None else scale
    T = q.shape[0]
    out = torch.full((T, n_head, hd), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    pieces = 3 if q.dtype == torch.float32 else 1
    u_p = 2.0 ** -22 if q.dtype == torch.float32 else \
        EPS_HALF[torch.bfloat16 if pages.k.dtype == torch.bfloat16 else torch.float16]
    floor = 0.0 if pages.k.dtype == torch.bfloat16 else \
        2.0 ** -(24 + (14 if q.dtype == torch.float32 else 6))
    tab = table.cpu()
    for s in range(len(kv_len)):
        n = start[s + 1] - start[s]
        if n == 0:
            continue
        ok = [(j, page_of(tab, s, j, page, n_pages)) for j in range(max(kv_len[s], 0))]
        ok = [(j, p) for j, p in ok if p >= 0]
        j = torch.tensor([a for a, _ in ok], dtype=torch.int64, device=q.device)
        ids = torch.tensor([b for _, b in ok], dtype=torch.int64, device=q.device)
        k = values(pages.k, pages.k_scale, ids, j % page)
        v = values(pages.v, pages.v_scale, ids, j % page)
        pos = torch.arange(kv_len[s] - n, kv_len[s], device=q.device)[:, None]
        see = j[None] <= pos
        if window:
            see &= (pos - j[None] < window) | (j[None] < n_sink)
        for h in range(n_head):
            qh = q[start[s]:start[s + 1], h * hd:(h + 1) * hd].double()
            kh, vh = k[:, h // g], v[:, h // g]
            sc = (qh @ kh.t()) * scale
            sc = torch.where(see, sc, torch.full_like(sc, -math.inf))
            any_ = see.any(-1, keepdim=True)
            top = torch.where(any_, sc.amax(-1, keepdim=True) if len(ok) else 0.0, 0.0)
            w = torch.where(see, torch.exp(sc - top), torch.zeros_like(sc))
            tot = torch.where(any_, w.sum(-1, keepdim=True), 1.0)
            w = w / tot
            # a weight of zero takes nothing from what it does not see
            o = torch.zeros((n, hd), dtype=torch.float64, device=q.device)
            fin = torch.isfinite(vh).all(-1)
            o += w[:, fin] @ vh[fin]
            for i in torch.nonzero(~fin).flatten().tolist():
                o += torch.where(see[:, i:i + 1], w[:, i:i + 1] * vh[i], 0.0)
            out[start[s]:start[s + 1], h] = o
            # rows that see a NaN or an infinity are compared as they are, and
            # their bound is not used
            ab = torch.where(see, (qh.abs() @ torch.nan_to_num(kh.abs(), 0, 0).t()) * scale, 0.0)
            a = ab.amax(-1, keepdim=True) if len(ok) else torch.zeros((n, 1), device=q.device)
            e = a * (2.0 ** -22 + (hd // 16) * pieces * 2.0 ** -22 + 6 * 2.0 ** -24)
            acc = ((len(ok) + 15) // 16 * pieces + 64) * 2.0 ** -22
            wabs = torch.nan_to_num(w, 0, 0) @ torch.nan_to_num(vh.abs(), 0, 0, 0)
            vmax = torch.nan_to_num(vh.abs(), 0, 0, 0).max() if len(ok) else 0.0
            bound[start[s]:start[s + 1], h] = (2 * e + u_p + acc) * wabs + \
                floor * len(ok) * vmax + EPS_HALF[q.dtype] * o.abs() + 1e-30
    if q.dtype == torch.float16:
        bound += 2.0 ** -25  # half a step of its subnormals
    return out.view(T, -1), bound.view(T, -1)
