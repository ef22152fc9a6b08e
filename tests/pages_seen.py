"""Attention over a paged cache in 64 bits, with the error that the kernels'
arithmetic may make counted over the positions that a row sees and no others:
whatever stands at a hidden position leaves a row's bound as it is."""
import math

import torch

import pages_ref as R


def attention(q, n_head, pages, table, start, kv_len, window=0, n_sink=0, scale=None):
    """(out, bound), [n_tokens, n_head * head_dim] in 64 bits; rows outside the
    batch are NaN in ``out``.

    The bound is that of pages_ref.attention, term by term, with its largest |v| and
    its number of positions taken per row, over the positions that the row
    sees.  An 8-bit row's products of weight and scale are held relative to the
    largest finite scale that this row sees, on a grid of 16-bit floats."""
    hd, nkv, page = pages.head_dim, pages.n_head_kv, pages.page_size
    n_pages = pages.k.shape[0]
    g = n_head // nkv
    scale = hd ** -0.5 if scale is None else scale
    out = torch.full((q.shape[0], n_head, hd), math.nan, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    f32 = q.dtype == torch.float32
    bf16_cache = pages.k.dtype == torch.bfloat16
    pieces = 3 if f32 else 1
    u_p = 2.0 ** -22 if f32 else R.EPS_HALF[torch.bfloat16 if bf16_cache else torch.float16]
    floor = 0.0 if bf16_cache else 2.0 ** -(24 + (14 if f32 else 6))
    tab = table.cpu()
    for s in range(len(kv_len)):
        n = start[s + 1] - start[s]
        if n == 0:
            continue
        at = [(j, R.page_of(tab, s, j, page, n_pages)) for j in range(max(kv_len[s], 0))]
        at = [x for x in at if x[1] >= 0]
        if not at:
            out[start[s]:start[s + 1]] = 0
            bound[start[s]:start[s + 1]] = 1e-30
            continue
        j = torch.tensor([x[0] for x in at], device=q.device)
        ids = torch.tensor([x[1] for x in at], device=q.device)
        k = R.values(pages.k, pages.k_scale, ids, j % page).permute(1, 0, 2)[:, None]
        v = R.values(pages.v, pages.v_scale, ids, j % page).permute(1, 0, 2)[:, None]
        x = q[start[s]:start[s + 1]].double().view(n, nkv, g, hd).permute(1, 2, 0, 3)
        pos = torch.arange(kv_len[s] - n, kv_len[s], device=q.device)[:, None]
        see = j[None] <= pos
        if window:
            see &= (pos - j[None] < window) | (j[None] < n_sink)
        any_ = see.any(-1, keepdim=True)
        sc = x @ k.transpose(-1, -2) * scale  # [nkv, g, n, len]
        sc = torch.where(see, sc, torch.full_like(sc, -math.inf))
        top = torch.where(any_, sc.amax(-1, keepdim=True), torch.zeros_like(sc[..., :1]))
        w = torch.where(see, torch.exp(sc - top), torch.zeros_like(sc))
        w = w / torch.where(any_, w.sum(-1, keepdim=True), torch.ones_like(sc[..., :1]))
        # what a row does not see has no part in its sum, finite or not
        fin = torch.isfinite(v)
        o = w @ torch.where(fin, v, torch.zeros_like(v))
        for i in torch.nonzero(~fin.all(-1).all(0)[0]).flatten().tolist():
            bad = torch.where(fin[:, :, i], torch.zeros_like(v[:, :, i]), v[:, :, i])
            term = w[..., i:i + 1] * bad[:, :, None]
            hit = see[:, i:i + 1] & ~fin[:, :, i][:, :, None]
            o = o + torch.where(hit, term, torch.zeros_like(term))
        out[start[s]:start[s + 1]] = o.permute(2, 0, 1, 3).reshape(n, n_head, hd)

        vabs = torch.nan_to_num(v.abs(), 0, 0)
        ab = torch.where(see, x.abs() @ torch.nan_to_num(k.abs(), 0, 0).transpose(-1, -2) * scale,
                         torch.zeros_like(sc))
        e = ab.amax(-1, keepdim=True) * \
            (2.0 ** -22 + (hd // 16) * pieces * 2.0 ** -22 + 6 * 2.0 ** -24)
        count = see.sum(-1)[:, None].double()  # [n, 1]
        acc = (torch.ceil(count / 16) * pieces + 64) * 2.0 ** -22
        big = vabs.amax(-1).expand(nkv, g, -1)[:, :, None]  # of a position, [nkv, g, 1, len]
        vmax = torch.where(see, big, torch.zeros_like(sc)).amax(-1, keepdim=True)
        b = (2 * e + u_p + acc) * (torch.nan_to_num(w, 0, 0) @ vabs) + floor * count * vmax + \
            R.EPS_HALF[q.dtype] * o.abs() + 1e-30
        bound[start[s]:start[s + 1]] = b.permute(2, 0, 1, 3).reshape(n, n_head, hd)
    if q.dtype == torch.float16:
        bound += 2.0 ** -25  # half a step of its subnormals
    return out.flatten(1), bound.flatten(1)
