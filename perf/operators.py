"""The paged KV cache operators: what is measured and against which plain form.

Three operators that a server of many requests calls per layer and step: storing the new K and V
rows in a paged cache (quantised to 8 bits, or rounded to 16), reading rows back, and the attention
of the new tokens over the pages, with or without a sliding window and sink tokens.

A case names the head layout, the types and the sequences.  Sequences are a text of groups
``COUNTxNEW@LO-HI``: COUNT sequences with NEW new tokens each, whose lengths after the write are
spread between LO and HI.
"""
import math

import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "q8": torch.int8}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2, "q8": 1}


def listed():
    return [
        # --- storing new rows -------------------------------------------------------------
        # one decode step of 48 users: the fp32 K/V rows the decode GEMV leaves (launch-bound).
        # 8-bit rows are returned as the values they stand for, so these passes store and read back
        dict(name="write_q8_decode48", op="write", n_head=32, n_kv=8, hd=128, page=16, q="f32",
             cache="q8", seqs="48x1@40-9000", window=0, sink=0),
        # a long prompt's rows from the prefill GEMM in bf16
        dict(name="write_q8_prompt8k", op="write", n_head=32, n_kv=8, hd=128, page=64, q="bf16",
             cache="q8", seqs="1x8192@8192-8192", window=0, sink=0),
        # ragged chunks of several requests, fp32 rows rounded to an f16 cache, small heads
        dict(name="write_f16_ragged", op="write", n_head=12, n_kv=4, hd=64, page=32, q="f32",
             cache="f16", seqs="3x1021@1021-5000,5x77@77-700,9x1@1-3001", window=0, sink=0),
        # --- reading rows back ------------------------------------------------------------
        # a prefix snapshot of four long requests leaves the cache in fp32
        dict(name="read_q8_snapshot", op="read", n_head=32, n_kv=8, hd=128, page=64, q="f32",
             cache="q8", seqs="4x7001@7001-9000", window=0, sink=0),
        # a short prefix of a bf16 cache
        dict(name="read_bf16_prefix", op="read", n_head=32, n_kv=8, hd=128, page=16, q="bf16",
             cache="bf16", seqs="1x333@333-333", window=0, sink=0),
        # --- attention over the pages -----------------------------------------------------
        # one user, short context, fp32 activations: latency
        dict(name="attn_decode1_q8", op="attn", n_head=32, n_kv=8, hd=128, page=16, q="f32",
             cache="q8", seqs="1x1@517-517", window=0, sink=0),
        # a serving step of 64 users with contexts of very different lengths: cache bandwidth
        dict(name="attn_decode64_q8", op="attn", n_head=32, n_kv=8, hd=128, page=64, q="bf16",
             cache="q8", seqs="64x1@100-16000", window=0, sink=0),
        # speculative verification: five tokens of eight users, 70B head layout, fp32 on f16
        dict(name="attn_verify5_f16", op="attn", n_head=64, n_kv=8, hd=128, page=32, q="f32",
             cache="f16", seqs="8x5@900-6000", window=0, sink=0),
        # a prefill chunk on top of what came before: tensor cores
        dict(name="attn_chunk2k_bf16", op="attn", n_head=32, n_kv=8, hd=128, page=64, q="bf16",
             cache="bf16", seqs="1x2048@16384-16384", window=0, sink=0),
        # chunked prefill beside decode in one batch, 8-bit cache
        dict(name="attn_mixed_q8", op="attn", n_head=32, n_kv=8, hd=128, page=16, q="f16",
             cache="q8", seqs="2x511@1300-7777,30x1@64-8000", window=0, sink=0),
        # --- sliding window and sinks -----------------------------------------------------
        # streaming decode far into long conversations
        dict(name="window_decode16_f16", op="attn", n_head=32, n_kv=8, hd=128, page=32, q="f32",
             cache="f16", seqs="16x1@20000-65000", window=4096, sink=4),
        # a long prompt under a window, small heads
        dict(name="window_prompt8k_bf16", op="attn", n_head=8, n_kv=2, hd=64, page=64, q="bf16",
             cache="bf16", seqs="1x8191@8191-8191", window=1024, sink=5),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    heads = [(32, 8, 128), (64, 8, 128), (12, 4, 64), (8, 2, 64), (16, 2, 256), (8, 8, 64)]
    most = [work(c) for c in listed()]
    most = {u: max(w[u] for w in most) for u in most[0]}
    while True:
        op = rng.choice(["write", "read", "attn", "attn", "attn"])
        nh, nkv, hd = rng.choice(heads)
        cache = rng.choice(["q8", "q8", "f16", "bf16"])
        q = rng.choice(["f32", "f16" if cache == "f16" else "bf16" if cache == "bf16"
                        else rng.choice(["f16", "bf16"])])
        groups = []
        kind = rng.choice(["decode", "chunk", "mixed", "verify"])
        if kind in ("decode", "mixed"):
            lo = log(1, 8000)
            groups.append(f"{log(1, 64)}x1@{lo}-{lo + log(1, 16000)}")
        if kind == "verify":
            n = rng.randint(2, 12)
            lo = n + log(1, 6000)
            groups.append(f"{log(1, 16)}x{n}@{lo}-{lo + log(1, 8000)}")
        if kind in ("chunk", "mixed"):
            n = log(17, 4096)
            lo = n + rng.choice([0, log(1, 12000)])
            groups.append(f"{rng.randint(1, 3)}x{n}@{lo}-{lo + log(1, 2000)}")
        windowed = op == "attn" and rng.random() < 0.4
        case = dict(op=op, n_head=nh, n_kv=nkv, hd=hd, page=rng.choice([16, 32, 64, 128]), q=q,
                    cache=cache, seqs=",".join(groups),
                    window=log(16, 5000) if windowed else 0,
                    sink=rng.randint(0, 70) if windowed else 0)
        w = work(case)
        held = sum(length for _, length in _seqs(case)) * 2 * nkv * hd * _SIZE[cache]
        if held <= 4 << 30 and all(w[u] <= most[u] for u in most):
            return case


def _seqs(case):
    """[(new tokens, length after the write)] of every sequence."""
    out = []
    for group in case["seqs"].split(","):
        count, rest = group.split("x")
        new, span = rest.split("@")
        lo, hi = (int(v) for v in span.split("-"))
        for i in range(int(count)):
            out.append((int(new), lo + int((hi - lo) * ((i + 1) * 0.6180339887498949 % 1.0))))
    return out


def _pairs(case, n, length):
    """Visible (query, position) pairs, and the positions that any query sees."""
    w, s = case["window"], case["sink"]
    first = length - n
    if not w:
        return n * first + n * (n + 1) // 2, length
    pairs = 0
    for p in range(first, length):
        lo = max(0, p - w + 1)
        pairs += p + 1 - lo + min(s, lo)
    lo = max(0, first - w + 1)
    return pairs, length - lo + min(s, lo)


def work(case):
    nkv, hd = case["n_kv"], case["hd"]
    cache_row = 2 * nkv * (hd * _SIZE[case["cache"]] + (4 if case["cache"] == "q8" else 0))
    x_row = 2 * nkv * hd * _SIZE[case["q"]]
    seqs = _seqs(case)
    rows = sum(n for n, _ in seqs)
    if case["op"] != "attn":
        # a pass that stores 8-bit rows also returns the values they stand for
        back = x_row if case["op"] == "write" and case["cache"] == "q8" else 0
        return {"bytes": rows * (cache_row + x_row + back), "flops": rows * nkv * hd * 4}
    pairs = seen = 0
    for n, length in seqs:
        a, b = _pairs(case, n, length)
        pairs += a
        seen += b
    q_row = case["n_head"] * hd * _SIZE[case["q"]]
    return {"bytes": 2 * rows * q_row + seen * cache_row, "flops": 4 * hd * case["n_head"] * pairs}


# ------------------------------------------------------------------------------------ inputs

def _inputs(case, seed):
    """Page pools with every slot filled, a shuffled page table and the new rows."""
    dev = torch.device("cuda", torch.cuda.current_device())
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    nkv, hd, page = case["n_kv"], case["hd"], case["page"]
    seqs = _seqs(case)
    rows = sum(n for n, _ in seqs)
    per = [-(-length // page) for _, length in seqs]
    n_pages = sum(per) + 3
    order = torch.randperm(n_pages, generator=g, device=dev, dtype=torch.int64)
    table = torch.full((len(seqs), max(per)), -1, dtype=torch.int64, device=dev)
    at = 0
    for s, c in enumerate(per):
        table[s, :c] = order[at:at + c]
        at += c
    # K rows carry a few strong channels, as rotated keys do
    channel = torch.ones(hd, device=dev)
    channel[hd // 8::hd // 4] = 4.0

    def rand(shape, gain):
        return torch.randn(shape, generator=g, device=dev) * gain

    st = {"case": case, "seqs": seqs, "table": table}
    for name, gain in (("k", channel), ("v", 1.0)):
        if case["cache"] == "q8":
            pool = torch.empty((n_pages, nkv, page, hd), dtype=torch.int8, device=dev)
            scale = torch.empty((n_pages, nkv, page), dtype=torch.float32, device=dev)
            step = max(1, (1 << 26) // (nkv * page * hd))
            for i in range(0, n_pages, step):
                x = rand((min(step, n_pages - i), nkv, page, hd), gain)
                d = x.abs().amax(-1) / 127
                pool[i:i + step] = (x / d[..., None]).round().clamp(-127, 127).to(torch.int8)
                scale[i:i + step] = d
            st[name + "_scale"] = scale
        else:
            pool = torch.empty((n_pages, nkv, page, hd), dtype=_DT[case["cache"]], device=dev)
            step = max(1, (1 << 26) // (nkv * page * hd))
            for i in range(0, n_pages, step):
                pool[i:i + step] = rand((min(step, n_pages - i), nkv, page, hd), gain)
        st[name] = pool
    if case["op"] == "write":
        st["k_new"] = rand((rows, nkv * hd), channel.repeat(nkv)).to(_DT[case["q"]])
        st["v_new"] = rand((rows, nkv * hd), 1.0).to(_DT[case["q"]])
    elif case["op"] == "attn":
        st["q"] = rand((rows, case["n_head"] * hd), 1.0).to(_DT[case["q"]])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    dev = st["table"].device
    starts, lens = [0], []
    for n, length in st["seqs"]:
        starts.append(starts[-1] + n)
        lens.append(length)
    st["rows"] = starts[-1]
    st["starts"] = starts
    # page and slot of every row of the batch, for the plain form
    page = case["page"]
    pos = torch.cat([torch.arange(length - n, length) for n, length in st["seqs"]]).to(dev)
    seq = torch.cat([torch.full((n,), i) for i, (n, _) in enumerate(st["seqs"])]).to(dev)
    st["row_page"] = st["table"][seq, pos // page]
    st["row_slot"] = pos % page
    if own:
        from xwfes_b200 import ftc
        st["pages"] = ftc.KvPages(st["k"], st["v"], st.get("k_scale"), st.get("v_scale"))
        st["batch"] = ftc.PageBatch(
            torch.tensor(starts, dtype=torch.int32, device=dev),
            torch.tensor(lens, dtype=torch.int32, device=dev), st["table"].to(torch.int32),
            n_tokens=st["rows"], max_new=max(n for n, _ in st["seqs"]))
    return st


# ------------------------------------------------------------------------------------ passes

def run(st):
    case = st["case"]
    if own:
        return _run_own(st, case)
    return {"write": _plain_write, "read": _plain_read, "attn": _plain_attn}[case["op"]](st, case)


def _run_own(st, case):
    from xwfes_b200 import ftc
    pages, batch = st["pages"], st["batch"]
    if case["op"] == "write":
        ftc.kv_pages_write(pages, st["k_new"], st["v_new"], batch)
        if case["cache"] != "q8":
            return [st["k"], st["v"]]
        return list(ftc.kv_pages_read(pages, batch, out_dtype=case["q"].upper()))
    if case["op"] == "read":
        return list(ftc.kv_pages_read(pages, batch, out_dtype=case["q"].upper()))
    return ftc.attention_pages(st["q"], case["n_head"], pages, batch, window=case["window"],
                               n_sink=case["sink"])


def _plain_write(st, case):
    page, slot = st["row_page"], st["row_slot"]
    out = []
    for name in ("k", "v"):
        x = st[name + "_new"].float().view(-1, case["n_kv"], case["hd"])
        if case["cache"] != "q8":
            st[name][page, :, slot] = x.to(_DT[case["cache"]])
            out.append(st[name])
            continue
        # quotients next to a half are decided in 64 bits
        d = (x.abs().amax(-1).double() / 127).float()
        code = (x.double() / d.double()[..., None]).round().clamp(-127, 127)
        code = torch.where(d[..., None] > 0, code, torch.zeros_like(code)).to(torch.int8)
        st[name][page, :, slot] = code
        st[name + "_scale"][page, :, slot] = d
        out.append((code.float() * d[..., None]).to(_DT[case["q"]]).view(st["rows"], -1))
    return out


def _plain_read(st, case):
    page, slot = st["row_page"], st["row_slot"]
    out = []
    for name in ("k", "v"):
        x = st[name][page, :, slot].float()
        if case["cache"] == "q8":
            x = x * st[name + "_scale"][page, :, slot][..., None]
        out.append(x.to(_DT[case["q"]]).reshape(st["rows"], -1))
    return out


def _plain_attn(st, case):
    nh, nkv, hd, page = case["n_head"], case["n_kv"], case["hd"], case["page"]
    gqa = nh // nkv
    w, sink = case["window"], case["sink"]
    q = st["q"]
    out = torch.empty((st["rows"], nkv, gqa, hd), dtype=q.dtype, device=q.device)
    for s, (n, length) in enumerate(st["seqs"]):
        r0 = st["starts"][s]
        first = length - n
        lo = max(0, first - w + 1) if w else 0
        j = torch.arange(lo, length, device=q.device)
        if min(sink, lo):
            j = torch.cat([torch.arange(min(sink, lo), device=q.device), j])
        pg, sl = st["table"][s, j // page], j % page
        k, v = st["k"][pg, :, sl].float(), st["v"][pg, :, sl].float()  # [len, n_kv, hd]
        if case["cache"] == "q8":
            k = k * st["k_scale"][pg, :, sl][..., None]
            v = v * st["v_scale"][pg, :, sl][..., None]
        p = torch.arange(first, length, device=q.device)[:, None]
        hidden = j[None, :] > p
        if w:
            hidden |= (p - j[None, :] >= w) & (j[None, :] >= sink)
        qs = q[r0:r0 + n].float().view(n, nkv, gqa, hd) * (1.0 / math.sqrt(hd))
        step = max(1, (1 << 28) // max(1, gqa * len(j)))
        for h in range(nkv):
            kt, vh = k[:, h].t(), v[:, h]
            for i in range(0, n, step):
                x = qs[i:i + step, h].reshape(-1, hd) @ kt
                x = x.view(-1, gqa, len(j)).masked_fill_(hidden[i:i + step, None], -math.inf)
                x = torch.exp(x - x.amax(-1, keepdim=True))
                tot = x.sum(-1, keepdim=True)
                y = (x.view(-1, len(j)) @ vh).view(-1, gqa, hd) / tot
                out[r0 + i:r0 + i + y.shape[0], h] = y.to(q.dtype)
    return out.view(st["rows"], nh * hd)


# ------------------------------------------------------------------------------------ exact

def exact(case, seed):
    """The definition in 64 bits, row by row of the page table, apart from the plain form."""
    st = _inputs(case, seed)
    if case["op"] == "attn":
        if work(case)["flops"] > 3e12:
            return None
        return _exact_attn(st, case)
    page, nkv, hd = case["page"], case["n_kv"], case["hd"]
    whole, outs = [], []
    for name in ("k", "v"):
        if case["op"] == "write" and case["cache"] != "q8":
            flat = st[name].double().permute(0, 2, 1, 3).reshape(-1, nkv, hd)
            new = st[name + "_new"].double().view(-1, nkv, hd)
            r = 0
            for s, (n, length) in enumerate(st["seqs"]):
                for a, b in _spans(length - n, length, page):
                    at = int(st["table"][s, a // page]) * page + a % page
                    flat[at:at + b - a] = new[r:r + b - a]
                    r += b - a
            whole.append(flat.view(-1, page, nkv, hd).permute(0, 2, 1, 3).contiguous())
        elif case["op"] == "write":
            x = st[name + "_new"].double().view(-1, nkv, hd)
            top = x.abs().max(dim=-1, keepdim=True).values
            d = (top / 127.0).float().double()
            level = torch.where(top > 0, torch.round(x / d), torch.zeros_like(x))
            outs.append((level * d).view(-1, nkv * hd))
        else:
            parts = []
            for s, (n, length) in enumerate(st["seqs"]):
                parts.append(_exact_rows(st, case, name, s, length - n, length))
            outs.append(torch.cat(parts).reshape(-1, nkv * hd))
    return whole or outs


def _spans(a, b, page):
    while a < b:
        e = min(b, (a // page + 1) * page)
        yield a, e
        a = e


def _exact_rows(st, case, name, s, a, b):
    """Cached rows [a, b) of sequence s in 64 bits, [b - a, n_kv, hd]."""
    page = case["page"]
    ids = st["table"][s, a // page:-(-b // page)]
    rows = st[name][ids].double()
    if case["cache"] == "q8":
        rows *= st[name + "_scale"][ids].double().unsqueeze(-1)
    rows = rows.transpose(1, 2).flatten(0, 1)
    return rows[a - a // page * page:][:b - a]


def _exact_attn(st, case):
    nh, nkv, hd = case["n_head"], case["n_kv"], case["hd"]
    group = nh // nkv
    rows = []
    at = 0
    for s, (n, length) in enumerate(st["seqs"]):
        keys = _exact_rows(st, case, "k", s, 0, length).permute(1, 2, 0)
        vals = _exact_rows(st, case, "v", s, 0, length).permute(1, 0, 2)
        where = torch.arange(length, device=keys.device)
        step = max(1, (1 << 27) // (nh * length))
        for i in range(0, n, step):
            m = min(step, n - i)
            pos = length - n + torch.arange(i, i + m, device=keys.device)
            seen = where <= pos[:, None]
            if case["window"]:
                seen &= (where > pos[:, None] - case["window"]) | (where < case["sink"])
            x = st["q"][at + i:at + i + m].double().view(m, nkv, group, hd)
            x = x.permute(1, 2, 0, 3).flatten(1, 2)
            score = torch.bmm(x, keys).view(nkv, group, m, length) * hd ** -0.5
            score = torch.where(seen, score, torch.full_like(score, -math.inf))
            prob = torch.softmax(score, dim=-1).view(nkv, group * m, length)
            y = torch.bmm(prob, vals).view(nkv, group, m, hd)
            rows.append(y.permute(2, 0, 1, 3).reshape(m, nh * hd))
        at += n
    return torch.cat(rows)
