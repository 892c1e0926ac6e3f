"""The paged KV cache's operators as they are measured: cases, inputs, plain forms.

A pool holds pages of 64 tokens for one KV head each.  A page is K then V, each
as panels of 64 rows of 128 bytes (F16: two panels, channels 0-63 and 64-127;
8 bits: one), the 16-byte chunk c of row r stored at c ^ (r & 7); the 8-bit
formats end with F32 scales, K[64] then V[64].  A sequence's position t lives
in row t % 64 of page table[t // 64].

Kinds of case:
  roundtrip  new K/V rows are written (quantised) into pages and read back
  read       listed positions are read back as F16 rows
  attend     decode attention of a batch over its pages, ragged lengths
  step       each sequence's new token is written, then the batch attends
  shared     decode attention of a batch whose sequences share a prefix
"""
import math

import torch

own = False

PAGE, DIM, GROUP = 64, 128, 4
TOP = {"int8": 127.0, "e4m3": 448.0}  # the largest code of a format


# ------------------------------------------------------------------- cases
def listed():
    return [
        # one decode step's K/V of 64 sequences: what every layer writes per token
        dict(name="write-step-64", kind="roundtrip", format="int8", heads=8, batch=64, tokens=1),
        # a whole prompt of the long-context workload entering the cache
        dict(name="write-prompt-32768", kind="roundtrip", format="e4m3", heads=8, batch=1, tokens=32768),
        # the selector's cap (20 %) of a 32768-token history read back for the packed attention
        dict(name="read-selected-6553", kind="read", format="int8", heads=8, tokens=32768, rows=6553),
        # a short selection
        dict(name="read-77", kind="read", format="e4m3", heads=8, tokens=1024, rows=77),
        # one short conversation: latency
        dict(name="attend-1x77", kind="attend", format="e4m3", heads=8, batch=1, tokens=77),
        # one long sequence, as a dense layer sees it
        dict(name="attend-1x32768", kind="attend", format="int8", heads=8, batch=1, tokens=32768),
        # a served batch of mixed lengths, one of them empty
        dict(name="attend-64x8192", kind="attend", format="e4m3", heads=8, batch=64, tokens=8192),
        # one KV head of eight (a shard), F16, 64 sequences
        dict(name="attend-shard-64x32768", kind="attend", format="f16", heads=1, batch=64, tokens=32768),
        # a decode step of an odd batch: write, then attend
        dict(name="step-48x4095", kind="step", format="int8", heads=8, batch=48, tokens=4095),
        # a few users of one short system prompt
        dict(name="shared-8x4097", kind="shared", format="f16", heads=8, batch=8, tokens=64, prefix=4097),
        # the served batch on one long document
        dict(name="shared-64x32768", kind="shared", format="int8", heads=8, batch=64, tokens=512, prefix=32768),
        # many samples of one prompt: the prefix is bound by its products
        dict(name="shared-256x16461", kind="shared", format="e4m3", heads=8, batch=256, tokens=256, prefix=16461),
    ]


def draw(rng):
    def spread(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["roundtrip", "read", "attend", "step", "shared"])
    case = dict(kind=kind, format=rng.choice(["f16", "int8", "e4m3"]), heads=rng.choice([1, 2, 4, 8]))
    if kind == "read":
        case["tokens"] = spread(64, 32768)
        case["rows"] = spread(1, case["tokens"])
        return case
    case["batch"] = spread(1, 64)
    if kind == "shared":
        case["batch"] = spread(1, 256)
        case["tokens"] = spread(1, 512)
        case["prefix"] = min(spread(1, 32768), 256 * 16461 // case["batch"])
    elif kind == "roundtrip":
        case["tokens"] = spread(1, max(1, 32768 // case["batch"]))
    else:  # attend, step: no more than the largest listed cache
        case["tokens"] = spread(1, min(32768, 64 * 32768 // (case["batch"] * case["heads"])))
    return case


def _lengths(case):
    """Ragged lengths up to case["tokens"]: the first has them all, one of a larger batch none."""
    b, top = case["batch"], case["tokens"]
    got = [top - int(top * (i * 0.6180339887498949 % 1.0)) for i in range(b)]
    if b >= 4:
        got[b // 2] = 0
    return got


# ------------------------------------------------------------------ inputs
def _panels(fmt):
    return 2 if fmt == "f16" else 1


def _page_bytes(fmt):
    return 32768 if fmt == "f16" else 16896


def _swizzle(x):
    """[..., 64 rows, 8 chunks, 16 bytes]: chunk c of row r to or from place c ^ (r & 7)."""
    row = torch.arange(PAGE, device=x.device)[:, None]
    place = torch.arange(8, device=x.device)[None, :] ^ (row & 7)
    return torch.gather(x, -2, place[..., None].expand(x.shape))


def _quantise(x, fmt):
    """Codes (as bytes, [..., bytes]) and scales ([...]) of the last axis of x."""
    if fmt == "f16":
        return x.contiguous().view(torch.uint8), None
    x = x.float()
    amax = x.abs().amax(-1)
    top = torch.full_like(amax, TOP[fmt])  # a tensor: both quotients are rounded once
    inv = torch.where(amax > 0, top / amax, torch.zeros_like(amax))
    y = x * inv[..., None]
    code = y.round().to(torch.int8) if fmt == "int8" else y.clamp(-448, 448).to(torch.float8_e4m3fn)
    return code.view(torch.uint8), amax / top


def _values(codes, scales, fmt):
    """F32 values of code bytes [..., bytes]."""
    if fmt == "f16":
        return codes.contiguous().view(torch.float16).float()
    code = codes.contiguous().view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn)
    return code.float() * scales[..., None]


def _store(pages, page, row, kv, fmt):
    """Writes rows kv [n, 2, heads, 128] F16 at (page, row)."""
    n, heads, per = kv.shape[0], kv.shape[2], _panels(fmt)
    codes, scales = _quantise(kv, fmt)
    chunk = torch.arange(8, device=kv.device)[None, :] ^ (row & 7)[:, None]
    codes = codes.view(n, 2, heads, per, 8, 16)
    area = pages[..., : 2 * per * PAGE * 128].view(-1, heads, 2, per, PAGE, 8, 16)
    # advanced indexes (page, row, chunk) of shape [n, 8]; what they pick is [n, 8, heads, 2, per, 16]
    area[page[:, None], :, :, :, row[:, None], chunk] = codes.permute(0, 4, 2, 1, 3, 5)
    if scales is not None:
        tail = pages[..., 2 * PAGE * 128:].view(torch.float32).view(-1, heads, 2, PAGE)
        tail[page, :, :, row] = scales.transpose(1, 2)


def _load(pages, page, row, fmt):
    """F32 rows [n, 2, heads, 128] at (page, row)."""
    n, heads, per = page.shape[0], pages.shape[1], _panels(fmt)
    chunk = torch.arange(8, device=pages.device)[None, :] ^ (row & 7)[:, None]
    area = pages[..., : 2 * per * PAGE * 128].view(-1, heads, 2, per, PAGE, 8, 16)
    codes = area[page[:, None], :, :, :, row[:, None], chunk].permute(0, 3, 2, 4, 1, 5).reshape(n, 2, heads, -1)
    if fmt == "f16":
        return _values(codes, None, fmt)
    tail = pages[..., 2 * PAGE * 128:].view(torch.float32).view(-1, heads, 2, PAGE)
    return _values(codes, tail[page, :, :, row].transpose(1, 2), fmt)


def _whole(pages, table, fmt):
    """F32 K and V [batch, heads, pages * 64, 128] of whole table rows."""
    heads, per = pages.shape[1], _panels(fmt)
    got = pages[table.clamp(min=0).long()]  # [batch, width, heads, bytes]
    b, w = table.shape
    codes = _swizzle(got[..., : 2 * per * PAGE * 128].view(b, w, heads, 2, per, PAGE, 8, 16))
    codes = codes.permute(0, 3, 2, 1, 5, 4, 6, 7).reshape(b, 2, heads, w * PAGE, -1)
    scales = None
    if fmt != "f16":
        scales = got[..., 2 * PAGE * 128:].view(torch.float32).view(b, w, heads, 2, PAGE)
        scales = scales.permute(0, 3, 2, 1, 4).reshape(b, 2, heads, w * PAGE)
    return _values(codes, scales, fmt).unbind(1)


def _rows(gen, n, heads):
    """K/V rows as a model gives them: F16, a few loud channels in K."""
    x = torch.randn((n, 2, heads, DIM), generator=gen, device="cuda")
    x[:, 0, :, 5::32] *= 6.0
    return x.half()


def _fill(gen, count, heads, fmt):
    """A pool of `count` pages, every row of it written, in pieces that bound the scratch."""
    pages = torch.zeros((count, heads, _page_bytes(fmt)), dtype=torch.uint8, device="cuda")
    step = max(1, 65536 // (PAGE * heads) * 8)
    for first in range(0, count, step):
        n = min(step, count - first)
        at = torch.arange(n * PAGE, device="cuda")
        _store(pages[first:first + n], at // PAGE, at % PAGE, _rows(gen, n * PAGE, heads), fmt)
    return pages


def _tables(gen, lengths):
    """Page tables of the lengths, pages in no order, -1 behind a sequence's last; and their number."""
    need = [-(-n // PAGE) for n in lengths]
    width, total = max(1, max(need)), sum(need)
    order = torch.randperm(max(1, total), generator=gen, device="cuda").int()
    table = torch.full((len(lengths), width), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = order[at:at + n]
        at += n
    return table, max(1, total)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    fmt, heads, kind = case["format"], case["heads"], case["kind"]
    s = dict(kind=kind, format=fmt, heads=heads)
    if kind == "read":
        s["table"], count = _tables(gen, [case["tokens"]])
        s["pages"] = _fill(gen, count, heads, fmt)
        at = torch.randperm(case["tokens"], generator=gen, device="cuda")[: case["rows"]]
        s["positions"] = at.sort().values.int()
    elif kind == "roundtrip":
        lengths = [case["tokens"]] * case["batch"]
        held = 100 if case["tokens"] == 1 else 0  # a decode step finds tokens there already
        s["table"], count = _tables(gen, [n + held for n in lengths])
        s["pages"] = torch.zeros((count, heads, _page_bytes(fmt)), dtype=torch.uint8, device="cuda")
        s["starts"] = torch.full((case["batch"],), held, dtype=torch.int32, device="cuda")
        s["rows"] = _rows(gen, sum(lengths), heads)
        s["offsets"] = torch.arange(case["batch"] + 1, dtype=torch.int32, device="cuda") * case["tokens"]
        s["seqs"] = torch.arange(case["batch"], dtype=torch.int32, device="cuda").repeat_interleave(case["tokens"])
        s["positions"] = torch.arange(case["tokens"], dtype=torch.int32, device="cuda").repeat(case["batch"]) + held
    else:
        lengths = _lengths(case)
        grow = 1 if kind == "step" else 0
        s["table"], count = _tables(gen, [n + grow for n in lengths])
        s["pages"] = _fill(gen, count, heads, fmt)
        s["lengths"] = torch.tensor([n + grow for n in lengths], dtype=torch.int32, device="cuda")
        q = torch.randn((case["batch"], GROUP * heads, DIM), generator=gen, device="cuda")
        s["q"] = q.half() if kind == "shared" else q
        if kind == "step":
            s["starts"] = s["lengths"] - 1
            s["rows"] = _rows(gen, case["batch"], heads)
        if kind == "shared":
            s["prefix_tokens"] = case["prefix"]
            table, count = _tables(gen, [case["prefix"]])
            s["prefix_table"], s["prefix"] = table[0].contiguous(), _fill(gen, count, heads, "f16")
    if own:
        import hillserve_b200 as hsb

        s["cache"] = hsb.KVPages(kv_heads=heads, format=fmt, data=s["pages"])
        if kind == "shared":
            s["prefix_cache"] = hsb.KVPages(kv_heads=heads, format="f16", data=s["prefix"])
    return s


# -------------------------------------------------------------- plain forms
def _softmax_sum(logits, v):
    """softmax(logits) . v over the last axis of logits; zero where every logit is -inf."""
    top = logits.amax(-1, keepdim=True)
    p = (logits - torch.where(top == -math.inf, torch.zeros_like(top), top)).exp()
    total = p.sum(-1, keepdim=True)
    return torch.matmul(p, v) / torch.where(total > 0, total, torch.ones_like(total))


def _own_tokens(s):
    """Masked logits [batch, heads, 4, tokens] and V of each sequence's own pages."""
    heads = s["heads"]
    k, v = _whole(s["pages"], s["table"], s["format"])
    q = s["q"].float().view(-1, heads, GROUP, DIM)
    live = torch.arange(k.shape[2], device=k.device)[None, :] < s["lengths"][:, None]
    logits = torch.matmul(q, k.transpose(-1, -2)) / math.sqrt(DIM)
    logits = logits.masked_fill(~live[:, None, None, :], -math.inf)
    return logits, v.masked_fill(~live[:, None, :, None], 0.0)


def _plain(s):
    fmt, heads, kind = s["format"], s["heads"], s["kind"]
    if kind in ("roundtrip", "read"):
        pos = s["positions"].long()
        seq = s["seqs"].long() if kind == "roundtrip" else torch.zeros_like(pos)
        page, row = s["table"][seq, pos // PAGE].long(), pos % PAGE
        if kind == "roundtrip":
            _store(s["pages"], page, row, s["rows"], fmt)
        return _load(s["pages"], page, row, fmt).half()
    if kind == "step":
        pos = s["starts"].long()
        page = s["table"].gather(1, (pos // PAGE)[:, None])[:, 0].long()
        _store(s["pages"], page, pos % PAGE, s["rows"], fmt)
        written = _load(s["pages"], page, pos % PAGE, fmt).half()
    logits, v = _own_tokens(s)
    if kind != "shared":
        out = _softmax_sum(logits, v).reshape(s["q"].shape)
        return (out, written) if kind == "step" else out
    n = s["prefix_tokens"]
    pk, pv = (x[0, :, :n] for x in _whole(s["prefix"], s["prefix_table"][None], "f16"))
    q = s["q"].float().view(-1, heads, GROUP, DIM)
    rows = q.transpose(0, 1).reshape(heads, -1, DIM)  # every sequence's rows against the one prefix
    before = (torch.matmul(rows, pk.transpose(-1, -2)) / math.sqrt(DIM)).view(heads, -1, GROUP, n).transpose(0, 1)
    top = torch.maximum(before.amax(-1, keepdim=True), logits.amax(-1, keepdim=True))
    a, b = (before - top).exp(), (logits - top).exp()
    joint = torch.matmul(a.transpose(0, 1).reshape(heads, -1, n), pv).view(heads, -1, GROUP, DIM).transpose(0, 1)
    out = (joint + torch.matmul(b, v)) / (a.sum(-1, keepdim=True) + b.sum(-1, keepdim=True))
    return out.half().reshape(s["q"].shape)


# --------------------------------------------------------- the library's own
def _own(s):
    cache, kind = s["cache"], s["kind"]
    if kind == "read":
        return cache.read(s["positions"], s["table"])
    if kind == "roundtrip":
        cache.append(s["rows"], s["table"], s["starts"], offsets=s["offsets"])
        return cache.read(s["positions"], s["table"], seqs=s["seqs"])
    if kind == "attend":
        return cache.attention(s["q"], s["table"], s["lengths"])
    if kind == "step":
        cache.append(s["rows"], s["table"], s["starts"])
        out = cache.attention(s["q"], s["table"], s["lengths"])
        return out, cache.read(s["starts"], s["table"], seqs=torch.arange(len(s["starts"]), dtype=torch.int32,
                                                                          device="cuda"))
    return cache.attention_shared(s["q"], s["table"], s["lengths"], s["prefix_cache"], s["prefix_table"],
                                  s["prefix_tokens"])


def run(state):
    return _own(state) if own else _plain(state)


# -------------------------------------------------------------------- floors
def _token_bytes(fmt, heads):
    """Bytes of one cached token: K and V codes, and their scales."""
    return heads * 2 * (DIM * (2 if fmt == "f16" else 1) + (0 if fmt == "f16" else 4))


def work(case):
    fmt, heads, kind = case["format"], case["heads"], case["kind"]
    row = heads * 2 * DIM * 2  # an F16 K||V row
    if kind == "read":
        n = case["rows"]
        return {"bytes": n * (_token_bytes(fmt, heads) + row + 4), "flops": n * heads * 2 * DIM}
    if kind == "roundtrip":
        n = case["batch"] * case["tokens"]
        return {"bytes": n * 2 * (_token_bytes(fmt, heads) + row), "flops": n * heads * 2 * DIM * 4}
    b = case["batch"]
    total = sum(_lengths(case))
    size, flops = b * GROUP * heads * DIM * 8, 4 * DIM * GROUP * heads * total
    size += total * _token_bytes(fmt, heads)
    if kind == "step":
        size += b * 2 * (_token_bytes(fmt, heads) + row)
        flops += 4 * DIM * GROUP * heads * b
    if kind == "shared":
        size += case["prefix"] * _token_bytes("f16", heads) - b * GROUP * heads * DIM * 4
        flops += 4 * DIM * GROUP * heads * b * case["prefix"]
    return {"bytes": size, "flops": flops}


# ------------------------------------------------------- the definition, 64 bits
def _sequence(pages, table, n, head, fmt):
    """K and V [n, 128] in 64 bits of one sequence's head, byte by byte from the page's definition."""
    per = 2 if fmt == "f16" else 1
    blocks = pages[table[: -(-n // 64)].long(), head]
    panels = blocks[:, : 2 * per * 8192].reshape(-1, 2, per, 64, 128)
    r = torch.arange(64, device=pages.device)[:, None]
    byte = torch.arange(128, device=pages.device)[None, :]
    plain = panels[:, :, :, r, ((byte // 16) ^ (r % 8)) * 16 + byte % 16]
    got = []
    for which in (0, 1):
        x = plain[:, which].transpose(1, 2).reshape(-1, per * 128)[:n].contiguous()  # a token's bytes in order
        if fmt == "f16":
            got.append(x.view(torch.float16).double())
            continue
        scale = blocks[:, 16384 + 256 * which: 16640 + 256 * which].contiguous().view(torch.float32)
        code = x.view(torch.int8 if fmt == "int8" else torch.float8_e4m3fn).float().double()
        got.append(code * scale.reshape(-1)[:n, None].double())
    return got


def _written64(rows, fmt):
    """What written rows stand for.  A code is what the format's F32 rule says
    (a border between two codes is its, not the real numbers'); its value is exact."""
    if fmt == "f16":
        return rows.double()
    a = rows.float().abs().max(-1, keepdim=True).values
    top = torch.full_like(a, TOP[fmt])
    y = rows.float() * torch.where(a > 0, top / a, a)
    code = torch.round(y) if fmt == "int8" else y.to(torch.float8_e4m3fn).float()
    return code.double() * (a / top).double()


def exact(case, seed):
    kind, heads, fmt = case["kind"], case["heads"], case["format"]
    s = prepare(case, seed)
    if kind == "roundtrip":
        return _written64(s["rows"], fmt)
    if kind == "read":
        kv = [torch.stack([_sequence(s["pages"], s["table"][0], case["tokens"], h, fmt)[w] for h in range(heads)], 1)
              for w in (0, 1)]
        return torch.stack(kv, 1)[s["positions"].long()]
    q = s["q"].double().view(-1, heads, GROUP, DIM)
    out = torch.zeros_like(q)
    lengths = s["lengths"].tolist()
    table = s["table"]
    first = [_sequence(s["prefix"], s["prefix_table"], case["prefix"], h, "f16") if kind == "shared" else None
             for h in range(heads)]
    for b, n in enumerate(lengths):
        held = n - 1 if kind == "step" else n
        for h in range(heads):
            k, v = _sequence(s["pages"], table[b], held, h, fmt)
            if kind == "step":
                new = _written64(s["rows"][b, :, h], fmt)
                k, v = torch.cat([k, new[:1]]), torch.cat([v, new[1:]])
            if kind == "shared":
                k, v = torch.cat([first[h][0], k]), torch.cat([first[h][1], v])
            if len(k):
                out[b, h] = torch.softmax(q[b, h] @ k.T / math.sqrt(128.0), -1) @ v
    out = out.view(s["q"].shape)
    return (out, _written64(s["rows"], fmt)) if kind == "step" else out
