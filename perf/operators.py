"""The operators of the cache in eight bits, and attention for trees of drafted tokens: the cases that they are measured on.

Keys and values of G heads of D values lie in pages [pages, 2, G, page, D] (keys, then values), in eight bits as codes of
float8_e4m3fn with one exponent a token, head and plane: a value is code * 2^(exponent - 127).  The exponent of a row of D values
is 127 + n with the smallest n for which max |x| <= 448 * 2^n, n in -60 .. 60 (127 for a row of zeros); codes are x * 2^-n rounded
to the nearest, ties to even.

  write    keys and values of new tokens, as float32 columns of a wider product or as bfloat16 rows, go into their slots
           (page * page size + place in the page; a negative slot: the row is not kept)
  read     pages come back as bfloat16 or float32, slots behind the last token as zeros
  attend   softmax attention of requests' new rows over what the cache holds of each: row i of a request with a history of h keys
           sees the keys up to h + i (the last `window` of them); one row a request when tokens are decoded, many for a prompt
  tree     the same where a request's rows are drafted tokens: row i sees the h keys of the history and those drafted
           tokens that its bits name (itself and what it was drafted from); over eight bits or over bfloat16

Head h of H reads key/value head h // (H / G).  The sizes of heads are those of the dense models that `bench.py` times (32 or 16
heads over 8 of 128) and generic ones of 64.
"""
import math

import numpy as np
import torch

own = False

DEVICE = "cuda:0"
LOWEST, HIGHEST = -60, 60


def _attend(name, **kw):
    c = dict(name=name, kind="attend", heads=32, kv_heads=8, dim=128, page=16, requests=1, rows=1, context=8192, ragged=False, window=0,
             dtype="bfloat16")
    c.update(kw)
    return c


def listed():
    return [
        # The new tokens of a decoding step of 8 requests: columns of the q/k/v product's float32 output.  Latency counts.
        dict(name="write_8_float32", kind="write", rows=8, heads=32, kv_heads=8, dim=128, page=16, dtype="float32"),
        # Rows of several prompts, made elsewhere as bfloat16, heads of 64, an odd number of them.
        dict(name="write_5001_bf16_64", kind="write", rows=5001, heads=0, kv_heads=16, dim=64, page=32, dtype="bfloat16"),
        # One request's cache read back whole, for a kernel that wants bfloat16 or for another process.
        dict(name="read_1x8192_bf16", kind="read", requests=1, context=8192, ragged=False, kv_heads=8, dim=128, page=16, dtype="bfloat16"),
        # Many requests of odd lengths, read back as float32.
        dict(name="read_16x4001_float32", kind="read", requests=16, context=4001, ragged=True, kv_heads=8, dim=64, page=16, dtype="float32"),
        # Decoding: one long request; the batch of the decode benchmark; many short ones of all lengths; the 32-bit path.
        _attend("decode_1x32768", context=32768),
        _attend("decode_8x8192", requests=8),
        _attend("decode_64x4096_ragged", requests=64, context=4096, ragged=True, heads=16, page=32),
        _attend("decode_4x2001_float32", requests=4, context=2001, heads=16, dtype="float32"),
        # A prompt's last portion after three others, and portions of several prompts under a window.
        _attend("prompt_2048_after_6144", rows=2048, context=8192),
        _attend("prompt_6x700_window", requests=6, rows=700, context=2500, ragged=True, heads=16, window=1024),
        # Drafts: 16 tokens for each of 8 requests over eight bits, one wide tree over bfloat16.
        _attend("tree_8x16_at_4096", kind="tree", requests=8, rows=16, context=4096, store="e4m3"),
        _attend("tree_1x63_at_8191_bf16", kind="tree", rows=63, context=8191, store="bfloat16"),
    ]


def _size(rng, low, high):
    """low .. high, spread over the logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "decode", "decode", "prompt", "tree"])
    dim = rng.choice([64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    page = rng.choice([16, 16, 32])
    if kind == "write":
        dtype = rng.choice(["float32", "bfloat16"])
        return dict(kind=kind, rows=_size(rng, 1, 8192), heads=rng.choice([0, 2, 4]) * kv_heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype)
    if kind == "read":
        requests = _size(rng, 1, 32)
        return dict(kind=kind, requests=requests, context=_size(rng, 1, 65536 // requests), ragged=rng.random() < 0.5, kv_heads=kv_heads, dim=dim, page=page,
                    dtype=rng.choice(["float32", "bfloat16"]))
    heads = kv_heads * rng.choice([1, 2, 4, 5, 8])
    case = dict(kind="attend", heads=heads, kv_heads=kv_heads, dim=dim, page=page, ragged=rng.random() < 0.5, window=0, dtype="bfloat16")
    if kind == "decode":
        requests = _size(rng, 1, 64)
        case.update(requests=requests, rows=1, context=_size(rng, 1, 65536 // requests), window=rng.choice([0, 0, 0, 500, 4096]))
        case["dtype"] = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    elif kind == "prompt":
        requests = _size(rng, 1, 6)
        case.update(requests=requests, rows=_size(rng, 2, 2048 // requests), window=rng.choice([0, 0, 777]))
        case["context"] = case["rows"] + _size(rng, 1, 6144) - 1
        if case["rows"] * requests * case["context"] * heads * dim > 2048 * 4096 * 4096:
            case["context"] = case["rows"] + case["context"] % 1000
            case["heads"] = kv_heads
    else:
        requests = _size(rng, 1, 8)
        case.update(kind="tree", requests=requests, rows=_size(rng, 2, 64), store=rng.choice(["e4m3", "bfloat16"]))
        case["context"] = case["rows"] + _size(rng, 1, 16384 // requests) - 1
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------------------------
def _lengths(case):
    """(rows, keys before them) of every request, from the case alone: ragged ones take fractions of the largest, none less than a row."""
    n, rows, context = case["requests"], case.get("rows", 0), case["context"]
    out = []
    for i in range(n):
        part = ((i * 37 + 11) % n + 1) / n if case["ragged"] else 1.0
        r = max(1, round(rows * part)) if rows else 0
        part = ((i * 53 + 7) % n + 1) / n if case["ragged"] else 1.0
        total = max(r, 1, round(context * part))
        out.append((r, total - r))
    return out


def _exponents(x):
    """n of every row of x (float32, [..., D]): the smallest with max |x| <= 448 * 2^n, in LOWEST .. HIGHEST; 0 for zeros."""
    m, e = torch.frexp(x.abs().amax(-1))                     # max = m 2^e, m in 1/2 .. 1
    n = torch.where(m <= 0.875, e - 9, e - 8)
    return torch.where(m == 0, torch.zeros_like(n), n.clamp(LOWEST, HIGHEST))


def _quantized(x):
    """(codes float8_e4m3fn [..., D], exponents uint8 [...]) of x, computed in 32 bits."""
    x = x.float()
    n = _exponents(x)
    codes = torch.ldexp(x, -n.unsqueeze(-1)).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
    return codes, (n + 127).to(torch.uint8)


def _keys_values(gen, shape, dim):
    """Keys and values as layers leave them: some channels of a head much larger than others, tokens of different size."""
    def normal(*s):
        return torch.randn(*s, generator=gen, device=DEVICE)
    channels = torch.exp(0.7 * normal(dim))
    k = normal(*shape, dim) * channels
    v = normal(*shape, dim) * torch.exp(0.8 * normal(*shape, 1))
    return k, v


def _paged(case, gen, lengths):
    """Block tables of pages in no order, and what the pages hold (stale values in slots that no request uses)."""
    page = case["page"]
    need = [max(1, -(-n // page)) for n in lengths]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device=DEVICE).int()
    tables = torch.full((len(need), max(need)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for r, n in enumerate(need):
        tables[r, :n] = order[at:at + n]
        at += n
    k, v = _keys_values(gen, (pages, case["kv_heads"], page), case["dim"])
    return tables, torch.stack([k, v], dim=1)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    kind, g, dim, page = case["kind"], case["kv_heads"], case["dim"], case["page"]
    s = dict(case)
    if kind == "write":
        rows, heads = case["rows"], case["heads"]
        k, v = _keys_values(gen, (rows, g), dim)
        if heads:                                     # columns of a product [rows, queries | keys | values]
            q = torch.randn(rows, heads * dim, generator=gen, device=DEVICE)
            product = torch.cat([q, k.reshape(rows, -1), v.reshape(rows, -1)], dim=1).to(getattr(torch, case["dtype"]))
            k = product[:, heads * dim:(heads + g) * dim].view(rows, g, dim)
            v = product[:, (heads + g) * dim:].view(rows, g, dim)
        else:
            k, v = k.to(getattr(torch, case["dtype"])), v.to(getattr(torch, case["dtype"]))
        pages = -(-rows // page) + 1
        slots = torch.randperm(pages * page, generator=gen, device=DEVICE)[:rows].int()
        if rows > 4:
            slots[rows // 3] = -1                     # a row of padding
        s.update(k=k, v=v, slots=slots)
        s["codes"] = torch.zeros(pages, 2, g, page, dim, dtype=torch.float8_e4m3fn, device=DEVICE)
        s["exponents"] = torch.full((pages, 2, g, page), 127, dtype=torch.uint8, device=DEVICE)
        return s
    lengths = _lengths(case)
    tables, values = _paged(case, gen, [r + h for r, h in lengths])
    if case.get("store") == "bfloat16":
        s["store_bf16"] = values.bfloat16()
    else:
        s["codes"], s["exponents"] = _quantized(values)
    s["tables"] = tables
    if kind == "read":
        need = [max(1, -(-h // page)) for _, h in lengths]
        s["pages"] = torch.cat([tables[r, :n] for r, n in enumerate(need)])
        used = [min(page, h - page * i) for (_, h), n in zip(lengths, need) for i in range(n)]
        s["used"] = torch.tensor(used, dtype=torch.int32, device=DEVICE)
        s["out"] = torch.empty(len(used), 2, g, page, dim, dtype=getattr(torch, case["dtype"]), device=DEVICE)
        return s
    counts, histories = [r for r, _ in lengths], [h for _, h in lengths]
    starts = np.concatenate([[0], np.cumsum(counts)[:-1]])
    s["row_start"], s["row_count"], s["history"] = (torch.tensor(np.asarray(x), dtype=torch.int32, device=DEVICE) for x in (starts, counts, histories))
    s["max_rows"], s["max_context"] = max(counts), max(r + h for r, h in lengths)
    rows = sum(counts)
    s["q"] = (1.5 * torch.randn(rows, case["heads"] * dim, generator=gen, device=DEVICE)).to(getattr(torch, case["dtype"]))
    s["out"] = torch.empty_like(s["q"])
    s["scale"] = 1.0 / math.sqrt(dim)
    if kind == "tree":
        # Every drafted token continues an earlier one of its request or the history; it sees itself and what it continues.
        rng = np.random.RandomState(seed % (1 << 31))
        words = -(-s["max_rows"] // 32)
        bits = np.zeros((rows, words), dtype=np.uint32)
        for a, n in zip(starts, counts):
            for i in range(n):
                parent = rng.randint(-1, i)
                if parent >= 0:
                    bits[a + i] = bits[a + parent]
                bits[a + i, i // 32] |= np.uint32(1 << (i % 32))
        s["tree"] = torch.from_numpy(bits.view(np.int32)).to(DEVICE)
    return s


# ---- one pass -------------------------------------------------------------------------------------------------------------------
def _own(s):
    from llmx_b200 import ops
    kind = s["kind"]
    if kind == "write":
        cache = ops.QuantizedPages(s["codes"], s["exponents"])
        ops.quantize_kv(s["k"], s["v"], s["slots"], cache)
        return s["codes"], s["exponents"]
    if kind == "read":
        return ops.dequantize_pages(ops.QuantizedPages(s["codes"], s["exponents"]), s["pages"], s["out"], used=s["used"])
    cache = s["store_bf16"] if "store_bf16" in s else ops.QuantizedPages(s["codes"], s["exponents"])
    rows = (s["row_start"], s["row_count"], s["history"], s["tables"])
    if kind == "tree":
        return ops.attention_tree(s["q"], cache, s["out"], *rows, s["tree"], s["heads"], s["kv_heads"], s["dim"], s["scale"], s["max_rows"], s["max_context"])
    return ops.attention_quantized(s["q"], cache, s["out"], *rows, s["heads"], s["kv_heads"], s["dim"], s["window"] or None, s["scale"], s["max_rows"],
                                   s["max_context"])


def _values(codes, exponents):
    return torch.ldexp(codes.float(), exponents.int().unsqueeze(-1) - 127)


def _plain_attention(s):
    g, dim, page = s["kv_heads"], s["dim"], s["page"]
    ratio, requests, top = s["heads"] // g, s["row_count"].numel(), s["max_rows"]
    pages = s["tables"].clamp(min=0).long()
    kv = s["store_bf16"][pages].float() if "store_bf16" in s else _values(s["codes"].view(torch.uint8)[pages].view(torch.float8_e4m3fn), s["exponents"][pages])
    kv = kv.permute(2, 0, 3, 1, 4, 5).reshape(2, requests, g, -1, dim)          # [keys and values, requests, heads, places, D]
    place = torch.arange(kv.shape[3], device=DEVICE)
    row = torch.arange(top, device=DEVICE)
    real = row < s["row_count"][:, None]                                        # [requests, rows]
    index = torch.where(real, s["row_start"][:, None] + row, 0).long()
    position = s["history"][:, None] + row                                      # [requests, rows]
    if s["kind"] == "tree":
        j = place - s["history"][:, None]                                       # [requests, places]: which drafted token a key is of
        word = (j.clamp(0, 32 * s["tree"].shape[1] - 1) // 32)[:, None, :].expand(-1, top, -1).long()
        bit = (s["tree"][index].gather(2, word) >> (j.clamp(min=0) % 32)[:, None, :]) & 1
        seen = ((j < 0)[:, None, :] | (bit == 1)) & (j < s["row_count"][:, None])[:, None, :]
    else:
        seen = place <= position[:, :, None]
        if s["window"]:
            seen = seen & (place > position[:, :, None] - s["window"])
    q = s["q"].float().view(-1, g, ratio, dim)[index].permute(0, 2, 1, 3, 4).reshape(requests, g, top * ratio, dim)
    seen = seen.repeat_interleave(ratio, dim=1)[:, None]
    scores = torch.where(seen, torch.matmul(q, kv[0].transpose(-1, -2)) * s["scale"], -math.inf)
    peak = scores.amax(-1, keepdim=True)
    weights = torch.where(seen, torch.exp(scores - torch.where(peak == -math.inf, 0.0, peak)), 0.0)
    total = weights.sum(-1, keepdim=True)
    o = torch.matmul(weights, torch.where(seen.any(2)[..., None], kv[1], 0.0)) / torch.where(total == 0, 1.0, total)
    o = o.view(requests, g, top, ratio, dim).permute(0, 2, 1, 3, 4).reshape(requests, top, -1)
    s["out"][index[real]] = o[real].to(s["out"].dtype)
    return s["out"]


def run(s):
    if own:
        return _own(s)
    if s["kind"] == "write":
        kept = s["slots"] >= 0
        slots = s["slots"][kept].long()
        page, place = slots // s["page"], slots % s["page"]
        for plane, x in enumerate((s["k"], s["v"])):
            codes, exponents = _quantized(x[kept])
            s["codes"].view(torch.uint8)[page, plane, :, place] = codes.view(torch.uint8)
            s["exponents"][page, plane, :, place] = exponents
        return s["codes"], s["exponents"]
    if s["kind"] == "read":
        pages = s["pages"].long()
        values = _values(s["codes"].view(torch.uint8)[pages].view(torch.float8_e4m3fn), s["exponents"][pages])
        live = torch.arange(s["page"], device=DEVICE) < s["used"][:, None]
        s["out"].copy_(torch.where(live[:, None, None, :, None], values, 0.0))
        return s["out"]
    return _plain_attention(s)


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def work(case):
    g, dim = case["kv_heads"], case["dim"]
    row = 2 * g * (dim + 1)                              # a token's codes and exponents
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] == "write":
        return {"bytes": case["rows"] * (2 * g * dim * size + 4 + row), "flops": case["rows"] * 2 * g * dim * 3}
    lengths = _lengths(case)
    if case["kind"] == "read":
        tokens = sum(h for _, h in lengths)
        pages = sum(max(1, -(-h // case["page"])) for _, h in lengths)
        return {"bytes": tokens * row + pages * (case["page"] * 2 * g * dim * size + 8), "flops": tokens * 2 * g * dim}
    if case.get("store") == "bfloat16":
        row = 2 * g * dim * 2
    keys = pairs = 0
    for r, h in lengths:
        w = case["window"] or r + h
        keys += min(r + h, w + r - 1)
        pairs += sum(min(w, h + i + 1) for i in range(r))
    rows = sum(r for r, _ in lengths)
    return {"bytes": keys * row + 2 * rows * case["heads"] * dim * size, "flops": pairs * case["heads"] * dim * 4}


# ---- the same in 64 bits ------------------------------------------------------------------------------------------------------------
def _decoded(code):
    """float64 values of codes: a sign, four bits of exponent (bias 7; 0: no leading one), three of mantissa."""
    c = code.view(torch.uint8).long()
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e == 0, m * 2.0 ** -9, (8.0 + m) * torch.pow(torch.tensor(2.0, dtype=torch.float64, device=c.device), (e - 10).double()))
    return torch.where(c >= 128, -v, v)


def _power(exponents):
    return torch.pow(torch.tensor(2.0, dtype=torch.float64, device=exponents.device), exponents.double() - 127.0)


def _nearest(x):
    """The nearest value that eight bits hold, ties to even, of x in -448 .. 448 (float64): steps of 2^-9 below 2^-6, then eight to
    each power of two."""
    a = x.abs()
    step = torch.pow(torch.tensor(2.0, dtype=torch.float64, device=x.device), torch.floor(torch.log2(a.clamp(min=2.0 ** -6))) - 3.0)
    return torch.sign(x) * torch.round(a / step) * step        # round() takes ties to even


def exact(case, seed):
    s = prepare(case, seed)
    g, dim, page = case["kv_heads"], case["dim"], case["page"]
    if case["kind"] == "write":
        values = torch.zeros(s["codes"].shape, dtype=torch.float64, device=DEVICE)
        slots = s["slots"].tolist()
        rows = [i for i, x in enumerate(slots) if x >= 0]
        where = torch.tensor([slots[i] for i in rows], device=DEVICE)
        for plane, x in enumerate((s["k"], s["v"])):
            x = x[rows].double()
            peak = x.abs().amax(-1, keepdim=True)
            n = torch.ceil(torch.log2(peak.clamp(min=1e-300) / 448.0) - 1e-10).clamp(LOWEST, HIGHEST)      # powers of two as themselves
            values.transpose(2, 3)[where // page, plane, where % page] = torch.where(peak > 0, _nearest(x * torch.exp2(-n)), 0.0)
        return values, None
    if case["kind"] == "read":
        out = torch.zeros(s["out"].shape, dtype=torch.float64, device=DEVICE)
        for i, (p, n) in enumerate(zip(s["pages"].tolist(), s["used"].tolist())):
            out[i, :, :, :n] = _decoded(s["codes"][p, :, :, :n]) * _power(s["exponents"][p, :, :, :n])[..., None]
        return out
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEVICE)
    at, heads = 0, case["heads"]
    for r, (n, h) in enumerate(_lengths(case)):
        at, first = at + n, at
        slots = torch.arange(h + n, device=DEVICE)
        page_of = s["tables"][r].long()[slots // page]
        for plane_head in range(g):
            if "store_bf16" in s:
                k, v = (s["store_bf16"][page_of, plane, plane_head, slots % page].double() for plane in (0, 1))
            else:
                k, v = (_decoded(s["codes"].view(torch.uint8)[page_of, plane, plane_head, slots % page])
                        * _power(s["exponents"][page_of, plane, plane_head, slots % page])[:, None] for plane in (0, 1))
            allowed = slots[None, :] <= h + torch.arange(n, device=DEVICE)[:, None]
            if case["window"]:
                allowed &= slots[None, :] + case["window"] > h + torch.arange(n, device=DEVICE)[:, None]
            if case["kind"] == "tree":
                words = s["tree"][first:at].cpu().numpy().view(np.uint32)
                drafted = np.array([[(words[i, j // 32] >> (j % 32)) & 1 for j in range(n)] for i in range(n)], dtype=bool)
                allowed[:, h:] = torch.from_numpy(drafted).to(DEVICE)
            for head in range(plane_head * (heads // g), (plane_head + 1) * (heads // g)):
                x = s["q"][first:at, head * dim:(head + 1) * dim].double()
                weights = torch.softmax((x @ k.T * s["scale"]).masked_fill(~allowed, -math.inf), dim=-1)
                out[first:at, head * dim:(head + 1) * dim] = weights @ v
    return out
