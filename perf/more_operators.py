"""The operators of a key and value cache held in MX formats, as timed cases: rows quantized as they are written, read
back as values, and the attention that reads the cache, for single tokens and for prompts.

A case is a dict of plain values.  `prepare` makes what a program holds before the call: the cache's bytes, the pages of
each sequence, rows to write or queries.  `run` makes one pass, through the package's entry points where `own` is true and
in elementary torch operations otherwise.  `exact` gives the 64-bit values from the definitions.

The cache is paged: codes pages x heads x page x bytes and E8M0 scales pages x heads x page x blocks, of keys and of
values.  A row is a head's vector in blocks of 32 columns, the last filled up with zeros; MXFP4 has two codes to a byte,
the even column in the low nibble.  Slot s is row s % page of page s / page.  A block's scale is the OCP one,
2^(floor(log2 amax) - emax), its elements go to the nearest, ties to even, saturated.
"""
import math
import os
import sys

import torch

sys.path.insert(0, os.path.join(os.getcwd(), "microscaling-quant_amd"))

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
# exponent bits, mantissa bits, largest exponent, largest code without its sign
FORMATS = {"MXFP8_E4M3": (4, 3, 8, 0x7E), "MXFP8_E5M2": (5, 2, 15, 0x7B), "MXFP4": (2, 1, 2, 0x7)}
BLOCK = 32


def listed():
    return [
        # a step of generation: one new row a sequence, written and read back; latency
        dict(name="write_step", kind="write", rows=64, heads=8, dim=128, page=16, fmt="MXFP4", dtype="bf16",
             padding=0.0),
        # a long prompt's rows
        dict(name="write_prompt", kind="write", rows=16384, heads=8, dim=128, page=64, fmt="MXFP8_E4M3", dtype="bf16",
             padding=0.0),
        # ragged sizes in float32, some rows padding without a slot
        dict(name="write_ragged", kind="write", rows=1021, heads=5, dim=80, page=16, fmt="MXFP4", dtype="f32",
             padding=0.1),
        # a shared prefix read back for a model that takes values
        dict(name="read_prefix", kind="read", rows=65536, heads=8, dim=128, page=32, fmt="MXFP4", dtype="bf16",
             padding=0.0),
        # a few rows of odd sizes
        dict(name="read_ragged", kind="read", rows=777, heads=3, dim=100, page=24, fmt="MXFP8_E5M2", dtype="f16",
             padding=0.05),
        # one token of one sequence, a head of keys for each of queries: latency
        dict(name="attend_one", kind="attend", seqs=1, tokens=1, ragged=False, context=1000, shortest=1.0, heads=16,
             kv_heads=16, dim=64, page=16, window=0, fmt="MXFP8_E4M3", dtype="bf16"),
        # a batch of generated tokens, contexts of unlike lengths: reading the cache
        dict(name="attend_decode", kind="attend", seqs=64, tokens=1, ragged=False, context=8192, shortest=0.5,
             heads=32, kv_heads=8, dim=128, page=16, window=0, fmt="MXFP4", dtype="bf16"),
        # one token at the end of a very long context
        dict(name="attend_long", kind="attend", seqs=1, tokens=1, ragged=False, context=131072, shortest=1.0, heads=64,
             kv_heads=8, dim=128, page=64, window=0, fmt="MXFP4", dtype="bf16"),
        # a few proposed tokens of each sequence looked at together, large heads, float16
        dict(name="attend_verify", kind="attend", seqs=12, tokens=4, ragged=False, context=4099, shortest=0.3,
             heads=16, kv_heads=2, dim=256, page=32, window=0, fmt="MXFP8_E5M2", dtype="f16"),
        # a long prompt against itself: the matrix cores' rate
        dict(name="attend_prompt", kind="attend", seqs=1, tokens=8192, ragged=False, context=8192, shortest=1.0,
             heads=32, kv_heads=8, dim=128, page=64, window=0, fmt="MXFP8_E4M3", dtype="bf16"),
        # prompts' pieces and single tokens in one batch, a window of positions, seven queries' heads to one of keys
        dict(name="attend_mixed", kind="attend", seqs=23, tokens=512, ragged=True, context=6001, shortest=0.1,
             heads=28, kv_heads=4, dim=80, page=16, window=2048, fmt="MXFP4", dtype="bf16"),
        # float32 queries on short contexts of odd lengths
        dict(name="attend_f32", kind="attend", seqs=5, tokens=67, ragged=True, context=531, shortest=0.2, heads=6,
             kv_heads=2, dim=96, page=48, window=0, fmt="MXFP4", dtype="f32"),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], its logarithm uniform."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    kind = rng.choice(("write", "read", "attend", "attend", "attend"))
    case = dict(kind=kind, fmt=rng.choice(tuple(FORMATS)), dtype=rng.choice(("bf16", "bf16", "f16", "f32")),
                page=rng.choice((1, 7, 16, 16, 32, 48, 64, 256)),
                dim=rng.choice((64, 80, 96, 128, 128, 192, 256, rng.randint(8, 256))))
    if kind != "attend":
        heads = _spread(rng, 1, 32)
        most = (2 ** 25 if kind == "write" else 2 ** 27) // (heads * case["dim"] * DTYPES[case["dtype"]].itemsize)
        return dict(case, heads=heads, rows=_spread(rng, 1, min(65536, most)), padding=rng.choice((0.0, 0.0, 0.1)))
    kv_heads = _spread(rng, 1, 16)
    heads = kv_heads * rng.choice((1, 2, 4, 4, 7, 8, 16))
    tokens = 1 if rng.random() < 0.4 else _spread(rng, 2, 2048)
    seqs = _spread(rng, 1, 64 if tokens < 64 else 8)
    tokens = min(tokens, max(1, 2 ** 25 // (seqs * heads * case["dim"])))
    context = _spread(rng, 1, 32768)
    context = min(context, 2 ** 27 // (seqs * kv_heads * case["dim"]), 2 ** 29 // (seqs * tokens * heads))
    return dict(case, seqs=seqs, tokens=min(tokens, context), ragged=rng.random() < 0.5, context=context,
                shortest=rng.choice((1.0, 0.5, 0.0)), heads=heads, kv_heads=kv_heads,
                window=rng.choice((0, 0, _spread(rng, 1, 4096))))


def _shape(case):
    """Lengths and numbers of queries of a case's sequences, before they are shuffled: spread evenly from the longest on."""
    S, n = case["seqs"], case["tokens"]
    part = [i / max(S - 1, 1) for i in range(S)]
    lengths = [round(case["context"] * (1 - p * (1 - case["shortest"]))) for p in part]
    if case["ragged"]:
        tokens = [max(1, round(n * (1 - p) ** 3)) for p in part[::-1]]
    else:
        tokens = [n] * S
    # a sequence may be shorter than its queries, the first of which then see nothing
    return lengths, tokens


# ------------------------------------------------------------------------------------------------ inputs

def _power(k, dtype=torch.float32):
    """2^k of whole numbers k that are exponents of normal values, by the fields: a library's power may be a unit off."""
    if dtype == torch.float64:
        return (k.long() + 1023 << 52).view(dtype)
    return (k.int() + 127 << 23).view(dtype)


def _quantized(x, fmt):
    """x (..., D) as code bytes (..., bytes) and scale bytes (..., blocks)."""
    e, m, emax, top = FORMATS[fmt]
    D = x.shape[-1]
    x = torch.nn.functional.pad(x.float(), (0, -D % BLOCK)).unflatten(-1, (-1, BLOCK))
    amax = x.abs().amax(-1, keepdim=True)
    power = torch.log2(torch.where(amax > 0, amax, 2.0 ** -126).double()).float().floor() - emax
    power = power.clamp_min(-127).int()
    x = x * _power(-power)
    low = 2 - 2 ** (e - 1)                                                            # the smallest normal's exponent
    exponent = torch.frexp(x.abs().clamp_min(2.0 ** low)).exponent - 1
    code = ((exponent - low) << m) + (x.abs() * _power(m - exponent)).round().int()
    code = (code.clamp_max(top) | (x < 0).int() << (e + m)).to(torch.uint8).flatten(-2)
    if fmt == "MXFP4":
        code = code[..., 0::2] | code[..., 1::2] << 4
    return code.contiguous(), (power.squeeze(-1) + 127).to(torch.uint8).contiguous()


def _tables(fmt):
    """The values of the 256 code bytes (of MXFP4, of both nibbles), float32."""
    e, m, _, _ = FORMATS[fmt]
    bias = 2 ** (e - 1) - 1

    def value(code):
        exponent, fraction = code >> m & (2 ** e - 1), code & (2 ** m - 1)
        whole = (1 + fraction / 2 ** m) * 2.0 ** (exponent - bias) if exponent else fraction / 2 ** m * 2.0 ** (1 - bias)
        return -whole if code >> (e + m) & 1 else whole

    if fmt == "MXFP4":
        return torch.tensor([[value(b & 15), value(b >> 4)] for b in range(256)], device="cuda")
    return torch.tensor([value(b) for b in range(256)], device="cuda")


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)

    def normal(*shape, dtype=torch.float32):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    def rows(n, heads, dtype=torch.float32):
        """A head's vectors: some columns larger than others, rows of unlike size."""
        size = torch.exp(0.6 * normal(heads, D)) * torch.exp(0.3 * normal(n, heads, 1))
        return (normal(n, heads, D) * size).to(dtype)

    dtype, fmt, D, page = DTYPES[case["dtype"]], case["fmt"], case["dim"], case["page"]
    kv_heads = case["kv_heads"] if case["kind"] == "attend" else case["heads"]
    state = dict(case=case, tables=_tables(fmt))
    if case["kind"] == "attend":
        lengths, tokens = _shape(case)
        order = torch.randperm(case["seqs"], generator=gen, device="cuda").tolist()
        lengths, tokens = [lengths[i] for i in order], [tokens[i] for i in order]
        need = [-(-l // page) for l in lengths]
        pages, width = sum(need) + 3, max(max(need), 1) + 2                            # tables have room left
    else:
        pages = -(-case["rows"] // page) + 3
    cache = []
    for _ in range(2):                                                                # keys, then values
        filled = rows(pages * page, kv_heads) if case["kind"] != "write" else normal(pages * page, kv_heads, D)
        for part in _quantized(filled, fmt):
            cache.append(part.unflatten(0, (pages, page)).transpose(1, 2).contiguous())
    state["cache"] = cache
    if case["kind"] != "attend":
        n = case["rows"]
        slots = torch.randperm(pages, generator=gen, device="cuda")[:, None] * page + torch.arange(page, device="cuda")
        slots = slots.flatten()[:n].int()
        if case["padding"]:
            slots[torch.rand(n, generator=gen, device="cuda") < case["padding"]] = -1
        state["slots"] = slots
        if case["kind"] == "write":
            state["k"], state["v"] = rows(n, kv_heads, dtype), rows(n, kv_heads, dtype)
        return state
    shuffled = torch.randperm(pages, generator=gen, device="cuda").int()
    table = torch.full((len(need), width), -1, dtype=torch.int32, device="cuda")
    first = 0
    for b, k in enumerate(need):
        table[b, :k] = shuffled[first:first + k]
        first += k
    state["table"], state["lengths"] = table, torch.tensor(lengths, dtype=torch.int32, device="cuda")
    total = sum(tokens)
    q = normal(total, case["heads"], D, dtype=dtype)
    if case["ragged"]:
        state["q"] = q
        state["starts"] = torch.tensor([0] + tokens, device="cuda").cumsum(0).int()
        state["most"] = max(tokens)
    else:
        state["q"] = q.unflatten(0, (case["seqs"], case["tokens"]))
    return state


# ------------------------------------------------------------------------------------------- plain forms

def _plain_values(codes, scales, table, D):
    values = table[codes.int()]
    if values.ndim > codes.ndim:
        values = values.flatten(-2)
    spread = _power(scales.int() - 127, torch.float64).float().repeat_interleave(BLOCK, -1)
    return (values * spread)[..., :D]


def _plain_read(s):
    c = s["case"]
    slots = s["slots"].long()
    there = slots >= 0
    page, at = slots.clamp_min(0) // c["page"], slots.clamp_min(0) % c["page"]
    out = []
    for codes, scales in (s["cache"][:2], s["cache"][2:]):
        values = _plain_values(codes[page, :, at], scales[page, :, at], s["tables"], c["dim"])
        out.append(torch.where(there[:, None, None], values, 0.0).to(DTYPES[c["dtype"]]))
    return out


def _plain_write(s):
    slots = s["slots"].long()
    there = slots >= 0
    kept = slots[there]
    page, at = kept // s["case"]["page"], kept % s["case"]["page"]
    for x, codes, scales in ((s["k"], *s["cache"][:2]), (s["v"], *s["cache"][2:])):
        c, f = _quantized(x[there], s["case"]["fmt"])
        codes[page, :, at] = c
        scales[page, :, at] = f
    return _plain_read(s)


def _plain_attend(s):
    """Every sequence filled up to the longest, its queries too, in one batched product."""
    c = s["case"]
    D, H, G = c["dim"], c["heads"], c["kv_heads"]
    q, lengths = s["q"].float(), s["lengths"].long()
    S, dev = len(lengths), q.device
    if c["ragged"]:
        n = s["most"]
        starts = s["starts"].long()
        count = starts.diff()
        row = starts[:-1, None] + torch.arange(n, device=dev)
        mine = torch.arange(n, device=dev) < count[:, None]
        q = q[row.clamp_max(len(q) - 1)]
    else:
        n = c["tokens"]
        count = torch.full((S,), n, device=dev)
    q = q.unflatten(2, (G, H // G)).permute(0, 2, 3, 1, 4).flatten(2, 3)              # S x G x (heads of a group, n) x D
    pages = s["table"].long().clamp_min(0)
    k, v = (_plain_values(codes[pages].transpose(1, 2).flatten(2, 3), scales[pages].transpose(1, 2).flatten(2, 3),
                          s["tables"], D) for codes, scales in (s["cache"][:2], s["cache"][2:]))
    L = k.shape[2]
    position = lengths[:, None] - count[:, None] + torch.arange(n, device=dev)        # S x n
    key = torch.arange(L, device=dev)
    seen = key <= position[..., None]
    if c["window"]:
        seen &= key > position[..., None] - c["window"]
    seen = seen & (key < lengths[:, None, None])
    scores = torch.matmul(q, k.transpose(2, 3)).mul_(D ** -0.5).unflatten(2, (H // G, n))
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top > -math.inf, top, 0.0)
    scores.sub_(top).exp_()
    total = scores.sum(-1, keepdim=True)
    out = torch.matmul(scores.flatten(2, 3), v).unflatten(2, (H // G, n))
    out = (out / torch.where(total > 0, total, 1.0)).permute(0, 3, 1, 2, 4).flatten(2, 3)    # S x n x H x D
    lse = (top + total.log())[..., 0].permute(0, 3, 1, 2).flatten(2, 3)
    if c["ragged"]:
        out, lse = out[mine], lse[mine]
    return [out.to(s["q"].dtype), lse]


# --------------------------------------------------------------------------------------------- own calls

def _own(s):
    from mxq import nn
    c = s["case"]
    cache = nn.PackedCache(*s["cache"], c["fmt"], c["dim"])
    if c["kind"] == "attend":
        return list(nn.cache_attend(s["q"], cache, s["table"], s["lengths"], s.get("starts"),
                                    window=c["window"] or None, return_lse=True))
    if c["kind"] == "write":
        nn.cache_write(s["k"], s["v"], cache, s["slots"])
    return list(nn.cache_read(cache, s["slots"], DTYPES[c["dtype"]]))


def run(state):
    if own:
        return _own(state)
    return {"write": _plain_write, "read": _plain_read, "attend": _plain_attend}[state["case"]["kind"]](state)


# -------------------------------------------------------------------------------------------------- work

def _row_bytes(case):
    blocks = -(-case["dim"] // BLOCK)
    return blocks * (17 if case["fmt"] == "MXFP4" else 33)


def work(case):
    """Bytes read and written once and the operations of the definition: of attention, the rows that some query sees and
    the pairs of a query and a key that it sees."""
    size, D = DTYPES[case["dtype"]].itemsize, case["dim"]
    if case["kind"] != "attend":
        rows = case["rows"] * (1 - case["padding"]) * case["heads"] * 2
        moved = rows * _row_bytes(case) + case["rows"] * (case["heads"] * 2 * D * size + 4)
        if case["kind"] == "write":                                                   # written, and read back
            moved += rows * (_row_bytes(case) + D * size)
        return {"bytes": int(moved), "flops": int(rows * D * (4 if case["kind"] == "write" else 1))}
    pairs = keys = queries = 0
    for length, n in zip(*_shape(case)):
        window = case["window"] or length + n
        # the j-th of n queries is at length - n + j and sees the window that ends there
        ends = [max(0, length - n + 1), length]
        first, last = min(ends[0], window), min(ends[1], window)
        ramp = last - first                                                           # queries that see one more each
        pairs += (first + last) * (ramp + 1) // 2 + last * max(0, ends[1] - ends[0] - ramp)
        keys += min(length, window + n - 1)
        queries += n
    H = case["heads"]
    moved = keys * case["kv_heads"] * 2 * _row_bytes(case) + queries * H * (2 * D * size + 4)
    return {"bytes": int(moved), "flops": int(4 * pairs * H * D)}


# ------------------------------------------------------------------------------------------------- exact

def _exact_values(codes, scales, fmt, D):
    """Code and scale bytes (..., bytes), (..., blocks) to float64 by their fields."""
    e, m, _, _ = FORMATS[fmt]
    if fmt == "MXFP4":
        codes = torch.stack((codes & 15, codes >> 4), -1).flatten(-2)
    exponent = (codes >> m & (2 ** e - 1)).int()
    fraction = (codes & (2 ** m - 1)).double() + (exponent > 0) * 2 ** m
    value = fraction * _power(exponent.clamp_min(1) - (2 ** (e - 1) - 1) - m, torch.float64)
    value = torch.where((codes >> (e + m) & 1).bool(), -value, value)
    return (value * _power(scales.int() - 127, torch.float64).repeat_interleave(BLOCK, -1))[..., :D]


def _exact_rounded(x, fmt):
    """x (n, heads, D) as the values that its blocks are quantized to."""
    e, m, emax, _ = FORMATS[fmt]
    D, largest = x.shape[-1], {"MXFP8_E4M3": 448.0, "MXFP8_E5M2": 57344.0, "MXFP4": 6.0}[fmt]
    out = torch.empty_like(x, dtype=torch.float64)
    for first in range(0, D, BLOCK):
        part = x[..., first:first + BLOCK].double()
        amax = part.abs().amax(-1, keepdim=True).clamp_min(2.0 ** -126)
        # the logarithm rounded to float32, as the quantizers of this package take it
        scale = _power((torch.log2(amax).to(torch.float32).floor() - emax).clamp_min(-127.0), torch.float64)
        z = (part / scale).clamp(-largest, largest)
        binade = torch.frexp(z.abs().clamp_min(2.0 ** (2 - 2 ** (e - 1)))).exponent - 1
        step = _power(binade - m, torch.float64)
        out[..., first:first + BLOCK] = torch.round(z / step) * step * scale
    return out


def exact(case, seed):
    s = prepare(case, seed)
    D, fmt, page = case["dim"], case["fmt"], case["page"]
    if case["kind"] == "write":
        there = (s["slots"] >= 0)[:, None, None]
        return [_exact_rounded(x, fmt) * there for x in (s["k"], s["v"])]
    if case["kind"] == "read":
        out = []
        for codes, scales in (s["cache"][:2], s["cache"][2:]):
            rows = [part.transpose(1, 2).flatten(0, 1)[s["slots"].clamp_min(0).long()] for part in (codes, scales)]
            out.append(_exact_values(*rows, fmt, D) * (s["slots"] >= 0)[:, None, None])
        return out
    q = s["q"].double()
    lengths = s["lengths"].tolist()
    flat = q.reshape(-1, case["heads"], D)
    starts = s["starts"].tolist() if case["ragged"] else [i * case["tokens"] for i in range(len(lengths) + 1)]
    out = torch.zeros(flat.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(flat.shape[:2], -math.inf, dtype=torch.float64, device="cuda")
    per = case["heads"] // case["kv_heads"]
    for b, length in enumerate(lengths):
        low, high = starts[b], starts[b + 1]
        if not length:
            continue
        at = torch.arange(length, device="cuda")
        slot = s["table"][b].long()[at // page] * page + at % page
        place = length - (high - low) + torch.arange(high - low, device="cuda")
        hidden = at[None] > place[:, None]
        if case["window"]:
            hidden |= at[None] <= place[:, None] - case["window"]
        for g in range(case["kv_heads"]):
            k, v = (_exact_values(codes[:, g].flatten(0, 1)[slot], scales[:, g].flatten(0, 1)[slot], fmt, D)
                    for codes, scales in (s["cache"][:2], s["cache"][2:]))
            for h in range(g * per, (g + 1) * per):
                z = (flat[low:high, h] @ k.t()) / math.sqrt(D)
                z.masked_fill_(hidden, -math.inf)
                total = torch.logsumexp(z, -1)
                lse[low:high, h] = total
                weights = torch.exp(z - total.masked_fill(total == -math.inf, 0.0)[:, None])
                out[low:high, h] = weights @ v
    return [out.reshape(q.shape), lse.reshape(q.shape[:-1])]
