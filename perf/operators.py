"""Performance cases of the paged key-value cache as a host with layers of its own uses it, next to the quantized GEMM
and the acceptance stage: writing new rows in the cache's format, reading rows back, and the attention of one new
token per sequence over the cache.

`listed()` names the regimes, `draw()` gives more of the same ranges:

  attend  attention_decode: one new token per sequence, grouped query heads, lengths on the device, any cache format
  write   kv_write: K and V rows of new tokens, quantised on their way into the pool
  read    kv_read: K and V rows of cached tokens as plain numbers

With `own` false the same results come from elementary torch operations in 32 bits; `exact()` computes them in 64.

Cache rows, all heads of a token behind one another (H heads of D values):
  f32, f16   the values; f16 rounds half up on the dropped bits
  q8_0       blocks of 32: f16 scale amax / 127 (rounded like f16 rows), 32 int8 round(x / scale)
  f8         H * D E4M3 values x * (448 / amax), then H f32 scales amax / 448 (amax over a head), padded to 16 bytes
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
FORMATS = {"f32": 0, "f16": 1, "q8_0": 2, "f8": 3}


# --------------------------------------------------------------------------- cases

def _attend(name, batch, lo, hi, fmt, heads, kv_heads, head_dim, dtype, block=16, window=0, gate=False, idle=0):
    """`lo`..`hi`: lengths of the sequences, `idle`: slots of the batch without a sequence (length zero)."""
    case = {"kind": "attend", "batch": batch, "lo": lo, "hi": hi, "format": fmt, "heads": heads, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "block": block, "window": window, "gate": gate, "idle": idle}
    return dict(case, name=name) if name else case


def _move(kind, name, rows, sequences, context, fmt, kv_heads, head_dim, dtype, block=16, padding=0):
    """`rows` tokens of `sequences` sequences that hold `context` others already, `padding` rows that name no token."""
    case = {"kind": kind, "rows": rows, "sequences": sequences, "context": context, "format": fmt, "kv_heads": kv_heads,
            "head_dim": head_dim, "dtype": dtype, "block": block, "padding": padding}
    return dict(case, name=name) if name else case


def listed():
    return [
        # a draft model or a test: one short sequence, latency is all of it
        _attend("attend 1x97 f16", 1, 97, 97, "f16", 4, 2, 64, "f32"),
        # plain decode behind a conversation, the 4B model's heads, activations as the library's GEMMs give them
        _attend("attend 1x1500 f16 gate", 1, 1500, 1500, "f16", 16, 4, 256, "f32", gate=True),
        # one long document, the mixture model's heads, a quantized cache
        _attend("attend 1x16000 q8_0", 1, 16000, 16000, "q8_0", 16, 2, 256, "f32", gate=True),
        # a full server with contexts of all lengths, two idle slots
        _attend("attend 32x256-4000 f16", 32, 256, 4000, "f16", 16, 4, 256, "bf16", gate=True, idle=2),
        # many users on an 8-bit cache
        _attend("attend 64x500-8000 f8", 64, 500, 8000, "f8", 32, 8, 128, "bf16", block=32),
        # long contexts on every slot: the largest
        _attend("attend 8x32768 f16", 8, 32768, 32768, "f16", 32, 8, 128, "bf16", block=64),
        # every head its own keys, unrounded cache, a sliding window, pages of an odd size
        _attend("attend 16x200-6000 f32 window", 16, 200, 6000, "f32", 12, 12, 64, "f32", block=24, window=1000),
        # the new token of one decode step
        _move("write", "write 1 f16", 1, 1, 700, "f16", 4, 256, "f32"),
        # a prompt of no round length into a quantized cache, the batch padded
        _move("write", "write 1837 q8_0", 1837, 1, 0, "q8_0", 4, 256, "f32", padding=11),
        # prompts of several requests at once into an 8-bit cache
        _move("write", "write 30000 f8", 30000, 9, 100, "f8", 8, 128, "bf16", block=32),
        # a prefix of a conversation taken out of the cache
        _move("read", "read 700 q8_0", 700, 1, 20, "q8_0", 4, 256, "f32"),
        # whole contexts moved off an 8-bit cache
        _move("read", "read 30000 f8", 30000, 5, 0, "f8", 8, 128, "bf16", block=32),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "write", "read"])
    fmt, dtype = rng.choice(["f16", "f16", "q8_0", "f8", "f32"]), rng.choice(["f32", "f16", "bf16"])
    head_dim, block = rng.choice([64, 128, 128, 256, 256]), rng.choice([16, 16, 32, 64, rng.randint(1, 100)])
    kv_heads = _log(rng, 1, 16)
    if kind == "attend":
        group = rng.choice([1, 2, 4, 4, 8, rng.randint(1, 20)])
        # keys of all sequences together: at most as many bytes as the largest listed case reads
        most = max(64, int((1 << 29) / (kv_heads * head_dim * {"f32": 4, "f16": 2, "q8_0": 1.0625, "f8": 1.04}[fmt])))
        most = min(most, int(2e10 / (2.0 * kv_heads * head_dim * max(group, 4))))
        batch = _log(rng, 1, 96)
        hi = min(_log(rng, 1, 32768), max(1, most // batch))
        lo = hi if batch == 1 else _log(rng, max(1, hi // 20), hi)
        window = rng.choice([0, 0, 0, _log(rng, 1, hi)])
        return _attend(None, batch, lo, hi, fmt, group * kv_heads, kv_heads, head_dim, dtype, block, window,
                       rng.random() < 0.4, rng.choice([0, 0, batch // 8]))
    rows = _log(rng, 1, 30000)
    rows = min(rows, max(1, 30000 * 1024 // (kv_heads * head_dim)))
    return _move(kind, None, rows, _log(rng, 1, min(rows, 40)), rng.choice([0, _log(rng, 1, 500)]), fmt, kv_heads, head_dim,
                 dtype, block, rng.choice([0, rng.randint(1, 16)]))


def _lengths(case):
    """Lengths of an attend case: spread evenly over the logarithm between the shortest and the longest, the idle slots at zero."""
    n, lo, hi = case["batch"], case["lo"], case["hi"]
    live = n - case["idle"]
    lens = [int(round(lo * (hi / lo) ** (i / max(1, live - 1)))) if live > 1 else hi for i in range(live)] + [0] * case["idle"]
    return [lens[(i * 7 + 3) % n] for i in range(n)] if n % 7 else lens


def _visible(case):
    return [min(n, case["window"]) if case["window"] else n for n in _lengths(case)]


def row_bytes(fmt, heads, dim):
    n = heads * dim
    return {"f32": 4 * n, "f16": 2 * n, "q8_0": n // 32 * 34, "f8": (n + 4 * heads + 15) // 16 * 16}[fmt]


def _payload(fmt, heads, dim):
    """Bytes of a row without its padding."""
    return heads * dim + 4 * heads if fmt == "f8" else row_bytes(fmt, heads, dim)


def work(case):
    h, d, size = case["kv_heads"], case["head_dim"], {"f32": 4, "f16": 2, "bf16": 2}[case["dtype"]]
    row = _payload(case["format"], h, d)
    if case["kind"] == "attend":
        seen = sum(_visible(case))
        io = case["batch"] * case["heads"] * d * size * (3 if case["gate"] else 2)
        pages = sum(-(-n // case["block"]) for n in _visible(case))
        return {"bytes": 2 * seen * row + io + 4 * pages + 4 * case["batch"] * (1 + case["heads"]), "flops": 4 * seen * case["heads"] * d}
    return {"bytes": case["rows"] * (2 * row + 2 * h * d * size + 8), "flops": 0}


# --------------------------------------------------------------------------- the formats in torch

def _half_up(x):
    """f32 -> the bits of f16, rounding half up on the dropped bits."""
    b = x.contiguous().view(torch.int32)
    sign, e, m = (b >> 16) & 0x8000, ((b >> 23) & 0xff) - 127, b & 0x7fffff
    normal = torch.clamp(((e + 15) << 10) + ((m + 0x1000) >> 13), max=0x7c00)
    shift = torch.clamp(-e - 14, 0, 11)
    one = torch.ones_like(shift)
    small = ((m | 0x800000) + torch.bitwise_left_shift(one, shift + 12)) >> (shift + 13)
    h = torch.where(e < -24, torch.zeros_like(b), torch.where(e < -14, small, normal))
    h = torch.where(e == 128, torch.where(m != 0, 0x7e00, 0x7c00).to(torch.int32), h)
    return (h | sign).to(torch.int16)


def _encode(x, fmt):
    """Rows [n, heads, dim] in f32 as cache rows, uint8 [n, row bytes]."""
    n, h, d = x.shape
    if fmt == "f32":
        return x.reshape(n, h * d).contiguous().view(torch.uint8)
    if fmt == "f16":
        return _half_up(x.reshape(n, h * d)).view(torch.uint8)
    if fmt == "q8_0":
        blocks = x.reshape(n, h * d // 32, 32)
        scale = blocks.abs().amax(-1, keepdim=True) / 127.0
        y = (blocks / torch.where(scale == 0, 1.0, scale)).double()
        q = (torch.floor(y.abs() + 0.5) * torch.sign(y)).to(torch.int8)
        s = _half_up(scale).view(torch.uint8).reshape(n, -1, 2)
        return torch.cat([s, q.view(torch.uint8)], -1).reshape(n, -1)
    amax = x.abs().amax(-1, keepdim=True)
    y = torch.clamp(x * torch.where(amax == 0, 0.0, 448.0 / torch.where(amax == 0, 1.0, amax)), -448.0, 448.0)
    q = y.to(torch.float8_e4m3fn).view(torch.uint8).reshape(n, h * d)
    s = (amax / 448.0).reshape(n, h).contiguous().view(torch.uint8)
    pad = torch.zeros(n, row_bytes(fmt, h, d) - h * d - 4 * h, dtype=torch.uint8, device=x.device)
    return torch.cat([q, s, pad], -1)


def _decode(rows, fmt, h, d):
    """Cache rows, uint8 [..., row bytes], as f32 [..., heads, dim]."""
    at = rows.shape[:-1]
    if fmt == "f32":
        return rows.view(torch.float32).reshape(*at, h, d)
    if fmt == "f16":
        return rows.view(torch.float16).float().reshape(*at, h, d)
    if fmt == "q8_0":
        b = rows.reshape(*at, h * d // 32, 34)
        s = b[..., :2].contiguous().view(torch.float16).float()
        return (s * b[..., 2:].contiguous().view(torch.int8).float()).reshape(*at, h, d)
    q = rows[..., : h * d].contiguous().view(torch.float8_e4m3fn).float().reshape(*at, h, d)
    return q * rows[..., h * d: h * d + 4 * h].contiguous().view(torch.float32).reshape(*at, h, 1)


def _values(pool, fmt, h, d):
    """What a pool stands for, without work: its numbers and scales where they lie."""
    if fmt in ("f32", "f16"):
        return [pool.view(DTYPES[fmt])]
    if fmt == "q8_0":
        b = pool.reshape(*pool.shape[:-1], h * d // 32, 34)
        return [b.view(torch.float16)[..., 0], b.view(torch.int8)[..., 2:]]
    return [pool[..., : h * d].view(torch.float8_e4m3fn), pool.view(torch.float32)[..., h * d // 4: h * d // 4 + h]]


# --------------------------------------------------------------------------- inputs

def _tables(lens, block, g):
    """Block tables of sequences of these lengths over a pool in which their pages lie in no order."""
    need = [max(1, -(-n // block)) for n in lens]
    blocks = sum(need) + 3
    order = torch.randperm(blocks, generator=g, device="cuda").to(torch.int32)
    tables = torch.zeros(len(lens), max(need), dtype=torch.int32)
    rows, at = order.cpu(), 0
    for i, k in enumerate(need):
        tables[i, :k] = rows[at: at + k]
        at += k
    return tables.cuda(), blocks


def _slots(tables, seq, pos, block):
    return tables[seq, pos // block].long() * block + pos % block


def _rows_of(lens):
    """Sequence and position of every token of sequences of these lengths."""
    n = torch.tensor(lens, device="cuda")
    seq = torch.repeat_interleave(torch.arange(len(lens), device="cuda"), n)
    return seq, torch.arange(int(sum(lens)), device="cuda") - (torch.cumsum(n, 0) - n)[seq]


def _fill(pool, slots, fmt, h, d, scale, g):
    """Random rows at the given slots; what no token has been written to keeps NaN."""
    flat = pool.view(-1, pool.shape[-1])
    for part in torch.split(slots, max(1, (1 << 26) // (h * d))):
        x = torch.randn(part.numel(), h, d, generator=g, device="cuda") * scale
        flat[part] = _encode(x, fmt)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    fmt, h, d, block, dtype = case["format"], case["kv_heads"], case["head_dim"], case["block"], DTYPES[case["dtype"]]
    state = dict(case)
    rb = row_bytes(fmt, h, d)
    if case["kind"] == "attend":
        lens, batch, heads = _lengths(case), case["batch"], case["heads"]
        tables, blocks = _tables(lens, block, g)
        state["k"], state["v"] = (torch.full((blocks, block, rb), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
        slots = _slots(tables, *_rows_of(lens), block)
        # keys of a normed head, queries that look for some of them: scores spread over a few units, as trained heads have it
        spread = torch.exp2(torch.linspace(-2, 1, h * d, device="cuda")).reshape(h, d)
        _fill(state["k"], slots, fmt, h, d, 1.0, g)
        _fill(state["v"], slots, fmt, h, d, spread, g)
        # queries and gates side by side, a head at a time, as the fused projection of the 4B model leaves them
        width = 2 * d if case["gate"] else d
        qg = torch.randn(batch, heads, width, generator=g, device="cuda")
        qg[..., :d] *= 1.0 + torch.rand(batch, heads, 1, generator=g, device="cuda")
        state["qg"] = qg.to(dtype)
        state["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        state["out"] = torch.zeros(batch, heads, d, dtype=dtype, device="cuda")
        state["lse"] = torch.zeros(batch, heads, dtype=torch.float32, device="cuda")
        state["longest"] = max(lens)
    else:
        n, count = case["rows"], case["sequences"]
        share = [n // count + (i < n % count) for i in range(count)]
        tables, blocks = _tables([case["context"] + s for s in share], block, g)
        seq, pos = _rows_of(share)
        pos = pos + case["context"]
        if case["kind"] == "write":
            state["k"], state["v"] = (torch.full((blocks, block, rb), 60, dtype=torch.uint8, device="cuda") for _ in range(2))
            # one projection's output: the queries' columns, then K, then V
            x = torch.randn(n + case["padding"], 4 * h, d, generator=g, device="cuda")
            x *= torch.exp2(torch.linspace(-6, 2, d, device="cuda")) * torch.exp2(4 * torch.rand(n + case["padding"], 1, 1, generator=g, device="cuda") - 2)
            state["x"] = x.to(dtype)
        else:
            state["k"], state["v"] = (torch.full((blocks, block, rb), 255, dtype=torch.uint8, device="cuda") for _ in range(2))
            slots = _slots(tables, seq, pos, block)
            _fill(state["k"], slots, fmt, h, d, 1.0, g)
            _fill(state["v"], slots, fmt, h, d, 0.3, g)
            state["to_k"], state["to_v"] = (torch.full((n + case["padding"], h, d), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        none = torch.full((case["padding"],), -1, device="cuda")
        state["seq"] = torch.cat([seq, torch.zeros_like(none)]).to(torch.int32)
        state["pos"] = torch.cat([pos, none]).to(torch.int32)
    state["tables"], state["blocks"] = tables, blocks
    if own:
        state["call"] = _handles(state)
    return state


# --------------------------------------------------------------------------- the framework's calls

_device, _scratch = None, None


def _view(t, offset=0):
    """A tensor's memory as the library sees it."""
    return _device.view(t.data_ptr() + offset, t.numel() * t.element_size() - offset)


def _handles(state):
    """What a program keeps from call to call: the cache, the rows or the step over it, the scratch area."""
    from yuuka_b200 import cuda
    global _device, _scratch
    if _device is None:
        _device = cuda.Device(0)
        _scratch = cuda.AttentionScratch(_device)
    stream = _device.stream_view(torch.cuda.current_stream().cuda_stream)
    h, d = state["kv_heads"], state["head_dim"]
    tables = state["tables"]
    cache = cuda.KvCache(_view(state["k"]), _view(state["v"]), _view(tables), FORMATS[state["format"]], h, d, state["block"],
                         state["blocks"], tables.shape[0], tables.shape[1])
    dtype = {"f32": cuda.F32, "f16": cuda.F16, "bf16": cuda.BF16}[state["dtype"]]
    if state["kind"] == "attend":
        qg, width = state["qg"], state["qg"].shape[-1]
        args = cuda.DecodeArgs(_view(qg), _view(state["out"]), _view(state["lens"]), state["batch"], state["heads"], dtype,
                               q_row_stride=state["heads"] * width, q_head_stride=width, window=state["window"],
                               gate=_view(qg, d * qg.element_size()) if state["gate"] else None, lse=_view(state["lse"]))
        return lambda: cuda.attention_decode(stream, _scratch, cache, args)
    seq, pos = _view(state["seq"]), _view(state["pos"])
    if state["kind"] == "write":
        x = state["x"]
        rows = cuda.KvRows(_view(x, 2 * h * d * x.element_size()), _view(x, 3 * h * d * x.element_size()), pos, x.shape[0], dtype,
                           seq=seq, k_stride=4 * h * d, v_stride=4 * h * d)
        return lambda: cuda.kv_write(stream, cache, rows)
    rows = cuda.KvRows(_view(state["to_k"]), _view(state["to_v"]), pos, state["to_k"].shape[0], dtype, seq=seq)
    return lambda: cuda.kv_read(stream, cache, rows)


# --------------------------------------------------------------------------- one pass

def _plain_attend(state):
    fmt, h, d, block, batch, heads = (state[k] for k in ("format", "kv_heads", "head_dim", "block", "batch", "heads"))
    lens = state["lens"].long()
    at = torch.arange(state["longest"], device="cuda")
    see = at[None, :] < lens[:, None]
    if state["window"]:
        see = see & (at[None, :] >= (lens - state["window"])[:, None])
    slots = torch.where(see, _slots(state["tables"], torch.arange(batch, device="cuda")[:, None], at[None, :], block), 0)
    rb = state["k"].shape[-1]
    hide = ~see[:, :, None, None]
    k = _decode(state["k"].view(-1, rb)[slots], fmt, h, d).masked_fill(hide, 0.0)
    q = state["qg"][..., :d].float().reshape(batch, h, heads // h, d)
    s = torch.matmul(q, k.permute(0, 2, 3, 1)) / math.sqrt(d)
    del k
    s = s.masked_fill(~see[:, None, None, :], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(torch.isinf(m), 0.0, m))
    l = p.sum(-1, keepdim=True)
    v = _decode(state["v"].view(-1, rb)[slots], fmt, h, d).masked_fill(hide, 0.0)
    out = (torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(l == 0, 1.0, l)).reshape(batch, heads, d)
    if state["gate"]:
        out = out / (1.0 + torch.exp(-state["qg"][..., d:].float()))
    return out.to(state["qg"].dtype), (m + torch.log(l)).reshape(batch, heads)


def run(state):
    fmt, h, d = state["format"], state["kv_heads"], state["head_dim"]
    if own:
        state["call"]()
        if state["kind"] == "attend":
            return state["out"], state["lse"]
    elif state["kind"] == "attend":
        return _plain_attend(state)
    elif state["kind"] == "write":
        n = state["rows"]
        slots = _slots(state["tables"], state["seq"][:n].long(), state["pos"][:n].long(), state["block"])
        for pool, first in ((state["k"], 2 * h), (state["v"], 3 * h)):
            pool.view(-1, pool.shape[-1])[slots] = _encode(state["x"][:n, first: first + h].float(), fmt)
    else:
        n = state["rows"]
        slots = _slots(state["tables"], state["seq"][:n].long(), state["pos"][:n].long(), state["block"])
        for pool, to in ((state["k"], state["to_k"]), (state["v"], state["to_v"])):
            to[:n] = _decode(pool.view(-1, pool.shape[-1])[slots], fmt, h, d).to(to.dtype)
    if state["kind"] == "write":
        return _values(state["k"], fmt, h, d) + _values(state["v"], fmt, h, d)
    return state["to_k"], state["to_v"]


# --------------------------------------------------------------------------- in 64 bits

def _numbers(raw, fmt, h, d):
    """Cache rows [n, row bytes] as 64-bit numbers [n, heads, dim]."""
    n = raw.shape[0]
    if fmt == "q8_0":
        blocks = raw.view(n, -1, 34)
        scale = blocks[:, :, 0:2].clone().view(torch.float16).double()
        return (blocks[:, :, 2:].clone().view(torch.int8).double() * scale).view(n, h, d)
    if fmt == "f8":
        scale = raw[:, h * d: h * d + 4 * h].clone().view(torch.float32).double()
        return raw[:, : h * d].clone().view(torch.float8_e4m3fn).double().view(n, h, d) * scale[:, :, None]
    return raw.view(DTYPES[fmt]).double().view(n, h, d)


def exact(case, seed):
    s = prepare(case, seed)
    fmt, h, d, block = case["format"], case["kv_heads"], case["head_dim"], case["block"]
    k_rows, v_rows = (s[x].view(-1, s[x].shape[-1]) for x in ("k", "v"))
    table = s["tables"].long()
    if case["kind"] != "attend":
        n = case["rows"]
        seq, pos = s["seq"][:n].long(), s["pos"][:n].long()
        where = table[seq, torch.div(pos, block, rounding_mode="floor")] * block + torch.remainder(pos, block)
        out = []
        for i, rows in enumerate((k_rows, v_rows)):
            if case["kind"] == "read":
                x = torch.full((n + case["padding"], h, d), 7.0, dtype=torch.float64, device="cuda")
                x[:n] = _numbers(rows[where], fmt, h, d)
                out.append(x)
                continue
            # before the rounding to the format; whole numbers have no such value
            x = s["x"][:n, (2 + i) * h: (3 + i) * h].double()
            old = [y.double() for y in _values(s["k" if i == 0 else "v"], fmt, h, d)]
            if fmt == "q8_0":
                old[0].view(-1, h * d // 32)[where] = x.view(n, -1, 32).abs().max(-1).values / 127
                old[1] = None
            elif fmt == "f8":
                top = x.abs().max(-1).values
                old[0].view(-1, h, d)[where] = torch.nan_to_num(x / top[..., None]) * 448
                old[1].view(-1, h)[where] = top / 448
            else:
                old[0].view(-1, h, d)[where] = x
            out += old
        return out if case["kind"] == "write" else tuple(out)
    group = case["heads"] // h
    out = torch.zeros(case["batch"], case["heads"], d, dtype=torch.float64, device="cuda")
    lse = torch.full((case["batch"], case["heads"]), -math.inf, dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lengths(case)):
        first = max(0, n - case["window"]) if case["window"] else 0
        if n == 0:
            continue
        where = torch.arange(first, n, device="cuda")
        where = table[b][torch.div(where, block, rounding_mode="floor")] * block + torch.remainder(where, block)
        k, v = _numbers(k_rows[where], fmt, h, d), _numbers(v_rows[where], fmt, h, d)
        for j in range(h):
            mine = slice(j * group, (j + 1) * group)
            score = (s["qg"][b, mine, :d].double() @ k[:, j].T) * d ** -0.5
            lse[b, mine] = torch.logsumexp(score, -1)
            out[b, mine] = torch.softmax(score, -1) @ v[:, j]
    if case["gate"]:
        out = out * torch.sigmoid(s["qg"][..., d:].double())
    return out, lse
