"""The operators of microscaled 4-bit serving, as measured cases.

The format: blocks of 32 values along one axis, each value a 4-bit float (1 sign, 2 exponent and 1 mantissa
bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6) times the block's scale, a power of two held as its biased exponent in a byte
(255: the block held a NaN or an infinity). The scale is 2^(floor(log2(largest magnitude)) - 2); values are rounded
to nearest, ties to the even code, and 6 is the largest. Two values share a byte, the first in its low half.

The kinds, each one traced program compiled once and launched on buffers in HBM:

* ``quantize``  a tensor quantised along its last axis, and read back;
* ``linear``    a projection: activations quantised, then their product with quantised weights [out, inner];
* ``cache``     the keys and values of new tokens quantised into a paged cache in place, and the cache read back;
* ``attend``    the newest queries of each sequence against its cached keys and values.

A cache is u8 [page, kv_head, bytes]. A page of T tokens and one key-value head of dimension d hold, in this
order, T rows of d/2 key codes, T rows of d/2 value codes, T rows of d/32 key scales, T rows of d/32 value scales.
"""
import math

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
PAGE = 64


def listed():
    return [
        # One token's activations, as a decode step quantises them before a projection: launch latency.
        {"name": "quantize-1x2048-bf16", "kind": "quantize", "rows": 1, "cols": 2048, "dtype": "bf16"},
        # A weight matrix quantised when a model is loaded.
        {"name": "quantize-8192x8192-f32", "kind": "quantize", "rows": 8192, "cols": 8192, "dtype": "f32"},
        # A decode step's MLP-up projection for sixteen sequences: the weights are read for few rows.
        {"name": "linear-16x2048x8192-bf16", "kind": "linear", "tokens": 16, "inner": 2048, "out": 8192, "dtype": "bf16"},
        # A general product off every tile grid.
        {"name": "linear-1000x992x1001-f32", "kind": "linear", "tokens": 1000, "inner": 992, "out": 1001, "dtype": "f32"},
        # The decoder block's MLP-up projection for one sequence of the benchmark's length.
        {"name": "linear-2048x2048x8192-f16", "kind": "linear", "tokens": 2048, "inner": 2048, "out": 8192, "dtype": "f16"},
        # The benchmark's contraction, the largest piece of work here.
        {"name": "linear-8192-bf16", "kind": "linear", "tokens": 8192, "inner": 8192, "out": 8192, "dtype": "bf16"},
        # A decode step of eight sequences: eight tokens' keys and values into a small cache.
        {"name": "cache-8x8x128-bf16", "kind": "cache", "tokens": 8, "pages": 8, "kv_heads": 8, "dim": 128, "dtype": "bf16"},
        # A prompt of 4000 tokens and some padding written at once.
        {"name": "cache-4000x8x128-f16", "kind": "cache", "tokens": 4000, "pages": 80, "kv_heads": 8, "dim": 128, "dtype": "f16"},
        # One short sequence, in full precision: launch latency.
        {"name": "attend-1x100-f32", "kind": "attend", "seqs": 1, "queries": 1, "kv_heads": 4, "group": 1, "dim": 64,
         "keys": 100, "dtype": "f32"},
        # A decode step's attention: eight sequences of sixteen heads, 4096 keys at most.
        {"name": "attend-8x16x4096-bf16", "kind": "attend", "seqs": 8, "queries": 1, "kv_heads": 16, "group": 1, "dim": 128,
         "keys": 4096, "dtype": "bf16"},
        # Many sequences of uneven lengths, eight query heads to a key-value head: the cache is larger than any on-chip memory.
        {"name": "attend-48x8x8-16000-bf16", "kind": "attend", "seqs": 48, "queries": 1, "kv_heads": 8, "group": 8, "dim": 128,
         "keys": 16000, "dtype": "bf16"},
        # A few drafted tokens per sequence checked at once.
        {"name": "attend-16x5x4-3001-f16", "kind": "attend", "seqs": 16, "queries": 5, "kv_heads": 4, "group": 4, "dim": 64,
         "keys": 3001, "dtype": "f16"},
    ]


# ---- drawn cases: the same kinds over the ranges their listed cases stand for ----

def _spread(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def _blocks(rng, lo, hi):
    """A blocked axis: a multiple of 32, most often of 128."""
    n = _spread(rng, lo, hi)
    step = 32 if rng.random() < 0.3 else 128
    return max(step, n // step * step)


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "cache", "attend", "attend"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind == "quantize":
        cols = _blocks(rng, 64, 16384)
        return {"kind": kind, "rows": _spread(rng, 1, min(16384, (1 << 26) // cols)), "cols": cols, "dtype": dtype}
    if kind == "linear":
        inner = _blocks(rng, 64, 8192)
        out = _spread(rng, 16, 8192)
        out = out if rng.random() < 0.3 else max(64, out // 64 * 64)
        return {"kind": kind, "tokens": _spread(rng, 1, 8192), "inner": inner, "out": out, "dtype": dtype}
    if kind == "cache":
        tokens = _spread(rng, 1, 4096)
        return {"kind": kind, "tokens": tokens, "pages": -(-tokens // PAGE) + rng.randint(0, 16),
                "kv_heads": rng.choice([1, 2, 4, 8, 16]), "dim": rng.choice([64, 96, 128, 256]), "dtype": dtype}
    kv_heads, dim, keys = rng.choice([1, 2, 4, 5, 8, 16]), rng.choice([64, 96, 128, 128, 256]), _spread(rng, 1, 32768)
    most = (1 << 29) // (kv_heads * dim * keys)
    return {"kind": kind, "seqs": _spread(rng, 1, max(1, min(64, most))), "queries": rng.choice([1, 1, 1, 2, 3, 8]),
            "kv_heads": kv_heads, "group": rng.choice([1, 2, 3, 4, 7, 8, 16]), "dim": dim, "keys": keys, "dtype": dtype}


# ---- the format, in elementary operations ----

def _power(e):
    """2^e in f32, e in -126 .. 127."""
    return ((e + 127) << 23).int().view(torch.float32)


def _scaled(blocks, e):
    """blocks [.., 32] times 2^e [..], in two exact steps so that neither power leaves the range of f32."""
    half = torch.div(e, 2, rounding_mode="floor")
    return blocks * _power(half).unsqueeze(-1) * _power(e - half).unsqueeze(-1)


def _scales(x):
    """The scale byte of every block of 32 of the last axis, and whether the block is finite."""
    blocks = x.float().unflatten(-1, (-1, 32))
    finite = torch.isfinite(blocks).all(-1)
    top = torch.where(finite, blocks.abs().amax(-1), 1.0)
    # frexp: top = m * 2^e with m in [0.5, 1), so floor(log2 top) = e - 1
    exponent = torch.where(top > 0, torch.frexp(top).exponent - 1, -1000)
    byte = (exponent - 2).clamp(-127, 127) + 127
    return torch.where(finite, byte, 255), blocks


def _codes(blocks, byte):
    """The 4-bit codes of blocks [.., 32] under their scale bytes."""
    y = _scaled(blocks, 127 - byte.clamp(max=254))
    a = torch.where((byte == 255).unsqueeze(-1), 0.0, y).abs()
    code = ((a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int() + (a > 2.5).int() + (a >= 3.5).int()
            + (a > 5.0).int())
    return code + 8 * torch.signbit(blocks).int()


def _pack(code):
    code = code.flatten(-2)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).to(torch.uint8)


def _quantize(x):
    """Codes [.., n/2] and scale bytes [.., n/32], both u8."""
    byte, blocks = _scales(x)
    return _pack(_codes(blocks, byte)), byte.to(torch.uint8)


def _dequantize(codes, scales):
    """The values, in f32."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    c = codes.int()
    v = grid[torch.stack([c & 15, c >> 4], -1).flatten(-2)].unflatten(-1, (-1, 32))
    v = _scaled(v, scales.clamp(max=254).int() - 127)
    return torch.where((scales == 255).unsqueeze(-1), math.nan, v).flatten(-2)


def _page_parts(cache, dim):
    """Key codes, value codes, key scales, value scales of a cache's pages, each [page, kv_head, token, bytes]; views."""
    tokens = cache.shape[-1] // (dim + dim // 16)
    sizes = [tokens * dim // 2, tokens * dim // 2, tokens * dim // 32, tokens * dim // 32]
    return [p.unflatten(-1, (tokens, -1)) for p in cache.split(sizes, -1)]


# ---- programs, as a user traces them ----

def _program(case):
    from accy_amd import tensor as T
    kind, dtype = case["kind"], case["dtype"]
    if kind == "quantize":
        def body(b, a):
            q = a[0].quantize_mx4("col")
            return [q.codes, q.scales, q.dequantize(dtype)]
        return T.define("quantize", [T.spec(dtype, row=case["rows"], col=case["cols"])], body)
    if kind == "linear":
        def body(b, a):
            return a[0].quantize_mx4("inner").contract(b.mx4(a[1], a[2], "inner"), dtype)
        return T.define("linear", [T.spec(dtype, token=case["tokens"], inner=case["inner"]),
                                   *T.mx4_specs("inner", out=case["out"], inner=case["inner"])], body)
    if kind == "cache":
        def body(b, a):
            cache = a[0].cache_write_mx4(a[1], a[2], a[3])
            return [cache, cache.cache_keys_mx4(a[4], ("dim", case["dim"]), dtype),
                    cache.cache_values_mx4(a[4], ("dim", case["dim"]), dtype)]
        token = T.spec(dtype, token=case["tokens"], kv_head=case["kv_heads"], dim=case["dim"])
        return T.define("cache", [T.cache_mx4_spec(case["pages"], case["kv_heads"], case["dim"], PAGE), token, token,
                                  T.spec("i32", token=case["tokens"]), T.spec("i32", slot=case["pages"] * PAGE)], body)

    def body(b, a):
        return a[0].attend_mx4(a[1], a[2], a[3])
    pages = -(-case["keys"] // PAGE)
    return T.define("attend", [T.spec(dtype, seq=case["seqs"], query=case["queries"], head=case["kv_heads"] * case["group"],
                                      dim=case["dim"]),
                               T.cache_mx4_spec(case["seqs"] * pages, case["kv_heads"], case["dim"], PAGE),
                               T.spec("i32", seq=case["seqs"], page_of=pages), T.spec("i32", seq=case["seqs"])], body)


# ---- inputs, in the programs' parameter order ----

def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], TORCH[case["dtype"]]

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(std).to(dtype)

    if kind == "quantize":
        # activations: some channels are much larger than the others
        x = normal(case["rows"], case["cols"])
        x[:, ::61] *= 20.0
        return [x]
    if kind == "linear":
        codes, scales = _quantize(normal(case["out"], case["inner"], std=0.02))
        return [normal(case["tokens"], case["inner"]), codes, scales]

    def cache_of(pages):
        cache = torch.empty(pages, case["kv_heads"], PAGE * (case["dim"] + case["dim"] // 16), dtype=torch.uint8, device="cuda")
        for first in range(0, pages, 256):
            parts = _page_parts(cache[first:first + 256], case["dim"])
            for codes, scales, std in ((parts[0], parts[2], 1.5), (parts[1], parts[3], 1.0)):
                c, s = _quantize(normal(*codes.shape[:-1], case["dim"], std=std))
                codes.copy_(c)
                scales.copy_(s)
        return cache

    if kind == "cache":
        n, slots = case["tokens"], case["pages"] * PAGE
        where = torch.randperm(slots, generator=gen, device="cuda")[:n].to(torch.int32)
        if n > 16:  # a padded batch: some tokens are no sequence's
            where[::17] = -1
        return [cache_of(case["pages"]), normal(n, case["kv_heads"], case["dim"]), normal(n, case["kv_heads"], case["dim"]),
                where, torch.arange(slots, device="cuda", dtype=torch.int32)]
    pages, seqs = -(-case["keys"] // PAGE), case["seqs"]
    table = torch.randperm(seqs * pages, generator=gen, device="cuda").to(torch.int32).view(seqs, pages)
    # lengths from half of the most to the most; the first sequence has them all
    lengths = torch.randint((case["keys"] + 1) // 2, case["keys"] + 1, (seqs,), generator=gen, device="cuda", dtype=torch.int32)
    lengths[0] = case["keys"]
    q = normal(seqs, case["queries"], case["kv_heads"] * case["group"], case["dim"])
    return [q, cache_of(seqs * pages), table, lengths]


def prepare(case, seed):
    state = {"case": case, "inputs": _inputs(case, seed)}
    if own:
        from accy_amd import hip
        names = dict(TORCH, u8=torch.uint8)
        state["executor"] = hip.Hip(_program(case))
        state["outputs"] = [torch.empty(tuple(e for _, e in d.dims), dtype=names[d.dtype], device="cuda")
                            for d in state["executor"].outputs]
        if case["kind"] == "cache":
            state["outputs"][0] = state["inputs"][0]  # written in place
    return state


def run(state):
    case, inputs = state["case"], state["inputs"]
    if own:
        state["executor"].launch_device([t.data_ptr() for t in inputs], [t.data_ptr() for t in state["outputs"]],
                                        torch.cuda.current_stream().cuda_stream)
        # what is held in 4 bits is returned as its values, which the program reads back
        return {"quantize": state["outputs"][2:], "cache": state["outputs"][1:]}.get(case["kind"], state["outputs"])
    return {"quantize": _plain_quantize, "linear": _plain_linear, "cache": _plain_cache, "attend": _plain_attend}[case["kind"]](case, *inputs)


def _plain_quantize(case, x):
    return [_dequantize(*_quantize(x)).to(x.dtype)]


def _plain_linear(case, x, codes, scales):
    return [(_dequantize(*_quantize(x)) @ _dequantize(codes, scales).t()).to(x.dtype)]


def _plain_cache(case, cache, keys, values, where, slots):
    parts, rows = _page_parts(cache, case["dim"]), []
    at = torch.where(where < 0, cache.shape[0] * PAGE, where).long()  # padding goes to a row of its own
    for codes, scales, new in ((parts[0], parts[2], keys), (parts[1], parts[3], values)):
        for old, fresh in zip((codes, scales), _quantize(new)):
            flat = old.transpose(1, 2).flatten(0, 1)  # [slot, kv_head, bytes]
            flat = torch.cat([flat, torch.zeros_like(flat[:1])])
            flat[at] = fresh
            rows.append(flat[:-1])
    keys_now, values_now = _dequantize(rows[0], rows[1]), _dequantize(rows[2], rows[3])
    return [keys_now[slots.long()].to(keys.dtype), values_now[slots.long()].to(values.dtype)]


def _plain_attend(case, q, cache, table, lengths):
    n, heads = case["queries"], case["kv_heads"]
    parts, out = _page_parts(cache, case["dim"]), []
    for b in range(case["seqs"]):
        # [kv_head, key, dim]
        k, v = (_dequantize(*(p[table[b].long()].transpose(0, 1).flatten(1, 2) for p in pair))
                for pair in ((parts[0], parts[2]), (parts[1], parts[3])))
        # [kv_head, query * group, dim]
        rows = q[b].float().unflatten(1, (heads, -1)).transpose(0, 1).flatten(1, 2)
        s = torch.matmul(rows, k.transpose(1, 2).contiguous()) / math.sqrt(case["dim"])
        sees = lengths[b] - (n - 1) + torch.arange(n, device=q.device).repeat_interleave(case["group"])
        hidden = torch.arange(k.shape[1], device=q.device) >= sees[:, None]
        s = s.masked_fill(hidden, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        total = p.sum(-1, keepdim=True)
        o = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
        out.append(o.unflatten(1, (n, -1)).transpose(0, 1).flatten(1, 2))
    return [torch.stack(out).to(q.dtype)]


# ---- the work ----

def work(case):
    size = SIZE[case["dtype"]]
    if case["kind"] == "quantize":
        n = case["rows"] * case["cols"]
        # the tensor in; codes, scales and the values read back out; a comparison, a scaling and a rounding each way
        return {"bytes": 2 * size * n + n // 2 + n // 32, "flops": 4 * n}
    if case["kind"] == "linear":
        m, k, n = case["tokens"], case["inner"], case["out"]
        return {"bytes": size * (m * k + m * n) + n * (k // 2 + k // 32), "flops": 2 * m * k * n}
    row = case["dim"] // 2 + case["dim"] // 32
    if case["kind"] == "cache":
        new, every = case["tokens"] * case["kv_heads"], case["pages"] * PAGE * case["kv_heads"]
        # new keys and values in, their codes out; the whole cache in, its values out
        return {"bytes": 2 * new * (size * case["dim"] + row) + 2 * every * (size * case["dim"] + row) + 4 * case["tokens"],
                "flops": 2 * case["dim"] * (3 * new + every)}
    # lengths are uniform from half of the most to the most, and the first is the most
    keys = case["keys"] + (case["seqs"] - 1) * 0.75 * case["keys"]
    q = case["seqs"] * case["queries"] * case["kv_heads"] * case["group"] * case["dim"]
    return {"bytes": int(2 * keys * case["kv_heads"] * row) + 2 * size * q,
            "flops": int(4 * keys * case["kv_heads"] * case["group"] * case["queries"] * case["dim"])}


# ---- the results in 64 bits, from the definitions ----

_GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])


def _exact_power(e):
    """2^e of whole numbers e held in f64."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_quantized(x):
    """The values that x's blocks of 32 are quantised to."""
    x = x.double()
    out = []
    grid = torch.tensor(_GRID, device=x.device)
    # a midpoint belongs to the neighbour of the even code
    middle = (grid[1:] + grid[:-1]) / 2
    even_above = torch.tensor([False, True, False, True, False, True, False], device=x.device)
    for part in x.reshape(-1, 32).split(1 << 20):
        top = part.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(torch.where(top == 0, 1.0, top)))
        e = e + (_exact_power(e + 1) <= top).double() - (_exact_power(e) > top).double()  # a logarithm may be a step off
        scale = _exact_power(e - 2)
        y = part / scale
        a = y.abs()
        at = torch.searchsorted(middle, a)  # the midpoints below a
        # a equal to midpoint `at` goes up where the even code is the upper one
        here = at.clamp(max=6)
        at = at + ((a == middle[here]) & even_above[here]).long()
        out.append(torch.copysign(grid[at], y) * scale)
    return torch.cat(out).view(x.shape)


def _exact_values(codes, scales):
    """The values that codes and scale bytes stand for."""
    table = torch.tensor(np.concatenate([_GRID, -_GRID]), device=codes.device)
    low, high = table[(codes % 16).long()], table[(codes // 16).long()]
    pairs = torch.cat([low[..., None], high[..., None]], -1).reshape(*codes.shape[:-1], -1)
    return pairs * _exact_power(scales.double() - 127.0).repeat_interleave(32, -1)


def _exact_rows(cache, dim, pages, value):
    """The keys (or values) of some pages, one after the other: [kv_head, token, dim]."""
    raw = cache[pages].transpose(0, 1)
    c0 = PAGE * dim // 2 if value else 0
    s0 = PAGE * dim + (PAGE * dim // 32 if value else 0)
    codes = raw[:, :, c0:c0 + PAGE * dim // 2].reshape(raw.shape[0], -1, dim // 2)
    return _exact_values(codes, raw[:, :, s0:s0 + PAGE * dim // 32].reshape(raw.shape[0], -1, dim // 32))


def exact(case, seed):
    args, kind = _inputs(case, seed), case["kind"]
    if kind == "quantize":
        return [_exact_quantized(args[0])]
    if kind == "linear":
        x, codes, scales = args
        return [_exact_quantized(x) @ _exact_values(codes, scales).t()]
    if kind == "cache":
        cache, keys, values, where, _ = args
        result = []
        for which, new in ((False, keys), (True, values)):
            rows = _exact_rows(cache, case["dim"], torch.arange(case["pages"], device=cache.device), which).transpose(0, 1).contiguous()
            kept = where >= 0
            rows[where[kept].long()] = _exact_quantized(new)[kept]
            result.append(rows)
        return result
    q, cache, table, lengths = args
    n, group = case["queries"], case["group"]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, length in enumerate(lengths.tolist()):
        if length == 0:
            continue
        pages = table[b, :-(-length // PAGE)].long()
        k, v = _exact_rows(cache, case["dim"], pages, False), _exact_rows(cache, case["dim"], pages, True)
        for i in range(n):
            seen = length - (n - 1 - i)
            if seen <= 0:
                continue
            for h in range(case["kv_heads"]):
                rows = q[b, i, h * group:(h + 1) * group].double()
                w = torch.softmax(rows @ k[h, :seen].t() * case["dim"] ** -0.5, 1)
                out[b, i, h * group:(h + 1) * group] = w @ v[h, :seen]
    return [out]
