"""The operators of sampling many answers to one prompt, as measured cases.

A prompt's keys and values lie once in the paged 4-bit cache; every answer has pages of its own behind it, sequences are forked,
freed and moved between steps, and the answers' log probabilities train the model that gave them.

* ``heads``           norms of each query and key head and the rotation by position, positions along one axis or several, in one pass;
* ``heads_grad``      its gradient: of queries, keys and both norms' gains;
* ``attend``          the newest queries of each sequence against a prefix that sequences share, and against their own keys;
* ``fork``            page tables for the next step: rows kept, freed and forked, the pages to come reserved, partly filled pages copied;
* ``compact``         pages moved to the lowest numbers, and the tables with them;
* ``log_probs``       log probabilities of given tokens, entropies and the top alternatives;
* ``log_probs_grad``  the gradient of log probabilities and entropies with respect to the logits.

The cache is u8 [page, kv_head, bytes] in microscaled 4-bit floats: a page of T tokens and one key-value head of dimension d
holds, in this order, T rows of d/2 key codes, T rows of d/2 value codes, T rows of d/32 key scales, T rows of d/32 value scales.
"""
import math

import numpy as np
import torch

own = False

TORCH = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16, "u8": torch.uint8, "i32": torch.int32}
SIZE = {"f32": 4, "bf16": 2, "f16": 2}
PAGE = 64
EPS = 1e-6


def listed():
    return [
        # One token of one sequence before its attention: launch latency.
        {"name": "heads-1x16-bf16", "kind": "heads", "tokens": 1, "heads": 16, "kv_heads": 4, "dim": 128, "rotated": 128, "axes": 1,
         "layout": "halves", "dtype": "bf16"},
        # The decoder block's queries and keys of four prompts of 2048 tokens.
        {"name": "heads-8192x16-bf16", "kind": "heads", "tokens": 8192, "heads": 16, "kv_heads": 16, "dim": 128, "rotated": 128, "axes": 1,
         "layout": "halves", "dtype": "bf16"},
        # Training on a video's tokens: three axes, part of the dims rotated, neighbours paired, sizes off every grid.
        {"name": "heads-grad-4001x12-f32", "kind": "heads_grad", "tokens": 4001, "heads": 12, "kv_heads": 3, "dim": 96, "rotated": 64,
         "axes": 3, "layout": "neighbours", "dtype": "f32"},
        # Four answers to a short prompt, in full precision.
        {"name": "attend-4x4-1000-f32", "kind": "attend", "seqs": 4, "queries": 1, "kv_heads": 4, "group": 1, "dim": 64, "prefixes": 1,
         "prefix_keys": 1000, "keys": 60, "dtype": "f32"},
        # A decode step of 64 answers to one long prompt.
        {"name": "attend-64x16-8192-bf16", "kind": "attend", "seqs": 64, "queries": 1, "kv_heads": 4, "group": 4, "dim": 128, "prefixes": 1,
         "prefix_keys": 8192, "keys": 1024, "dtype": "bf16"},
        # Drafted tokens of answers to three prompts checked at once.
        {"name": "attend-48x40-3001-f16", "kind": "attend", "seqs": 48, "queries": 5, "kv_heads": 8, "group": 5, "dim": 64, "prefixes": 3,
         "prefix_keys": 3001, "keys": 500, "dtype": "f16"},
        # Between two steps of a small batch: a few rows forked, a few freed.
        {"name": "fork-8x64", "kind": "fork", "seqs": 8, "rows": 8, "slots": 64, "pages": 1024, "kv_heads": 4, "dim": 128},
        # A large batch of long sequences.
        {"name": "fork-256x512", "kind": "fork", "seqs": 256, "rows": 256, "slots": 512, "pages": 16384, "kv_heads": 4, "dim": 128},
        # Pages of a half empty cache moved together.
        {"name": "compact-64x256", "kind": "compact", "seqs": 64, "slots": 256, "pages": 16384, "moves": 4096, "kv_heads": 4, "dim": 128},
        # A decode step's sampled tokens, with five alternatives each.
        {"name": "log_probs-8x32000-f32", "kind": "log_probs", "rows": 8, "vocab": 32000, "top": 5, "dtype": "f32"},
        # A batch of answers scored at once.
        {"name": "log_probs-2048x50257-bf16", "kind": "log_probs", "rows": 2048, "vocab": 50257, "top": 20, "dtype": "bf16"},
        # The gradient of a policy's loss.
        {"name": "log_probs-grad-1001x50257-f16", "kind": "log_probs_grad", "rows": 1001, "vocab": 50257, "dtype": "f16"},
    ]


# ---- drawn cases: the same kinds over the ranges their listed cases stand for ----

def _spread(rng, lo, hi):
    """A whole number of [lo, hi], uniform in its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def draw(rng):
    kind = rng.choice(["heads", "heads", "heads_grad", "attend", "attend", "attend", "fork", "compact", "log_probs", "log_probs", "log_probs_grad"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    if kind in ("heads", "heads_grad"):
        kv_heads, dim = rng.choice([1, 2, 3, 4, 8, 16]), rng.choice([64, 80, 96, 128, 128, 192, 256])
        heads = kv_heads * rng.choice([1, 1, 2, 4, 7])
        most = (1 << 28) // ((heads + kv_heads) * dim * SIZE[dtype] * (2 if kind == "heads" else 3))
        return {"kind": kind, "tokens": _spread(rng, 1, max(1, min(16384, most))), "heads": heads, "kv_heads": kv_heads, "dim": dim,
                "rotated": rng.choice([dim, dim, dim // 2]), "axes": rng.choice([1, 1, 2, 3]), "layout": rng.choice(["halves", "halves", "neighbours"]),
                "dtype": dtype}
    if kind == "attend":
        kv_heads, group, dim = rng.choice([1, 2, 4, 5, 8]), rng.choice([1, 2, 3, 4, 5, 8]), rng.choice([64, 96, 128, 128, 256])
        prefixes, queries = rng.choice([1, 1, 2, 3]), rng.choice([1, 1, 1, 2, 5])
        prefix_keys, keys = _spread(rng, 1, 16384), _spread(rng, queries, 2048)
        most = min((1 << 31) // (kv_heads * group * queries * dim * (prefixes * prefix_keys + keys)), (1 << 25) // (kv_heads * dim * keys))
        return {"kind": kind, "seqs": _spread(rng, 1, max(1, min(128, most))), "queries": queries, "kv_heads": kv_heads, "group": group, "dim": dim,
                "prefixes": prefixes, "prefix_keys": prefix_keys, "keys": keys, "dtype": dtype}
    if kind in ("fork", "compact"):
        seqs, slots, kv_heads, dim = _spread(rng, 1, 256), _spread(rng, 1, 512), rng.choice([1, 2, 4]), rng.choice([64, 128])
        pages = _spread(rng, max(32, seqs * slots // 8), max(64, min(16384, seqs * slots * 2)))
        case = {"kind": kind, "seqs": seqs, "slots": slots, "pages": pages, "kv_heads": kv_heads, "dim": dim}
        return case | ({"rows": _spread(rng, 1, 256)} if kind == "fork" else {"moves": _spread(rng, 1, max(1, pages // 4))})
    vocab = _spread(rng, 500, 131072)
    most = (1 << 28) // (vocab * SIZE[dtype] * (1 if kind == "log_probs" else 2))
    case = {"kind": kind, "rows": _spread(rng, 1, max(1, min(4096, most))), "vocab": vocab, "dtype": dtype}
    return case | ({"top": rng.choice([1, 2, 5, 8, 20, 32])} if kind == "log_probs" else {})


# ---- programs, as a user traces them ----

def _program(case):
    from accy_amd import tensor as T
    kind, dtype = case["kind"], case.get("dtype")
    if kind in ("heads", "heads_grad"):
        q, k = (T.spec(dtype, token=case["tokens"], head=case["heads"], dim=case["dim"]),
                T.spec(dtype, token=case["tokens"], kv_head=case["kv_heads"], dim=case["dim"]))
        several = case["axes"] > 1
        position = T.spec("i32", token=case["tokens"], axis=case["axes"]) if several else T.spec("i32", token=case["tokens"])
        pairs = case["rotated"] // 2
        rest = [position, T.spec("f32", pair=pairs), *([T.spec("i32", pair=pairs)] if several else []), *[T.spec(dtype, dim=case["dim"])] * 2]

        def body(b, a):
            n = 2 if kind == "heads" else 4
            rotation = T.Rotation(a[n], a[n + 1], a[n + 2] if several else None, case["layout"])
            norm = T.HeadNorm(a[-2], a[-1], EPS)
            if kind == "heads":
                return list(b.rotate_heads(a[0], a[1], rotation, norm))
            return list(b.rotate_heads_grad(a[0], a[1], a[2], a[3], rotation, norm))
        return T.define(kind, [q, k] * (1 if kind == "heads" else 2) + rest, body)
    if kind == "attend":
        own_pages, prefix_pages = -(-case["keys"] // PAGE), -(-case["prefix_keys"] // PAGE)

        def body(b, a):
            return a[0].attend_mx4(a[1], a[2], a[3], shared=(a[4], a[5], a[6]))
        return T.define("attend", [T.spec(dtype, seq=case["seqs"], query=case["queries"], head=case["kv_heads"] * case["group"], dim=case["dim"]),
                                   T.cache_mx4_spec(case["seqs"] * own_pages + case["prefixes"] * prefix_pages, case["kv_heads"], case["dim"], PAGE),
                                   T.spec("i32", seq=case["seqs"], page_of=own_pages), T.spec("i32", seq=case["seqs"]),
                                   T.spec("i32", prefix=case["prefixes"], prefix_page=prefix_pages), T.spec("i32", prefix=case["prefixes"]),
                                   T.spec("i32", seq=case["seqs"])], body)
    if kind in ("fork", "compact"):
        cache = T.cache_mx4_spec(case["pages"], case["kv_heads"], case["dim"], PAGE)
        table = T.spec("i32", seq=case["seqs"], slot=case["slots"])
        if kind == "fork":
            def body(b, a):
                f = b.fork_pages(a[0], a[1], a[2], a[3], a[4], PAGE)
                return [f.pages, f.lengths, f.source, f.target, f.left, a[5].copy_pages(f.source, f.target)]
            row = T.spec("i32", row=case["rows"])
            return T.define("fork", [table, T.spec("i32", seq=case["seqs"]), row, row, T.spec("i1", page=case["pages"]), cache], body)

        def body(b, a):
            c = b.compact_pages(a[0], a[1], ("move", case["moves"]))
            return [c.pages, c.source, c.target, a[2].copy_pages(c.source, c.target)]
        return T.define("compact", [table, T.spec("i1", page=case["pages"]), cache], body)
    logits, tokens = T.spec(dtype, row=case["rows"], vocab=case["vocab"]), T.spec("i32", row=case["rows"])
    if kind == "log_probs":
        def body(b, a):
            p = a[0].log_probs(a[1], "vocab", top=case["top"])
            return [p.token, p.entropy, p.top, p.top_tokens]
        return T.define("log_probs", [logits, tokens], body)

    def body(b, a):
        return a[0].log_probs_grad(a[1], a[2], a[3], "vocab")
    return T.define("log_probs_grad", [logits, tokens, *[T.spec("f32", row=case["rows"])] * 2], body)


# ---- inputs, in the programs' parameter order ----

def _axis_of(case):
    """The axis of every pair: the first half of the pairs go by the first axis, the others by the rest in turn."""
    pairs, axes = case["rotated"] // 2, case["axes"]
    i = torch.arange(pairs, device="cuda")
    return torch.where(i < pairs // 2, 0, 1 + i % (axes - 1)).to(torch.int32)


def _positions(case, gen):
    n, axes = case["tokens"], case["axes"]
    at = torch.randint(0, 100000, (1,), generator=gen, device="cuda")
    t = torch.arange(n, device="cuda")
    if axes == 1:
        # sequences of 2048 tokens at most, one after the other, each going on from where it was
        return (at + t % 2048 + 17 * (t // 2048)).to(torch.int32)
    # frames of 24 x 32 patches
    parts = [at + t // 768, t // 32 % 24, t % 32]
    return torch.stack(parts[:axes], 1).to(torch.int32)


def _random_cache(gen, pages, kv_heads, dim):
    """Pages of random codes whose scales are those of values of about one."""
    bytes_ = PAGE * (dim + dim // 16)
    cache = torch.randint(0, 256, (pages, kv_heads, bytes_), generator=gen, device="cuda", dtype=torch.uint8)
    cache[:, :, PAGE * dim:].clamp_(126, 127)
    return cache


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, dtype = case["kind"], TORCH.get(case.get("dtype"))

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=gen, device="cuda").mul_(std).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda", dtype=torch.int32)

    if kind in ("heads", "heads_grad"):
        shapes = [(case["tokens"], case[h], case["dim"]) for h in ("heads", "kv_heads")]
        pairs = case["rotated"] // 2
        freq = torch.tensor(10000.0 ** (-np.arange(pairs) / pairs), dtype=torch.float32, device="cuda")
        gains = [(1 + 0.1 * torch.randn(case["dim"], generator=gen, device="cuda")).to(dtype) for _ in range(2)]
        rows = [normal(*s, std=3.0) for s in shapes]
        if kind == "heads_grad":
            rows = [normal(*s) for s in shapes] + rows  # the gradients of the results come first
        return [*rows, _positions(case, gen), freq, *([_axis_of(case)] if case["axes"] > 1 else []), *gains]
    if kind == "attend":
        seqs, own_pages, prefix_pages = case["seqs"], -(-case["keys"] // PAGE), -(-case["prefix_keys"] // PAGE)
        pages = seqs * own_pages + case["prefixes"] * prefix_pages
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table, prefix_table = order[:seqs * own_pages].view(seqs, own_pages), order[seqs * own_pages:].view(case["prefixes"], prefix_pages)
        # answers of any length, the new tokens' keys among them; one prompt has them all
        lengths = whole(min(case["queries"], case["keys"]), case["keys"] + 1, seqs)
        prefix_lengths = whole((case["prefix_keys"] + 1) // 2, case["prefix_keys"] + 1, case["prefixes"])
        prefix_lengths[0] = case["prefix_keys"]
        of = whole(0, case["prefixes"], seqs)
        if seqs > 8:
            of[seqs // 2] = -1  # a sequence without a shared prompt
        q = normal(seqs, case["queries"], case["kv_heads"] * case["group"], case["dim"])
        return [q, _random_cache(gen, pages, case["kv_heads"], case["dim"]), table.clone(), lengths, prefix_table.clone(), prefix_lengths, of]
    if kind in ("fork", "compact"):
        seqs, slots, pages = case["seqs"], case["slots"], case["pages"]
        held = torch.rand(pages, generator=gen, device="cuda") < 0.02
        # every sequence has pages of its own, as many as there are for each, and with them a shared beginning
        each = max(1, min(slots, pages // (2 * seqs)))
        order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
        table = torch.full((seqs, slots), -1, dtype=torch.int32, device="cuda")
        mine = torch.arange(seqs * each, device="cuda").view(seqs, each) % pages
        table[:, :each] = order[mine]
        table[:, :each // 2] = table[0, :each // 2].clone()
        lengths = whole(each * PAGE // 2, each * PAGE + 1, seqs)
        if kind == "compact":
            return [table, held, _random_cache(gen, pages, case["kv_heads"], case["dim"])]
        parents = whole(0, seqs, case["rows"])
        parents[1::2] = torch.arange(case["rows"], device="cuda", dtype=torch.int32)[1::2] % seqs  # half of the rows go on
        parents[3::8] = -1  # and some are done
        return [table, lengths, parents, whole(0, PAGE + 1, case["rows"]), held, _random_cache(gen, pages, case["kv_heads"], case["dim"])]
    rows, vocab = case["rows"], case["vocab"]
    logits = normal(rows, vocab, std=2.5)
    logits[::7, ::3] = -math.inf  # rows whose grammar allows some tokens only
    tokens = whole(0, vocab // 3, rows) * 3 + 1
    if rows > 16:
        tokens[::13] = -1  # padding
    if kind == "log_probs":
        return [logits, tokens]
    return [logits, tokens, torch.randn(rows, generator=gen, device="cuda"), torch.randn(rows, generator=gen, device="cuda") * 0.01]


def prepare(case, seed):
    state = {"case": case, "inputs": _inputs(case, seed)}
    if own:
        from accy_amd import hip
        state["executor"] = hip.Hip(_program(case))
        state["outputs"] = [torch.empty(tuple(e for _, e in d.dims), dtype=TORCH[d.dtype], device="cuda") for d in state["executor"].outputs]
        if case["kind"] in ("fork", "compact"):
            state["outputs"][-1] = state["inputs"][-1]  # pages are copied in place
    return state


def run(state):
    case, inputs = state["case"], state["inputs"]
    if own:
        state["executor"].launch_device([t.data_ptr() for t in inputs], [t.data_ptr() for t in state["outputs"]],
                                        torch.cuda.current_stream().cuda_stream)
        return state["outputs"]
    return {"heads": _plain_heads, "heads_grad": _plain_heads_grad, "attend": _plain_attend, "fork": _plain_fork, "compact": _plain_compact,
            "log_probs": _plain_log_probs, "log_probs_grad": _plain_log_probs_grad}[case["kind"]](case, *inputs)


# ---- heads ----

def _turns(case, rest):
    """cos and sin [token, 1, pair] of the angles, which are formed in 64 bits: positions go to the hundred thousands."""
    position, freq = rest[0].double(), rest[1].double()
    angle = position[:, rest[2].long()] * freq if case["axes"] > 1 else position[:, None] * freq
    return angle.cos().float()[:, None], angle.sin().float()[:, None]


def _rotate(case, x, cos, sin):
    """x [token, head, dim] with its pairs turned; what lies beyond the rotated dims stays."""
    n = case["rotated"]
    if case["layout"] == "halves":
        a, b = x[..., :n // 2], x[..., n // 2:n]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., n:]], -1)
    a, b = x[..., 0:n:2], x[..., 1:n:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., n:]], -1)


def _plain_heads(case, q, k, *rest):
    cos, sin = _turns(case, rest)

    def one(x, gain):
        f = x.float()
        f = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * gain.float()
        return _rotate(case, f, cos, sin).to(x.dtype)
    return [one(q, rest[-2]), one(k, rest[-1])]


def _plain_heads_grad(case, dq, dk, q, k, *rest):
    cos, sin = _turns(case, rest)

    def one(dy, x, gain):
        f = x.float()
        r = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
        n = f * r
        g = _rotate(case, dy.float(), cos, -sin)  # turned back
        gw = g * gain.float()
        return (r * (gw - n * (gw * n).mean(-1, keepdim=True))).to(x.dtype), (g * n).sum((0, 1)).to(gain.dtype)
    (dq, gq), (dk, gk) = one(dq, q, rest[-2]), one(dk, k, rest[-1])
    return [dq, dk, gq, gk]


# ---- attention ----

def _dequantize(codes, scales):
    """The f32 values of codes [.., n/2] and scale bytes [.., n/32]."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0], device=codes.device)
    c = codes.int()
    v = grid[torch.stack([c & 15, c >> 4], -1).flatten(-2)].unflatten(-1, (-1, 32))
    return (v * (scales.int() << 23).view(torch.float32).unsqueeze(-1)).flatten(-2)


def _rows_of(cache, table, dim):
    """Keys and values of the pages of every row of a table: [row, kv_head, key, dim]."""
    sizes = [PAGE * dim // 2, PAGE * dim // 2, PAGE * dim // 32, PAGE * dim // 32]
    parts = [p.unflatten(-1, (PAGE, -1)).flatten(2, 3) for p in cache[table.long()].transpose(1, 2).split(sizes, -1)]
    return _dequantize(parts[0], parts[2]), _dequantize(parts[1], parts[3])


def _plain_attend(case, q, cache, table, lengths, prefix_table, prefix_lengths, of):
    S, n, H, G, dim = case["seqs"], case["queries"], case["kv_heads"], case["group"], case["dim"]
    # rows of a key-value head, query by query: [seq, kv_head, query * group, dim]
    rows = q.float().unflatten(2, (H, G)).permute(0, 2, 1, 3, 4).flatten(2, 3) / math.sqrt(dim)
    k, v = _rows_of(cache, table, dim)
    pk, pv = _rows_of(cache, prefix_table, dim)
    own_scores = torch.matmul(rows, k.transpose(2, 3).contiguous())
    sees = lengths[:, None] - (n - 1) + torch.arange(n, device=q.device).repeat_interleave(G)
    own_scores = own_scores.masked_fill((torch.arange(k.shape[2], device=q.device) >= sees[..., None])[:, None], -math.inf)
    # all rows against every prefix, those of its own kept
    flat = rows.transpose(0, 1).flatten(1, 2)  # [kv_head, seq * query * group, dim]
    shared = torch.matmul(flat, pk.transpose(2, 3).contiguous())  # [prefix, kv_head, seq * query * group, key]
    shared = shared.unflatten(2, (S, n * G)).permute(2, 1, 3, 0, 4)  # [seq, kv_head, query * group, prefix, key]
    hidden = (of[:, None] != torch.arange(pk.shape[0], device=q.device))[..., None] | (torch.arange(pk.shape[2], device=q.device) >= prefix_lengths[:, None])
    shared = shared.masked_fill(hidden[:, None, None], -math.inf).flatten(3)
    top = torch.maximum(own_scores.amax(-1, keepdim=True), shared.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    p, ps = torch.exp(own_scores - top), torch.exp(shared - top)
    total = p.sum(-1, keepdim=True) + ps.sum(-1, keepdim=True)
    values = pv.transpose(0, 1).flatten(1, 2)  # [kv_head, prefix * key, dim]
    o = torch.matmul(p, v) + torch.matmul(ps.transpose(0, 1).flatten(1, 2), values).unflatten(1, (S, n * G)).transpose(0, 1)
    o = o / torch.where(total == 0, 1.0, total)
    return [o.unflatten(2, (n, G)).permute(0, 2, 1, 3, 4).flatten(2, 3).to(q.dtype)]


# ---- pages ----

def _copy_pages(cache, source, target):
    """cache[target] = cache[source] in place; a copy without a page repeats the first one that has both, or none."""
    flat, pages = cache.view(cache.shape[0], -1), cache.shape[0]
    valid = (source >= 0) & (source < pages) & (target >= 0) & (target < pages)
    first, some = valid.int().argmax(), valid.any()
    s, t = (torch.where(valid, x, torch.where(some, x[first], 0)).long() for x in (source, target))
    flat.index_copy_(0, t, flat.index_select(0, s))


def _first_of(mask, count):
    """The positions that are true, in order, `count` of them, and how many there are; what follows is of no meaning."""
    return torch.sort((~mask).int(), stable=True).indices[:count], mask.sum()


def _plain_fork(case, table, lengths, parents, room, held, cache):
    S, W, R, P = case["seqs"], case["slots"], case["rows"], case["pages"]
    here = (parents >= 0) & (parents < S)
    parent = torch.where(here, parents, 0).long()
    length = torch.where(here, lengths[parent].clamp(0, W * PAGE), 0)
    kept = (length + PAGE - 1) // PAGE
    want = torch.where(here, ((length.long() + room.clamp(min=0)).clamp(max=W * PAGE) + PAGE - 1) // PAGE, 0)
    j = torch.arange(W, device=table.device)
    rows = torch.where(j < kept[:, None], table[parent], -1)
    rows = torch.where((rows >= 0) & (rows < P), rows, -1)
    partial = length % PAGE != 0
    last = torch.where(partial, rows.gather(1, (kept - 1).clamp(min=0).long()[:, None])[:, 0], -1)
    # pages in whole use, and the first row that holds a page partly filled; P takes what is no page
    whole = torch.zeros(P + 1, dtype=torch.bool, device=table.device)
    full = (j < (kept - partial.int())[:, None]) & (rows >= 0)
    whole[torch.where(full, rows, P).long()] = True
    at = torch.where(last >= 0, last, P).long()
    first = torch.full((P + 1,), R, device=table.device).scatter_reduce_(0, at, torch.arange(R, device=table.device), "amin")
    mine = ~whole[at] & ~held[at.clamp(max=P - 1)] & (first[at] == torch.arange(R, device=table.device))
    copied = (last >= 0) & ~mine
    used = whole.clone()
    used[at] = True
    free, count = _first_of(~(used[:P] | held), P)
    asked = ((j == (kept - 1)[:, None]) & copied[:, None]) | ((j >= kept[:, None]) & (j < want[:, None]))
    k = asked.flatten().cumsum(0).view(R, W) - 1
    fresh = torch.where(k < count, free[k.clamp(0, P - 1)], -1)
    pages = torch.where(asked, fresh, rows).to(torch.int32)
    new = torch.where(copied, pages.gather(1, (kept - 1).clamp(min=0).long()[:, None])[:, 0], -1)
    source, target = torch.where(new >= 0, last, -1), new
    left = (count - asked.sum()).to(torch.int32)
    _copy_pages(cache, source, target)
    return [pages, length.to(torch.int32), source, target, left, cache]


def _plain_compact(case, table, held, cache):
    P, M = case["pages"], case["moves"]
    valid = (table >= 0) & (table < P)
    used = torch.zeros(P + 1, dtype=torch.bool, device=table.device)
    used[torch.where(valid, table, P).long()] = True
    used = used[:P]
    in_use = used | held
    at, count = torch.arange(P, device=table.device), in_use.sum()
    (source, moving), (target, _) = _first_of(used & ~held & (at >= count), M), _first_of(~in_use & (at < count), M)
    moved = torch.arange(M, device=table.device) < moving
    number = torch.cat([at, at[:1]])
    number[torch.where(moved, source, P)] = torch.where(moved, target, 0)
    source, target = (torch.where(moved, x, -1).to(torch.int32) for x in (source, target))
    table = torch.where(valid, number[table.clamp(0, P - 1).long()], -1).to(torch.int32)
    _copy_pages(cache, source, target)
    return [table, source, target, cache]


# ---- log probabilities ----

def _statistics(x):
    """log of the sum of exponentials, the entropy, and the shift and the sum they come from, of f32 rows."""
    top = x.amax(-1, keepdim=True)
    base = torch.where(top == -math.inf, 0.0, top)
    e = torch.exp(x - base)
    total = e.sum(-1, keepdim=True)
    weighed = torch.where(e > 0, e * (x - base), 0.0).sum(-1, keepdim=True)
    entropy = torch.where(total > 0, total.log() - weighed / total, 0.0)
    return base, total, entropy


def _plain_log_probs(case, logits, tokens):
    x = logits.float()
    base, total, entropy = _statistics(x)
    log_total = total.log()
    inside = (tokens >= 0) & (tokens < case["vocab"])
    chosen = x.gather(1, torch.where(inside, tokens, 0).long()[:, None])
    chosen = torch.where(total > 0, chosen - base - log_total, -math.inf)[:, 0]
    # ties go to the lowest index: whole numbers in the order of the values, then against that of the indices
    bits = (x + 0.0).view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long()
    order = (order << 32) + (0xFFFFFFFF - torch.arange(case["vocab"], device=x.device))
    best = torch.topk(order, case["top"]).values
    top_tokens = 0xFFFFFFFF - (best & 0xFFFFFFFF)
    top = x.gather(1, top_tokens)
    top = torch.where(total > 0, top - base - log_total, -math.inf)
    return [torch.where(inside, chosen, 0.0), entropy[:, 0], top, top_tokens.to(torch.int32)]


def _plain_log_probs_grad(case, logits, tokens, d_token, d_entropy):
    x = logits.float()
    base, total, entropy = _statistics(x)
    p = torch.where(total > 0, torch.exp(x - base) / total, 0.0)
    inside = (tokens >= 0) & (tokens < case["vocab"])
    g = torch.where(inside, d_token, 0.0)[:, None]
    slope = torch.where(p > 0, p * (g + d_entropy[:, None] * (x - base - total.log() + entropy)), 0.0)
    here = torch.arange(case["vocab"], device=x.device) == tokens[:, None]
    return [(torch.where(here & (total > 0), g, 0.0) - slope).to(logits.dtype)]


# ---- the work ----

def work(case):
    kind = case["kind"]
    if kind in ("heads", "heads_grad"):
        n = case["tokens"] * (case["heads"] + case["kv_heads"]) * case["dim"]
        size, small = SIZE[case["dtype"]], 4 * case["tokens"] * case["axes"]
        # rows in and out, gradients too for the second; squares, gain, rotation
        return {"bytes": size * n * 2 + small, "flops": 8 * n} if kind == "heads" else {"bytes": size * n * 3 + small, "flops": 18 * n}
    if kind == "attend":
        rows = case["seqs"] * case["queries"] * case["kv_heads"] * case["group"]
        # a prompt's keys are read once; lengths are uniform, and the first prompt has the most
        shared = case["prefix_keys"] * (1 + 0.75 * (case["prefixes"] - 1))
        mine = case["seqs"] * (case["keys"] + case["queries"]) / 2
        row = case["dim"] // 2 + case["dim"] // 32
        return {"bytes": int(2 * (shared + mine) * case["kv_heads"] * row) + 2 * SIZE[case["dtype"]] * rows * case["dim"],
                "flops": int(4 * case["dim"] * rows * (shared / case["prefixes"] + mine / case["seqs"]))}
    if kind in ("fork", "compact"):
        page = case["kv_heads"] * PAGE * (case["dim"] + case["dim"] // 16)
        each = max(1, min(case["slots"], case["pages"] // (2 * case["seqs"])))
        if kind == "fork":
            # kept entries in, whole tables out; about three of eight rows share their last page with another
            return {"bytes": 4 * case["rows"] * (each * 3 // 4 + case["slots"]) + case["pages"] + 2 * page * (case["rows"] * 3 // 8), "flops": 0}
        # about half of the pages in use lie above as many as there are
        in_use = min(case["seqs"] * each * 51 // 100, case["pages"])
        moved = min(case["moves"], in_use * (case["pages"] - in_use) // case["pages"])
        return {"bytes": 8 * case["seqs"] * case["slots"] + case["pages"] + 2 * page * moved, "flops": 0}
    n, size = case["rows"] * case["vocab"], SIZE[case["dtype"]]
    if kind == "log_probs":
        return {"bytes": n * size + case["rows"] * (12 + 8 * case["top"]), "flops": 6 * n}
    return {"bytes": 2 * n * size + 12 * case["rows"], "flops": 12 * n}


# ---- the results in 64 bits, from the definitions ----

def _exact_rotation(case, position, freq, axis):
    """e^(i angle) of each token's pairs."""
    per_pair = position.double().reshape(case["tokens"], -1).t()
    per_pair = per_pair[axis.long()] if axis is not None else per_pair.expand(freq.numel(), -1)
    angle = per_pair.t() * freq.double()
    return torch.polar(torch.ones_like(angle), angle)


def _exact_pairs(case, x):
    n = case["rotated"]
    if case["layout"] == "halves":
        return torch.complex(x[..., :n // 2].contiguous(), x[..., n // 2:n].contiguous())
    return torch.view_as_complex(x[..., :n].contiguous().unflatten(-1, (-1, 2)))


def _exact_turned(case, x, turn):
    z, n = _exact_pairs(case, x) * turn[:, None, :], case["rotated"]
    out = x.clone()
    if case["layout"] == "halves":
        out[..., :n // 2], out[..., n // 2:n] = z.real, z.imag
    else:
        out[..., :n] = torch.view_as_real(z).flatten(-2)
    return out


def _exact_heads(case, args):
    rows = args[:2] if case["kind"] == "heads" else args[:4]
    rest = args[len(rows):]
    turn = _exact_rotation(case, rest[0], rest[1], rest[2] if case["axes"] > 1 else None)
    out, gains = [], []
    for i, gain in enumerate(rest[-2:]):
        x, w = rows[i - 2].double(), gain.double()
        size = torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)
        if case["kind"] == "heads":
            out.append(_exact_turned(case, x / size * w, turn))
            continue
        g = _exact_turned(case, rows[i].double(), turn.conj())
        inner = (g * w * x).sum(-1, keepdim=True) / case["dim"]
        out.append(g * w / size - x * inner / size ** 3)
        gains.append((g * x / size).sum(0).sum(0))
    return out + gains


def _exact_values(codes, scales):
    table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=codes.device)
    table = torch.cat([table, -table])
    pairs = torch.stack([table[(codes % 16).long()], table[(codes // 16).long()]], -1).reshape(*codes.shape[:-1], -1)
    return pairs * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _exact_keys(cache, pages, count, dim, value):
    """The first `count` keys (or values) of some pages: [kv_head, key, dim]."""
    raw = cache[pages.long()].transpose(0, 1)
    c0, s0 = (PAGE * dim // 2, PAGE * dim + PAGE * dim // 32) if value else (0, PAGE * dim)
    codes, scales = raw[:, :, c0:c0 + PAGE * dim // 2], raw[:, :, s0:s0 + PAGE * dim // 32]
    return _exact_values(codes.reshape(raw.shape[0], -1, dim // 2), scales.reshape(raw.shape[0], -1, dim // 32))[:, :count]


def _exact_attend(case, q, cache, table, lengths, prefix_table, prefix_lengths, of):
    n, group, dim = case["queries"], case["group"], case["dim"]
    prefix = [[_exact_keys(cache, prefix_table[p], int(prefix_lengths[p]), dim, value) for value in (False, True)] for p in range(case["prefixes"])]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (length, p) in enumerate(zip(lengths.tolist(), of.tolist())):
        mine = [_exact_keys(cache, table[b], length, dim, value) for value in (False, True)]
        for i in range(n):
            seen = max(0, length - (n - 1 - i))
            k, v = ([torch.cat([prefix[p][w], mine[w][:, :seen]], 1) if 0 <= p < case["prefixes"] else mine[w][:, :seen] for w in (0, 1)])
            if k.shape[1] == 0:
                continue
            rows = q[b, i].double().unflatten(0, (-1, group))  # [kv_head, group, dim]
            w = torch.softmax(torch.matmul(rows, k.transpose(1, 2).contiguous()) * dim ** -0.5, -1)
            out[b, i] = torch.matmul(w, v).flatten(0, 1)
    return [out]


def _exact_log_probs(case, args):
    logits, tokens = args[:2]
    parts = []
    for first in range(0, case["rows"], 256):
        x, t = logits[first:first + 256].double(), tokens[first:first + 256].long()
        logp = x - torch.logsumexp(x, -1, keepdim=True)
        p = logp.exp()
        entropy = -torch.special.xlogy(p, p).sum(-1)
        chosen = torch.where(t >= 0, logp[torch.arange(len(t), device=x.device), t.clamp(min=0)], 0.0)
        if case["kind"] == "log_probs":
            parts.append([chosen, entropy, logp.topk(case["top"]).values])
            continue
        da, dh = (a[first:first + 256].double()[:, None] for a in args[2:])
        da = torch.where(t[:, None] >= 0, da, 0.0)
        g = -p * da - dh * (torch.special.xlogy(p, p) + p * entropy[:, None])
        g[torch.arange(len(t), device=x.device), t.clamp(min=0)] += da[:, 0]
        parts.append([g])
    whole = [torch.cat(p) for p in zip(*parts)]
    return whole + [None] if case["kind"] == "log_probs" else whole


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None  # whole numbers and bytes, which have no other value
    args = _inputs(case, seed)
    if case["kind"] in ("heads", "heads_grad"):
        return _exact_heads(case, args)
    return _exact_attend(case, *args) if case["kind"] == "attend" else _exact_log_probs(case, args)
