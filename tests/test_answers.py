"""Heads, shared-prefix attention, page tables and log probabilities, against the same in float64 (numpy) or with loops over
plain Python numbers, on identical inputs.

Tolerances count roundings. u = eps / 2 of the result's type is its one rounding; an f32 operation errs by 2^-24 of its result, a hardware
reciprocal square root, exponential or logarithm by 2^-22 at most, a sum of n terms in any order by n 2^-24 of the sum of their magnitudes.
"""
import ctypes
import random
import re
from fractions import Fraction

import numpy as np
import pytest

from accy_amd import hip
from accy_amd import tensor as T
from accy_amd import workloads as W
from conftest import hip_run
from test_mutated_programs import _mutate, _plan_status
from test_mx4 import HALF_STEP, _error, assert_within, cache_parts, decoded, encoded, finite_cache, floats, say, wide
from test_zz_no_alloc import _Bound, _capture, _hip_runtime, _same

E24 = 2.0 ** -24


# ---- recording and planning (no device) ----

def _rotation(b, tokens=5, pairs=8, axes=0, layout="halves"):
    if axes:
        return T.Rotation(b.input("i32", token=tokens, axis=axes), b.input("f32", pair=pairs), b.input("i32", pair=pairs), layout)
    return T.Rotation(b.input("i32", token=tokens), b.input("f32", pair=pairs), None, layout)


def test_recorded_types():
    b = T.Builder("p")
    q, k = b.input("bf16", token=5, head=6, dim=32), b.input("bf16", token=5, kv_head=2, dim=32)
    gain = b.input("f32", dim=32)
    norm = T.HeadNorm(gain, gain)
    assert [x.ty for x in b.rotate_heads(q, k, _rotation(b), norm)] == [q.ty, k.ty]
    assert [x.ty for x in b.rotate_heads(q, k, _rotation(b, axes=3, layout="neighbours"))] == [q.ty, k.ty]
    assert [x.ty for x in b.rotate_heads_grad(q, k, q, k, _rotation(b), norm)] == [q.ty, k.ty, gain.ty, gain.ty]
    assert len(b.rotate_heads_grad(q, k, q, k, _rotation(b))) == 2
    table, lengths, held = b.input("i32", seq=4, slot=7), b.input("i32", seq=4), b.input("i1", page=30)
    parents, room = b.input("i32", row=3), b.input("i32", row=3)
    f = b.fork_pages(table, lengths, parents, room, held, 64, tokens=2)
    assert f.pages.ty == T.Type("i32", (("row", 3), ("slot", 7))) and f.left.ty == T.Type("i32", ())
    assert f.lengths.ty == f.source.ty == f.target.ty == parents.ty and f.slots.ty == T.Type("i32", (("row", 3), ("token", 2)))
    c = b.compact_pages(table, held, ("move", 9))
    assert c.pages.ty == table.ty and c.source.ty == c.target.ty == T.Type("i32", (("move", 9),))
    cache = b.input_spec(T.cache_mx4_spec(30, 2, 64))
    assert cache.copy_pages(f.source, f.target).ty == cache.ty
    qs = b.input("f16", seq=4, query=2, head=6, dim=64)
    shared = (b.input("i32", prefix=2, at=3), b.input("i32", prefix=2), b.input("i32", seq=4))
    assert qs.attend_mx4(cache, table, lengths, shared=shared).ty == qs.ty
    x, tokens = b.input("bf16", row=4, vocab=50), b.input("i32", row=4)
    p = x.log_probs(tokens, "vocab", top=3)
    assert p.token.ty == p.entropy.ty == T.Type("f32", (("row", 4),)) and p.top.ty == T.Type("f32", (("row", 4), ("top", 3)))
    assert p.top_tokens.ty == T.Type("i32", (("row", 4), ("top", 3))) and x.log_probs(tokens, "vocab").top is None
    assert x.log_probs_grad(tokens, p.token, p.entropy, "vocab").ty == x.ty


def test_recording_refuses_what_does_not_fit():
    b = T.Builder("p")
    q, k = b.input("bf16", token=5, head=6, dim=32), b.input("bf16", token=5, kv_head=2, dim=32)
    rotation, gain = _rotation(b), b.input("bf16", dim=32)
    heads = lambda *a, **kw: _error(lambda: b.rotate_heads(*a, **kw))  # noqa: E731
    assert heads(q, b.input("f16", token=5, kv_head=2, dim=32), rotation) == "DTypeMismatch"
    assert heads(q, b.input("bf16", token=4, kv_head=2, dim=32), rotation) == "ShapeMismatch"
    assert heads(q, b.input("bf16", token=5, kv_head=2, dim=64), rotation) == "ShapeMismatch"
    assert heads(b.input("i32", token=5, head=6, dim=32), k, rotation) == "DTypeMismatch"
    assert heads(q, k, _rotation(b, tokens=4)) == "ShapeMismatch" and heads(q, k, _rotation(b, pairs=17)) == "InvalidDimension"
    assert heads(q, k, _rotation(b, pairs=0)) == "InvalidDimension" and heads(q, k, _rotation(b, layout="thirds")) == "InvalidDimension"
    assert heads(q, k, T.Rotation(b.input("f32", token=5), rotation.frequencies)) == "DTypeMismatch"
    assert heads(q, k, T.Rotation(rotation.positions, rotation.frequencies, b.input("i32", pair=8))) == "ShapeMismatch"
    assert heads(q, k, rotation, T.HeadNorm(gain, b.input("f16", dim=32))) == "DTypeMismatch"
    assert heads(q, k, rotation, T.HeadNorm(gain, b.input("bf16", dim=31))) == "ShapeMismatch"
    wide_head = b.input("bf16", token=5, head=1, dim=514)
    assert heads(wide_head, wide_head, rotation) == "InvalidDimension"
    assert _error(lambda: b.rotate_heads_grad(k, k, q, k, rotation)) == "ShapeMismatch"
    table, lengths, held = b.input("i32", seq=4, slot=7), b.input("i32", seq=4), b.input("i1", page=30)
    rows = b.input("i32", row=3)
    assert _error(lambda: b.fork_pages(table, lengths, rows, b.input("i32", row=4), held, 64)) == "ShapeMismatch"
    assert _error(lambda: b.fork_pages(table, rows, rows, rows, held, 64)) == "ShapeMismatch"
    assert _error(lambda: b.fork_pages(table, lengths, rows, rows, rows, 64)) == "DTypeMismatch"
    assert _error(lambda: b.fork_pages(table, lengths, rows, rows, held, 0)) == "InvalidDimension"
    assert _error(lambda: b.fork_pages(table, lengths, rows, rows, held, 64, tokens=0)) == "InvalidDimension"
    assert _error(lambda: b.compact_pages(table, held, ("move", 31))) == "InvalidDimension"
    assert _error(lambda: b.compact_pages(lengths, held, ("move", 3))) == "RankMismatch"
    assert _error(lambda: held.copy_pages(rows, lengths)) == "ShapeMismatch"
    assert _error(lambda: held.copy_pages(gain, gain)) == "DTypeMismatch"
    x, tokens, d = b.input("f32", row=4, vocab=50), b.input("i32", row=4), b.input("f32", row=4)
    assert _error(lambda: x.log_probs(tokens, "row")) == "InvalidPermutation" and _error(lambda: x.log_probs(tokens, "no")) == "AxisNotFound"
    assert _error(lambda: x.log_probs(tokens, "vocab", top=51)) == "InvalidDimension"
    assert _error(lambda: b.input("f32", row=4, vocab=99).log_probs(tokens, "vocab", top=65)) == "InvalidDimension"
    assert _error(lambda: x.log_probs(d, "vocab")) == "DTypeMismatch" and _error(lambda: x.log_probs(lengths, "vocab")) == "ShapeMismatch"
    assert _error(lambda: x.log_probs_grad(tokens, tokens, d, "vocab")) == "DTypeMismatch"
    cache, qs = b.input_spec(T.cache_mx4_spec(30, 2, 64)), b.input("f16", seq=4, head=6, dim=64)
    pre = b.input("i32", prefix=2, at=3), b.input("i32", prefix=2), b.input("i32", seq=4)
    assert _error(lambda: qs.attend_mx4(cache, table, lengths, shared=pre[:2])) == "InvalidDimension"
    assert _error(lambda: qs.attend_mx4(cache, table, lengths, shared=(pre[0], pre[1], pre[1]))) == "ShapeMismatch"
    assert _error(lambda: qs.attend_mx4(cache, table, lengths, shared=(pre[0], d, pre[2]))) == "DTypeMismatch"


I32 = lambda *e: ("i32", e)  # noqa: E731
F32 = lambda *e: ("f32", e)  # noqa: E731


@pytest.mark.parametrize("call,operands,groups,result,reason", [
    ("heads.queries", [F32(3, 2, 8), F32(3, 1, 8), I32(3), F32(4)], [(0,), (1,), (2, 3)], F32(3, 2, 9), "operand's type"),
    ("heads.queries", [F32(3, 2, 8), F32(3, 1, 8), I32(3), F32(4)], [(0,), (1,), (2,)], F32(3, 2, 8), "group of 2 to 3"),
    ("heads.queries", [F32(3, 2, 8), F32(3, 1, 8), I32(3), F32(5)], [(0,), (1,), (2, 3)], F32(3, 2, 8), "one to dim / 2"),
    ("heads.keys", [F32(3, 2, 8), F32(3, 1, 6), I32(3), F32(3)], [(0,), (1,), (2, 3)], F32(3, 1, 6), "of one type"),
    ("heads.keys_neighbours", [F32(3, 2, 8), F32(3, 1, 8), I32(4), F32(3)], [(0,), (1,), (2, 3)], F32(3, 1, 8), "position for every token"),
    ("heads.queries", [F32(3, 2, 8), F32(3, 1, 8), I32(3), F32(4), F32(8), F32()], [(0,), (1,), (2, 3), (4, 4, 5)], F32(3, 2, 8), "f32 constant"),
    ("heads.d_queries", [F32(3, 2, 8), F32(3, 1, 8), I32(3), F32(4)], [(0, 1), (1, 0), (2, 3)], F32(3, 2, 8), "gradients of the results"),
    ("heads.d_key_gain", [F32(3, 2, 8), F32(3, 1, 8), I32(3), F32(4)], [(0, 1), (0, 1), (2, 3)], F32(8), "without a norm"),
    ("heads.thirds", [F32(3, 2, 8)], [(0,)], F32(3, 2, 8), "not supported"),
    ("pages.copy", [F32(3, 2), I32(2), I32(3)], [(0,), (1,), (2,)], F32(3, 2), "source and target"),
    ("pages.copy", [F32(3, 2), I32(2), I32(2)], [(0,), (1,), (2,)], F32(4, 2), "cache's type"),
    ("pages.fork_table", [I32(3, 2), I32(3), I32(4), ("i1", (9,)), I32()], [(0, 1), (2, 2), (3,), (4,)], I32(4, 2), "i32 constant"),
    ("pages.fork_table", [I32(3, 2), I32(3), I32(4), ("i1", (9,)), I32()], [(0,), (2, 2), (3,), (4,)], I32(4, 2), "group of 2"),
    ("pages.compact_table", [I32(3, 2), ("i1", (9,)), 5], [(0,), (1,), (2,)], I32(3, 3), "as the table"),
    ("pages.compact_source", [I32(3, 2), ("i1", (9,)), 5], [(0,), (1,), (2,)], I32(4), "i32 [move]"),
    ("pages.compact_source", [I32(3, 2), ("i1", (9,)), 10], [(0,), (1,), (2,)], I32(10), "as many as pages"),
    ("pages.compact_target", [I32(3, 2), ("i1", (9,)), I32()], [(0,), (1,), (2,)], I32(9), "i32 constant"),
    ("pages.compact_target", [I32(3, 2), ("i1", (9,))], [(0,), (1,)], I32(9), "3 operands"),
    ("pages.compact_source", [I32(3, 2), ("i1", ((1 << 24) + 1,)), 5], [(0,), (1,), (2,)], I32(5), "2^24 pages"),
    ("logits.token", [F32(3, 9), I32(3)], [(0,), (1,)], F32(3, 1), "f32 [row"),
    ("logits.top", [F32(3, 9), I32(3)], [(0,), (1,)], F32(3, 10), "1 to 64 alternatives"),
    ("logits.top_tokens", [F32(3, 9), I32(3)], [(0,), (1,)], F32(3, 2), "of tokens i32"),
    ("logits.entropy", [F32(3, 0), I32(3)], [(0,), (1,)], F32(3), "1 to 2^30"),
    ("logits.grad", [F32(3, 9), I32(3), F32(3)], [(0,), (1,), (2,), (2,)], F32(3, 8), "logits' type"),
    ("mx4.attend_shared", [F32(3, 2, 64), ("u8", (4, 2, 32 * 68)), I32(3, 2), I32(3), I32(2, 5)], [(0,), (1,), (2, 3), (4, 3, 3)], F32(3, 2, 64), "shared lengths"),
    ("mx4.attend_shared", [F32(3, 2, 64), ("u8", (4, 2, 32 * 68)), I32(3, 2), I32(3), I32(1025, 5), I32(1025)], [(0,), (1,), (2, 3), (4, 5, 3)], F32(3, 2, 64),
     "1 to 1024 prefixes"),
    ("mx4.attend_shared", [F32(3, 2, 64), ("u8", (4, 2, 32 * 68)), I32(3, 2), I32(3)], [(0,), (1,), (2,), (3,)], F32(3, 2, 64), "group of 2"),
])
def test_planning_refuses_what_the_wire_may_carry(call, operands, groups, result, reason):
    dims = lambda i, e: [(f"a{i}_{j}", n) for j, n in enumerate(e)]  # noqa: E731

    def body(b, a):
        a = [a.pop(0) if isinstance(o, tuple) else b.full("i32", o) for a in [list(a)] for o in operands]
        args = [a[g[0]] if len(g) == 1 else b._group(*(a[i] for i in g)) for g in groups]
        return b.custom_call(f"accy.{call}", 1, args, T.Type(result[0], tuple(dims("r", result[1]))))
    prog = T.define("bad", [T.spec(o[0], *dims(i, o[1])) for i, o in enumerate(operands) if isinstance(o, tuple)], body)
    with pytest.raises(hip.HipError) as e:
        hip.plan_source(prog)
    assert e.value.status == hip.COMPILE_FAILED and reason in e.value.message and f"accy.{call}" in e.value.message


@pytest.mark.parametrize("name", ["fork_page", "fork_", "fork_tables", "compact_left", "compact_"])
def test_a_name_that_is_none_is_refused_beside_those_that_are(name):
    """A call of a set without such a result, on the operands of one that there is: neither may be passed over."""
    def body(b, a):
        fork = name.startswith("fork")
        args = [b._group(a[0], a[1]), b._group(a[2], a[2]), a[3], b.full("i32", 64)] if fork else [a[0], a[3], b.full("i32", 5)]
        there = "fork_lengths" if fork else "compact_source"
        calls = [b.custom_call(f"accy.pages.{n}", 1, args, T.Type("i32", (("row", 5),))) for n in (name, there)]
        return calls if first else calls[::-1]
    for first in (True, False):
        prog = T.define("p", [T.spec("i32", seq=4, slot=7), T.spec("i32", seq=4), T.spec("i32", row=5), T.spec("i1", page=30)], body)
        with pytest.raises(hip.HipError) as e:
            hip.plan_source(prog)
        assert e.value.status == hip.COMPILE_FAILED and f"accy.pages.{name}" in e.value.message


def test_groups_are_operands_only():
    spec = [T.spec("f32", r=2)]
    for body in (lambda b, a: b._group(a[0], a[0]), lambda b, a: b.broadcast(b._group(a[0], a[0]), [("r", 2)]),
                 lambda b, a: b.scan(2, [b._group(a[0], a[0])], lambda bb, c: c)):
        with pytest.raises(hip.HipError) as e:
            hip.plan_source(T.define("p", spec, body))
        assert e.value.status == hip.COMPILE_FAILED


def _labels(prog):
    return [line.split()[1].split(":")[0] for line in hip.plan_source(prog).splitlines() if line.startswith("// ") and " grid " in line]


def test_results_of_one_call_are_one_kernel():
    row, spec = T.spec("i32", row=3), [T.spec("f32", row=3, vocab=40), T.spec("i32", row=3)]

    def both(b, a):
        p, more = a[0].log_probs(a[1], "vocab", top=4), a[0].log_probs(a[1], "vocab", top=2)
        return [p.token, p.entropy, p.top, p.top_tokens, more.top]
    assert _labels(T.define("p", spec, both)) == ["log_probs", "log_probs"]  # (the second for two alternatives)
    fork = T.define("p", [T.spec("i32", seq=4, slot=7), T.spec("i32", seq=4), row, row, T.spec("i1", page=30)],
                    lambda b, a: [x for f in [b.fork_pages(*a, 64)] for x in (f.pages, f.lengths, f.source, f.target, f.left, f.slots)])
    assert _labels(fork) == ["fork"]
    # two updates in a row are one buffer's: nothing is copied between them
    step = W.answers_step_mx4_program(8, 8, 128, 4, 2, 64, 300, 40, 32, 6, 2, 3, 4)
    assert _labels(step) == ["fork", "copy_pages", "row", "quantize", "mx4", "mx4", "heads", "mx4", "cache_write", "mx4_attend", "mx4_join", "quantize", "mx4", "row",
                             "quantize", "mx4", "log_probs"]


ALTERNATIVES = [((1, 5), ("x.top_tokens", "y.top")), ((5, 3), ("x.top_tokens", "y.top")), ((2, 4), ("y.top", "x.top_tokens", "y.top_tokens", "x.token")), ((4, 2), ("x.top", "y.top_tokens")),
                ((3, 7), ("x.entropy", "y.top_tokens", "x.top")), ((6, 6), ("x.top", "y.top_tokens", "y.top"))]


def _two_numbers_program(numbers, names, rows=3, vocab=40):
    def body(b, a):
        both = dict(zip("xy", (a[0].log_probs(a[1], "vocab", top=n) for n in numbers)))
        return [getattr(both[n[0]], n[2:]) for n in names]
    return T.define("two", [T.spec("f32", row=rows, vocab=vocab), T.spec("i32", row=rows)], body)


@pytest.mark.parametrize("numbers,names", ALTERNATIVES)
def test_every_result_of_two_numbers_of_alternatives_has_a_kernel(numbers, names):
    """Results of two calls on the same logits that differ in their alternatives alone: each is written, by a kernel of its own number."""
    source = hip.plan_source(_two_numbers_program(numbers, names))
    # (results are the pointers of a kernel that are not const)
    results = [len(re.findall(r"(?<!const )(?:float|int|i32_t)\* __restrict__ a\d+", line)) for line in source.splitlines() if "__global__" in line]
    assert sum(results) == len(names), source


def test_every_mutated_program_gets_a_status():
    lib, rng = hip.library(), random.Random(4)
    spec = [T.spec("f32", r=2, v=9), T.spec("i32", r=2), *[T.spec("f32", r=2)] * 2]
    bases = [p.encode() for p in (W.answers_step_mx4_program(2, 3, 64, 2, 1, 32, 40, 6, 32, 2, 1, 1, 2), _grad_program(3, 2, 1, 8, 4, 2, "halves", "f32", True),
                                  T.define("g", spec, lambda b, a: a[0].log_probs_grad(*a[1:], "v")))]
    seen = {_plan_status(lib, _mutate(rng.choice(bases), rng)) for _ in range(1500)}
    assert seen <= set(range(9)) and {0, 1} <= seen


# ---- heads ----

def _heads_specs(tokens, hq, hk, dim, pairs, axes, dtype, norm, gains=None):
    position = T.spec("i32", token=tokens, axis=axes) if axes else T.spec("i32", token=tokens)
    return [T.spec(dtype, token=tokens, head=hq, dim=dim), T.spec(dtype, token=tokens, kv_head=hk, dim=dim), position, T.spec("f32", pair=pairs),
            *([T.spec("i32", pair=pairs)] if axes else []), *([T.spec(gains or dtype, dim=dim)] * 2 if norm else [])]


def _operands(b, a, axes, layout, norm, eps):
    return T.Rotation(a[0], a[1], a[2] if axes else None, layout), T.HeadNorm(a[-2], a[-1], eps) if norm else None


def _heads_program(tokens, hq, hk, dim, pairs, axes, layout, dtype, norm, gains=None, eps=1e-5):
    return T.define("heads", _heads_specs(tokens, hq, hk, dim, pairs, axes, dtype, norm, gains),
                    lambda b, a: list(b.rotate_heads(a[0], a[1], *_operands(b, a[2:], axes, layout, norm, eps))))


def _grad_program(tokens, hq, hk, dim, pairs, axes, layout, dtype, norm, gains=None, eps=1e-5):
    specs = _heads_specs(tokens, hq, hk, dim, pairs, axes, dtype, norm, gains)
    return T.define("heads_grad", specs[:2] + specs, lambda b, a: list(b.rotate_heads_grad(*a[:4], *_operands(b, a[4:], axes, layout, norm, eps))))


def _angles(position, freq, axes):
    position = position.astype(np.float64)
    if axes is None:
        return position[:, None] * freq.astype(np.float64)
    inside = (axes >= 0) & (axes < position.shape[1])
    return np.where(inside, position[:, np.clip(axes, 0, position.shape[1] - 1)], 0.0) * freq.astype(np.float64)


def _pairs(x, pairs, layout):
    return (x[..., :pairs], x[..., pairs:2 * pairs]) if layout == "halves" else (x[..., 0:2 * pairs:2], x[..., 1:2 * pairs:2])


def _turned(x, angle, pairs, layout):
    """x with its pairs turned, and the sum of both magnitudes of a pair at each of its places."""
    out, size = x.copy(), np.abs(x)
    (a, b), (oa, ob), (sa, sb) = (_pairs(v, pairs, layout) for v in (x, out, size))
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = a.copy(), b.copy()
    oa[...], ob[...] = a * c - b * s, b * c + a * s
    sa[...] = sb[...] = np.abs(a) + np.abs(b)
    return out, size


def _heads_want(x, gain, angle, pairs, layout, norm, eps):
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps) if norm else 1.0
    return _turned(x * r * (gain if norm else 1.0), angle, pairs, layout)


def _grad_want(dy, x, gain, angle, pairs, layout, norm, eps):
    """dx, d gain and bounds of the magnitudes that they are sums of."""
    g, size = _turned(dy, -angle, pairs, layout)
    if not norm:
        return g, None, size, None
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    n, gw, sw = x * r, g * gain, size * np.abs(gain)
    dx = r * (gw - n * (gw * n).mean(-1, keepdims=True))
    return dx, (g * n).sum((0, 1)), r * (sw + np.abs(n) * (sw * np.abs(n)).mean(-1, keepdims=True)), (size * np.abs(n)).sum((0, 1))


HEADS = [(1, 1, 1, 2, 1, 0, "halves"), (1, 16, 4, 128, 64, 0, "halves"), (3, 5, 1, 10, 3, 0, "neighbours"), (7, 12, 3, 96, 32, 3, "neighbours"),
         (2, 3, 2, 80, 20, 2, "halves"), (65, 2, 2, 64, 32, 1, "halves"), (33, 4, 1, 256, 128, 0, "neighbours"), (5, 1, 3, 250, 125, 0, "halves"),
         (2, 2, 1, 512, 255, 4, "halves"), (4, 2, 1, 7, 3, 0, "halves"), (3, 0, 2, 32, 16, 0, "halves"), (3, 2, 0, 32, 12, 0, "neighbours"), (4500, 1, 1, 24, 8, 0, "neighbours"), (2100, 3, 2, 32, 16, 0, "halves")]


def _heads_inputs(tokens, hq, hk, dim, pairs, axes, dtype, gains, rng):
    q, k = (floats(rng.standard_normal((tokens, h, dim)) * 3, dtype) for h in (hq, hk))
    far = np.array([0, 1, -1, 131071, 2 ** 31 - 1, -2 ** 31])
    position = rng.integers(0, 200000, (tokens, axes) if axes else tokens).astype(np.int32)
    position.reshape(-1)[:6] = far[:position.size].astype(np.int32)[:6]
    freq = (10000.0 ** (-np.arange(pairs) / pairs)).astype(np.float32)
    axis = rng.integers(-1, axes + 1, pairs).astype(np.int32) if axes else None
    gain = [floats(rng.standard_normal(dim), gains) for _ in range(2)]
    return q, k, position, freq, axis, gain


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,norm,gains", [("bf16", True, "bf16"), ("f16", True, "f32"), ("f32", True, "f32"), ("f32", False, "f32"), ("bf16", False, "bf16")])
@pytest.mark.parametrize("tokens,hq,hk,dim,pairs,axes,layout", HEADS)
def test_heads_and_their_gradient(tokens, hq, hk, dim, pairs, axes, layout, dtype, norm, gains):
    """A row's sum of squares errs by dim 2^-24, its root by 2^-22, n and the gain's product by two roundings, the turn by two products, their sum and
    cosines off by 2^-22: dim + 24 steps of 2^-24 of the pair's magnitudes. The gradient twice that; a gain's sum over rows by as many
    more steps as there are rows."""
    rng = np.random.default_rng(tokens + dim)
    eps = float(np.float32(1e-5))
    q, k, position, freq, axis, gain = _heads_inputs(tokens, hq, hk, dim, pairs, axes, dtype, gains, rng)
    angle = _angles(position, freq, axis)
    rest = [position, freq, *([axis] if axes else []), *(gain if norm else [])]
    args = (tokens, hq, hk, dim, pairs, axes, layout, dtype, norm, gains)
    least = 2.0 ** -25 if dtype == "f16" else 1e-37
    say(f"heads {args}")
    got = hip_run(_heads_program(*args), [q, k, *rest])
    for y, x, g in zip(got, (q, k), gain):
        want, size = _heads_want(wide(x, dtype), wide(g, gains), angle, pairs, layout, norm, eps)
        assert_within(wide(y, dtype), want, HALF_STEP[dtype] * np.abs(want) + (dim + 24) * E24 * size + least)
    dq, dk = (floats(rng.standard_normal(x.shape), dtype) for x in (q, k))
    say(f"heads' gradient {args}")
    got = hip_run(_grad_program(*args), [dq, dk, q, k, *rest])
    for i, (dy, x, g) in enumerate(((dq, q, gain[0]), (dk, k, gain[1]))):
        dx, dg, size, total = _grad_want(wide(dy, dtype), wide(x, dtype), wide(g, gains), angle, pairs, layout, norm, eps)
        assert_within(wide(got[i], dtype), dx, HALF_STEP[dtype] * np.abs(dx) + 2 * (dim + 24) * E24 * size + least, "dx")
        if norm:
            rows = tokens * x.shape[1]
            assert_within(wide(got[2 + i], gains), dg, HALF_STEP[gains] * np.abs(dg) + (dim + 24 + rows) * E24 * total + least, "d gain")


def test_the_formulas_gradients_are_differences():
    """Gradients that the kernels are checked against, against central differences of the formulas in 64 bits: error h^2 of a function of order 1."""
    rng = np.random.default_rng(3)
    for layout in ("halves", "neighbours"):
        x, dy, gain = rng.standard_normal((3, 2, 10)), rng.standard_normal((3, 2, 10)), rng.standard_normal(10)
        angle = rng.standard_normal((3, 4))
        f = lambda x, gain: (_heads_want(x, gain, angle, 4, layout, True, 1e-5)[0] * dy).sum()  # noqa: E731
        dx, dg, _, _ = _grad_want(dy, x, gain, angle, 4, layout, True, 1e-5)
        _differences(f, (x, gain), (dx, dg))
    x, t = rng.standard_normal((4, 7)) * 2, np.array([3, 0, -1, 6])
    a, h = rng.standard_normal(4), rng.standard_normal(4)

    def loss(x):
        token, entropy, _ = _log_probs_want(x, t)
        return (np.where(t >= 0, a * token, 0) + h * entropy).sum()
    _differences(loss, (x,), (_grad_logits_want(x, t, a, h)[0],))


def _differences(f, at, grads, step=1e-5):
    for i, (x, g) in enumerate(zip(at, grads)):
        for j in np.ndindex(x.shape):
            lo, hi = [v.copy() for v in at], [v.copy() for v in at]
            lo[i][j] -= step
            hi[i][j] += step
            assert abs((f(*hi) - f(*lo)) / (2 * step) - g[j]) <= 1e-7 * (1 + np.abs(g).max())


def _turns_exactly(position, freq):
    """cos and sin of position * freq for whole positions and f32 frequencies, reduced in fractions with 80 digits of pi."""
    pi = Fraction("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899")
    turns = np.array([[float((lambda t: t - round(t))(int(p) * Fraction(float(f)) / (2 * pi))) for f in freq] for p in position])
    return np.cos(2 * np.pi * turns), np.sin(2 * np.pi * turns)


@pytest.mark.gpu
@pytest.mark.parametrize("layout", ["halves", "neighbours"])
def test_heads_of_far_positions_and_of_fast_pairs(layout):
    """Every 32-bit position is exact, at frequencies from 1e-4 to 2e4. A cosine is off by its argument's rounding, an ulp and a half of the polynomial
    and the rounding of the reduced angle, 4 steps of 2^-24; two products and a sum are 3 more."""
    position = np.array([2 ** 31 - 1, -2 ** 31, 2 ** 31 - 2, 2 ** 30 + 12345, -1999999999, 123456789, 16777217, -99999, 1, 0], np.int32)
    freq = np.float32([1, 0.7, 0.999, 0.1, 1e-4, 3.3, 10, 100.1, 1000.7, 19999.9])
    rng = np.random.default_rng(4)
    q, k = (rng.standard_normal((10, h, 22)).astype(np.float32) for h in (3, 1))
    c, s = (x[:, None] for x in _turns_exactly(position, freq))
    say(f"far positions {layout}")
    got = hip_run(_heads_program(10, 3, 1, 22, 10, 0, layout, "f32", False), [q, k, position, freq])
    back = hip_run(_grad_program(10, 3, 1, 22, 10, 0, layout, "f32", False), [q, k, q, k, position, freq])
    for x, there, here in zip((q, k), got, back):
        x = x.astype(np.float64)
        a, b = _pairs(x, 10, layout)
        size = np.abs(a) + np.abs(b)
        for y, sign in ((there, 1), (here, -1)):
            ya, yb = _pairs(y.astype(np.float64), 10, layout)
            assert_within(ya, a * c - sign * b * s, 7 * E24 * size, "first of a pair")
            assert_within(yb, b * c + sign * a * s, 7 * E24 * size, "second of a pair")
            assert np.array_equal(y[..., 20:], x[..., 20:].astype(np.float32))


@pytest.mark.gpu
def test_heads_one_result_alone_and_rows_that_are_no_numbers():
    """Only the keys asked for; a row with a NaN or an infinity is one by itself; a row of zeros stays zeros; repeated calls give the same bits."""
    rng = np.random.default_rng(8)
    args = (9, 3, 2, 48, 16, 0, "halves", "f32", True, "f32")
    q, k, position, freq, _, gain = _heads_inputs(9, 3, 2, 48, 16, 0, "f32", "f32", rng)
    k[0, 0, 5], k[1, 1, 47], k[2, 0] = np.nan, np.inf, 0.0
    ins = [q, k, position, freq, *gain]
    both = hip_run(_heads_program(*args), ins)
    alone = hip_run(T.define("keys", _heads_specs(9, 3, 2, 48, 16, 0, "f32", True),
                             lambda b, a: b.rotate_heads(a[0], a[1], *_operands(b, a[2:], 0, "halves", True, 1e-5))[1]), ins)[0]
    assert np.array_equal(both[1], alone, equal_nan=True)
    assert np.isnan(alone[0, 0]).all() and np.isnan(alone[1, 1]).any() and not alone[2, 0].any()
    assert np.isfinite(np.delete(alone.reshape(18, 48), [0, 3], 0)).all()
    k[:3] = 1
    grads = [hip_run(_grad_program(*args), [q, k, q, k, position, freq, *gain]) for _ in range(2)]
    _same(grads[0], grads[1])
    # no tokens: nothing of them, and sums of nothing
    none = (0, 3, 2, 48, 16, 0, "halves", "f32", True, "f32")
    ins = [q[:0], k[:0], q[:0], k[:0], position[:0], freq, *gain]
    got = hip_run(_grad_program(*none), ins)
    assert got[0].shape == (0, 3, 48) and not got[2].any() and not got[3].any()


# ---- log probabilities ----

def _log_probs_want(x, tokens):
    """Log probabilities of tokens, entropies and all log probabilities in float64; rows of no number are NaN."""
    with np.errstate(all="ignore"):
        bad = np.isnan(x).any(-1) | (x == np.inf).any(-1)
        m = np.where(np.isneginf(x).all(-1), 0.0, np.where(bad, 0.0, np.nan_to_num(x, nan=0.0, neginf=-np.inf).max(-1)))[..., None]
        e = np.exp(x - m)
        total = e.sum(-1, keepdims=True)
        logp = np.where(total > 0, (x - m) - np.log(total), -np.inf)
        p = np.where(total > 0, e / total, 0.0)
        entropy = -np.where(p > 0, p * np.where(np.isfinite(logp), logp, 0.0), 0.0).sum(-1)
        logp[bad], entropy[bad] = np.nan, np.nan
        inside = (tokens >= 0) & (tokens < x.shape[-1])
        token = np.where(inside, logp[np.arange(len(x)), np.clip(tokens, 0, x.shape[-1] - 1)], 0.0)
    return token, entropy, logp


def _grad_logits_want(x, tokens, a, h):
    """The gradient and the magnitudes that it is a sum of."""
    _, entropy, logp = _log_probs_want(x, tokens)
    with np.errstate(all="ignore"):
        p = np.where(np.isneginf(logp), 0.0, np.exp(logp))
        inside = (tokens >= 0) & (tokens < x.shape[-1])
        g = np.where(inside, a, 0.0)[:, None]
        here = (np.arange(x.shape[-1]) == tokens[:, None]) & ~np.isneginf(x).all(-1)[:, None]
        lp = np.where(p > 0, logp, 0.0)
        out = here * g - p * (g + h[:, None] * (lp + entropy[:, None]))
        size = here * np.abs(g) + p * (np.abs(g) + np.abs(h)[:, None] * (np.abs(lp) + np.abs(entropy)[:, None]))
    return out, size


def _steps(x):
    """How far a log probability may be off: two roundings of the largest magnitudes that are subtracted and one of their logarithm's, the exponents'
    of terms that weigh, and sums of at most 64 terms a thread and batch, of the batches and of the joins."""
    finite = np.where(np.isfinite(x), x, 0.0)
    n = x.shape[-1]
    return E24 * (200 + n / 2048 + 4 * np.abs(finite).max(-1, initial=0.0).clip(max=1e6) + 8 * np.log(n + 1))


def _check_log_probs(x, tokens, top, dtype):
    rows, n = x.shape
    prog = T.define("log_probs", [T.spec(dtype, row=rows, vocab=n), T.spec("i32", row=rows)],
                    lambda b, a: [v for p in [a[0].log_probs(a[1], "vocab", top=top)] for v in (p.token, p.entropy, p.top, p.top_tokens)][:4 if top else 2])
    got = hip_run(prog, [x, tokens])
    v = wide(x, dtype)
    token, entropy, logp = _log_probs_want(v, tokens)
    tol = _steps(v)
    assert_within(got[0], token, tol + 2 * E24 * np.abs(token), "token")
    assert_within(got[1], entropy, 4 * tol * (2 + np.log(n + 1)), "entropy")
    if not top:
        return got
    for r in range(rows):
        order = np.argsort(np.where(np.isnan(v[r]), np.inf, -v[r]), kind="stable")[:top]
        order = np.where(np.isnan(v[r][order]), -1, order)
        assert np.array_equal(got[3][r], order), (r, got[3][r], order)
        want = np.where(order < 0, np.nan, logp[r][order])
        assert_within(got[2][r], want, tol[r] + 2 * E24 * np.abs(want), "top")
    return got


LOGITS = [(1, 1, 1), (3, 2, 2), (5, 7, 3), (4, 9, 9), (2, 63, 20), (7, 500, 32), (3, 1031, 64), (2, 4096, 1), (5, 20011, 5), (1, 131073, 8), (600, 515, 4), (513, 5003, 20),
          (530, 9000, 0), (3, 40000, 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,n,top", LOGITS)
def test_log_probs(rows, n, top, dtype):
    rng = np.random.default_rng(rows + n)
    x = rng.standard_normal((rows, n)) * 2.5
    x[::3, 1::2] = -np.inf  # (the first place stays)
    tokens = rng.integers(-2, n + 2, rows).astype(np.int32)
    tokens[-1] = 2 ** 31 - 1
    say(f"log_probs {rows} {n} {top} {dtype}")
    _check_log_probs(floats(x, dtype), tokens, top, dtype)


def _hard_rows(n, dtype):
    """Rows where it can go wrong, each of n logits."""
    low = {"bf16": -3.3895313892515355e38, "f16": -65504.0, "f32": -3.4028234663852886e38}[dtype]
    rng = np.random.default_rng(6)
    base = rng.standard_normal(n)
    rows = {"masked": np.full(n, -np.inf), "lowest": np.full(n, low), "equal": np.full(n, 1.5), "rising": np.arange(n) * (60000.0 / n), "falling": -np.arange(n) * (60000.0 / n),
            "one": np.where(np.arange(n) == n // 2, 3.0, -np.inf), "peak": np.where(np.arange(n) == n - 1, 40000.0, base), "low peak": np.where(np.arange(n) == n // 3, -7.0, low),
            "zeros": np.where(np.arange(n) % 2 == 0, -0.0, 0.0), "masked low": np.where(np.arange(n) % 3 == 0, low, base), "nan": np.where(np.arange(n) == 5, np.nan, base),
            "infinity": np.where(np.arange(n) == n - 2, np.inf, base), "all nan": np.full(n, np.nan), "few": np.where(np.arange(n) < 3, 1.0, np.nan),
            "negative": -100 - np.abs(base), "two heights": np.where(np.arange(n) < n // 2, -5.0, 30000.0), "bottom": np.full(n, -50000.0)}
    return np.stack([np.asarray(v, np.float64) for v in rows.values()])


@pytest.mark.gpu
@pytest.mark.parametrize("numbers,names", ALTERNATIVES)
@pytest.mark.parametrize("rows,vocab", [(3, 40), (2, 9000)])
def test_results_of_two_numbers_of_alternatives(rows, vocab, numbers, names):
    rng = np.random.default_rng(vocab)
    x, tokens = rng.standard_normal((rows, vocab)).astype(np.float32), rng.integers(0, vocab, rows).astype(np.int32)
    token, entropy, logp = _log_probs_want(x.astype(np.float64), tokens)
    order = np.argsort(-x, axis=1, kind="stable")
    say(f"two numbers {numbers} {names} {rows} {vocab}")
    for got, name in zip(hip_run(_two_numbers_program(numbers, names, rows, vocab), [x, tokens]), names):
        best = order[:, :numbers[name[0] == "y"]]
        want = {"token": token, "entropy": entropy, "top": np.take_along_axis(logp, best, 1), "top_tokens": best}[name[2:]]
        if name[2:] == "top_tokens":
            assert np.array_equal(got, want)
            continue
        # as in _check_log_probs
        tol = _steps(x)[:, None] * (4 * (2 + np.log(vocab + 1)) if name[2:] == "entropy" else 1)
        assert_within(got.reshape(rows, -1), want.reshape(rows, -1), tol + 2 * E24 * np.abs(want.reshape(rows, -1)), name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("n,copies", [(100, 1), (2500, 1), (12001, 1), (2500, 31), (12001, 31)])
def test_log_probs_of_hard_rows(n, copies, dtype):
    """Everything masked or of the type's lowest value, equal, rising (a list of alternatives is full at once) and falling rows, zeros of both signs, NaN and
    infinities, in a few rows (several workgroups each) and in more than 512 (one)."""
    x = floats(np.tile(_hard_rows(n, dtype), (copies, 1)), dtype)
    tokens = np.arange(len(x)).astype(np.int32) * 7 % n
    say(f"hard rows {n} {copies} {dtype}")
    for top in (1, 20):
        _check_log_probs(x, tokens, top, dtype)
    if copies == 1:
        _check_grad(x, tokens, dtype)


def _check_grad(x, tokens, dtype):
    rows, n = x.shape
    rng = np.random.default_rng(rows)
    a, h = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    prog = T.define("grad", [T.spec(dtype, row=rows, vocab=n), T.spec("i32", row=rows), *[T.spec("f32", row=rows)] * 2], lambda b, x: x[0].log_probs_grad(*x[1:], "vocab"))
    got = wide(hip_run(prog, [x, tokens, a, h])[0], dtype)
    v = wide(x, dtype)
    want, size = _grad_logits_want(v, tokens, a.astype(np.float64), h.astype(np.float64))
    # (an f16 gradient below 2^-14 is off by half of f16's smallest step)
    tol = HALF_STEP[dtype] * np.abs(want) + 8 * (_steps(v) * (2 + np.log(n + 1)))[:, None] * size + (2.0 ** -25 if dtype == "f16" else 1e-37)
    assert_within(got, want, tol, "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 2), (4, 9), (7, 500), (300, 1031), (2, 20011), (260, 40000), (257, 70001), (1, 131073)])
def test_log_probs_gradient(rows, n, dtype):
    rng = np.random.default_rng(rows + n)
    x = rng.standard_normal((rows, n)) * 2.5
    x[::3, 1::2] = -np.inf
    tokens = (rng.integers(0, (n + 1) // 2, rows) * 2).astype(np.int32)
    tokens[::4] = -1
    say(f"gradient {rows} {n} {dtype}")
    _check_grad(floats(x, dtype), tokens, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n", [(3, 512), (260, 9000), (2, 20011)])
def test_log_probs_of_a_chunk_far_below(rows, n, dtype):
    """Logits near -2.5e38, whose distance from the maximum is beyond the type in powers of two, in chunks whose own maximum is -4e37 or -1e19."""
    x = np.random.default_rng(n).standard_normal((rows, n))
    for r, high in ((0, -4e37), (1, -1e19)):
        x[r, 16:32] = -2.5e38
        x[r, 16:32:4] = high
        x[r, 40] = high
    x = floats(x, dtype)
    tokens = np.full(rows, 17, np.int32)
    say(f"far below {rows} {n} {dtype}")
    _check_log_probs(x[2:], tokens[2:], 3, dtype)
    _check_grad(x[2:], tokens[2:], dtype)
    _check_log_probs(x[:2], tokens[:2], 3, dtype)
    _check_grad(x, tokens, dtype)


def _steps_of_weight(x):
    """As _steps, but for the logits' own size: a softmax depends on differences from the maximum alone, and those are formed with one rounding, so
    that what counts of them is the mean over the row's probabilities (a sum's relative error) and, beside a result, the result's own size."""
    with np.errstate(all="ignore"):
        bad = ~(np.isfinite(x) | np.isneginf(x)).all(-1) | np.isneginf(x).all(-1)
        x = np.where(bad[:, None], 0.0, x)
        far = x.max(-1, keepdims=True) - x
        p = np.exp(-far)
        mean = (p * np.where(p > 0, far, 0.0)).sum(-1) / p.sum(-1)
    return E24 * (200 + x.shape[-1] / 2048 + 4 * mean + 8 * np.log(x.shape[-1] + 1))


def _check_large(x, tokens, top, dtype):
    """log_probs and its gradient with tolerances that do not grow with the logits."""
    rows, n = x.shape
    spec = [T.spec(dtype, row=rows, vocab=n), T.spec("i32", row=rows)]
    prog = T.define("log_probs", spec, lambda b, a: [v for p in [a[0].log_probs(a[1], "vocab", top=top)] for v in (p.token, p.entropy, p.top, p.top_tokens)])
    got = hip_run(prog, [x, tokens])
    v = wide(x, dtype)
    token, entropy, logp = _log_probs_want(v, tokens)
    tol = _steps_of_weight(v)
    best = np.argsort(-v, axis=1, kind="stable")[:, :top]
    assert np.array_equal(got[3], best)
    # (beyond f32 a log probability is -inf)
    least = lambda w: np.where(w < -3.4028235e38, -np.inf, w)  # noqa: E731
    assert_within(got[0], least(token), tol + 2 * E24 * np.abs(token), "token")
    assert_within(got[1], entropy, 4 * tol * (2 + np.log(n + 1)), "entropy")
    want = np.take_along_axis(logp, best, 1)
    assert_within(got[2], least(want), tol[:, None] + 2 * E24 * np.abs(want), "top")
    rng = np.random.default_rng(rows)
    a, h = (rng.standard_normal(rows).astype(np.float32) for _ in range(2))
    prog = T.define("grad", spec + [T.spec("f32", row=rows)] * 2, lambda b, x: x[0].log_probs_grad(*x[1:], "vocab"))
    got = wide(hip_run(prog, [x, tokens, a, h])[0], dtype)
    want, size = _grad_logits_want(v, tokens, a.astype(np.float64), h.astype(np.float64))
    assert_within(got, want, HALF_STEP[dtype] * np.abs(want) + 8 * (tol * (2 + np.log(n + 1)))[:, None] * size + (2.0 ** -25 if dtype == "f16" else 1e-37), "gradient")


def _shifted_rows(n, dtype):
    """Ordinary rows at a distance from 0, rows of one large value, and ordinary rows of which a third, or whole stretches at the beginning, in the middle or at
    the ends, are masked with a large finite value."""
    rng = np.random.default_rng(n)
    offsets = [1e3, -1e3, 3e4, -3e4] + ([] if dtype == "f16" else [1e5, -1e5, 1e6, -1e7, 1e7, 2.0 ** 24, -2.0 ** 24, 1e8, -1e8, 1e10, -1e10, 1e12, -1e12])
    base, rows = rng.standard_normal(n) * 2.5, []
    for o in offsets:
        rows += [base + o, np.full(n, o), np.where(np.arange(n) % 3 == 0, base, -abs(o))]
        rows += [np.where(part, base, -abs(o)) for part in (np.arange(n) >= n // 2, np.arange(n) < n // 2, np.abs(np.arange(n) - n // 2) > n // 4, np.arange(n) == n // 2)]
        # the largest ones alone in what lies beside the whole chunks
        rows += [np.where((np.arange(n) == 0) | (np.arange(n) == n - 1), base + abs(o), base + abs(o) - 3)]
    return np.stack(rows)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("n,copies", [(7, 1), (100, 1), (2501, 1), (12001, 1), (40003, 1), (2501, 40), (12001, 10)])
def test_log_probs_do_not_depend_on_a_shift(n, copies, dtype):
    """Rows at distances of 1e3 to 1e12 from 0, and masks of -1e3 to -1e12: in a few rows (several workgroups each), in a workgroup's registers, and in more than 512."""
    rows = _shifted_rows(n, dtype)
    x = floats(np.tile(rows, (max(1, -(-copies * 32 // len(rows))) if copies > 1 else 1, 1)), dtype)
    tokens = (np.arange(len(x)).astype(np.int32) * 7) % n
    say(f"shifted {len(x)} {n} {dtype}")
    _check_large(x, tokens, min(n, 5), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,n", [(12, 5), (12, 700), (260, 9001), (6, 20011)])
def test_a_certain_token_has_an_entropy_whose_gradient_is_none(rows, n):
    """Rows in which one logit lies 1000 above all others, wherever that is: its probability is 1, the entropy 0 and the entropy's gradient none at all."""
    at = np.arange(rows) % n
    x = np.resize(np.float32([0, 0.3, 7.1, -300.7, 3000.1, -1e5 - 0.3]), rows)[:, None] - np.full(n, 1000, np.float32)
    x[np.arange(rows), at] += 1000
    tokens, zero, h = np.full(rows, -1, np.int32), np.zeros(rows, np.float32), np.linspace(-3, 2, rows).astype(np.float32)
    spec = [T.spec("f32", row=rows, vocab=n), T.spec("i32", row=rows), *[T.spec("f32", row=rows)] * 2]
    say(f"certain {rows} {n}")
    got = hip_run(T.define("grad", spec, lambda b, v: v[0].log_probs_grad(*v[1:], "vocab")), [x, tokens, zero, h])[0]
    assert not got.any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("rows,n", [(600, 20011), (9, 9001), (600, 70)])
def test_entropies_of_peaked_rows(rows, n, dtype):
    """One logit 12 to 40 above the others: entropies near 0, none below, and no log probability above 0. A thread's sum of 2^y y may be of y up to 46, from an m 32 lower in units of log 2: the
    sum's roundings, one of y, three where it is measured from another maximum, and log2 l's, are 2^-24 of that each, times ln 2."""
    rng = np.random.default_rng(rows + n)
    x = rng.standard_normal((rows, n)) * 2.5
    x[np.arange(rows), rng.integers(0, n, rows)] = x.max(-1) + rng.uniform(12, 40, rows)
    x = floats(x, dtype)
    tokens = np.zeros(rows, np.int32)
    say(f"peaked {rows} {n} {dtype}")
    got, top = hip_run(T.define("p", [T.spec(dtype, row=rows, vocab=n), T.spec("i32", row=rows)],
                                lambda b, a: [v for p in [a[0].log_probs(a[1], "vocab", top=1)] for v in (p.entropy, p.top)]), [x, tokens])
    _, want, logp = _log_probs_want(wide(x, dtype), tokens)
    assert (got >= 0).all() and (top <= 0).all()
    assert_within(top[:, 0], logp.max(-1), _steps_of_weight(wide(x, dtype)) + 2 * E24 * np.abs(logp.max(-1)), "top")
    assert_within(got, want, 6 * 46 * E24 * np.log(2) + 2 * E24 * want, "entropy")


@pytest.mark.gpu
@pytest.mark.parametrize("shift", [0.0, 1e5, -1e7])
def test_the_gradient_of_a_row_does_not_depend_on_how_many_there_are(shift):
    """One row by itself, in two kernels, and among 300, in one kernel: the same but for roundings."""
    rng = np.random.default_rng(9)
    x = (rng.standard_normal((300, 20011)) * 2.5 + shift).astype(np.float32)
    tokens, a, h = rng.integers(0, 20011, 300).astype(np.int32), *(rng.standard_normal(300).astype(np.float32) for _ in range(2))

    def grad(rows):
        spec = [T.spec("f32", row=rows, vocab=20011), T.spec("i32", row=rows), *[T.spec("f32", row=rows)] * 2]
        return hip_run(T.define("grad", spec, lambda b, v: v[0].log_probs_grad(*v[1:], "vocab")), [x[:rows], tokens[:rows], a[:rows], h[:rows]])[0]
    say(f"gradient alone and among others, {shift}")
    alone, among = grad(1).astype(np.float64), grad(300)[:1].astype(np.float64)
    _, size = _grad_logits_want(x[:1].astype(np.float64), tokens[:1], a[:1].astype(np.float64), h[:1].astype(np.float64))
    assert_within(among, alone, 16 * (_steps_of_weight(x[:1].astype(np.float64)) * (2 + np.log(20012)))[:, None] * size + 1e-37)


@pytest.mark.gpu
@pytest.mark.parametrize("n,dtype", [(65536, "f16"), (90103, "bf16"), (106496, "f16"), (131072, "bf16"), (131063, "f16"), (65531, "f32"), (151936, "bf16"), (180215, "f16"), (90112, "f32"), (200001, "bf16")])
def test_log_probs_gradient_of_long_rows(n, dtype):
    """Rows that fill a workgroup's registers, whole chunks and not, and longer ones: four different rows 64 times over, each the same wherever it lies."""
    rng = np.random.default_rng(n)
    x = rng.standard_normal((4, n)) * 2.5
    x[1, ::3], x[2] = -np.inf, x[2] + 300
    x = floats(x, dtype)
    tokens, a, h = np.array([n - 1, 4, 0, -1], np.int32), *(rng.standard_normal(4).astype(np.float32) for _ in range(2))
    spec = [T.spec(dtype, row=256, vocab=n), T.spec("i32", row=256), *[T.spec("f32", row=256)] * 2]
    say(f"gradient 256 {n} {dtype}")
    got = hip_run(T.define("grad", spec, lambda b, v: v[0].log_probs_grad(*v[1:], "vocab")), [np.tile(v, (64, 1)[:v.ndim]) for v in (x, tokens, a, h)])[0].reshape(64, 4, n)
    v = wide(x, dtype)
    want, size = _grad_logits_want(v, tokens, a.astype(np.float64), h.astype(np.float64))
    tol = HALF_STEP[dtype] * np.abs(want) + 8 * (_steps_of_weight(v) * (2 + np.log(n + 1)))[:, None] * size + (2.0 ** -25 if dtype == "f16" else 1e-37)
    # (a row's place decides which of its elements are whole chunks': eight rows on, the same again)
    for first in (0, 1):
        assert_within(wide(got[first], dtype), want, tol, "gradient")
        assert (got[first] == got[first::2]).all()


@pytest.mark.gpu
def test_log_probs_without_rows_and_of_a_vector():
    got = hip_run(T.define("p", [T.spec("f32", row=0, vocab=9), T.spec("i32", row=0)], lambda b, a: a[0].log_probs(a[1], "vocab", top=2).top), [np.zeros((0, 9), np.float32), np.zeros(0, np.int32)])[0]
    assert got.shape == (0, 2)
    x, t = np.float32([1, 3, 2]), np.array(1, np.int32)
    got = hip_run(T.define("p", [T.spec("f32", vocab=3), T.spec("i32")], lambda b, a: [a[0].log_probs(a[1], "vocab", top=1).token, a[0].log_probs(a[1], "vocab", top=1).top_tokens]), [x, t])
    assert abs(got[0] - _log_probs_want(x[None].astype(np.float64), t[None])[0][0]) < 1e-6 and got[1][0] == 1


# ---- pages ----

def fork_want(table, lengths, parents, room, held, page, tokens):
    S, W_ = table.shape
    P = len(held)
    rows = []
    for p, more in zip(parents.tolist(), room.tolist()):
        if not 0 <= p < S:
            rows.append(([], 0, 0))
            continue
        n = min(max(int(lengths[p]), 0), W_ * page)
        kept = [x if 0 <= x < P else -1 for x in table[p, :-(-n // page)].tolist()]
        rows.append((kept, n, -(-min(n + max(more, 0), W_ * page) // page)))
    full = {x for kept, n, _ in rows for x in (kept[:-1] if n % page else kept)}
    seen, used, copies = set(), set(full) | set(np.flatnonzero(held).tolist()), []
    for kept, n, _ in rows:
        last = kept[-1] if n % page else -1
        copies.append(last if last >= 0 and (last in full or held[last] or last in seen) else -1)
        if last >= 0:
            seen.add(last)
    used |= seen
    free = [x for x in range(P) if x not in used]
    asked = 0

    def fresh():
        nonlocal asked
        asked += 1
        return free[asked - 1] if asked <= len(free) else -1
    out = np.full((len(rows), W_), -1, np.int32)
    source, target, slots = (np.full(s, -1, np.int32) for s in (len(rows), len(rows), (len(rows), tokens)))
    for r, ((kept, n, want), old) in enumerate(zip(rows, copies)):
        now = list(kept)
        if old >= 0:
            now[-1] = fresh()
            if now[-1] >= 0:
                source[r], target[r] = old, now[-1]
        now += [fresh() for _ in range(want - len(kept))]
        out[r, :len(now)] = now
        for i in range(min(tokens, max(int(room[r]), 0))):
            if want and n + i < W_ * page and now[(n + i) // page] >= 0:
                slots[r, i] = now[(n + i) // page] * page + (n + i) % page
    return out, np.array([n for _, n, _ in rows], np.int32), source, target, np.array(len(free) - asked, np.int32), slots


FORKS = [(1, 1, 1, 1, 32), (4, 6, 5, 40, 64), (8, 8, 64, 300, 64), (3, 40, 9, 64, 1), (5, 300, 20, 900, 16), (20, 7, 700, 3000, 64), (6, 1100, 3, 5000, 32), (9, 30, 4, 140000, 64),
         (4, 1500, 5, 135000, 7), (2, 3, 0, 10, 32), (0, 4, 3, 10, 32), (3, 0, 4, 10, 32), (2, 3, 4, 0, 32)]


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,rows,slots,pages,page", FORKS)
def test_fork_pages(seqs, rows, slots, pages, page):
    """Rows kept, freed and forked; pages that are none; lengths and rooms of any size; pages that run out; more rows than a workgroup's threads, more pages than
    LDS holds; large tables, which other workgroups write."""
    rng = np.random.default_rng(rows + pages)
    for case in range(3):
        table = rng.integers(0, max(pages, 1), (seqs, slots)).astype(np.int32)
        if case and pages:  # pages of their own but for a beginning, as in earnest
            table[...] = rng.permutation(max(pages, seqs * slots))[:seqs * slots].reshape(seqs, slots) % pages
            table[:, :slots // 3] = table[:1, :slots // 3]
        else:
            table[rng.random(table.shape) < 0.1] = -1
            table[rng.random(table.shape) < 0.1] = pages + 5
        lengths = rng.integers(0, slots * page + 1, seqs).astype(np.int32)
        if seqs > 2:
            lengths[:3] = [-4, 2 ** 31 - 1, slots * page // 2 // page * page]
        parents = rng.integers(-1, seqs + 1, rows).astype(np.int32)
        room = rng.integers(-2, 2 * page + 2, rows).astype(np.int32)
        if rows > 2:
            parents[0], room[1] = -2 ** 31, 2 ** 31 - 1
        held = rng.random(pages) < (0.05, 0.3, 0.97)[case]
        prog = T.define("fork", [T.spec("i32", seq=seqs, slot=slots), T.spec("i32", seq=seqs), T.spec("i32", row=rows), T.spec("i32", row=rows), T.spec("i1", page=pages)],
                        lambda b, a: [v for f in [b.fork_pages(*a, page, tokens=2)] for v in (f.pages, f.lengths, f.source, f.target, f.left, f.slots)])
        say(f"fork {seqs} {rows} {slots} {pages} {page} {case}")
        ins = [table, lengths, parents, room, held]
        for got, want in zip(hip_run(prog, ins), fork_want(*ins, page, 2)):
            assert np.array_equal(got, want), (got, want)


def compact_want(table, held, moves):
    P = len(held)
    used = {x for x in table.reshape(-1).tolist() if 0 <= x < P}
    both = used | set(np.flatnonzero(held).tolist())
    movers = [x for x in range(len(both), P) if x in used and not held[x]]
    holes = [x for x in range(len(both)) if x not in both]
    pairs = list(zip(movers, holes))[:moves]
    new = dict(pairs)
    out = np.array([new.get(x, x) if 0 <= x < P else -1 for x in table.reshape(-1).tolist()], np.int32).reshape(table.shape)
    ends = np.full((2, moves), -1, np.int32)
    for i, (a, b) in enumerate(pairs):
        ends[:, i] = a, b
    return out, ends[0], ends[1]


@pytest.mark.gpu
@pytest.mark.parametrize("seqs,slots,pages,moves", [(1, 1, 1, 1), (4, 6, 40, 10), (8, 64, 3000, 600), (100, 90, 20000, 20000), (7, 9, 140000, 50), (3, 0, 10, 4), (5, 5, 30, 0), (9, 600, 200000, 4000), (2, 3, 0, 0)])
def test_compact_pages(seqs, slots, pages, moves):
    rng = np.random.default_rng(pages)
    for case in range(2):
        table = rng.integers(-1, pages + 1, (seqs, slots)).astype(np.int32)
        held = rng.random(pages) < (0.02, 0.5)[case]
        prog = T.define("compact", [T.spec("i32", seq=seqs, slot=slots), T.spec("i1", page=pages)],
                        lambda b, a: [v for c in [b.compact_pages(*a, ("move", moves))] for v in (c.pages, c.source, c.target)])
        say(f"compact {seqs} {slots} {pages} {moves} {case}")
        for got, want in zip(hip_run(prog, [table, held]), compact_want(table, held, moves)):
            assert np.array_equal(got, want)
    if slots:
        alone = hip_run(T.define("table", [T.spec("i32", seq=seqs, slot=slots), T.spec("i1", page=pages)], lambda b, a: b.compact_pages(*a, ("move", moves)).pages), [table, held])[0]
        assert np.array_equal(alone, compact_want(table, held, moves)[0])


@pytest.mark.gpu
@pytest.mark.parametrize("pages", [32768, 32769, 40000, 65536, 131071, 131072, 131073])
def test_large_tables_among_pages_of_several_words_a_thread(pages):
    """Bitmaps of more words than a workgroup has threads, up to where they leave LDS, and tables that another kernel writes: the counts
    that it reads are those of all words. Pages in use, holes and moves lie in words all over; rows forked from the same tables."""
    rng = np.random.default_rng(pages)
    for used, held_share, moves in ((pages // 4, 0.02, 9000), (pages, 0.4, 700)):
        table = rng.integers(0, used, (64, 256)).astype(np.int32) * (pages // used)
        table[rng.random(table.shape) < 0.05] = -1
        held = rng.random(pages) < held_share
        prog = T.define("compact", [T.spec("i32", seq=64, slot=256), T.spec("i1", page=pages)],
                        lambda b, a: [v for c in [b.compact_pages(*a, ("move", moves))] for v in (c.pages, c.source, c.target)])
        want = compact_want(table, held, moves)
        assert len(np.unique(want[1] // 32)) > 90 and (want[0] != table).any()
        say(f"compact 64 x 256 of {pages}")
        for got, w in zip(hip_run(prog, [table, held]), want):
            assert np.array_equal(got, w)
        ins = [table, rng.integers(0, 256 * 16 + 1, 64).astype(np.int32), rng.integers(-1, 65, 40).astype(np.int32), rng.integers(0, 400, 40).astype(np.int32), held]
        row = T.spec("i32", row=40)
        prog = T.define("fork", [T.spec("i32", seq=64, slot=256), T.spec("i32", seq=64), row, row, T.spec("i1", page=pages)],
                        lambda b, a: [v for f in [b.fork_pages(*a, 16, tokens=2)] for v in (f.pages, f.lengths, f.source, f.target, f.left, f.slots)])
        say(f"fork 64 x 256 of {pages}")
        for got, w in zip(hip_run(prog, ins), fork_want(*ins, 16, 2)):
            assert np.array_equal(got, w)


@pytest.mark.gpu
def test_compact_pages_of_two_numbers_of_moves():
    """Results of two calls on one table that differ in their moves alone, each by its own."""
    rng = np.random.default_rng(3)
    table, held = rng.integers(0, 400, (6, 20)).astype(np.int32), rng.random(400) < 0.1
    prog = T.define("compact", [T.spec("i32", seq=6, slot=20), T.spec("i1", page=400)],
                    lambda b, a: [v for x, y in [(b.compact_pages(*a, ("move", 9)), b.compact_pages(*a, ("move", 70)))] for v in (x.pages, y.source, y.pages, x.target)])
    few, many = compact_want(table, held, 9), compact_want(table, held, 70)
    for got, want in zip(hip_run(prog, [table, held]), (few[0], many[1], many[0], few[2])):
        assert np.array_equal(got, want)


def copied(cache, source, target):
    out = cache.copy()
    for s, t in zip(source.tolist(), target.tolist()):
        if 0 <= s < len(cache) and 0 <= t < len(cache):
            out[t] = cache[s]
    return out


COPIES = [("u8", (6, 3), 9), ("f32", (40, 2, 5), 30), ("u8", (30, 2, 32 * 68), 25), ("u16", (50, 4099), 64), ("i64", (5, 1), 1), ("u8", (300, 16), 5000), ("f32", (7, 0), 3), ("f32", (4,), 6), ("u8", (3, 20000), 0)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shape,n", COPIES)
def test_copy_pages(dtype, shape, n):
    """Any list: to one page twice, from a page that is a target, round in a circle, to itself, from and to no page; the cache in a buffer of its own
    and in place, twice over."""
    rng = np.random.default_rng(n + shape[0])
    cache = rng.integers(0, 250, shape).astype(T.NUMPY_DTYPE[dtype])
    source, target = (rng.integers(-1, shape[0] + 1, n).astype(np.int32) for _ in range(2))
    if n > 4 and shape[0] > 3:
        source[:4], target[:4] = [0, 1, 2, 2 ** 31 - 1], [1, 2, 0, -2 ** 31]
    prog = T.define("copy", [T.spec(dtype, *[(f"d{i}", e) for i, e in enumerate(shape)]), T.spec("i32", copy=n), T.spec("i32", copy=n)], lambda b, a: a[0].copy_pages(a[1], a[2]))
    want = copied(cache, source, target)
    say(f"copy {dtype} {shape} {n}")
    assert np.array_equal(hip_run(prog, [cache, source, target])[0], want)
    if not cache.nbytes or not n:
        return
    stream = hip.Stream()
    bufs = [hip.DeviceBuffer.from_array(x) for x in (cache, source, target)]
    with hip.Hip(prog) as ex:
        for _ in range(2):
            bufs[0].upload(cache)
            ex.launch_device([b.ptr for b in bufs], [bufs[0].ptr], stream.handle)
            stream.synchronize()
            assert np.array_equal(bufs[0].download(np.empty_like(cache)), want)
    stream.destroy()


@pytest.mark.gpu
def test_copies_of_pages_one_after_the_other():
    """Three in a row over one buffer, in place and into another; a cache that is its own lists, and one read again after it was copied, stay what they were."""
    rng = np.random.default_rng(5)
    cache = rng.integers(0, 250, (40, 3, 17)).astype(np.uint8)
    lists = [rng.integers(-1, 41, n).astype(np.int32) for n in (25, 25, 60, 60, 5, 5)]
    want = cache
    for i in (0, 2, 4):
        want = copied(want, *lists[i:i + 2])
    specs = [T.spec("u8", page=40, r=3, c=17), *[T.spec("i32", **{f"copy{i // 2}": len(x)}) for i, x in enumerate(lists)]]
    prog = T.define("row", specs, lambda b, a: a[0].copy_pages(*a[1:3]).copy_pages(*a[3:5]).copy_pages(*a[5:7]))
    say("copies in a row")
    assert np.array_equal(hip_run(prog, [cache, *lists])[0], want)
    stream, bufs = hip.Stream(), [hip.DeviceBuffer.from_array(x) for x in (cache, *lists)]
    with hip.Hip(prog) as ex:
        for _ in range(2):
            bufs[0].upload(cache)
            ex.launch_device([b.ptr for b in bufs], [bufs[0].ptr], stream.handle)
            stream.synchronize()
            assert np.array_equal(bufs[0].download(np.empty_like(cache)), want)
    stream.destroy()
    numbers, other = rng.permutation(64).astype(np.int32), rng.permutation(64).astype(np.int32)
    one = copied(numbers, numbers, other)
    prog = T.define("own", [T.spec("i32", page=64)] * 2, lambda b, a: [a[0].copy_pages(a[0], a[1]).copy_pages(b.full("i32", 3, ("page", 64)), a[1]), a[0].copy_pages(a[1], a[0])])
    say("a cache as its own lists")
    got = hip_run(prog, [numbers, other])
    assert np.array_equal(got[0], copied(one, np.full(64, 3, np.int32), other)) and np.array_equal(got[1], copied(numbers, other, numbers))
    first = lambda b, a: a[0].copy_pages(a[0], a[1])  # noqa: E731
    prog = T.define("again", [T.spec("i32", page=64)] * 2, lambda b, a: [v for c in [first(b, a)] for v in (c.copy_pages(c, a[1]), c.copy_pages(a[1], c))])
    got = hip_run(prog, [numbers, other])
    assert np.array_equal(got[0], copied(one, one, other)) and np.array_equal(got[1], copied(one, other, one))


# ---- attention with shared keys ----

def shared_attention(q, cache, pages, lengths, prefix_pages, prefix_lengths, of):
    """(output, sum of p |v|, largest sum of |q k|) in float64: every query sees the whole prefix."""
    S, Q, heads, dim = q.shape
    kc, ks, vc, vs = cache_parts(cache, dim)
    K, V = decoded(kc, ks), decoded(vc, vs)
    P, H, page, _ = K.shape
    out, mass, most = np.zeros(q.shape), np.zeros(q.shape), 0.0

    def places(table, n):
        n = min(max(int(n), 0), len(table) * page)
        return [(table[j // page], j % page) for j in range(n) if 0 <= table[j // page] < P]
    for b in range(S):
        before = places(prefix_pages[of[b]], prefix_lengths[of[b]]) if 0 <= of[b] < len(prefix_pages) else []
        n = min(max(int(lengths[b]), 0), pages.shape[1] * page)
        for i in range(Q):
            keys = before + places(pages[b], n - (Q - 1 - i))
            if not keys:
                continue
            at = np.array(keys)
            for h in range(heads):
                k, v = (x[at[:, 0], h // (heads // H), at[:, 1]] for x in (K, V))
                s = k @ q[b, i, h] / np.sqrt(dim)
                p = np.exp(s - s.max())
                p /= p.sum()
                out[b, i, h], mass[b, i, h] = p @ v, p @ np.abs(v)
                most = max(most, np.nanmax(np.abs(k) @ np.abs(q[b, i, h])) / np.sqrt(dim))
    return out, mass, most


def _shared_program(q, cache, pages, prefix_pages, dtype):
    S, N = ("seq", q.shape[0]), ("prefix", prefix_pages.shape[0])
    specs = [T.spec(dtype, S, ("query", q.shape[1]), ("head", q.shape[2]), ("dim", q.shape[3])), T.spec("u8", page=cache.shape[0], kv_head=cache.shape[1], byte=cache.shape[2]),
             T.spec("i32", S, ("at", pages.shape[1])), T.spec("i32", S), T.spec("i32", N, ("there", prefix_pages.shape[1])), T.spec("i32", N), T.spec("i32", S)]
    return T.define("attend", specs, lambda b, a: a[0].attend_mx4(a[1], a[2], a[3], shared=a[4:]))


def _check_shared(q, cache, pages, lengths, prefix_pages, prefix_lengths, of, dtype):
    ins = [q, cache, pages, lengths, prefix_pages, prefix_lengths, of]
    got = hip_run(_shared_program(q, cache, pages, prefix_pages, dtype), ins)[0]
    want, mass, most = shared_attention(wide(q, dtype), *ins[1:])
    dim = q.shape[3]
    n = (pages.shape[1] + prefix_pages.shape[1]) * (cache.shape[2] // (dim + dim // 16))
    # as for attention without shared keys, over the keys of both, and twice as many joins
    rel = 2 * ((3 * dim + 4) * 2.0 ** -23 * most + 2.0 ** -21 + (n + 128) * 2.0 ** -23 * 3)
    least = 2.0 ** -25 if dtype == "f16" else 1e-37
    assert_within(wide(got, dtype), want, HALF_STEP[dtype] * np.abs(want) + (1 + HALF_STEP[dtype]) * rel * mass + least)
    return wide(got, dtype)


SHARED = [(1, 1, 1, 1, 32, 32, 1, 1, 1), (3, 1, 4, 4, 64, 64, 2, 1, 3), (20, 1, 8, 2, 128, 64, 1, 1, 9), (9, 2, 6, 3, 64, 32, 3, 3, 2), (5, 3, 10, 2, 96, 64, 2, 2, 5), (7, 1, 3, 1, 256, 32, 2, 4, 4),
          (40, 1, 2, 2, 64, 32, 0, 2, 6), (6, 33, 2, 2, 32, 64, 2, 2, 1), (270, 1, 2, 1, 32, 32, 1, 300, 1), (2, 5, 16, 2, 160, 32, 2, 1, 40)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("seqs,query,heads,kv,dim,page,slots,prefixes,prefix_slots", SHARED)
def test_attend_shared(seqs, query, heads, kv, dim, page, slots, prefixes, prefix_slots, dtype):
    """Sequences with and without a prefix, prefixes of many, of one and of no sequence, keys of their own or none."""
    rng = np.random.default_rng(seqs * 10 + dim)
    P = seqs * slots + prefixes * prefix_slots + 2
    cache = finite_cache(P, kv, dim, page, rng)
    q = floats(rng.standard_normal((seqs, query, heads, dim)) * 2, dtype)
    order = rng.permutation(P).astype(np.int32)
    pages, prefix_pages = order[:seqs * slots].reshape(seqs, slots), order[seqs * slots:P - 2].reshape(prefixes, prefix_slots)
    lengths = rng.integers(0, slots * page + 1, seqs).astype(np.int32)
    prefix_lengths = rng.integers(0, prefix_slots * page + 1, prefixes).astype(np.int32)
    prefix_lengths[0] = prefix_slots * page
    of = rng.integers(-1, prefixes + 1, seqs).astype(np.int32)
    of[0] = 0
    say(f"attend shared {seqs} {query} {heads} {kv} {dim} {page} {slots} {prefixes} {prefix_slots} {dtype}")
    got = _check_shared(q, cache, pages, lengths, prefix_pages, prefix_lengths, of, dtype)
    assert not got[(lengths <= 0) & ((of < 0) | (of >= prefixes))].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,query", [("bf16", 1), ("f32", 3)])
def test_attend_shared_places_that_nobody_sees(dtype, query):
    """Rows behind the ends and other pages hold NaN; pages outside the cache hold no keys; lengths of any size; a NaN in one prefix reaches its own sequences only."""
    rng = np.random.default_rng(5)
    cache = finite_cache(16, 2, 64, 32, rng)
    _, ks, _, vs = cache_parts(cache, 64)
    pages, prefix_pages = np.arange(12).reshape(6, 2).astype(np.int32), np.arange(12, 16).reshape(2, 2).astype(np.int32)
    lengths, prefix_lengths, of = np.array([40, 3, 0, -7, 64, 33], np.int32), np.array([45, 31], np.int32), np.array([0, 1, 0, 1, -1, 2 ** 31 - 1], np.int32)
    for table, count in list(zip(pages, lengths)) + list(zip(prefix_pages, prefix_lengths)):
        for j in range(max(int(count), 0), 64):
            ks[table[j // 32], :, j % 32] = vs[table[j // 32], :, j % 32] = 255
    pages[5, 1], prefix_pages[1, 1] = -1, 2 ** 31 - 1
    q = floats(rng.standard_normal((6, query, 4, 64)), dtype)
    _check_shared(q, cache, pages, lengths, prefix_pages, prefix_lengths, of, dtype)
    prefix_lengths[0] = 2 ** 31 - 1  # all of its pages, NaN among them
    got = wide(hip_run(_shared_program(q, cache, pages, prefix_pages, dtype), [q, cache, pages, lengths, prefix_pages, prefix_lengths, of])[0], dtype)
    assert np.isnan(got[[0, 2]]).all() and np.isfinite(got[[1, 3, 4, 5]]).all()


# ---- a step of them together ----

STEPS = [(3, 5, 64, 2, 1, 32, 300, 40, 32, 4, 1, 3, 4, "f32"), (6, 9, 128, 6, 2, 64, 1001, 60, 64, 5, 3, 2, 20, "bf16"), (4, 4, 96, 4, 4, 96, 77, 30, 32, 3, 2, 2, 1, "f16")]


def _step(seqs, rows, model, heads, kv, hd, vocab, pages, page, slots, prefixes, prefix_pages, top, dtype, seed=3):
    rng = np.random.default_rng(seed)
    prog = W.answers_step_mx4_program(seqs, rows, model, heads, kv, hd, vocab, pages, page, slots, prefixes, prefix_pages, top, dtype)
    weight = lambda n, k: list(encoded(rng.standard_normal((n, k)) * k ** -0.5))  # noqa: E731
    shaped = lambda w, *rows: [x.reshape(*rows, x.shape[-1]) for x in w]  # noqa: E731
    gains = lambda n: floats(1 + 0.1 * rng.standard_normal(n), dtype)  # noqa: E731
    order = rng.permutation(pages).astype(np.int32)
    n = prefixes * prefix_pages
    table = np.full((seqs, slots), -1, np.int32)
    each = slots - 1
    table[:, :each] = order[n:n + seqs * each].reshape(seqs, each)
    held = np.zeros(pages, bool)
    held[order[:n]] = True
    parents = rng.integers(0, seqs, rows).astype(np.int32)
    parents[-1] = -1
    ins = [floats(rng.standard_normal((rows, model)), dtype), gains(model), *shaped(weight(heads * hd, model), heads, hd), *shaped(weight(kv * hd, model), kv, hd),
           *shaped(weight(kv * hd, model), kv, hd), *weight(model, heads * hd), gains(hd), gains(hd), rng.integers(0, 5000, rows).astype(np.int32),
           (10000.0 ** (-np.arange(hd // 2) / (hd // 2))).astype(np.float32), gains(model), *weight(vocab, model), finite_cache(pages, kv, hd, page, rng), table,
           rng.integers(1, each * page + 1, seqs).astype(np.int32), parents, np.ones(rows, np.int32), held, order[:n].reshape(prefixes, prefix_pages),
           rng.integers(1, prefix_pages * page + 1, prefixes).astype(np.int32), rng.integers(0, prefixes, rows).astype(np.int32), rng.integers(-1, vocab, rows).astype(np.int32)]
    for v, t in zip(ins, prog.input_types()):
        assert v.shape == t.shape and v.dtype == T.NUMPY_DTYPE[t.dtype], (t, v.shape, v.dtype)
    return prog, ins


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", STEPS)
def test_answers_step_is_its_operators_one_by_one(sizes):
    """The program against programs of a part each, bit for bit, whose results are checked by themselves on the way."""
    seqs, rows, model, heads, kv, hd, vocab, pages, page, slots, prefixes, prefix_pages, top, dtype = sizes
    prog, ins = _step(*sizes)
    (x, g, qg, kg, positions, freq, g2, cache, table, lengths, parents, room, held, pre_table, pre_lengths, of, tokens) = (
        ins[0], ins[1], ins[10], ins[11], ins[12], ins[13], ins[14], ins[17], *ins[18:27])
    say(f"answers step {sizes}")
    got = hip_run(prog, ins)
    forked = fork_want(table, lengths, parents, room, held, page, 1)
    assert np.array_equal(got[4], forked[0]) and np.array_equal(got[5], forked[1] + 1)
    specs, R = prog.input_types(), ("row", rows)
    spec = lambda i: T.Spec(specs[i].dtype, specs[i].dims)  # noqa: E731
    alone = lambda body, ids, values: hip_run(T.define("alone", [s if isinstance(s, T.Spec) else spec(s) for s in ids], body), values)  # noqa: E731

    def project(b, a):
        h = W.rms_norm(b, a[0], a[1], "model", dtype).quantize_mx4("model")
        return [h.contract(b.mx4(a[i], a[i + 1], "model"), dtype) for i in (2, 4, 6)]
    q, k, v = alone(project, range(8), ins[:8])
    qs, ks = T.Spec(dtype, (R, ("head", heads), ("dim", hd))), T.Spec(dtype, (R, ("kv_head", kv), ("dim", hd)))
    q, k = alone(lambda b, a: list(b.rotate_heads(a[0], a[1], T.Rotation(a[4], a[5]), T.HeadNorm(a[2], a[3]))), [qs, ks, 10, 11, 12, 13], [q, k, qg, kg, positions, freq])
    after = copied(cache, forked[2], forked[3])
    after = alone(lambda b, a: a[0].cache_write_mx4(a[1], a[2], a[3]), [17, ks, ks, T.Spec("i32", (R,))], [after, k, v, forked[5][:, 0]])[0]
    assert np.array_equal(after, got[6])
    o = alone(lambda b, a: a[0].attend_mx4(*a[1:4], shared=a[4:]), [qs, 17, T.Spec("i32", (R, ("slot", slots))), T.Spec("i32", (R,)), 23, 24, 25],
              [q, after, forked[0], forked[1] + 1, pre_table, pre_lengths, of])[0]
    want, mass, _ = shared_attention(wide(q, dtype)[:, None], after, forked[0], forked[1] + 1, pre_table, pre_lengths, of)
    assert_within(wide(o, dtype)[:, None], want, HALF_STEP[dtype] * np.abs(want) + 1e-3 * mass + 2.0 ** -25)

    def rest(b, a):
        y = a[0].add(a[1].merge(("head", "dim"), "att").quantize_mx4("att").contract(b.mx4(a[2], a[3], "att"), dtype))
        logits = W.rms_norm(b, y, a[4], "model", dtype).quantize_mx4("model").contract(b.mx4(a[5], a[6], "model"), "f32")
        p = logits.log_probs(a[7], "vocab", top=top)
        return [p.token, p.entropy, p.top, p.top_tokens]
    last = alone(rest, [0, qs, 8, 9, 14, 15, 16, 26], [x, o, ins[8], ins[9], g2, ins[15], ins[16], tokens])
    _same(got[:4], last)


CACHE = 17  # the step's input; its last output


def _step_bound(prog, ins, in_place):
    bound = _Bound(prog, ins)
    if in_place:
        bound.op[6] = bound.ip[CACHE]

    def restore():
        bound.clear()
        bound.dins[CACHE].upload(ins[CACHE])

    def outputs():
        out = bound.read()
        return out[:6] + [bound.dins[CACHE].download(np.empty_like(ins[CACHE])) if in_place else out[6]]
    return bound, restore, outputs


@pytest.mark.gpu
@pytest.mark.parametrize("scratch", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_answers_step_captured_into_hip_graphs(scratch, in_place):
    """Steps of two models captured and replayed in turn, with eager steps of the other between the replays; every replay equals run_hip bit for bit."""
    rt, s, stream = _hip_runtime(), hip.Session(), hip.Stream()
    progs = [_step(*STEPS[0]), _step(*STEPS[1], seed=4)]
    refs = [hip_run(*p) for p in progs]
    handles = [s.compile(p) for p, _ in progs]
    bounds = [_step_bound(*p, in_place) for p in progs]
    graphs, exes = [], []
    try:
        for h, (bound, restore, outputs), ref in zip(handles, bounds, refs):
            bound.call(h, scratch, stream)
            stream.synchronize()
            _same(outputs(), ref)
            graphs.append(_capture(rt, stream, lambda: bound.call(h, scratch, stream)))
            exes.append(ctypes.c_void_p())
            assert rt.hipGraphInstantiate(ctypes.byref(exes[-1]), graphs[-1], None, None, 0) == 0
        for r in range(3):
            for i in (0, 1):
                say(f"replay {r} of {i}, scratch={scratch}, in place={in_place}")
                bounds[i][1]()
                assert rt.hipGraphLaunch(exes[i], ctypes.c_void_p(stream.handle)) == 0
                stream.synchronize()
                _same(bounds[i][2](), refs[i])
                bounds[1 - i][1]()
                bounds[1 - i][0].call(handles[1 - i], scratch, stream)
                stream.synchronize()
                _same(bounds[1 - i][2](), refs[1 - i])
        for exe, graph in zip(exes, graphs):
            rt.hipGraphExecDestroy(exe)
            rt.hipGraphDestroy(graph)
    finally:
        for b, _, _ in bounds:
            b.free()
        for h in handles:
            s.release(h)
        stream.destroy()


def _training_programs():
    """Gradients of heads and of logits in both of their forms, and pages moved, copied in any order and twice to one page."""
    rng = np.random.default_rng(12)
    heads = _heads_specs(300, 3, 2, 48, 16, 2, "bf16", True)
    logits = lambda rows, n, dtype: [T.spec(dtype, **{f"r{n}": rows, f"v{n}": n}), T.spec("i32", **{f"r{n}": rows}), *[T.spec("f32", **{f"r{n}": rows})] * 2]  # noqa: E731

    def train(b, a):
        grads = list(b.rotate_heads_grad(*a[:4], *_operands(b, a[4:9], 2, "neighbours", True, 1e-5)))
        return grads + [a[9].log_probs_grad(*a[10:13], "v700"), a[13].log_probs_grad(*a[14:17], "v20011"), a[13].log_probs(a[14], "v20011", top=3).top]
    q, k, position, freq, axis, gain = _heads_inputs(300, 3, 2, 48, 16, 2, "bf16", "bf16", rng)
    ins = [q[::-1].copy(), k[::-1].copy(), q, k, position, freq, axis, *gain]
    for rows, n, dtype in ((270, 700, "f16"), (3, 20011, "f32")):
        ins += [floats(rng.standard_normal((rows, n)) * 2, dtype), rng.integers(0, n, rows).astype(np.int32), *(rng.standard_normal(rows).astype(np.float32) for _ in range(2))]
    yield T.define("train", heads[:2] + heads + logits(270, 700, "f16") + logits(3, 20011, "f32"), train), ins
    table, held = rng.integers(-1, 900, (70, 64)).astype(np.int32), rng.random(900) < 0.1
    cache, lists = rng.integers(0, 256, (900, 3, 40)).astype(np.uint8), [rng.integers(-1, 901, n).astype(np.int32) for n in (50, 50, 5000, 5000)]

    def pages(b, a):
        c = b.compact_pages(a[0], a[1], ("move", 300))
        return [c.pages, c.source, c.target, a[2].copy_pages(c.source, c.target).copy_pages(a[3], a[4]).copy_pages(a[5], a[6])]
    yield T.define("pages", [T.spec("i32", seq=70, slot=64), T.spec("i1", page=900), T.spec("u8", page=900, r=3, c=40),
                             *[T.spec("i32", **{f"copy{len(x)}": len(x)}) for x in lists]], pages), [table, held, cache, *lists]


@pytest.mark.gpu
@pytest.mark.parametrize("scratch", [False, True])
def test_gradients_and_moved_pages_captured_into_hip_graphs(scratch):
    """Two programs captured and replayed in turn on one stream, each run eagerly on another between its replays."""
    rt, s, stream, other = _hip_runtime(), hip.Session(), hip.Stream(), hip.Stream()
    progs = list(_training_programs())
    refs = [hip_run(*p) for p in progs]
    table, held, cache, *lists = progs[1][1]
    moved = compact_want(table, held, 300)
    want = copied(copied(copied(cache, *moved[1:]), *lists[:2]), *lists[2:])
    assert all(np.array_equal(g, w) for g, w in zip(refs[1], (*moved, want)))
    handles, bounds, graphs, exes = [s.compile(p) for p, _ in progs], [_Bound(*p) for p in progs], [], []
    try:
        for h, bound, ref in zip(handles, bounds, refs):
            bound.call(h, scratch, stream)
            stream.synchronize()
            _same(bound.read(), ref)
            graphs.append(_capture(rt, stream, lambda: bound.call(h, scratch, stream)))
            exes.append(ctypes.c_void_p())
            assert rt.hipGraphInstantiate(ctypes.byref(exes[-1]), graphs[-1], None, None, 0) == 0
        for r in range(3):
            for i in (0, 1):
                say(f"replay {r} of {i}, scratch={scratch}")
                bounds[i].clear()
                assert rt.hipGraphLaunch(exes[i], ctypes.c_void_p(stream.handle)) == 0
                stream.synchronize()
                _same(bounds[i].read(), refs[i])
                bounds[i].clear()
                bounds[i].call(handles[i], scratch, other)
                other.synchronize()
                _same(bounds[i].read(), refs[i])
        for exe, graph in zip(exes, graphs):
            rt.hipGraphExecDestroy(exe)
            rt.hipGraphDestroy(graph)
    finally:
        for b in bounds:
            b.free()
        for h in handles:
            s.release(h)
        stream.destroy()
        other.destroy()
