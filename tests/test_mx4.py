"""Microscaled 4-bit floats on an MI355X: quantisation, products, the paged cache and its attention, against the same
in float64 (numpy) on identical inputs.

Tolerances are sums of what the operators' arithmetic allows. u = eps / 2 of the result's type is its one rounding.
A product is exact, so a sum of n products in f32, in any order, is within n 2^-23 sum |a b| (each addition errs by at
most an ulp, truncating ones included). Quantised values are exact: codes and scales are compared byte for byte.
"""
import ctypes
import itertools
import random
import re

import numpy as np
import pytest

from accy_amd import hip
from accy_amd import tensor as T
from accy_amd import workloads as W
from conftest import hip_run, to_f32
from test_mutated_programs import _mutate, _plan_status
from test_zz_no_alloc import _Bound, _capture, _hip_runtime, _same

GRID = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
HALF_STEP = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}


def say(msg):
    print(msg, flush=True)


def floats(x, dtype):
    """Values of a type from float64, nearest even."""
    return W.to_dtype(np.asarray(x, np.float64), dtype)


def wide(x, dtype):
    return to_f32(np.asarray(x), dtype).astype(np.float64)


def quantized(x):
    """(codes as 0 .. 15, scale bytes, values) of float64 x blocked along its last axis, from the definition."""
    b = np.asarray(x, np.float64).reshape(*x.shape[:-1], -1, 32)
    finite = np.isfinite(b).all(-1)
    top = np.where(finite, np.abs(np.where(np.isfinite(b), b, 0.0)).max(-1), 1.0)
    e = np.where(top > 0, np.frexp(np.where(top > 0, top, 1.0))[1] - 1, -10000)
    byte = np.clip(e - 2, -127, 127) + 127
    y = np.where(finite[..., None], np.ldexp(np.where(np.isfinite(b), b, 0.0), (127 - byte)[..., None]), 0.0)
    # the nearest grid value, ties to the even code
    d = np.abs(np.abs(y)[..., None] - GRID)
    best = d.min(-1)
    code = np.argmin(d, -1)
    above = np.minimum(code + 1, 7)
    tie = (np.take_along_axis(d, above[..., None], -1)[..., 0] == best) & (above != code) & (code % 2 == 1)
    code = np.where(tie, above, code)
    value = np.where(finite[..., None], np.copysign(np.ldexp(GRID[code], (byte - 127)[..., None]), b), np.nan)
    return code + 8 * np.signbit(b), np.where(finite, byte, 255), value.reshape(x.shape)


def packed(code):
    c = code.reshape(*code.shape[:-2], -1).astype(np.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4)


def encoded(x):
    """Codes and scale bytes, u8, of float64 x."""
    code, byte, _ = quantized(x)
    return packed(code), byte.astype(np.uint8)


def decoded(codes, scales):
    table = np.concatenate([GRID, -GRID])
    v = np.stack([table[codes & 15], table[codes >> 4]], -1).reshape(*codes.shape[:-1], -1, 32)
    v = np.where((scales == 255)[..., None], np.nan, np.ldexp(v, scales.astype(np.int64)[..., None] - 127))
    return v.reshape(*codes.shape[:-1], -1)


def assert_within(got, want, tol, what=""):
    bad = ~((np.abs(got - want) <= tol) | (np.isnan(got) & np.isnan(want)) | (got == want))
    assert not bad.any(), f"{what}: {bad.sum()} of {bad.size} off, first {np.argwhere(bad)[0]}: {got[bad][0]} for {want[bad][0]} (tolerance {np.broadcast_to(tol, want.shape)[bad][0]})"


# ---- recording and planning (no device) ----

def _error(fn):
    with pytest.raises(T.TensorError) as e:
        fn()
    return e.value.name


def test_recorded_types():
    b = T.Builder("p")
    x = b.input("bf16", col=64, row=5)
    q = x.quantize_mx4("col")  # moved to the end
    assert q.codes.ty == T.Type("u8", (("row", 5), ("col.codes", 32))) and q.scales.ty == T.Type("u8", (("row", 5), ("col.scales", 2)))
    assert q.dims == (("row", 5), ("col", 64)) and q.dequantize("f32").ty == T.Type("f32", (("row", 5), ("col", 64)))
    w = b.mx4(*b.inputs(T.mx4_specs("col", out=7, col=64)), "col")
    assert q.contract(w, "f16").ty == T.Type("f16", (("row", 5), ("out", 7)))
    cache = b.input_spec(T.cache_mx4_spec(3, 2, 96, 32))
    assert cache.ty.shape == (3, 2, 32 * 102)
    slots = b.input("i32", token=9)
    k = b.input("f32", token=9, kv_head=2, dim=96)
    assert cache.cache_write_mx4(k, k, slots).ty == cache.ty
    assert cache.cache_keys_mx4(slots, ("dim", 96), "f16").ty == T.Type("f16", (("token", 9), ("kv_head", 2), ("dim", 96)))
    qs = b.input("f32", seq=4, head=6, dim=96)
    assert qs.attend_mx4(cache, b.input("i32", seq=4, p=2), b.input("i32", seq=4)).ty == qs.ty


def test_recording_refuses_what_does_not_fit():
    b = T.Builder("p")
    x, i = b.input("f32", row=4, col=64), b.input("i32", row=4, col=64)
    assert _error(lambda: x.quantize_mx4("nope")) == "AxisNotFound"
    assert _error(lambda: x.quantize_mx4("row")) == "InvalidDimension"  # 4 is no multiple of 32
    assert _error(lambda: i.quantize_mx4("col")) == "DTypeMismatch"
    assert _error(lambda: T.mx4_specs("col", col=64, row=4)) == "InvalidPermutation"
    assert _error(lambda: T.mx4_specs("col", row=4, col=40)) == "InvalidDimension"
    codes, scales = b.inputs(T.mx4_specs("col", out=8, col=64))
    q = x.quantize_mx4("col")
    w = b.mx4(codes, scales, "col")
    assert _error(lambda: b.mx4(codes, codes, "col")) == "AxisExtentMismatch"
    assert _error(lambda: b.mx4(x, scales, "col")) == "DTypeMismatch"
    assert _error(lambda: b.mx4(codes, q.scales, "col")) == "ShapeMismatch"
    assert _error(lambda: q.contract(w, "f64")) == "DTypeMismatch"
    assert _error(lambda: q.contract(q, "f32")) == "DuplicateAxis"
    assert _error(lambda: q.contract(b.mx4(codes, scales, "other"), "f32")) == "AxisNotFound"
    assert _error(lambda: q.contract(b.mx4(*b.inputs(T.mx4_specs("col", out=8, col=32)), "col"), "f32")) == "AxisExtentMismatch"
    assert _error(lambda: T.cache_mx4_spec(1, 1, 48)) == "InvalidDimension"
    assert _error(lambda: T.cache_mx4_spec(1, 1, 64, 48)) == "InvalidDimension"
    cache = b.input_spec(T.cache_mx4_spec(3, 2, 64))
    k, slots = b.input("f32", token=9, kv_head=2, dim=64), b.input("i32", token=9)
    assert _error(lambda: cache.cache_write_mx4(k, b.input("f16", token=9, kv_head=2, dim=64), slots)) == "DTypeMismatch"
    assert _error(lambda: cache.cache_write_mx4(k, k, b.input("i32", token=8))) == "ShapeMismatch"
    assert _error(lambda: cache.cache_write_mx4(k, k, b.input("i64", token=9))) == "DTypeMismatch"
    many = b.input("f32", token=9, kv_head=4, dim=64)
    assert _error(lambda: cache.cache_write_mx4(many, many, slots)) == "AxisExtentMismatch"
    assert _error(lambda: cache.cache_keys_mx4(slots, ("dim", 96), "f32")) == "AxisExtentMismatch"
    pages, lengths = b.input("i32", seq=5, p=2), b.input("i32", seq=5)
    assert _error(lambda: b.input("f32", seq=5, head=3, dim=64).attend_mx4(cache, pages, lengths)) == "AxisExtentMismatch"
    assert _error(lambda: b.input("f32", seq=4, head=4, dim=64).attend_mx4(cache, pages, lengths)) == "ShapeMismatch"
    assert _error(lambda: b.input("f32", seq=5, dim=64).attend_mx4(cache, pages, lengths)) == "RankMismatch"
    assert _error(lambda: b.input("i32", seq=5, head=4, dim=64).attend_mx4(cache, pages, lengths)) == "DTypeMismatch"


U8 = lambda *e: ("u8", e)  # noqa: E731


@pytest.mark.parametrize("call,operands,result,reason", [
    ("codes", [("f32", (4, 40))], U8(4, 20), "multiple of 32"),
    ("codes", [("i32", (4, 64))], U8(4, 32), "i32 values"),
    ("codes", [("f32", (4, 64))], U8(4, 64), "K / 2 to a row"),
    ("scales", [("f32", (4, 64))], U8(3, 2), "K / 32 to a row"),
    ("scales", [("f32", (4, 64)), ("f32", (4, 64))], U8(4, 2), "1 operands"),
    ("values", [U8(4, 32), U8(4, 3)], ("f32", (4, 64)), "K / 32 scales"),
    ("values", [U8(4, 32), U8(4, 2)], ("f64", (4, 64)), "f64 values"),
    ("values", [U8(4, 32), U8(4, 2)], ("f32", (4, 96)), "two values for each"),
    ("contract", [U8(4, 32), U8(4, 2), U8(5, 16), U8(5, 1)], ("f32", (4, 5)), "different K"),
    ("contract", [U8(4, 32), U8(4, 2), U8(5, 32), U8(5, 2)], ("f32", (5, 4)), "rows of the first"),
    ("contract", [U8(4, 0), U8(4, 0), U8(5, 0), U8(5, 0)], ("f32", (4, 5)), "empty contraction"),
    ("cache_write", [U8(2, 1, 32 * 68), ("f32", (3, 1, 64)), ("f16", (3, 1, 64)), ("i32", (3,))], U8(2, 1, 32 * 68), "one type and shape"),
    ("cache_write", [U8(2, 1, 33 * 68), ("f32", (3, 1, 64)), ("f32", (3, 1, 64)), ("i32", (3,))], U8(2, 1, 33 * 68), "multiple of 32 tokens"),
    ("cache_write", [U8(2, 1, 32 * 68), ("f32", (3, 1, 64)), ("f32", (3, 1, 64)), ("i32", (4,))], U8(2, 1, 32 * 68), "slot for every token"),
    ("cache_write", [U8(2, 1, 32 * 68), ("f32", (3, 1, 64)), ("f32", (3, 1, 64)), ("i32", (3,))], U8(3, 1, 32 * 68), "cache's type"),
    ("cache_write", [U8(2, 2, 32 * 68), ("f32", (3, 1, 64)), ("f32", (3, 1, 64)), ("i32", (3,))], U8(2, 2, 32 * 68), "holds 2 heads"),
    ("cache_keys", [U8(2, 1, 32 * 34), ("i32", (3,))], ("f32", (3, 1, 288)), "head dimensions"),
    ("cache_values", [U8(1 << 27, 1, 32 * 34), ("i32", (3,))], ("f32", (3, 1, 32)), "2^31 slots"),
    ("attend", [("f32", (5, 4, 64)), U8(2, 3, 32 * 68), ("i32", (5, 2)), ("i32", (5,))], ("f32", (5, 4, 64)), "4 query heads over 3"),
    ("attend", [("f32", (5, 4, 64)), U8(2, 2, 32 * 68), ("i32", (5, 2)), ("i32", (4,))], ("f32", (5, 4, 64)), "lengths"),
    ("attend", [("f32", (5, 4, 64)), U8(2, 2, 32 * 68), ("i32", (4, 2)), ("i32", (5,))], ("f32", (5, 4, 64)), "pages"),
    ("attend", [("f32", (5, 4, 64)), U8(2, 2, 32 * 68), ("i32", (5, 2)), ("i32", (5,))], ("f16", (5, 4, 64)), "queries' type"),
    ("attend", [("f32", (5, 64)), U8(2, 2, 32 * 68), ("i32", (5, 2)), ("i32", (5,))], ("f32", (5, 64)), "queries are"),
    ("attend", [("f32", (5, 4, 64)), U8(2, 2, 32 * 68), ("i32", (5, 1 << 27)), ("i32", (5,))], ("f32", (5, 4, 64)), "2^31 keys"),
    ("nothing", [("f32", (4, 64))], ("f32", (4, 64)), "is not supported"),
])
def test_planning_refuses_what_the_wire_may_carry(call, operands, result, reason):
    """The wire carries a custom call's result type, so a program that was not recorded here is checked again."""
    dims = lambda i, e: [(f"a{i}_{j}", n) for j, n in enumerate(e)]  # noqa: E731

    def body(b, a):
        return b.custom_call(f"accy.mx4.{call}", 1, a, T.Type(result[0], tuple(dims("r", result[1]))))
    prog = T.define("bad", [T.spec(d, *dims(i, e)) for i, (d, e) in enumerate(operands)], body)
    with pytest.raises(hip.HipError) as e:
        hip.plan_source(prog)
    assert e.value.status == hip.COMPILE_FAILED and reason in e.value.message and f"accy.mx4.{call}" in e.value.message


def test_planning_refuses_other_versions():
    p = T.define("v2", [T.spec("f32", r=2, c=32)], lambda b, a: b.custom_call("accy.mx4.scales", 2, a, T.Type("u8", (("r", 2), ("s", 1)))))
    with pytest.raises(hip.HipError) as e:
        hip.plan_source(p)
    assert e.value.status == hip.COMPILE_FAILED and "version 2" in e.value.message


def test_codes_and_scales_are_one_kernel_that_evaluates_its_operand():
    def body(b, a):
        q = a[0].mul(a[1]).quantize_mx4("k")
        return [q.codes, q.scales]
    src = hip.plan_source(T.define("p", [T.spec("bf16", m=8, k=64), T.spec("bf16", k=64)], body), compile=True)
    assert src.count("__global__") == 1


def test_values_of_new_codes_are_stored_by_their_kernel():
    def source(body):
        return hip.plan_source(T.define("p", [T.spec("bf16", m=8, k=64), T.spec("f32", m=8, k=64)], body), compile=True)

    def both(b, a):
        q = a[0].quantize_mx4("k")
        return [q.codes, q.scales, q.dequantize("bf16"), q.dequantize("f32")]
    assert source(both).count("__global__") == 1

    def back(b, a):
        return [a[1].quantize_mx4("k").dequantize("f16")]  # nobody else reads codes and scales
    src = source(back)
    assert src.count("__global__") == 1 and "i0 / 2)" not in src and "[i0 / 32]" not in src

    def mixed(b, a):  # codes of one tensor with scales of another are no tensor's own
        q, r = a[0].quantize_mx4("k"), a[1].quantize_mx4("k")
        return [b.mx4(q.codes, r.scales, "k").dequantize("bf16"), q.scales, r.codes]
    assert source(mixed).count("__global__") == 3


# ---- quantisation ----

def _roundtrip(shape, dtype):
    def body(b, a):
        q = a[0].quantize_mx4("k")
        return [q.codes, q.scales, q.dequantize(dtype)]
    return T.define("roundtrip", [T.spec(dtype, **{f"r{i}": n for i, n in enumerate(shape[:-1])}, k=shape[-1])], body)


def _check_roundtrip(x, dtype):
    codes, scales, values = hip_run(_roundtrip(x.shape, dtype), [x])
    code, byte, value = quantized(wide(x, dtype))
    finite = byte != 255
    want = packed(code)
    ok = np.repeat(finite, 16, -1)
    assert np.array_equal(scales, byte)
    assert np.array_equal(codes[ok], want[ok])
    got, rounded = wide(values, dtype), wide(floats(np.where(np.isnan(value), 0.0, value), dtype), dtype)
    assert np.array_equal(np.isnan(got), np.isnan(value))
    assert np.array_equal(got[~np.isnan(value)], rounded[~np.isnan(value)])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("shape", [(32,), (1, 32), (3, 96), (7, 5, 64), (1000, 224), (129, 4096)])
def test_quantize_and_back(shape, dtype):
    rng = np.random.default_rng(1)
    x = rng.standard_normal(shape) * np.exp(rng.uniform(-6, 6, shape[:-1] + (1,)))
    x.reshape(-1)[::53] *= 30.0
    _check_roundtrip(floats(x, dtype), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_quantize_borders(dtype):
    """Ties, saturation, signed zeros, powers of two, the largest and smallest values, NaN and infinity in one block only."""
    ties = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.2500001, 0.74999, 6.0, 6.9, 7.5, 0.0, 0.5, 1.0, 4.0])
    rows = []
    tiny = {"bf16": -133, "f16": -24, "f32": -149}[dtype]
    top = {"bf16": 125, "f16": 13, "f32": 125}[dtype]
    for e in (0, 1, -3, top - 2, tiny + 2, tiny + 5, tiny + 9, tiny + 24 if dtype != "f16" else -10):
        rows.append(np.concatenate([np.ldexp(ties, e), -np.ldexp(ties, e)]))
    rows.append(np.zeros(32))
    rows.append(-np.zeros(32))
    for special in (np.nan, np.inf, -np.inf):
        r = np.linspace(-1, 1, 32)
        r[17] = special
        rows.append(r)
    rows.append(np.full(32, 2.0 ** tiny))
    with np.errstate(over="ignore", invalid="ignore"):
        x = np.stack(rows)
        f = x.astype(np.float16) if dtype == "f16" else x.astype(np.float32)
        if dtype == "bf16":
            f = (f.view(np.uint32) >> 16).astype(np.uint16)
            f = np.where(np.isnan(x), np.uint16(0x7fc0), f)
    _check_roundtrip(f, dtype)


@pytest.mark.gpu
def test_quantize_evaluates_its_operand_and_moves_the_axis():
    rng = np.random.default_rng(2)
    x, g = rng.standard_normal((64, 9)).astype(np.float32), rng.standard_normal(64).astype(np.float32)

    def body(b, a):
        q = a[0].mul(a[1]).quantize_mx4("k")
        return [q.codes, q.scales]
    codes, scales = hip_run(T.define("p", [T.spec("f32", k=64, m=9), T.spec("f32", k=64)], body), [x, g])
    want = encoded((x * g[:, None]).T.astype(np.float64))
    assert np.array_equal(codes, want[0]) and np.array_equal(scales, want[1])


def test_index_width():
    """Beyond 2^30 elements an index and a grid's stride no longer fit 32 bits together."""
    def body(b, a):
        m = a[0].quantize_mx4("c")
        return [m.codes, m.scales, b.mx4(a[1], a[2], "c").dequantize("f16"), a[0].add(a[0])]
    for rows, index in ((1 << 15, "i32_t"), ((1 << 15) + 1, "i64_t")):
        source = hip.plan_source(T.define("p", [T.spec("bf16", r=rows, c=1 << 15), *T.mx4_specs("c", r=rows, c=1 << 15)], body))
        assert set(re.findall(r"typedef (i\d\d_t) I;", source)) == {index} and f"values<1, {index}," in source


@pytest.mark.gpu
def test_values_read_back_in_other_types():
    """Values of new codes in three types, alone and beside the codes; codes of one tensor under another's scales."""
    rng = np.random.default_rng(23)
    x, y = floats(rng.standard_normal((7, 96)) * 3, "bf16"), floats(rng.standard_normal((7, 96)), "bf16")
    x[3, 40] = floats(np.array(np.nan), "bf16")
    specs = [T.spec("bf16", m=7, k=96)] * 2

    def three(b, a):
        q = a[0].quantize_mx4("k")
        return [q.dequantize(t) for t in ("bf16", "f16", "f32")]

    def mixed(b, a):
        q, r = a[0].quantize_mx4("k"), a[1].quantize_mx4("k")
        return [q.codes, r.scales, b.mx4(q.codes, r.scales, "k").dequantize("f32"), r.dequantize("f32"), q.scales]
    want = quantized(wide(x, "bf16"))[2]
    for got, t in zip(hip_run(T.define("p", specs, three), [x, y]), ("bf16", "f16", "f32")):
        assert np.array_equal(wide(got, t), want, equal_nan=True)
    codes, scales, got, back, own = hip_run(T.define("p", specs, mixed), [x, y])
    assert np.array_equal(got.astype(np.float64), decoded(codes, scales), equal_nan=True)
    assert np.array_equal(back.astype(np.float64), quantized(wide(y, "bf16"))[2]) and np.array_equal(scales, quantized(wide(y, "bf16"))[1])
    assert np.array_equal(own, quantized(wide(x, "bf16"))[1])


@pytest.mark.gpu
def test_quantize_more_than_2_to_the_30():
    """1.1 G values, rows that repeat: so do codes, scales and values."""
    rows, cols = 33600, 1 << 15
    row = floats(np.random.default_rng(19).standard_normal((25, cols)), "bf16")
    spec = T.spec("bf16", g=rows // 25, r=25, c=cols)
    x = np.broadcast_to(row, (rows // 25, 25, cols))

    def body(b, a):
        m = a[0].quantize_mx4("c")
        return [m.codes, m.scales, m.dequantize("bf16")]
    say("quantize 1.1 G")
    got = hip_run(T.define("p", [spec], body), [np.ascontiguousarray(x)])
    want = hip_run(T.define("p", [T.spec("bf16", g=1, r=25, c=cols)], body), [row[None]])
    for g, w in zip(got, want):
        for i in range(len(g)):
            assert np.array_equal(g[i], w[0])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_values_of_every_code_and_scale(dtype):
    codes = np.tile(np.arange(256, dtype=np.uint8).reshape(16, 16), (256, 1))
    scales = np.repeat(np.arange(256, dtype=np.uint8), 16)[:, None]
    prog = T.define("v", list(T.mx4_specs("k", r=4096, k=32)), lambda b, a: b.mx4(a[0], a[1], "k").dequantize(dtype))
    got = wide(hip_run(prog, [codes, scales])[0], dtype)
    want = decoded(codes, scales)
    with np.errstate(over="ignore", invalid="ignore"):
        limit = {"bf16": 3.39e38, "f16": 65519.0, "f32": 3.41e38}[dtype]
        rounded = np.where(np.abs(want) > limit, np.copysign(np.inf, want), wide(floats(np.clip(np.nan_to_num(want), -limit, limit), dtype), dtype))
    rounded = np.where(np.isnan(want), np.nan, rounded)
    assert np.array_equal(got, rounded, equal_nan=True)


# ---- products ----

def _product(m, n, k, dtype, tail=None, rows=None):
    def body(b, a):
        y = b.mx4(a[0], a[1], "k").contract(b.mx4(a[2], a[3], "k"), dtype)
        return y if tail is None else tail(b, y, a[4:])
    return T.define("product", [*T.mx4_specs("k", m=m, k=k), *T.mx4_specs("k", n=n, k=k), *(rows or [])], body)


def _operands(m, n, k, seed, spread=3):
    rng = np.random.default_rng(seed)
    out = []
    for r in (m, n):
        out += [rng.integers(0, 256, (r, k // 2), dtype=np.uint8), rng.integers(127 - spread, 128 + spread, (r, k // 32)).astype(np.uint8)]
    return out


def _check_product(got, ops, dtype, what=""):
    a, b = decoded(ops[0], ops[1]), decoded(ops[2], ops[3])
    want, mass = a @ b.T, np.abs(a) @ np.abs(b).T
    k = a.shape[1]
    assert_within(wide(got, dtype), want, HALF_STEP[dtype] * np.abs(want) + (1 + HALF_STEP[dtype]) * k * 2.0 ** -23 * mass, what)


# every kernel's sizes: single rows, fewer and more than a tile in each direction, K of one block, odd numbers of blocks, and long
PRODUCTS = [(1, 1, 32), (1, 7, 64), (16, 33, 96), (5, 1000, 160), (17, 64, 2048), (33, 65, 224), (64, 31, 1056), (100, 257, 512),
            (129, 129, 544), (256, 256, 1024), (300, 511, 1184), (513, 260, 4096), (1, 4096, 8192), (48, 520, 4128)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_contract(m, n, k, dtype):
    ops = _operands(m, n, k, m + n + k)
    say(f"contract {m} {n} {k} {dtype}")
    _check_product(hip_run(_product(m, n, k, dtype), ops)[0], ops, dtype)


# the large tiles, ragged: 128 x 128 and 256 x 256, K in whole steps of 512, of 128 and neither, K split
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,dtype,tile,splits", [
    (1100, 4100, 672, "bf16", 128, 1), (260, 4100, 1280, "f16", 128, 1), (1000, 4100, 128, "f32", 256, 1), (1000, 4000, 256, "f32", 128, 1), (2500, 4100, 1184, "f32", 256, 1),
    (2100, 4200, 1664, "bf16", 256, 1), (2100, 4200, 2048, "f16", 256, 1), (200, 1000, 28672, "bf16", 128, 8), (1024, 1000, 8320, "f32", 128, 1)])
def test_contract_large(m, n, k, dtype, tile, splits):
    prog = _product(m, n, k, dtype)
    src = hip.plan_source(prog)
    assert f"BM = {tile}, BN = {tile}" in src and f"SPLITS = {splits};" in src
    ops = _operands(m, n, k, m + n + k)
    say(f"contract {m} {n} {k} {dtype}")
    _check_product(hip_run(prog, ops)[0], ops, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(3, 40, 96), (130, 300, 544), (600, 2600, 1056)])
def test_contract_keeps_nan_blocks_to_their_rows(m, n, k):
    """A NaN scale makes the sums it is in NaN and no others, whatever the other scales are."""
    ops = _operands(m, n, k, 5)
    ops[1][m // 2, k // 64], ops[3][n - 1, 0] = 255, 255
    ops[1][0, :], ops[3][0, :] = 20, 230
    got = wide(hip_run(_product(m, n, k, "f32"), ops)[0], "f32")
    nan = np.zeros((m, n), bool)
    nan[m // 2, :], nan[:, n - 1] = True, True
    assert np.array_equal(np.isnan(got), nan)
    a, b = decoded(ops[0], ops[1]), decoded(ops[2], ops[3])
    assert_within(np.where(nan, 0, got), np.where(nan, 0, np.nan_to_num(a) @ np.nan_to_num(b).T),
                  k * 2.0 ** -23 * (np.abs(np.nan_to_num(a)) @ np.abs(np.nan_to_num(b)).T))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(4, 48, 64), (70, 300, 1024), (520, 2512, 512), (200, 1000, 8192)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_contract_with_a_fused_epilogue(m, n, k, dtype):
    """An elementwise region after the product runs in its kernel: a bias, an activation and a residual."""
    rng = np.random.default_rng(3)
    ops = _operands(m, n, k, 4, 1)
    bias, res = floats(rng.standard_normal(n), dtype), floats(rng.standard_normal((m, n)) * 4, dtype)

    def tail(b, y, a):
        return y.add(a[0]).max(b.full_float(T.Type(dtype, ()), 0.0)).add(a[1])
    prog = _product(m, n, k, dtype, tail, [T.spec(dtype, n=n), T.spec(dtype, m=m, n=n)])
    # the elementwise operations evaluate the product's rounded value: apart from it, they are the same program
    y = hip_run(_product(m, n, k, dtype), ops)[0]
    after = T.define("tail", [T.spec(dtype, m=m, n=n), T.spec(dtype, n=n), T.spec(dtype, m=m, n=n)], lambda b, a: tail(b, a[0], a[1:]))
    want = hip_run(after, [y, bias, res])[0]
    got = hip_run(prog, ops + [bias, res])[0]
    assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    assert "map" not in {line.split()[1].split(":")[0] for line in hip.plan_source(prog).splitlines() if line.startswith("// ") and " grid " in line}


@pytest.mark.gpu
def test_contract_of_several_axes_and_empty_rows():
    rng = np.random.default_rng(6)
    x = rng.standard_normal((3, 5, 64)).astype(np.float32)
    w = rng.standard_normal((4, 6, 64)).astype(np.float32)

    def body(b, a):
        return a[0].quantize_mx4("k").contract(a[1].quantize_mx4("k"), "f32")
    got = hip_run(T.define("p", [T.spec("f32", b=3, t=5, k=64), T.spec("f32", h=4, d=6, k=64)], body), [x, w])[0]
    a, b = quantized(x.astype(np.float64))[2], quantized(w.astype(np.float64))[2]
    want, mass = np.einsum("btk,hdk->bthd", a, b), np.einsum("btk,hdk->bthd", np.abs(a), np.abs(b))
    assert_within(got.astype(np.float64), want, 64 * 2.0 ** -22 * mass)
    none = hip_run(T.define("p", [T.spec("f32", b=0, t=5, k=64), T.spec("f32", h=4, d=6, k=64)], body), [x[:0], w])[0]
    assert none.shape == (0, 5, 4, 6)


# ---- the cache ----

def empty_cache(pages, heads, dim, page, rng):
    """Bytes that a cache might hold: any codes, scales around 1, some blocks NaN (rows never written)."""
    c = rng.integers(0, 256, (pages, heads, page * (dim + dim // 16)), dtype=np.uint8)
    s = c[..., page * dim:]
    s[...] = np.where(rng.random(s.shape) < 0.1, 255, rng.integers(120, 132, s.shape))
    return c


def cache_parts(cache, dim):
    """(key codes, key scales, value codes, value scales), views [page, head, token, bytes]."""
    page = cache.shape[2] // (dim + dim // 16)
    at = np.cumsum([0, page * dim // 2, page * dim // 2, page * dim // 32, page * dim // 32])
    kc, vc, ks, vs = (cache[..., at[i]:at[i + 1]].reshape(*cache.shape[:2], page, -1) for i in range(4))
    return kc, ks, vc, vs


def written(cache, keys, values, slots):
    """The cache after the tokens, one after the other."""
    out = cache.copy()
    kc, ks, vc, vs = cache_parts(out, keys.shape[-1])
    page = kc.shape[2]
    for t, s in enumerate(slots.reshape(-1)):
        if 0 <= s < cache.shape[0] * page:
            for x, codes, scales in ((keys, kc, ks), (values, vc, vs)):
                codes[s // page, :, s % page], scales[s // page, :, s % page] = encoded(x.reshape(-1, *x.shape[-2:])[t])
    return out


def _write_program(pages, heads, dim, page, tokens, dtype):
    row = T.spec(dtype, token=tokens, kv_head=heads, dim=dim)
    return T.define("write", [T.cache_mx4_spec(pages, heads, dim, page), row, row, T.spec("i32", token=tokens)],
                    lambda b, a: a[0].cache_write_mx4(a[1], a[2], a[3]))


@pytest.mark.gpu
@pytest.mark.parametrize("pages,heads,dim,page,tokens,dtype", [
    (1, 1, 32, 32, 1, "f32"), (2, 3, 64, 64, 5, "bf16"), (3, 8, 128, 64, 70, "f16"), (4, 2, 96, 32, 128, "bf16"), (5, 16, 256, 128, 33, "f32"),
    (40, 1, 64, 256, 9000, "f16"), (2, 2, 64, 32, 0, "bf16")])
def test_cache_write_and_read(pages, heads, dim, page, tokens, dtype):
    rng = np.random.default_rng(tokens + dim)
    n = pages * page
    cache = empty_cache(pages, heads, dim, page, rng)
    keys, values = (floats(rng.standard_normal((tokens, heads, dim)) * 3, dtype) for _ in range(2))
    # any slots: some of them twice, some outside on either side
    slots = rng.integers(-3, n + 3, tokens).astype(np.int32)
    if tokens > 3:
        slots[-1], slots[1], slots[2] = slots[0], 2 ** 31 - 1, -2 ** 31
    say(f"cache write {pages} {heads} {dim} {page} {tokens} {dtype}")
    got = hip_run(_write_program(pages, heads, dim, page, tokens, dtype), [cache, keys, values, slots])[0]
    want = written(cache, wide(keys, dtype), wide(values, dtype), slots)
    assert np.array_equal(got, want)
    ask = np.concatenate([rng.integers(-3, n + 3, 37), [0, n - 1, n, -1, 2 ** 31 - 1, -2 ** 31]]).astype(np.int32)
    prog = T.define("read", [T.cache_mx4_spec(pages, heads, dim, page), T.spec("i32", slot=len(ask))],
                    lambda b, a: [a[0].cache_keys_mx4(a[1], ("dim", dim), dtype), a[0].cache_values_mx4(a[1], ("dim", dim), dtype)])
    kc, ks, vc, vs = cache_parts(want, dim)
    for back, codes, scales in zip(hip_run(prog, [want, ask]), (kc, vc), (ks, vs)):
        rows = decoded(codes, scales).transpose(0, 2, 1, 3).reshape(n, heads, dim)
        inside = (ask >= 0) & (ask < n)
        exact = np.where(inside[:, None, None], rows[np.clip(ask, 0, n - 1)], 0.0)
        assert np.array_equal(wide(back, dtype), exact, equal_nan=True)


def _device_run(prog, buffers, outputs, stream):
    with hip.Hip(prog) as ex:
        ex.launch_device([b.ptr for b in buffers], [o.ptr for o in outputs], stream.handle)
        stream.synchronize()


@pytest.mark.gpu
def test_cache_write_in_place():
    """A cache that comes in and goes out may be one buffer, which then changes only in the tokens' rows; where something
    else of the program reads what was in it, it may not."""
    rng = np.random.default_rng(9)
    cache = empty_cache(4, 2, 64, 32, rng)
    keys, values = (floats(rng.standard_normal((6, 2, 64)), "bf16") for _ in range(2))
    slots = np.array([5, 40, -1, 127, 128, 64], np.int32)
    want = written(cache, wide(keys, "bf16"), wide(values, "bf16"), slots)
    stream = hip.Stream()
    bufs = [hip.DeviceBuffer.from_array(x) for x in (cache, keys, values, slots)]
    prog = _write_program(4, 2, 64, 32, 6, "bf16")
    _device_run(prog, bufs, bufs[:1], stream)
    assert np.array_equal(bufs[0].download(np.empty_like(cache)), want)
    # another buffer: the input stays as it is
    bufs[0].upload(cache)
    other = hip.DeviceBuffer(cache.nbytes)
    _device_run(prog, bufs, [other], stream)
    assert np.array_equal(other.download(np.empty_like(cache)), want) and np.array_equal(bufs[0].download(np.empty_like(cache)), cache)

    def both(b, a):
        return [a[0].cache_write_mx4(a[1], a[2], a[3]), a[0].cache_keys_mx4(a[3], ("dim", 64), "bf16")]
    row = T.spec("bf16", token=6, kv_head=2, dim=64)
    reads = T.define("reads", [T.cache_mx4_spec(4, 2, 64, 32), row, row, T.spec("i32", token=6)], both)
    out = hip.DeviceBuffer(6 * 2 * 64 * 2)
    for outputs in ([bufs[0], out], [bufs[1], out]):
        with pytest.raises(hip.HipError) as e:
            _device_run(reads, bufs, outputs, stream)
        assert e.value.status == hip.INVALID_BUFFER
    # nor may the cache be bound again as another input, nor to a part of itself
    for p, ins in ((bufs[0].ptr, [bufs[0], bufs[0], bufs[2], bufs[3]]), (bufs[0].ptr + 64, bufs)):
        with hip.Hip(prog) as ex, pytest.raises(hip.HipError) as e:
            ex.launch_device([b.ptr for b in ins], [p], stream.handle)
        assert e.value.status == hip.INVALID_BUFFER
    stream.destroy()


# ---- attention over the cache ----

def attention(q, cache, pages, lengths):
    """(output, sum of p |v|, largest sum of |q k|) in float64; q [seq, query, head, dim]."""
    S, Q, heads, dim = q.shape
    kc, ks, vc, vs = cache_parts(cache, dim)
    K, V = decoded(kc, ks), decoded(vc, vs)
    P, H, page, _ = K.shape
    out, mass, most = np.zeros(q.shape), np.zeros(q.shape), 0.0
    for b, i, h in itertools.product(range(S), range(Q), range(heads)):
        n = min(max(int(lengths[b]), 0), pages.shape[1] * page) - (Q - 1 - i)
        keys = [(pages[b, j // page], j % page) for j in range(max(n, 0)) if 0 <= pages[b, j // page] < P]
        if not keys:
            continue
        kh = h // (heads // H)
        k, v = (np.stack([x[p, kh, r] for p, r in keys]) for x in (K, V))
        s = k @ q[b, i, h] / np.sqrt(dim)
        p = np.exp(s - s.max())
        p /= p.sum()
        out[b, i, h], mass[b, i, h] = p @ v, p @ np.abs(v)
        most = max(most, np.nanmax(np.abs(k) @ np.abs(q[b, i, h])) / np.sqrt(dim))
    return out, mass, most


def finite_cache(pages, heads, dim, page, rng):
    c = np.zeros((pages, heads, page * (dim + dim // 16)), np.uint8)
    for x in np.split(np.arange(4), 2):
        codes, scales = (cache_parts(c, dim)[i] for i in x)
        codes[...], scales[...] = encoded(rng.standard_normal((pages, heads, page, dim)) * 1.5)
    return c


def _attend_program(q, cache, pages, dtype):
    dims = [("seq", q.shape[0]), ("query", q.shape[1]), ("head", q.shape[2]), ("dim", q.shape[3])]
    return T.define("attend", [T.spec(dtype, *dims), T.spec("u8", page=cache.shape[0], kv_head=cache.shape[1], byte=cache.shape[2]),
                               T.spec("i32", seq=q.shape[0], at=pages.shape[1]), T.spec("i32", seq=q.shape[0])],
                    lambda b, a: a[0].attend_mx4(a[1], a[2], a[3]))


def _check_attend(q, cache, pages, lengths, dtype, got=None):
    if got is None:
        got = hip_run(_attend_program(q, cache, pages, dtype), [q, cache, pages, lengths])[0]
    want, mass, most = attention(wide(q, dtype), cache, pages, lengths)
    dim, n = q.shape[3], pages.shape[1] * (cache.shape[2] // (q.shape[3] + q.shape[3] // 16))
    # A score errs by its sum's (3 dim) 2^-23 and three roundings, of the sum of |q k| at most, which is also a bound of its
    # largest distance to the running maximum; a probability by that, 2^-21 of the hardware's exponential and the parts it is
    # split into (2^-17 for two, less for three); the sums over n keys by n 2^-23, the joins' scalings by 2^-18 of 64 or fewer. Numerator and
    # denominator both. An f16 result below 2^-14 is off by half of f16's smallest step, 2^-24, and no longer by a share of itself.
    rel = 2 * ((3 * dim + 4) * 2.0 ** -23 * most + 2.0 ** -21 + 2.0 ** -17 * (dtype != "f32") + (n + 64) * 2.0 ** -23 * 3)
    least = 2.0 ** -25 if dtype == "f16" else 1e-37
    assert_within(wide(got, dtype), want, HALF_STEP[dtype] * np.abs(want) + (1 + HALF_STEP[dtype]) * rel * mass + least)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("seqs,query,heads,kv,dim,page,slots", [
    (1, 1, 1, 1, 32, 32, 1), (3, 1, 4, 4, 64, 64, 2), (4, 1, 8, 2, 128, 64, 5), (2, 1, 12, 1, 96, 32, 9), (3, 4, 6, 3, 64, 128, 3),
    (2, 3, 7, 1, 256, 32, 4), (2, 5, 16, 2, 128, 64, 3), (1, 33, 2, 1, 64, 64, 2), (5, 1, 5, 5, 160, 96, 2), (2, 1, 40, 1, 128, 64, 20)])
def test_attend(seqs, query, heads, kv, dim, page, slots, dtype):
    rng = np.random.default_rng(seqs * 100 + dim + slots)
    P = seqs * slots + 2
    cache = finite_cache(P, kv, dim, page, rng)
    q = floats(rng.standard_normal((seqs, query, heads, dim)) * 2, dtype)
    pages = rng.permutation(P)[:seqs * slots].reshape(seqs, slots).astype(np.int32)
    lengths = rng.integers(0, slots * page + 1, seqs).astype(np.int32)
    lengths[0] = slots * page
    say(f"attend {seqs} {query} {heads} {kv} {dim} {page} {slots} {dtype}")
    _check_attend(q, cache, pages, lengths, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,query,kv", [("bf16", 1, 2), ("f16", 3, 1), ("f32", 2, 4)])
def test_attend_lengths(dtype, query, kv):
    """Every length around a page's and a step's ends; none, negative and too large; fewer keys than queries."""
    rng = np.random.default_rng(11)
    lengths = np.array([0, 1, 2, 3, 31, 32, 33, 63, 64, 65, 95, 96, 97, 127, 128, -5, 1000, 2 ** 31 - 1, -2 ** 31], np.int32)
    S = len(lengths)
    cache = finite_cache(2 * S, kv, 64, 64, rng)
    q = floats(rng.standard_normal((S, query, 4, 64)), dtype)
    got = _check_attend(q, cache, rng.permutation(2 * S).reshape(S, 2).astype(np.int32), lengths, dtype)
    assert not wide(got, dtype)[lengths <= 0].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,query", [("bf16", 1), ("f16", 4), ("f32", 3)])
def test_attend_masked_places_hold_anything(dtype, query):
    """Rows behind a sequence's end and pages of others hold NaN; pages outside the cache hold no keys; a NaN among a
    sequence's own keys reaches the queries that see it and no others."""
    rng = np.random.default_rng(12)
    page, dim, kv, heads = 32, 64, 2, 6
    cache = finite_cache(12, kv, dim, page, rng)
    kc, ks, vc, vs = cache_parts(cache, dim)
    pages = np.arange(12).reshape(3, 4).astype(np.int32)
    lengths = np.array([70, 33, 100], np.int32)
    for b, n in enumerate(lengths):
        for j in range(n, 4 * page):
            ks[pages[b, j // page], :, j % page], vs[pages[b, j // page], :, j % page] = 255, 255
    pages[0, 1], pages[1, 3], pages[2, 0], pages[2, 3] = -1, 12, 2 ** 31 - 1, -2 ** 31
    q = floats(rng.standard_normal((3, query, heads, dim)), dtype)
    _check_attend(q, cache, pages, lengths, dtype)
    # the newest key of sequence 1 is NaN: its value for one head only, and, for another, its key
    vs[pages[1, 1], 0, 0, 1] = 255
    got = wide(_check_attend(q, cache, pages, lengths, dtype), dtype)
    seen = np.isnan(got)
    assert seen[1, -1, :3, 32:].all() and not seen[1, -1, :3, :32].any()
    assert not seen[1, :-1].any() and not seen[1, :, 3:].any() and not seen[[0, 2]].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attend_with_very_different_scores(dtype):
    """One key far above the rest at the end, or at the start; scores of both signs, hundreds apart."""
    rng = np.random.default_rng(13)
    cache = finite_cache(8, 1, 128, 64, rng)
    kc, ks, vc, vs = cache_parts(cache, 128)
    q = floats(rng.standard_normal((2, 1, 3, 128)) * 8, dtype)
    pages = np.arange(8).reshape(2, 4).astype(np.int32)
    kc[pages[0, 3], 0, 60], ks[pages[0, 3], 0, 60] = encoded(wide(q, dtype)[0, 0, 0] * 4)
    kc[pages[1, 0], 0, 0], ks[pages[1, 0], 0, 0] = encoded(wide(q, dtype)[1, 0, 1] * 4)
    _check_attend(q, cache, pages, np.array([256, 250], np.int32), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("below", [2, 8, 13])
def test_attend_small_queries_beside_large_ones(dtype, below):
    """One dim of each block is 2^below or more times the others; every key has the same large value there, so what tells
    the keys apart is the small ones' part of the score."""
    rng = np.random.default_rng(15)
    cache = finite_cache(4, 2, 64, 32, rng)
    kc, ks, vc, vs = cache_parts(cache, 64)
    kc[...] |= 0x11  # no zeros
    kc[..., 0::16] |= 7
    ks[...] = 127
    q = rng.uniform(1, 2, (2, 3, 4, 64)) * 2.0 ** -below
    q[..., 0::32] = 1.9
    pages = np.arange(4).reshape(2, 2).astype(np.int32)
    _check_attend(floats(q * 8, dtype), cache, pages, np.array([64, 40], np.int32), dtype)


@pytest.mark.gpu
def test_attend_without_sequences_pages_or_cache():
    rng = np.random.default_rng(14)
    cache = finite_cache(2, 1, 64, 32, rng)
    q = rng.standard_normal((3, 1, 2, 64)).astype(np.float32)
    for c, pages in ((cache, np.zeros((3, 0), np.int32)), (cache[:0], np.zeros((3, 4), np.int32))):
        got = hip_run(_attend_program(q, c, pages, "f32"), [q, c, pages, np.full(3, 50, np.int32)])[0]
        assert got.shape == q.shape and not got.any()
    none = hip_run(_attend_program(q[:0], cache, np.zeros((0, 4), np.int32), "f32"), [q[:0], cache, np.zeros((0, 4), np.int32), np.zeros(0, np.int32)])[0]
    assert none.shape == (0, 1, 2, 64)


@pytest.mark.gpu
def test_cache_beyond_32_bits():
    """A cache of 4.5 GB, its last pages in use, against a small one that holds the same tokens."""
    rng = np.random.default_rng(16)
    pages, kv, dim, page, tokens, dtype = 64000, 8, 128, 64, 100, "f16"
    keys, values = (floats(rng.standard_normal((tokens, kv, dim)), dtype) for _ in range(2))
    q = floats(rng.standard_normal((1, 1, 16, dim)), dtype)
    row = T.spec(dtype, token=tokens, kv_head=kv, dim=dim)

    def body(b, a):
        cache = a[0].cache_write_mx4(a[1], a[2], a[3])
        return [cache, cache.cache_keys_mx4(a[3], ("dim", dim), dtype), cache.cache_values_mx4(a[3], ("dim", dim), dtype),
                a[4].attend_mx4(cache, a[5], a[6])]
    out = []
    for n in (2, pages):
        prog = T.define("far", [T.cache_mx4_spec(n, kv, dim, page), row, row, T.spec("i32", token=tokens), T.spec(dtype, seq=1, query=1, head=16, dim=dim),
                                T.spec("i32", seq=1, at=2), T.spec("i32", seq=1)], body)
        table = np.array([[n - 1, n - 2]], np.int32)
        at = np.arange(tokens)
        slots = (table[0, at // page] * page + at % page).astype(np.int32)
        say(f"{n} pages")
        stream = hip.Stream()
        cache = hip.DeviceBuffer(n * kv * page * (dim + dim // 16))
        ins = [cache] + [hip.DeviceBuffer.from_array(x) for x in (keys, values, slots, q, table, np.array([tokens], np.int32))]
        got = [np.zeros_like(keys), np.zeros_like(keys), np.zeros_like(q)]
        outs = [hip.DeviceBuffer(x.nbytes) for x in got]
        _device_run(prog, ins, [cache] + outs, stream)
        out.append([o.download(x) for o, x in zip(outs, got)])
        for x in ins + outs:
            x.free()
        stream.destroy()
    _same(out[1], out[0])
    for got, want in zip(out[0], (keys, values)):
        assert np.array_equal(wide(got, dtype), quantized(wide(want, dtype))[2])


@pytest.mark.gpu
def test_operands_used_twice():
    """One quantised tensor on both sides of a product; one tensor as keys and values."""
    rng = np.random.default_rng(17)
    x = floats(rng.standard_normal((70, 96)), "f32")

    def gram(b, a):
        m = a[0].quantize_mx4("k")
        return m.contract(b.mx4(m.codes.rename("m", "n"), m.scales.rename("m", "n"), "k"), "f32")
    got = hip_run(T.define("gram", [T.spec("f32", m=70, k=96)], gram), [x])[0]
    v = quantized(wide(x, "f32"))[2]
    assert_within(got.astype(np.float64), v @ v.T, 2 * 96 * 2.0 ** -23 * (np.abs(v) @ np.abs(v).T))
    cache = finite_cache(2, 3, 32, 32, rng)
    slots = np.array([63, 0, 5], np.int32)
    prog = T.define("both", [T.cache_mx4_spec(2, 3, 32, 32), T.spec("f32", token=3, kv_head=3, dim=32), T.spec("i32", token=3)],
                    lambda b, a: a[0].cache_write_mx4(a[1], a[1], a[2]))
    rows = x.reshape(-1)[:3 * 3 * 32].reshape(3, 3, 32)
    assert np.array_equal(hip_run(prog, [cache, rows, slots])[0], written(cache, wide(rows, "f32"), wide(rows, "f32"), slots))


@pytest.mark.gpu
def test_cache_grows_in_a_scan():
    """Tokens made one after the other inside a scan, each from the attention over those before: as single programs."""
    rng = np.random.default_rng(18)
    S, H, D, page, per, dtype = 3, 2, 64, 32, 2, "bf16"
    cache = finite_cache(S * per, H, D, page, rng)
    table = rng.permutation(S * per).reshape(S, per).astype(np.int32)
    lengths = np.array([5, 31, 32], np.int32)
    x = floats(rng.standard_normal((S, H, D)), dtype)
    specs = [T.spec(dtype, seq=S, head=H, dim=D), T.cache_mx4_spec(S * per, H, D, page), T.spec("i32", seq=S, at=per), T.spec("i32", seq=S)]

    def step(b, c):
        x, cache, table, lengths = c
        one, width = b.full("i32", 1, ("seq", S)), b.full("i32", page, ("seq", S))
        at = lengths.div(width)
        second = at.compare("ge", one)
        pages = [table.mul(b.iota("i32", "at", ("seq", S), ("at", per)).compare("eq", b.full("i32", i, ("seq", S), ("at", per))).select(
            b.full("i32", 1, ("seq", S), ("at", per)), b.full("i32", 0, ("seq", S), ("at", per)))).sum("at") for i in range(per)]
        slots = second.select(pages[1], pages[0]).mul(width).add(lengths.sub(at.mul(width)))
        rows = x.rename("head", "kv_head")
        cache = cache.cache_write_mx4(rows, rows, slots)
        return [x.attend_mx4(cache, table, lengths.add(one)).add(x), cache, table, lengths.add(one)]
    ins = [x, cache, table, lengths]
    loop = T.define("loop", specs, lambda b, a: (lambda l: [l, b.projection(l, 1)])(b.scan(4, a, step)))
    one = T.define("one", specs, lambda b, a: step(b, a))
    want = ins
    for _ in range(4):
        want = hip_run(one, want)
    got = hip_run(loop, ins)
    _same(got, want[:2])


# ---- the operators together: one token of every sequence through a decoder block ----

STEPS = [  # seqs, model, heads, kv, hd, ffn, page, pages per sequence, dtype
    (5, 256, 4, 2, 64, 512, 32, 4, "bf16"), (33, 160, 6, 1, 96, 288, 64, 3, "f16"), (1, 128, 2, 2, 32, 256, 32, 1, "f32"),
    (8, 512, 8, 2, 128, 1024, 64, 40, "bf16")]


def _step(seqs, model, heads, kv, hd, ffn, page, per, dtype, seed=20):
    """The program and its inputs; each sequence's own pages in some order, its new token the last of its length."""
    rng = np.random.default_rng(seed)
    pages = seqs * per + 1
    prog = W.decoder_step_mx4_program(seqs, model, heads, kv, hd, ffn, pages, page, per, dtype)

    def weight(*shape):
        return list(encoded(rng.standard_normal(shape) * shape[-1] ** -0.5))

    def gains():
        return floats(1 + 0.1 * rng.standard_normal(model), dtype)
    x = floats(rng.standard_normal((seqs, model)), dtype)
    table = rng.permutation(pages)[:seqs * per].reshape(seqs, per).astype(np.int32)
    lengths = rng.integers(1, per * page + 1, seqs).astype(np.int32)
    lengths[-1] = per * page
    slots = (table[np.arange(seqs), (lengths - 1) // page] * page + (lengths - 1) % page).astype(np.int32)
    ins = ([x, gains()] + weight(heads, hd, model) + weight(kv, hd, model) + weight(kv, hd, model) + weight(model, heads * hd) + [gains()] +
           weight(ffn, model) + weight(model, ffn) + [finite_cache(pages, kv, hd, page, rng), slots, table, lengths])
    for v, t in zip(ins, prog.input_types()):
        assert v.shape == t.shape and v.dtype == T.NUMPY_DTYPE[t.dtype]
    return prog, ins


def _alone(body, specs, ins):
    return hip_run(T.define("alone", specs, body), ins)


@pytest.mark.gpu
@pytest.mark.parametrize("sizes", STEPS)
def test_decoder_step_is_its_operators_one_by_one(sizes):
    """The program, with what it fuses, against programs of one operator each, bit for bit; and its attention and products
    against 64 bits on the way."""
    seqs, model, heads, kv, hd, ffn, page, per, dtype = sizes
    prog, ins = _step(*sizes)
    x, g1, g2, cache, slots, table, lengths = ins[0], ins[1], ins[10], ins[15], ins[16], ins[17], ins[18]
    say(f"decoder step {sizes}")
    y, after = hip_run(prog, ins)
    S, M = ("seq", seqs), ("model", model)

    def codes(v, axis, n):
        return _alone(lambda b, a: list(_pair(a[0].quantize_mx4(axis))), [T.spec(dtype, S, (axis, n))], [v])

    def normed(v, g):
        return codes(_alone(lambda b, a: W.rms_norm(b, a[0], a[1], "model", dtype), [T.spec(dtype, S, M), T.spec(dtype, M)], [v, g])[0], "model", model)

    def product(v, w, axis, n, *rows):
        specs = [*T.mx4_specs(axis, S, (axis, n)), *T.mx4_specs(axis, *rows, (axis, n))]
        got = _alone(lambda b, a: b.mx4(a[0], a[1], axis).contract(b.mx4(a[2], a[3], axis), dtype), specs, v + w)[0]
        p, q = decoded(*v), decoded(*w).reshape(-1, n)
        want, mass = p @ q.T, np.abs(p) @ np.abs(q).T
        assert_within(wide(got, dtype).reshape(seqs, -1), want, HALF_STEP[dtype] * np.abs(want) + 2 * n * 2.0 ** -23 * mass + (2.0 ** -25 if dtype == "f16" else 0))
        return got
    h = normed(x, g1)
    q = product(h, ins[2:4], "model", model, ("head", heads), ("dim", hd))
    k, v = (product(h, ins[i:i + 2], "model", model, ("kv_head", kv), ("dim", hd)) for i in (4, 6))
    row = T.spec(dtype, S, ("kv_head", kv), ("dim", hd))
    filled = _alone(lambda b, a: a[0].cache_write_mx4(a[1], a[2], a[3]),
                    [T.cache_mx4_spec(len(cache), kv, hd, page), row, row, T.spec("i32", S)], [cache, k, v, slots])[0]
    assert np.array_equal(filled, after) and np.array_equal(filled, written(cache, wide(k, dtype), wide(v, dtype), slots))
    o = _alone(lambda b, a: a[0].attend_mx4(a[1], a[2], a[3]), [T.spec(dtype, S, ("head", heads), ("dim", hd)),
               T.cache_mx4_spec(len(cache), kv, hd, page), T.spec("i32", S, ("at", per)), T.spec("i32", S)], [q, filled, table, lengths])[0]
    _check_attend(q[:, None], filled, table, lengths, dtype, o[:, None])
    back = product(codes(o.reshape(seqs, -1), "att", heads * hd), ins[8:10], "att", heads * hd, M)
    two = [T.spec(dtype, S, M)] * 2
    x1 = _alone(lambda b, a: a[0].add(a[1]), two, [x, back])[0]
    f = product(normed(x1, g2), ins[11:13], "model", model, ("ffn", ffn))
    f = _alone(lambda b, a: W.gelu(b, a[0], dtype), [T.spec(dtype, S, ("ffn", ffn))], [f])[0]
    last = product(codes(f, "ffn", ffn), ins[13:15], "ffn", ffn, M)
    want = _alone(lambda b, a: a[0].add(a[1]), two, [x1, last])[0]
    assert np.array_equal(y.view(np.uint8), want.view(np.uint8))


def _pair(q):
    return q.codes, q.scales


def test_decoder_step_plan():
    """Elementwise work is part of the operators' kernels: norms' sums, codes, products, the cache, attention and nothing else;
    the cache may be updated in place."""
    source = hip.plan_source(_step(*STEPS[0])[0])
    labels = [line.split()[1].split(":")[0] for line in source.splitlines() if line.startswith("// ") and " grid " in line]
    assert labels == ["row", "quantize", "mx4", "mx4", "mx4", "cache_write", "mx4_attend", "quantize", "mx4", "row", "quantize", "mx4", "quantize", "mx4"]


CACHE = 15  # the step's input; its second output


def _step_bound(prog, ins, in_place):
    bound = _Bound(prog, ins)
    if in_place:
        bound.op[1] = bound.ip[CACHE]

    def restore():
        """The outputs cleared, the cache as it came in."""
        bound.clear()
        bound.dins[CACHE].upload(ins[CACHE])

    def outputs():
        y, cache = bound.read()
        return [y, bound.dins[CACHE].download(np.empty_like(ins[CACHE])) if in_place else cache]
    return bound, restore, outputs


@pytest.mark.gpu
@pytest.mark.parametrize("scratch", [False, True])
@pytest.mark.parametrize("in_place", [False, True])
def test_decoder_step_captured_into_hip_graphs(scratch, in_place):
    """The steps of two models captured on a stream of their own and replayed in turn, with eager steps of the other between the
    replays; the cache in a buffer of its own and in place. Every replay equals run_hip bit for bit."""
    rt, s, stream = _hip_runtime(), hip.Session(), hip.Stream()
    progs = [_step(*STEPS[0]), _step(*STEPS[3], seed=21)]
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


@pytest.mark.gpu
def test_decoder_steps_on_two_streams_at_once():
    """Two executors of one program on two streams, their steps submitted in turn without waiting; then every step of both has
    run: the caches hold the tokens of all, the outputs the last step's."""
    sizes = STEPS[0]
    prog, ins = _step(*sizes)
    rng = np.random.default_rng(22)
    tokens = [floats(rng.standard_normal(ins[0].shape), sizes[-1]) for _ in range(3)]
    want = []
    for order in ((0, 1, 2), (2, 1, 0)):
        cache = ins[CACHE]
        for t in order:
            y, cache = hip_run(prog, [tokens[t]] + ins[1:CACHE] + [cache] + ins[CACHE + 1:])
        want.append([y, cache])
    s, streams = hip.Session(), [hip.Stream(), hip.Stream()]
    handles = [s.compile(prog) for _ in streams]
    bounds = [_step_bound(prog, ins, True) for _ in streams]
    xs = [hip.DeviceBuffer.from_array(t) for t in tokens]
    try:
        for again in range(3):
            for _, restore, _ in bounds:
                restore()
            for step in range(3):
                for i, (bound, _, _) in enumerate(bounds):
                    bound.ip[0] = xs[step if i == 0 else 2 - step].ptr
                    bound.call(handles[i], False, streams[i])
            for i in (0, 1):
                streams[i].synchronize()
                _same(bounds[i][2](), want[i])
    finally:
        for b in [b for b, _, _ in bounds] + xs:
            b.free()
        for h in handles:
            s.release(h)
        for st in streams:
            st.destroy()


@pytest.mark.parametrize("program", [
    lambda: W.decoder_step_mx4_program(0, 256, 4, 2, 64, 512, 24, 32, 4), lambda: W.decoder_program(0, 32, 64, 2, 32, 128),
    lambda: T.define("sums", [T.spec("bf16", m=0, k=64)] * 2, lambda b, a: a[0].mul(a[1]).sum("k"))])
def test_no_sequences_are_planned(program):
    """Nothing to compute for a batch of none."""
    hip.plan_source(program())


def test_every_mutated_program_gets_a_status():
    lib, rng = hip.library(), random.Random(1)
    bases = [p.encode() for p in (_step(*STEPS[0])[0], _step(*STEPS[1])[0], _product(1000, 4000, 256, "bf16"), _product(40, 50, 96, "f32"),
                                  _write_program(4, 2, 64, 32, 9000, "f16"))]
    seen = {_plan_status(lib, _mutate(rng.choice(bases), rng)) for _ in range(1500)}
    assert seen <= set(range(9)) and {0, 1} <= seen


@pytest.mark.gpu
def test_decoder_step_tuned_and_profiled():
    """Launch tuning of a program with custom calls keeps its results; profiling names their kernels."""
    prog, ins = _step(*STEPS[1])
    want = hip_run(prog, ins)
    hip.tuning_clear()
    try:
        hip.tune(prog, ins, repeats=2)
        _same(hip_run(prog, ins), want)
    finally:
        hip.tuning_clear()
    bound, _, outputs = _step_bound(prog, ins, False)
    stream = hip.Stream()
    with hip.Hip(prog) as ex:
        ex.set_profiling(True)
        ex.launch_device(list(bound.ip), list(bound.op), stream.handle)
        kernels = ex.kernels()
        assert {"quantize", "gemm", "attention", "row"} == {k.klass for k in kernels} and all(k.last_ms > 0 for k in kernels)
        _same(outputs(), want)
    bound.free()
    stream.destroy()


@pytest.mark.gpu
def test_decoder_step_of_no_sequences():
    prog, ins = _step(*STEPS[0])
    none = W.decoder_step_mx4_program(0, *STEPS[0][1:6], len(ins[CACHE]), *STEPS[0][6:])
    y, cache = hip_run(none, [x[:0] if i in (0, 16, 17, 18) else x for i, x in enumerate(ins)])
    assert y.shape == (0, STEPS[0][1]) and np.array_equal(cache, ins[CACHE])
