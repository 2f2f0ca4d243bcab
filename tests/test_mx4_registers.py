"""Kernels of the 4-bit operators fit in their registers (CPU test, see test_kernel_registers.py): none uses scratch memory, whatever
its head dimension, type, number of queries, tile or epilogue. A spill in attention over several queries has cost a factor of two."""
import re
from concurrent.futures import ThreadPoolExecutor

import pytest

from accy_amd import hip, tensor as T, workloads as W
from accy_amd.build import KERNELS
from test_kernel_registers import HIPCC, _resources

pytestmark = pytest.mark.skipif(not HIPCC.exists(), reason="needs the ROCm compiler")


def _kernels(prog):
    """(label, source) of each kernel of a program, with the template texts in place of its #include lines."""
    out = []
    for part in re.split(r"^// (?=\S+ grid \d+ block \d+\n)", hip.plan_source(prog), flags=re.M)[1:]:
        label, body = part.split("\n", 1)
        body = re.sub(r'^#include "(gemm|mx4|mx4_contract)"\n', lambda m: (KERNELS / f"{m.group(1)}.h").read_text() + "\n", body, flags=re.M)
        out.append((label.split(":")[0], (KERNELS / "common.h").read_text() + "\n" + body))
    return out


def _attend(dim, dtype, queries):
    specs = [T.spec(dtype, seq=24, query=queries, head=32, dim=dim), T.cache_mx4_spec(1600, 8, dim), T.spec("i32", seq=24, at=64), T.spec("i32", seq=24)]
    return T.define("attend", specs, lambda b, a: a[0].attend_mx4(a[1], a[2], a[3]))


ATTENTION = [(d, t, q) for d in (32, 64, 96, 128, 160, 192, 224, 256) for t in ("bf16", "f16", "f32") for q in (1, 5)]


def test_attention_uses_no_scratch(tmp_path):
    with ThreadPoolExecutor(8) as ex:
        kernels = {c: [s for label, s in _kernels(_attend(*c)) if label == "mx4_attend"][0] for c in ATTENTION}
        used = dict(zip(kernels, ex.map(lambda c: _resources("attend_%d_%s_%d" % c, kernels[c], tmp_path), kernels)))
    assert not {c: r for c, r in used.items() if r["scratch"]}
    # one query of up to 128 dims in 16 bits: three workgroups to a CU
    assert not {c: r for c, r in used.items() if c[0] <= 128 and c[1] != "f32" and c[2] == 1 and r["vgpr"] + r["agpr"] > 168}


def _product(m, n, k, dtype, tail):
    def body(b, a):
        y = b.mx4(a[0], a[1], "k").contract(b.mx4(a[2], a[3], "k"), dtype)
        return y.add(a[4]) if tail == "residual" else W.gelu(b, y, dtype) if tail == "gelu" else y
    return T.define("product", [*T.mx4_specs("k", m=m, k=k), *T.mx4_specs("k", n=n, k=k), *([T.spec(dtype, m=m, n=n)] if tail == "residual" else [])], body)


# small tiles of four and two waves along K, large ones in whole steps of 128 and not, K split
PRODUCTS = [((16, 8192, 2048), 16), ((300, 2048, 8224), 32), ((1000, 1001, 992), 32), ((1100, 4100, 672), 128), ((1000, 4000, 256), 128), ((2048, 8192, 2048), 256),
            ((2500, 4100, 1184), 256), ((300, 2048, 8192), 128)]


def test_products_use_no_scratch(tmp_path):
    sources = []
    for (m, n, k), tile in PRODUCTS:
        for dtype, tail in (("bf16", "none"), ("f32", "residual"), ("bf16", "gelu")):
            found = _kernels(_product(m, n, k, dtype, tail))
            assert any(f"BM = {tile}," in s for _, s in found), (m, n, k)
            sources += [(f"{m} {n} {k} {dtype} {tail} {label}", s) for label, s in found]
    with ThreadPoolExecutor(8) as ex:
        used = list(ex.map(lambda c: (c[0], _resources(c[0], c[1], tmp_path)), sources))
    assert not [u for u in used if u[1]["scratch"]]


def test_decoder_step_uses_no_scratch(tmp_path):
    sources = list({s: (label, s) for label, s in _kernels(W.decoder_step_mx4_program())}.values())
    with ThreadPoolExecutor(8) as ex:
        used = list(ex.map(lambda c: (c[1][0], _resources(f"step_{c[0]}", c[1][1], tmp_path)), enumerate(sources)))
    assert len(used) >= 10 and not [u for u in used if u[1]["scratch"]]
