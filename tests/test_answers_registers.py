"""Kernels of heads, pages and log probabilities fit in their registers (CPU test, see test_kernel_registers.py): none uses scratch memory."""
import re
from concurrent.futures import ThreadPoolExecutor

import pytest

from accy_amd import hip, tensor as T, workloads as W
from accy_amd.build import KERNELS
from test_answers import _grad_program, _heads_program
from test_kernel_registers import HIPCC, _resources

pytestmark = pytest.mark.skipif(not HIPCC.exists(), reason="needs the ROCm compiler")


def _kernels(prog):
    """(label, source) of each kernel of a program, with the template texts in place of its #include lines."""
    out = []
    for part in re.split(r"^// (?=\S+ grid \d+ block \d+\n)", hip.plan_source(prog), flags=re.M)[1:]:
        label, body = part.split("\n", 1)
        body = re.sub(r'^#include "(\w+)"\n', lambda m: (KERNELS / f"{m.group(1)}.h").read_text() + "\n", body, flags=re.M)
        out.append((label.split(":")[0], (KERNELS / "common.h").read_text() + "\n" + body))
    return out


def _no_scratch(programs, tmp_path):
    sources = list({s: (label, s) for p in programs for label, s in _kernels(p)}.values())
    with ThreadPoolExecutor(8) as ex:
        used = list(ex.map(lambda c: (c[1][0], _resources(f"k{c[0]}", c[1][1], tmp_path)), enumerate(sources)))
    assert used and not [u for u in used if u[1]["scratch"]]
    return used


def test_heads_use_no_scratch(tmp_path):
    sizes = [(4001, 12, 3, 96, 32, 3, "neighbours", "f32", True), (8192, 16, 4, 128, 64, 0, "halves", "bf16", True), (64, 8, 2, 256, 128, 0, "halves", "f16", True),
             (9, 3, 2, 250, 125, 0, "halves", "f32", True), (100, 2, 2, 512, 256, 0, "halves", "f32", False), (100, 2, 2, 512, 256, 0, "neighbours", "bf16", True)]
    _no_scratch([p(*s) for s in sizes for p in (_heads_program, _grad_program)], tmp_path)


def _logits(rows, vocab, top, dtype):
    return T.define("p", [T.spec(dtype, row=rows, vocab=vocab), T.spec("i32", row=rows)],
                    lambda b, a: [v for p in [a[0].log_probs(a[1], "vocab", top=top)] for v in (p.token, p.entropy, p.top, p.top_tokens) if v is not None])


def _logits_grad(rows, vocab, dtype):
    return T.define("g", [T.spec(dtype, row=rows, vocab=vocab), T.spec("i32", row=rows), *[T.spec("f32", row=rows)] * 2], lambda b, a: a[0].log_probs_grad(*a[1:], "vocab"))


def test_log_probabilities_use_no_scratch(tmp_path):
    _no_scratch([_logits(*s, d) for s in ((8, 32000, 5), (2048, 50257, 20), (600, 515, 0), (1, 131073, 64)) for d in ("bf16", "f16", "f32")] +
                [_logits_grad(*s, d) for s in ((1001, 50257), (300, 1031), (8, 50257), (512, 65500)) for d in ("bf16", "f16", "f32")], tmp_path)


@pytest.mark.parametrize("chunks", [8, 11, 13, 16, 17, 19, 22])
def test_the_gradient_of_rows_that_fill_the_registers_uses_no_scratch(tmp_path, chunks):
    """Rows of 8 to 22 chunks of 16 bytes for each of 1024 threads, whole ones and such that start anywhere, in the registers of one workgroup."""
    used = _no_scratch([_logits_grad(300, chunks * 1024 * per - less, d) for d, per in (("bf16", 8), ("f16", 8), ("f32", 4)) for less in (0, per + 1)], tmp_path)
    assert [label for label, _ in used] == ["log_probs_grad"] * 6


def test_pages_and_the_step_use_no_scratch(tmp_path):
    row = T.spec("i32", row=9)
    fork = lambda slots, pages: T.define("f", [T.spec("i32", seq=4, slot=slots), T.spec("i32", seq=4), row, row, T.spec("i1", page=pages), T.spec("u8", page=pages, byte=4352)],  # noqa: E731
                                         lambda b, a: [v for f in [b.fork_pages(*a[:5], 64)] for v in (f.pages, f.slots, a[5].copy_pages(f.source, f.target))])
    used = _no_scratch([fork(7, 300), fork(2000, 200000), W.answers_step_mx4_program(), W.answers_step_mx4_program(dtype="f32")], tmp_path)
    # attention over shared keys: three workgroups to a CU for a row of 16 bits and 128 dims
    assert [u["vgpr"] + u["agpr"] for label, u in used if label == "mx4_attend"][0] <= 168
