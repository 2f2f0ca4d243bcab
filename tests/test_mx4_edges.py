"""Microscaled 4-bit floats where their values lie far apart and where a kernel's rarer paths run, against float64 (helpers and
tolerances: test_mx4.py)."""
import re

import numpy as np
import pytest

from accy_amd import hip
from accy_amd import tensor as T
from accy_amd import workloads as W
from conftest import hip_run
from test_mx4 import _attend_program, _check_attend, _write_program, cache_parts, empty_cache, finite_cache, floats, say, wide, written


# ---- attention: queries of any spread ----

@pytest.mark.gpu
@pytest.mark.parametrize("dtype,apart", [("bf16", 13), ("bf16", 17), ("bf16", 20), ("bf16", 60), ("f16", 13), ("f16", 15), ("f32", 24), ("f32", 40)])
def test_attend_small_queries_beside_large_ones_that_meet_zeros(dtype, apart):
    """Two dims of each block are 2^apart times the others, and every key is 0 there: the small ones are all of the score."""
    rng = np.random.default_rng(31)
    cache = finite_cache(4, 2, 64, 32, rng)
    cache_parts(cache, 64)[0][..., 0::8] &= 0xf0
    q = rng.uniform(1, 2, (2, 3, 4, 64)) * rng.choice([-1.0, 1.0], (2, 3, 4, 64))
    q[..., 0::16] = 2.0 ** apart
    pages = np.arange(4).reshape(2, 2).astype(np.int32)
    _check_attend(floats(q, dtype), cache, pages, np.array([64, 40], np.int32), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_tiny_queries_and_huge_keys(dtype):
    """Queries around 2^-105 against keys as much above 1: scores of ordinary size."""
    rng = np.random.default_rng(32)
    cache = finite_cache(4, 2, 96, 32, rng)
    cache_parts(cache, 96)[1][...] += 100
    q = rng.standard_normal((2, 2, 4, 96)) * 2.0 ** -100
    pages = np.arange(4).reshape(2, 2).astype(np.int32)
    _check_attend(floats(q, dtype), cache, pages, np.array([64, 40], np.int32), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("below", [2, 8, 13])
def test_attend_small_queries_beside_a_large_one_that_all_keys_share(dtype, below):
    """One dim of each block is 2^below or more times the others; every key is 6 there, so only the small ones tell keys apart."""
    rng = np.random.default_rng(15)
    cache = finite_cache(4, 2, 64, 32, rng)
    kc, ks, vc, vs = cache_parts(cache, 64)
    kc[...] |= 0x11  # no zeros
    kc[..., 0::16] = kc[..., 0::16] & 0xf0 | 7
    ks[...] = 127
    q = rng.uniform(1, 2, (2, 3, 4, 64)) * 2.0 ** -below
    q[..., 0::32] = 1.9
    pages = np.arange(4).reshape(2, 2).astype(np.int32)
    _check_attend(floats(q * 8, dtype), cache, pages, np.array([64, 40], np.int32), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("seqs,query,heads,kv,dim,page,slots", [(3, 1, 8, 2, 128, 64, 20), (2, 3, 6, 2, 96, 32, 5), (1, 1, 4, 4, 32, 32, 2), (2, 1, 16, 1, 256, 32, 12)])
def test_attend_in_16_bits_is_rounded_once(seqs, query, heads, kv, dim, page, slots, dtype):
    """Scores, probabilities and sums are f32's whatever the type: results are the bits of the f32 ones, rounded."""
    rng = np.random.default_rng(dim)
    cache = finite_cache(seqs * slots, kv, dim, page, rng)
    q = floats(rng.standard_normal((seqs, query, heads, dim)) * 2, dtype)
    pages = rng.permutation(seqs * slots).reshape(seqs, slots).astype(np.int32)
    lengths = rng.integers(1, slots * page + 1, seqs).astype(np.int32)
    full = wide(q, dtype).astype(np.float32)
    got, want = (hip_run(_attend_program(x, cache, pages, t), [x, cache, pages, lengths])[0] for x, t in ((q, dtype), (full, "f32")))
    assert np.array_equal(got, floats(want, dtype))


# ---- the cache ----

# tokens per workgroup of 5, 10, 21, 12 and 1
@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,dtype", [(8, 96, "bf16"), (4, 96, "f16"), (2, 96, "f32"), (5, 64, "bf16"), (5, 128, "f32"), (17, 256, "bf16")])
def test_cache_write_of_a_padded_batch(heads, dim, dtype):
    """Most tokens are padding, some slots come twice; workgroups whose tokens are no multiple of the four searched at a time."""
    rng = np.random.default_rng(heads + dim)
    pages, page, tokens = 3, 32, 333
    cache = empty_cache(pages, heads, dim, page, rng)
    keys, values = (floats(rng.standard_normal((tokens, heads, dim)), dtype) for _ in range(2))
    slots = np.where(rng.random(tokens) < 0.7, -1, rng.integers(0, pages * page, tokens)).astype(np.int32)
    got = hip_run(_write_program(pages, heads, dim, page, tokens, dtype), [cache, keys, values, slots])[0]
    assert np.array_equal(got, written(cache, wide(keys, dtype), wide(values, dtype), slots))


# ---- 32-bit and 64-bit indices ----

def _index_types(program):
    return set(re.findall(r"typedef (i\d\d_t) I;", hip.plan_source(program)))


def test_a_large_cache_leaves_other_kernels_their_indices():
    """A cache that only cache calls take is indexed by none of the generated kernels: a step over 1.3 GB of it, and a scan of steps,
    index their norms and codes in 32 bits; arithmetic on the cache itself does not."""
    assert _index_types(W.decoder_step_mx4_program(pages=40000)) == {"i32_t"}
    row = T.spec("bf16", token=4, kv_head=4, dim=128)
    specs = [T.cache_mx4_spec(80000, 4, 128), row, T.spec("i32", token=4)]

    def step(b, c):
        cache = c[0].cache_write_mx4(c[1], c[1], c[2])
        return [cache, c[1].add(cache.cache_keys_mx4(c[2], ("dim", 128), "bf16")), c[2]]
    assert _index_types(T.define("loop", specs, lambda b, a: (lambda l: [l, b.projection(l, 1).add(a[1])])(b.scan(4, a, step)))) == {"i32_t"}
    assert _index_types(T.define("sum", specs, lambda b, a: [step(b, a)[1], a[0].add(a[0])])) == {"i64_t"}


def test_row_kernels_and_folds_of_more_than_2_to_the_30():
    """Kernels whose grids stride by rows or single elements take 32 bits up to 1.75 x 2^30 elements."""
    def body(b, a):
        return [a[0].max("c"), a[0].max("r")]
    for rows, index in (((1 << 15) + 32, "i32_t"), (57000, "i32_t"), (57400, "i64_t")):
        assert _index_types(T.define("p", [T.spec("bf16", r=rows, c=1 << 15)], body)) == {index}


@pytest.mark.gpu
def test_row_kernel_and_fold_more_than_2_to_the_30():
    """1.8 G values in rows that repeat, indexed in 32 bits: the largest of each row and of each column."""
    group, cols = 25, 1 << 15
    groups = 2276  # 1.736 x 2^30
    row = floats(np.random.default_rng(33).standard_normal((group, cols)), "bf16")

    prog = T.define("p", [T.spec("bf16", r=groups * group, c=cols)], lambda b, a: [a[0].max("c"), a[0].max("r")])
    assert _index_types(prog) == {"i32_t"}
    say("rows of 1.8 G")
    top, columns = hip_run(prog, [np.tile(row, (groups, 1))])
    want = wide(row, "bf16")
    assert np.array_equal(wide(top, "bf16"), np.tile(want.max(1), groups)) and np.array_equal(wide(columns, "bf16"), want.max(0))
