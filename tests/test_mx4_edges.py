"""Microscaled 4-bit floats where their values lie far apart and where a kernel's rarer paths run, against float64 (helpers and
tolerances: test_mx4.py)."""
import re

import numpy as np
import pytest

from accy_amd import hip
from accy_amd import tensor as T
from accy_amd import workloads as W
from conftest import hip_run
from test_mx4 import (HALF_STEP, _attend_program, _check_attend, _operands, _product, _write_program, assert_within, cache_parts, decoded,
                      empty_cache, finite_cache, floats, say, wide, written)


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
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_attend_huge_queries_and_tiny_keys(dtype):
    """Keys of the four smallest scales, 2^-127 on, many of them below the smallest normal number."""
    rng = np.random.default_rng(34)
    cache = finite_cache(4, 2, 64, 32, rng)
    ks = cache_parts(cache, 64)[1]
    ks[...] = rng.integers(0, 4, ks.shape)
    q = rng.standard_normal((2, 2, 4, 64)) * 2.0 ** 124
    _check_attend(floats(q, dtype), cache, np.arange(4).reshape(2, 2).astype(np.int32), np.array([64, 40], np.int32), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
def test_attend_of_queries_that_are_no_numbers(dtype):
    """A NaN or an infinity in a query makes its own outputs NaN, and 0 where it sees no key."""
    rng = np.random.default_rng(35)
    cache = finite_cache(6, 2, 64, 32, rng)
    lengths = np.array([64, 40, 1], np.int32)
    x = rng.standard_normal((3, 2, 4, 64))
    f = floats(x, dtype)
    bad = [(0, 0, 1, 5, np.nan), (0, 1, 2, 63, np.inf), (1, 1, 3, 0, -np.inf), (2, 0, 0, 7, np.nan)]
    for *at, v in bad:
        f[tuple(at)] = floats(np.array(v), dtype) if dtype != "bf16" else (0x7fc0 if np.isnan(v) else 0x7f80 if v > 0 else 0xff80)
    pages = np.arange(6).reshape(3, 2).astype(np.int32)
    got = wide(hip_run(_attend_program(f, cache, pages, dtype), [f, cache, pages, lengths])[0], dtype)
    nan = np.isnan(got)
    for b, i, h in np.ndindex(3, 2, 4):
        assert nan[b, i, h].all() if (b, i, h) in [(0, 0, 1), (0, 1, 2), (1, 1, 3)] else not nan[b, i, h].any()
    assert not got[2, 0].any()
    for *at, v in bad:
        f[tuple(at)] = 0
    clean = hip_run(_attend_program(f, cache, pages, dtype), [f, cache, pages, lengths])[0]
    assert np.array_equal(got[~nan], wide(_check_attend(f, cache, pages, lengths, dtype, clean), dtype)[~nan])


@pytest.mark.gpu
def test_attend_to_one_key_is_its_value():
    """Of every code under scales at both ends of the range, the smallest values below the smallest normal number."""
    scales = np.array([0, 1, 2, 3, 100, 127, 251, 252], np.uint8)
    cache = np.zeros((8, 1, 32 * 34), np.uint8)
    kc, ks, vc, vs = cache_parts(cache, 32)
    vc[:, 0, 0] = [0x10, 0x32, 0x54, 0x76, 0x98, 0xba, 0xdc, 0xfe, 0x01, 0x23, 0x45, 0x67, 0x89, 0xab, 0xcd, 0xef]
    vs[:, 0, 0, 0] = scales
    ks[...] = 127
    q = np.ones((8, 1, 1, 32), np.float32)
    got = hip_run(_attend_program(q, cache, np.zeros((8, 1)), "f32"), [q, cache, np.arange(8, dtype=np.int32)[:, None], np.ones(8, np.int32)])[0]
    assert np.array_equal(got[:, 0, 0].astype(np.float64), decoded(vc[:, 0, 0], vs[:, 0, 0]))


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


# ---- attention: paths that only some sizes take ----

# head dims whose scales take two load instructions, and others, over more steps than a wave has stages; several queries over splits;
# more than eight sequences and heads with more than one group of rows, the last set of eight not full
@pytest.mark.gpu
@pytest.mark.parametrize("seqs,query,heads,kv,dim,page,slots,dtype,splits", [
    (2, 1, 3, 1, 160, 64, 30, "bf16", 3), (1, 1, 2, 1, 224, 32, 50, "f32", 3), (1, 1, 4, 2, 256, 64, 26, "bf16", 3), (2, 1, 2, 2, 96, 32, 60, "f16", 3),
    (1, 3, 2, 1, 192, 32, 48, "f16", 3), (2, 4, 6, 2, 64, 64, 24, "f16", 3), (1, 5, 8, 2, 128, 32, 40, "f32", 2), (1, 40, 2, 1, 64, 32, 36, "bf16", 2),
    (3, 5, 16, 4, 64, 32, 6, "bf16", 1), (5, 3, 28, 4, 64, 32, 33, "f32", 2)])
def test_attend_long_ranges_splits_and_sets(seqs, query, heads, kv, dim, page, slots, dtype, splits):
    rng = np.random.default_rng(dim + slots)
    P = seqs * slots + 1
    cache = finite_cache(P, kv, dim, page, rng)
    q = floats(rng.standard_normal((seqs, query, heads, dim)) * 2, dtype)
    pages = rng.permutation(P)[:seqs * slots].reshape(seqs, slots).astype(np.int32)
    lengths = rng.integers(slots * page // 2, slots * page + 1, seqs).astype(np.int32)
    lengths[0] = slots * page - 3
    prog = _attend_program(q, cache, pages, dtype)
    assert f"SPLITS = {splits};" in hip.plan_source(prog)
    say(f"attend {seqs} {query} {heads} {kv} {dim} {page} {slots} {dtype}")
    _check_attend(q, cache, pages, lengths, dtype, hip_run(prog, [q, cache, pages, lengths])[0])


@pytest.mark.gpu
def test_attend_of_a_prompt_with_nan_values():
    """Each of 2048 queries among 2048 keys, eight of whose values are NaN: the queries from a NaN on are NaN in its block's dims, those
    before it as without it, and the call takes a few times as long, not as many times as there are queries."""
    rng = np.random.default_rng(36)
    n, dim, page = 2048, 64, 64
    cache = finite_cache(n // page, 1, dim, page, rng)
    q = floats(rng.standard_normal((1, n, 1, dim)), "bf16")
    pages, lengths = np.arange(n // page, dtype=np.int32)[None], np.array([n], np.int32)
    prog = _attend_program(q, cache, pages, "bf16")
    at = np.sort(rng.choice(n, 8, replace=False))
    dirty = cache.copy()
    for j in at:
        cache_parts(dirty, dim)[3][j // page, 0, j % page, 1] = 255
    got, took, stream = [], [], hip.Stream()
    with hip.Hip(prog) as ex:
        for c in (cache, dirty):
            bufs = [hip.DeviceBuffer.from_array(x) for x in (q, c, pages, lengths)]
            out = hip.DeviceBuffer(q.nbytes)
            times = []
            for _ in range(3):
                a, b = hip.Event(), hip.Event()
                a.record(stream)
                ex.launch_device([x.ptr for x in bufs], [out.ptr], stream.handle)
                b.record(stream)
                stream.synchronize()
                times.append(a.elapsed_ms(b))
            got.append(wide(out.download(np.empty_like(q)), "bf16")[0, :, 0])
            took.append(min(times))
            for x in bufs + [out]:
                x.free()
    stream.destroy()
    say(f"{took[0]:.3f} ms without, {took[1]:.3f} ms with NaN")
    nan = np.zeros((n, dim), bool)
    nan[at[0]:, 32:] = True
    assert np.array_equal(np.isnan(got[1]), nan) and np.array_equal(got[1][~nan], got[0][~nan])
    # a workgroup's sixteen queries weigh one after the other in the steps that hold a NaN
    assert took[1] < 20 * took[0]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("byte", [253, 254, 255])
def test_attend_keeps_values_beyond_f32_to_the_queries_that_see_them(dtype, byte):
    """The newest value is infinite (6 under the largest scales) or NaN: the last of three queries sees it, the others are as without it."""
    rng = np.random.default_rng(37)
    cache = finite_cache(2, 1, 64, 32, rng)
    q = floats(rng.standard_normal((1, 3, 4, 64)), dtype)
    pages, lengths = np.array([[1, 0]], np.int32), np.array([50], np.int32)
    prog = _attend_program(q, cache, pages, dtype)
    kc, ks, vc, vs = cache_parts(cache, 64)
    vc[0, 0, 17] = 0x77
    clean = wide(hip_run(prog, [q, cache, pages, lengths])[0], dtype)
    vs[0, 0, 17, 0] = byte
    got = wide(hip_run(prog, [q, cache, pages, lengths])[0], dtype)
    same = got == clean
    assert same[0, :2].all() and same[0, 2, :, 32:].all()
    assert not np.isfinite(got[0, 2, :, :32]).any(), got[0, 2, 0, :4]


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


# ---- products ----

def _tile(program):
    """(rows of a tile, waves along K or 0, workgroups along K)."""
    return tuple(int(x) for x in re.search(r"BM = (\d+), BN = \d+, GROUP_M = \d+, WK = (\d+), SPLITS = (\d+);", hip.plan_source(program)).groups())


# K split into 8, 4 and 2: the last share one group of four steps, shorter than the others or not, ending in one to three steps; K in
# whole steps of 128 and not
@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,dtype,splits", [(200, 1000, 18048, "f32", 8), (390, 1000, 24832, "bf16", 4), (257, 1500, 20000, "f16", 4), (513, 2048, 13152, "f32", 2)])
def test_contract_split_along_k(m, n, k, dtype, splits):
    prog = _product(m, n, k, dtype)
    assert _tile(prog) == (128, 0, splits)
    ops = _operands(m, n, k, m + n + k)
    say(f"contract {m} {n} {k} {dtype}")
    got = wide(hip_run(prog, ops)[0], dtype)
    a, b = decoded(*ops[:2]), decoded(*ops[2:])
    want, mass = a @ b.T, np.abs(a) @ np.abs(b).T
    tol = HALF_STEP[dtype] * np.abs(want) + (1 + HALF_STEP[dtype]) * k * 2.0 ** -23 * mass
    # f16 rounds to infinity from 65520 on (65504 and half of its step of 32)
    over = np.abs(got) == np.inf
    assert np.all(np.abs(want)[over] >= (65520.0 if dtype == "f16" else np.inf) - tol[over]) and np.array_equal(np.sign(got[over]), np.sign(want[over]))
    assert_within(np.where(over, 0, got), np.where(over, 0, want), tol)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,splits", [(300, 2048, 8192, 4), (257, 1500, 20000, 4), (1100, 4100, 672, 1), (2500, 4100, 1184, 1)])
@pytest.mark.parametrize("dtype", ["bf16", "f32"])
def test_contract_of_large_tiles_with_a_fused_epilogue(m, n, k, splits, dtype):
    """A bias, an activation and a residual in the kernel of a split product's sum, and in those of 128 x 128 and 256 x 256 tiles."""
    rng = np.random.default_rng(3)
    ops = _operands(m, n, k, 4, 1)
    bias, res = floats(rng.standard_normal(n), dtype), floats(rng.standard_normal((m, n)) * 4, dtype)

    def tail(b, y, a):
        return y.add(a[0]).max(b.full_float(T.Type(dtype, ()), 0.0)).add(a[1])
    rows = [T.spec(dtype, n=n), T.spec(dtype, m=m, n=n)]
    prog = _product(m, n, k, dtype, tail, rows)
    bm, wk, s = _tile(prog)
    assert bm >= 128 and not wk and s == splits
    say(f"contract {m} {n} {k} {dtype} with an epilogue")
    y = hip_run(_product(m, n, k, dtype), ops)[0]
    want = hip_run(T.define("tail", [T.spec(dtype, m=m, n=n)] + rows, lambda b, a: tail(b, a[0], a[1:])), [y, bias, res])[0]
    got = hip_run(prog, ops + [bias, res])[0]
    assert np.array_equal(got.view(np.uint8), want.view(np.uint8))
    assert "map" not in {line.split()[1].split(":")[0] for line in hip.plan_source(prog).splitlines() if line.startswith("// ") and " grid " in line}


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,tile", [(1100, 4100, 672, (128, 0, 1)), (1024, 1000, 8320, (128, 0, 1)), (2500, 4100, 1184, (256, 0, 1)), (2100, 4200, 1664, (256, 0, 1)),
                                        (300, 2048, 8192, (128, 0, 4)), (513, 2048, 13152, (128, 0, 2))])
def test_contract_of_large_tiles_keeps_nan_blocks_to_their_rows(m, n, k, tile):
    """NaN scales in the first and the last block of a row, beside rows of scales near both ends of the range."""
    prog = _product(m, n, k, "f32")
    assert _tile(prog) == tile
    ops = _operands(m, n, k, 5)
    ops[1][0, :], ops[3][0, :] = 20, 230
    ops[1][m // 2, k // 32 - 1], ops[3][n - 1, 0], ops[3][n // 3, k // 32 - 1] = 255, 255, 255
    say(f"contract {m} {n} {k} with NaN")
    got = wide(hip_run(prog, ops)[0], "f32")
    nan = np.zeros((m, n), bool)
    nan[m // 2, :], nan[:, n - 1], nan[:, n // 3] = True, True, True
    assert np.array_equal(np.isnan(got), nan)
    a, b = (np.nan_to_num(decoded(*ops[i:i + 2])) for i in (0, 2))
    assert_within(np.where(nan, 0, got), np.where(nan, 0, a @ b.T), k * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k,tile", [(5, 40, 64, 16), (33, 65, 128, 32), (130, 300, 256, 32), (1000, 4000, 256, 128), (1000, 4100, 128, 256), (2500, 4100, 256, 256)])
def test_contract_of_blocks_far_apart(m, n, k, tile):
    """Scales 2^20 apart within a row, so that an instruction's blocks are up to 2^40 apart. A block's 32 products are multiples of a
    quarter of its scale below 2^11 of it and so is their sum, exact in f32; a sum over B blocks then errs by an ulp of each of its B additions, and
    of those of up to 4 waves."""
    prog = _product(m, n, k, "f32")
    assert _tile(prog)[0] == tile
    ops = _operands(m, n, k, 7, 10)
    a, b = decoded(*ops[:2]), decoded(*ops[2:])
    tol = (k // 32 + 4) * 2.0 ** -23 * (np.abs(a) @ np.abs(b).T)
    assert_within(wide(hip_run(prog, ops)[0], "f32"), a @ b.T, tol)
