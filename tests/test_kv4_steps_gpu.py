"""Attention over a 4-bit cache whose value vectors have no step, or one far below their offset:
the weights, which such vectors do not scale, stay finite however the scores rise, and so do the
sums of weights times offsets."""
import numpy as np
import pytest

import ammon_b200 as ab

import kv4_ref as ref
from test_kv4_gpu import attend, check_attention, rt  # noqa: F401

pytestmark = pytest.mark.gpu

ROUND = {ab.F32: 0.0, ab.BF16: 2.0 ** -8}


def scales_of(step, offset):
    bits = [ref.bf16_bits(np.asarray(a, np.float32)).astype(np.uint32) for a in (step, offset)]
    return bits[0] | bits[1] << np.uint32(16)


def constant(values, head):
    """Codes and scales of vectors [...] that hold one number (a bf16 value) throughout."""
    values = np.asarray(values, np.float32)
    assert np.array_equal(ref.bf16_values(ref.bf16_bits(values)), values)
    return (np.zeros(values.shape + (ref.words_of(head),), np.uint32),
            scales_of(np.zeros_like(values), values))


def rising(lead, kv, seq, head, octaves):
    """Key vectors of one number each and the nats a unit of it is to be worth, by which scores
    rise by `octaves` of base 2 over the cache, in 256 steps."""
    level = np.floor(np.arange(seq) * 256.0 / seq) - 128
    return constant(np.broadcast_to(level, lead + (kv, seq)), head), octaves / 256 * np.log(2)


def query_for(per, rows, heads, head):
    """Equal components whose score against a key vector of ones is `per` nats."""
    return np.full((rows, heads, head), per / np.sqrt(head), np.float32)


def constant_bound(value, n, out_dtype):
    """The weights cancel: what is left is the f32 sums of n weights and of their products (random
    roundings, six standard deviations), the division, and the output's own rounding."""
    return abs(value) * (6 * np.sqrt(n) * 2.0 ** -24 + 2.0 ** -21 + ROUND[out_dtype])


SHAPES = [  # rows, heads, kv, head, seq: units of eight warps, more of them than blocks (four
    # warps), eight slots a unit, eight slots at head 128
    (3, 4, 1, 64, 4100), (310, 2, 2, 32, 900), (160, 8, 2, 48, 1300), (1, 8, 1, 128, 9000)]


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("octaves", [10, 30, 60, 200, -200])
@pytest.mark.parametrize("rows,heads,kv,head,seq", SHAPES)
@pytest.mark.parametrize("value", [0.0, 1.0, -3.0, 999424.0, 2.0 ** 100])
def test_one_value_throughout(rt, rows, heads, kv, head, seq, octaves, out_dtype, value):
    """The output is that value, whatever the scores."""
    rng = np.random.default_rng(rows)
    keys, per = rising((rows,), kv, seq, head, octaves)
    layer = list(keys) + list(constant(np.full((rows, kv, seq), value), head))
    positions = [seq - 1 - int(p) for p in rng.integers(0, 20, rows)]
    got = attend(rt, query_for(per, rows, heads, head), layer, positions, out_dtype)
    assert np.isfinite(got).all()
    assert np.abs(got - value).max() <= constant_bound(value, seq, out_dtype)
    rt.synchronize()


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("octaves", [30, 60, 200])
@pytest.mark.parametrize("rows,heads,kv,head,seq", SHAPES)
def test_rows_without_a_step_before_and_between_others(rt, rows, heads, kv, head, seq, octaves,
                                                       out_dtype):
    """The first half has no steps, then every third vector has none; scores rise throughout, so
    what counts is the cache's end."""
    rng = np.random.default_rng(rows + octaves)
    keys, per = rising((rows,), kv, seq, head, octaves)
    codes, scales = ref.quantise(rng.standard_normal((rows, kv, seq, head)).astype(np.float32))
    flat = np.zeros(seq, bool)
    flat[:seq // 2] = True
    flat[::3] = True
    codes[:, :, flat], scales[:, :, flat] = constant(
        ref.bf16_values(ref.bf16_bits(rng.standard_normal((rows, kv, flat.sum()))
                                      .astype(np.float32))), head)
    layer = list(keys) + [codes, scales]
    positions = [seq - 1 - int(p) for p in rng.integers(0, 20, rows)]
    some = slice(0, 12)  # the 64-bit attention of so many rows
    q = query_for(per, rows, heads, head)
    got = attend(rt, q, layer, positions, out_dtype)
    assert np.isfinite(got).all()
    check_attention(got[some], q[some], [a[some] for a in layer], positions[some], out_dtype, False)
    rt.synchronize()


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("octaves", [100, 140, 300, -140, -300])
@pytest.mark.parametrize("step", [0.0, 0.5])
def test_scores_far_from_zero_from_the_first_position_on(rt, octaves, step, out_dtype):
    """All scores equal, their exponential alone past the range of f32 or below it."""
    rows, heads, kv, head, seq = 5, 4, 1, 64, 700
    rng = np.random.default_rng(3)
    codes = rng.integers(0, 2 ** 32, (rows, kv, seq, 8), dtype=np.uint32)
    scales = scales_of(np.full((rows, kv, seq), step), rng.integers(-8, 8, (rows, kv, seq)))
    layer = list(constant(np.ones((rows, kv, seq)), head)) + [codes, scales]
    positions = [699, 0, 31, 300, 255]
    q = query_for(octaves * np.log(2), rows, heads, head)
    got = attend(rt, q, layer, positions, out_dtype)
    assert np.isfinite(got).all()
    check_attention(got, q, layer, positions, out_dtype, False)
    rt.synchronize()


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("value,seq", [(2560.0, 131072), (3008.0, 131072), (2.0 ** 18, 1000),
                                       (1.0 * 2 ** 20, 131072), (-2.0 ** 60, 50000)])
def test_large_offsets_of_equal_weights(rt, value, seq, out_dtype):
    head = 16
    layer = (list(constant(np.ones((1, seq)), head)) + list(constant(np.full((1, seq), value), head)))
    got = attend(rt, np.zeros((1, 2, head), np.float32), layer, [seq - 1], out_dtype)
    assert np.isfinite(got).all()
    assert np.abs(got - value).max() <= constant_bound(value, seq, out_dtype)
    rt.synchronize()


def test_rows_whose_bf16_minimum_is_above_their_largest(rt):
    """Rows within 3003 .. 3003.4 have offset 3008 and no step."""
    head, seq = 64, 40000
    rng = np.random.default_rng(4)
    codes, scales = ref.quantise((3003 + 0.4 * rng.random((1, seq, head))).astype(np.float32))
    assert (scales == scales[0, 0]).all() and scales[0, 0] == scales_of(0.0, 3008.0)
    keys = ref.quantise(rng.standard_normal((1, seq, head)).astype(np.float32))
    q = rng.standard_normal((1, 3, head)).astype(np.float32)
    got = attend(rt, q, list(keys) + [codes, scales], [seq - 1])
    assert np.abs(got - 3008).max() <= constant_bound(3008.0, seq, ab.F32)


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
def test_head_size_one_of_bf16_values(rt, out_dtype):
    """Vectors of one bf16 element are all offset; scores as they come, of several hundred."""
    rows, heads, kv, seq = 4, 6, 2, 3000
    rng = np.random.default_rng(5)
    k, v = (ref.bf16_values(ref.bf16_bits(rng.standard_normal((rows, kv, seq)).astype(np.float32)))
            for _ in range(2))
    layer = list(constant(k, 1)) + list(constant(v, 1))
    q = (rng.standard_normal((rows, heads, 1)) * 100).astype(np.float32)
    positions = [2999, 1500, 256, 31]
    got = attend(rt, q, layer, positions, out_dtype)
    check_attention(got, q, layer, positions, out_dtype, False)
    rt.synchronize()


@pytest.mark.parametrize("exponent", [-30, -60, -75])
def test_values_of_tiny_steps_keep_their_digits(rt, exponent):
    """The norm of the difference against the result's: f32 scores of up to 40 and their sums,
    40 x 2^-23 + 6 sqrt(n) 2^-24 at most, as at any other size of the values."""
    rng = np.random.default_rng(6)
    heads, kv, head, seq = 8, 2, 64, 2000
    keys = ref.quantise(rng.standard_normal((kv, seq, head)).astype(np.float32))
    vals = ref.quantise((rng.standard_normal((kv, seq, head)) * 2.0 ** exponent).astype(np.float32))
    q = rng.standard_normal((1, heads, head)).astype(np.float32)
    got = attend(rt, q, list(keys) + list(vals), [seq - 1])[0]
    want = ref.attention(q[0], ref.values(*keys, head), ref.values(*vals, head), seq - 1)
    assert np.linalg.norm(got - want) <= np.linalg.norm(want) * (40 * 2.0 ** -23 + 6 * seq ** 0.5 * 2.0 ** -24)


@pytest.mark.parametrize("octaves", [30, 200, -200])
@pytest.mark.parametrize("value", [0.0, -3.0, 999424.0, 2.0 ** 100])
def test_prompt_rows_over_one_value_throughout(rt, octaves, value):
    rows, heads, kv, head, seq = 270, 2, 1, 64, 2000
    keys, per = rising((), kv, seq, head, octaves)
    layer = list(keys) + list(constant(np.full((kv, seq), value), head))
    positions = list(range(seq - rows, seq))
    got = attend(rt, query_for(per, rows, heads, head), layer, positions, ab.BF16)
    assert np.isfinite(got).all()
    assert np.abs(got - value).max() <= constant_bound(value, seq, ab.BF16)
    rt.synchronize()
