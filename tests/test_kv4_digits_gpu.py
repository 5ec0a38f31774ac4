"""How many digits attention over the 4-bit cache keeps, and that every position counts: bounds on
the norm of the error, far below what a lost tile, position or operand column would cost."""
import numpy as np
import pytest

import ammon_b200 as ab

import kv4_ref as ref
from test_kv4_gpu import attend, packed, rt, spoil  # noqa: F401

pytestmark = pytest.mark.gpu

# Norm of the difference over the result's. Scores are at most about 35 and off by 2^-23 of that
# with the queries' 22 bits, 4e-6, which moves weights, and with them a mean of values, by no more;
# the sums add some 1e-6 of random sign. fp16 weights would be 5e-5 off, fp16 queries 1e-3, a tile
# of 256 positions less of 70001 2e-2. A rounding to bf16 is at most 2^-8 of each value.
DIGITS = {ab.F32: 1e-5, ab.BF16: 1e-5 + 2.0 ** -8}


def check_norm(got, q, layer, positions, out_dtype, shared):
    head = q.shape[-1]
    for r, pos in enumerate(positions):
        kc, ks, vc, vs = layer if shared else [a[r] for a in layer]
        want = ref.attention(q[r], ref.values(kc[:, :pos + 1], ks[:, :pos + 1], head),
                             ref.values(vc[:, :pos + 1], vs[:, :pos + 1], head), pos)
        off = np.linalg.norm(got[r] - want) / np.linalg.norm(want)
        assert off <= DIGITS[out_dtype], (r, pos, off)


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("heads,kv,head", [(6, 6, 48), (32, 8, 128), (5, 1, 80), (12, 12, 64),
                                           (16, 1, 128), (24, 2, 96), (9, 3, 33), (14, 2, 32)])
def test_digits_of_rows_with_their_own_caches(rt, heads, kv, head, out_dtype):
    rng = np.random.default_rng(heads + head)
    positions = [0, 7, 31, 64, 127, 300, 900]
    layer = packed(rng, (len(positions),), kv, 901, head)
    spoil(layer, positions, False)
    q = (rng.standard_normal((len(positions), heads, head)) * 1.5).astype(np.float32)
    check_norm(attend(rt, q, layer, positions, out_dtype), q, layer, positions, out_dtype, False)


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("heads,kv,head,rows,last", [(32, 8, 128, 37, 236), (12, 2, 64, 70, 1500),
                                                     (8, 2, 128, 100, 2000), (6, 6, 48, 260, 300),
                                                     (4, 1, 96, 80, 700), (3, 1, 33, 100, 400)])
def test_digits_of_rows_over_one_cache(rt, heads, kv, head, rows, last, out_dtype):
    """Both kernels: up to 256 query slots of a kv head, and more of them with bf16 outputs."""
    rng = np.random.default_rng(heads + head + rows)
    positions = list(range(last + 1 - rows, last + 1))
    layer = packed(rng, (), kv, last + 2, head)
    spoil(layer, positions, True)
    q = (rng.standard_normal((rows, heads, head)) * 1.5).astype(np.float32)
    got = attend(rt, q, layer, positions, out_dtype)
    some = [0, 1, rows // 2, rows - 2, rows - 1]
    check_norm(got[some], q[some], layer, [positions[i] for i in some], out_dtype, True)


@pytest.mark.parametrize("heads,kv,head,pos", [(32, 8, 128, 70000), (2, 2, 64, 30001)])
def test_digits_over_a_long_cache(rt, heads, kv, head, pos):
    rng = np.random.default_rng(pos)
    layer = packed(rng, (), kv, pos + 1, head)
    q = rng.standard_normal((1, heads, head)).astype(np.float32)
    check_norm(attend(rt, q, layer, [pos]), q, layer, [pos], ab.F32, True)


# ---- every position counts -------------------------------------------------------------------
def even(rt, rng, rows, heads, kv, head, positions, out_dtype, shared, seq=None):
    """Attention of queries of zero, so all weights alike, against the plain mean of values of up
    to 1: a position lost or met twice moves the row by 1 / n of its values.

    f32: sums of about 1 in chains of at most some hundred additions, random roundings, offsets
    and codes apart: 64 x 2^-24. bf16: sums of codes stay in the tensor unit, whose additions cut
    off, 2^-16 over such chains, and the output's rounding."""
    seq = seq or max(positions) + 1
    lead = () if shared else (rows,)
    keys = packed(rng, lead, kv, seq, head)[:2]
    codes, scales = ref.quantise(rng.uniform(-1, 1, lead + (kv, seq, head)).astype(np.float32))
    layer = keys + [codes, scales]
    spoil(layer, positions, shared)
    got = attend(rt, np.zeros((rows, heads, head), np.float32), layer, positions, out_dtype)
    for r in range(rows) if rows <= 64 else list(range(0, rows, rows // 40)) + [rows - 1]:
        n = positions[r] + 1
        c, s = (codes, scales) if shared else (codes[r], scales[r])
        want = np.repeat(ref.values(c[:, :n], s[:, :n], head).mean(1), heads // kv, 0)
        bound = 64 * 2.0 ** -24
        if out_dtype == ab.BF16:
            bound = 2.0 ** -16 + np.abs(want) * 2.0 ** -8
        assert (np.abs(got[r] - want) <= bound).all(), (r, n, np.abs(got[r] - want).max())
    rt.synchronize()


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("heads,kv,head", [(4, 4, 32), (8, 2, 128), (16, 2, 64), (3, 1, 96)])
def test_every_position_of_rows_with_their_own_caches(rt, heads, kv, head, out_dtype):
    rng = np.random.default_rng(head)
    positions = [0, 1, 30, 31, 32, 33, 127, 128, 129, 254, 255, 256, 257, 511, 512, 513, 767, 1023,
                 1024, 1025, 1791, 1792, 2047, 2048]
    even(rt, rng, len(positions), heads, kv, head, positions, out_dtype, False)


@pytest.mark.parametrize("heads,kv,head,rows", [(2, 2, 32, 700), (8, 1, 64, 700), (8, 1, 128, 400)])
def test_every_position_of_many_rows(rt, heads, kv, head, rows):
    rng = np.random.default_rng(rows + head)
    positions = [int(p) for p in rng.integers(0, 700, rows)]
    even(rt, rng, rows, heads, kv, head, positions, ab.F32, False, 700)


@pytest.mark.parametrize("pos", [8191, 8192, 20001, 37887, 37888, 70000])
def test_every_position_of_one_long_row(rt, pos):
    rng = np.random.default_rng(pos)
    even(rt, rng, 1, 8, 2, 32, [pos], ab.F32, True)


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("heads,kv,head,rows,last", [(4, 1, 128, 70, 129), (4, 2, 64, 140, 2100),
                                                     (1, 1, 32, 300, 640), (8, 8, 96, 257, 1025)])
def test_every_position_of_prompt_rows(rt, heads, kv, head, rows, last, out_dtype):
    rng = np.random.default_rng(rows)
    even(rt, rng, rows, heads, kv, head, list(range(last + 1 - rows, last + 1)), out_dtype, True,
         last + 40)
