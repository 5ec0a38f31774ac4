"""Prompts over one 4-bit cache with bf16 outputs (matrix products on the tensor cores' own
memory): head sizes, groups, positions in any order, rows without an end, NaN, splits, replays."""
import numpy as np
import pytest

import ammon_b200 as ab
from ammon_b200 import kernels as K

from test_kv4_gpu import (NAN_WORD, attend, check_attention, packed, rt, spoil,  # noqa: F401
                          steps, upload)
from test_kv4_calls_gpu import shifted

pytestmark = pytest.mark.gpu


def query(rng, *shape):
    return (rng.standard_normal(shape) * 1.5).astype(np.float32)


@pytest.mark.parametrize("heads,kv,head", [(4, 1, 128), (3, 3, 64), (8, 8, 128), (6, 2, 33),
                                           (5, 1, 80), (2, 2, 32), (14, 2, 100), (1, 1, 1),
                                           (9, 3, 17), (130, 1, 64)])
@pytest.mark.parametrize("last", [63, 64, 700])
def test_prompt_rows(rt, heads, kv, head, last):
    rng = np.random.default_rng(heads * 100 + head + last)
    rows = 260 // (heads // kv) + 3
    first = max(0, last + 1 - rows)
    positions = [min(last, first + i) for i in range(rows)]
    layer = packed(rng, (), kv, last + 2, head)
    spoil(layer, positions, True)
    q = query(rng, rows, heads, head)
    check_attention(attend(rt, q, layer, positions, ab.BF16), q, layer, positions, ab.BF16, True)
    rt.synchronize()


def test_prompt_positions_in_any_order_and_past_the_end(rt):
    """Rows of unlike, repeated and unordered positions; those past the end give zeros and are
    reported, and the call after them is unharmed."""
    rng = np.random.default_rng(31)
    heads, kv, head, seq, rows = 8, 2, 128, 500, 90
    positions = rng.integers(0, seq, rows)
    positions[:4] = [0, 0, 499, 1]
    layer = packed(rng, (), kv, seq, head)
    q = query(rng, rows, heads, head)
    check_attention(attend(rt, q, layer, positions, ab.BF16), q, layer, positions, ab.BF16, True)
    bad = positions.copy()
    bad[[3, 40, 41]] = [500, 2 ** 31, 2 ** 32 - 1]
    got = attend(rt, q, layer, bad, ab.BF16, past_the_end=True)
    assert (got[[3, 40, 41]] == 0).all()
    keep = [r for r in range(rows) if r not in (3, 40, 41)]
    check_attention(got[keep], q[keep], layer, positions[keep], ab.BF16, True)
    got = attend(rt, q, layer, [seq] * rows, ab.BF16, past_the_end=True)
    assert (got == 0).all()
    check_attention(attend(rt, q, layer, positions, ab.BF16), q, layer, positions, ab.BF16, True)
    rt.synchronize()


def test_prompt_over_rows_that_are_not_finite(rt):
    """A key or value vector that is NaN reaches exactly the rows at or past its position."""
    rng = np.random.default_rng(32)
    heads, kv, head, rows, seq = 16, 4, 64, 80, 200
    for which in (1, 3):
        layer = packed(rng, (), kv, seq, head)
        positions = list(range(100, 180))
        layer[which][1, 150] = NAN_WORD
        layer[which][1, 181:] = NAN_WORD
        q = query(rng, rows, heads, head)
        got = attend(rt, q, layer, positions, ab.BF16)
        nan = np.isnan(got)
        assert nan[50:, 4:8].all() and not nan[:50].any()
        assert not nan[:, :4].any() and not nan[:, 8:].any()
    layer = packed(rng, (), kv, seq, head)
    q[7, 3, 5], q[9, 6, 0] = np.nan, np.inf
    nan = np.isnan(attend(rt, q, layer, positions, ab.BF16))
    assert nan[7, 3].all() and nan[9, 6].all()
    nan[7, 3] = nan[9, 6] = False
    assert not nan.any()
    rt.synchronize()


def test_prompt_where_maxima_grow_along_the_cache(rt):
    """Scores that rise by thousands over the positions move every running maximum; the weights'
    own order of size changes with the steps of V."""
    rng = np.random.default_rng(33)
    heads, kv, head, rows, seq = 4, 1, 64, 90, 640
    k = rng.standard_normal((kv, seq, head)).astype(np.float32)
    k *= np.linspace(0.01, 40, seq, dtype=np.float32)[None, :, None]
    v = rng.standard_normal((kv, seq, head)).astype(np.float32)
    v *= np.exp2(rng.integers(-20, 20, seq)).astype(np.float32)[None, :, None]
    import kv4_ref as ref
    kc, vc = ref.quantise(k), ref.quantise(v)
    layer = [kc[0], kc[1], vc[0], vc[1]]
    q = query(rng, rows, heads, head)
    positions = list(range(seq - rows, seq))
    check_attention(attend(rt, q, layer, positions, ab.BF16), q, layer, positions, ab.BF16, True)
    rt.synchronize()


@pytest.mark.parametrize("heads,kv,rows,last", [(8, 1, 64, 40000), (4, 4, 300, 9000),
                                                (4, 4, 1500, 1600)])
def test_prompt_split_and_not(rt, heads, kv, rows, last):
    """One slot block over a long cache (a hundred parts), a few, and more blocks than the device
    takes at once; the same bits every time."""
    rng = np.random.default_rng(last)
    head = 64
    layer = packed(rng, (), kv, last + 1, head)
    positions = [last - rows + 1 + i for i in range(rows)]
    q = query(rng, rows, heads, head)
    got = attend(rt, q, layer, positions, ab.BF16)
    check_attention(got[::7], q[::7], layer, positions[::7], ab.BF16, True)
    assert np.array_equal(got, attend(rt, q, layer, positions, ab.BF16))
    rt.synchronize()


def test_prompt_replays_at_changing_positions(rt):
    """One recorded call whose rows move, so that its parts are one, some and none of theirs; beside
    it a call of another kind that uses the same scratch."""
    rng = np.random.default_rng(34)
    heads, kv, head, rows, seq = 8, 2, 128, 70, 3000
    layer = packed(rng, (), kv, seq, head)
    q, q1 = query(rng, rows, heads, head), query(rng, 1, heads, head)
    up = upload(rt, layer)
    out = ab.Tensor.zeros(rt, (rows, heads * head), ab.BF16)
    out1 = ab.Tensor.zeros(rt, (1, heads * head))
    parcel, parcel1 = steps(rt, [0] * rows), steps(rt, [0])
    s = rt.scheme()
    kernel = K.Kv4AttentionKernel.prepare(rt)
    kernel.record(s, "one", ab.Tensor.from_array(rt, q1), up, out1, parcel1)
    kernel.record(s, "prompt", ab.Tensor.from_array(rt, q), up, out, parcel)
    kernel.record(s, "one", ab.Tensor.from_array(rt, q1), up, out1, parcel1)
    for first in (0, 2930, 500, 25, 1900):
        positions = [first + i for i in range(rows)]
        rt.deposit(parcel, [ab.DecodeStep(0, p) for p in positions])
        rt.deposit(parcel1, [ab.DecodeStep(0, first)])
        s.submit()
        got = out.read_f32().reshape(rows, heads, head)
        check_attention(got, q, layer, positions, ab.BF16, True)
        assert np.array_equal(got, attend(rt, q, layer, positions, ab.BF16))
        check_attention(out1.read().reshape(1, heads, head), q1, layer, [first], ab.F32, True)
    rt.synchronize()


@pytest.mark.parametrize("head", [128, 72, 50])
def test_prompt_at_odd_addresses(rt, head):
    rng = np.random.default_rng(35)
    rows, heads, kv, seq = 33, 32, 2, 333
    positions = list(range(300, 333))
    layer = packed(rng, (), kv, seq, head)
    q = query(rng, rows, heads, head)
    keep = [shifted(rt, layer[i], 1, ab.U32) for i in (1, 3)]
    codes = [ab.Tensor.from_array(rt, layer[i], ab.U32) for i in (0, 2)]
    qt, _ = shifted(rt, q, 1)
    out, base = shifted(rt, np.zeros((rows, heads * head), np.uint16), 1, ab.BF16)
    s = rt.scheme()
    K.Kv4AttentionKernel.prepare(rt).record(
        s, "prompt", qt, ab.Kv4Layer(codes[0], keep[0][0], codes[1], keep[1][0]), out,
        steps(rt, positions))
    s.submit()
    got = base.read_f32()
    assert got[0] == 0
    check_attention(got[1:].reshape(rows, heads, head), q, layer, positions, ab.BF16, True)
    rt.synchronize()
