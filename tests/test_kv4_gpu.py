"""The 4-bit key/value cache against its 64-bit definition: rows quantised as they are written,
rows read back, attention over the packed cache, and the three as one run."""
import numpy as np
import pytest

import ammon_b200 as ab
from ammon_b200 import kernels as K

import kv4_ref as ref

pytestmark = pytest.mark.gpu

NAN_WORD = np.uint32(0x7FFF7FFF)


@pytest.fixture(scope="module")
def rt():
    r = ab.create_runtime(0)
    yield r
    r.synchronize()


def steps(rt, positions):
    p = ab.DecodeStep.parcel(rt, len(positions))
    rt.deposit(p, [ab.DecodeStep(0, int(x)) for x in positions])
    return p


def upload(rt, layer):
    """Kv4Layer of four uint32 arrays (key codes, key scales, value codes, value scales)."""
    return ab.Kv4Layer(*[ab.Tensor.from_array(rt, a, ab.U32) for a in layer])


def download(layer):
    return [t.read() for t in (layer.key_codes, layer.key_scales, layer.value_codes,
                               layer.value_scales)]


def rows_like(rng, shape):
    """Rows with an offset and a width of their own per channel and per row."""
    x = rng.standard_normal(shape) + rng.standard_normal(shape[-2:])
    return (x * rng.uniform(0.1, 4, shape[:-1] + (1,))).astype(np.float32)


def tensor(rt, x, dtype):
    if dtype == ab.BF16:
        bits = ref.bf16_bits(x)
        return ab.Tensor.from_array(rt, bits, ab.BF16), ref.bf16_values(bits)
    return ab.Tensor.from_array(rt, x), x


# ---- writing ---------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("kv,head", [(1, 1), (6, 48), (8, 128), (3, 33), (2, 64), (5, 20),
                                     (4, 96), (1, 32), (2, 112)])
@pytest.mark.parametrize("shared", [True, False])
def test_store_writes_the_defined_codes_and_nothing_else(rt, kv, head, dtype, shared):
    rng = np.random.default_rng(head * 100 + kv)
    rows, seq = 13, 29
    w = ref.words_of(head)
    lead = () if shared else (rows + 1,)
    before = [rng.integers(0, 2 ** 32, lead + (kv, seq) + ((w,) if i % 2 == 0 else ()),
                           dtype=np.uint32) for i in range(4)]
    at = rng.permutation(seq)[:rows] if shared else rng.integers(0, seq, rows)
    x = [rows_like(rng, (rows, kv, head)) for _ in range(2)]
    (kt, kx), (vt, vx) = (tensor(rt, a, dtype) for a in x)
    layer = upload(rt, before)
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", kt, vt, layer, steps(rt, at))
    s.submit()
    want = [a.copy() for a in before]
    for which, a in ((0, kx), (2, vx)):
        codes, scales = ref.quantise(a)
        for r in range(rows):
            for arr, new in ((want[which], codes), (want[which + 1], scales)):
                (arr if shared else arr[r])[:, at[r]] = new[r]
    for got, exp in zip(download(layer), want):
        assert np.array_equal(got, exp)
    rt.synchronize()


def test_store_single_row_without_a_row_axis(rt):
    rng = np.random.default_rng(2)
    x = rows_like(rng, (4, 40))
    c = ab.Kv4Cache(rt, 2, 9, 4, 40)
    c.zero()
    layer = c.layer(1)
    t = ab.Tensor.from_array(rt, x)
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", t, t, layer, steps(rt, [8]))
    s.submit()
    codes, scales = ref.quantise(x)
    got = download(layer)
    assert np.array_equal(got[0][:, 8], codes) and np.array_equal(got[3][:, 8], scales)
    assert not got[0][:, :8].any() and not got[1][:, :8].any()
    assert not any(a.any() for a in download(c.layer(0)))


def test_store_halves_constants_and_extremes(rt):
    """Quotients that are exactly halves, or next to them by one unit in the last place, rows of
    one value, tiny and huge ranges, and rows that are not finite."""
    head = 32
    half = np.arange(head, dtype=np.float32) % 16
    half[1:15] += 0.5  # m = 0, s = 1: 1.5, 2.5, ... are ties
    rows = [half, np.nextafter(half, np.float32(-9)), np.nextafter(half, np.float32(99)),
            half * np.float32(3 * 2.0 ** -20), half * np.float32(2.0 ** -127),
            np.full(head, 1.2345678, np.float32), np.full(head, -0.0, np.float32),
            np.zeros(head, np.float32), np.float32(1e4) + half * np.float32(1e-3),
            np.linspace(-3e38, 3e38, head).astype(np.float32),
            np.linspace(-1.6e38, 1.6e38, head).astype(np.float32),
            np.full(head, 3.4e38, np.float32), np.linspace(0, 1e-44, head).astype(np.float32)]
    for bad in (np.nan, np.inf, -np.inf):
        r = half.copy()
        r[17] = bad
        rows.append(r)
    x = np.stack(rows)[:, None]
    layer = upload(rt, [np.zeros((1, 16, 4), np.uint32), np.zeros((1, 16), np.uint32)] * 2)
    t = ab.Tensor.from_array(rt, x)
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", t, t, layer, steps(rt, range(len(rows))))
    s.submit()
    codes, scales = ref.quantise(x)
    got = download(layer)
    for r in range(len(rows)):
        assert got[1][0, r] == scales[r, 0], r
        assert np.array_equal(got[0][0, r], codes[r, 0]), r
    assert (got[1][0, -3:] == NAN_WORD).all() and not got[0][0, -3:].any()


@pytest.mark.parametrize("rows,kv,head", [(40, 2, 32), (700, 8, 16), (5000, 1, 8)])
def test_store_of_equal_positions_keeps_the_last_row(rt, rows, kv, head):
    rng = np.random.default_rng(rows)
    seq = rows
    at = rng.integers(0, rows // 2, rows)
    x = rows_like(rng, (rows, kv, head))
    layer = upload(rt, [np.zeros((kv, seq, ref.words_of(head)), np.uint32),
                        np.zeros((kv, seq), np.uint32)] * 2)
    t = ab.Tensor.from_array(rt, x)
    parcel = steps(rt, at)
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", t, t, layer, parcel)
    for turn in range(2):
        s.submit()
        codes, scales = ref.quantise(x)
        want_c, want_s = np.zeros_like(download(layer)[0]), np.zeros((kv, seq), np.uint32)
        for r in range(rows):
            want_c[:, at[r]], want_s[:, at[r]] = codes[r], scales[r]
        got = download(layer)
        used = np.unique(at)
        assert np.array_equal(got[0][:, used], want_c[:, used])
        assert np.array_equal(got[3][:, used], want_s[:, used])
        at = np.arange(rows)  # the same recorded call, now at rising positions
        rt.deposit(parcel, [ab.DecodeStep(0, int(p)) for p in at])


def test_store_past_the_end_writes_nothing_and_is_reported(rt):
    x = ab.Tensor.from_array(rt, np.ones((3, 2, 32), np.float32))
    layer = upload(rt, [np.full((2, 8, 4), 7, np.uint32), np.full((2, 8), 9, np.uint32)] * 2)
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", x, x, layer, steps(rt, [2, 8, 2 ** 32 - 1]))
    s.submit()
    with pytest.raises(ab.DeviceError, match="position"):
        rt.synchronize()
    got = download(layer)
    rest = [i for i in range(8) if i != 2]
    assert (got[0][:, rest] == 7).all() and (got[1][:, rest] == 9).all()
    assert (got[1][:, 2] == 0x3F800000).all()  # one value throughout: step 0, offset 1


# ---- reading back -----------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("kv,head", [(1, 1), (6, 48), (8, 128), (3, 33), (2, 64), (4, 96)])
@pytest.mark.parametrize("batch,n", [(None, 1), (None, 21), (3, 7)])
def test_load_gives_the_values_that_codes_stand_for(rt, kv, head, dtype, batch, n):
    rng = np.random.default_rng(head + n)
    seq, b = 21, batch or 1
    lead = (b,) if batch else ()
    layer = []
    for _ in range(2):
        codes, scales = ref.quantise(rows_like(rng, lead + (kv, seq, head)))
        layer += [codes, scales]
    first = rng.integers(0, seq - n + 1, b)
    shape = lead + (n, kv, head)
    out = [ab.Tensor.zeros(rt, shape, dtype) for _ in range(2)]
    s = rt.scheme()
    K.Kv4LoadKernel.prepare(rt).record(s, "load", upload(rt, layer), steps(rt, first), *out)
    s.submit()
    for which in range(2):
        want = ref.values(layer[2 * which], layer[2 * which + 1], head)
        want = want.reshape((b, kv, seq, head)).astype(np.float32)  # one rounding of m + s c
        want = np.stack([want[i][:, f:f + n].transpose(1, 0, 2) for i, f in enumerate(first)])
        if dtype == ab.BF16:
            want = ref.bf16_values(ref.bf16_bits(want))
        assert np.array_equal(out[which].read_f32(), want.reshape(shape))
    rt.synchronize()


def test_load_past_the_end_gives_zeros_and_is_reported(rt):
    codes, scales = ref.quantise(np.ones((2, 6, 16), np.float32))
    out = [ab.Tensor.from_array(rt, np.full((4, 2, 16), 5, np.float32)) for _ in range(2)]
    s = rt.scheme()
    K.Kv4LoadKernel.prepare(rt).record(s, "load", upload(rt, [codes, scales] * 2),
                                       steps(rt, [4]), *out)
    s.submit()
    with pytest.raises(ab.DeviceError, match="position"):
        rt.synchronize()
    got = out[0].read()
    assert (got[:2] == 1).all() and (got[2:] == 0).all()


# ---- attention --------------------------------------------------------------------------
def packed(rng, lead, kv, seq, head):
    layer = []
    for _ in range(2):
        codes, scales = ref.quantise(rows_like(rng, lead + (kv, seq, head)))
        layer += [codes, scales]
    return layer


def check_attention(got, q, layer, positions, out_dtype, shared):
    """got [rows, heads, head] against the 64-bit attention of every row."""
    head = q.shape[-1]
    for r, pos in enumerate(positions):
        kc, ks, vc, vs = layer if shared else [a[r] for a in layer]
        k = ref.values(kc[:, :pos + 1], ks[:, :pos + 1], head)
        v = ref.values(vc[:, :pos + 1], vs[:, :pos + 1], head)
        want = ref.attention(q[r], k, v, pos)
        bound = ref.attention_bound(q[r], kc, ks, v, pos)
        if out_dtype == ab.BF16:
            bound = bound + np.abs(want) * 2.0 ** -8 + bound * 2.0 ** -8
        off = np.abs(got[r] - want)
        assert np.isfinite(got[r]).all() and (off <= bound).all(), (r, pos, (off / bound).max())


def attend(rt, q, layer, positions, out_dtype=ab.F32, past_the_end=False):
    rows, heads, head = q.shape
    out = ab.Tensor.from_array(rt, np.full((rows, heads * head), 0x7FC0 if out_dtype == ab.BF16
                                           else np.nan,
                                           np.uint16 if out_dtype == ab.BF16 else np.float32))
    s = rt.scheme()
    K.Kv4AttentionKernel.prepare(rt).record(s, "attend", ab.Tensor.from_array(rt, q),
                                            upload(rt, layer), out, steps(rt, positions))
    s.submit()
    if past_the_end:
        with pytest.raises(ab.DeviceError, match="position"):
            rt.synchronize()
    return out.read_f32().reshape(rows, heads, head)


def spoil(layer, positions, shared):
    """Fills what lies past each row's position with codes of ones and NaN scales."""
    for r, pos in enumerate([max(positions)] if shared else positions):
        for i, a in enumerate(layer):
            (a if shared else a[r])[:, pos + 1:] = np.uint32(0xFFFFFFFF) if i % 2 == 0 else NAN_WORD


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("heads,kv,head", [(1, 1, 1), (6, 6, 48), (32, 8, 128), (5, 1, 80),
                                           (12, 12, 64), (16, 1, 128), (24, 2, 96), (9, 3, 33),
                                           (14, 2, 32), (8, 1, 112), (3, 3, 31)])
def test_attention_rows_with_their_own_caches(rt, heads, kv, head, out_dtype):
    rng = np.random.default_rng(heads * 1000 + head)
    positions = [0, 1, 7, 8, 15, 16, 31, 63, 64, 65, 127, 300, 40]
    seq = 301
    layer = packed(rng, (len(positions),), kv, seq, head)
    spoil(layer, positions, False)
    q = (rng.standard_normal((len(positions), heads, head)) * 1.5).astype(np.float32)
    got = attend(rt, q, layer, positions, out_dtype)
    check_attention(got, q, layer, positions, out_dtype, False)
    rt.synchronize()


@pytest.mark.parametrize("out_dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("heads,kv,head,positions", [
    (32, 8, 128, list(range(200, 237))), (6, 6, 48, [9, 3, 40, 0]), (12, 2, 64, [511]),
    (2, 1, 96, list(range(70))), (16, 1, 33, [5, 5, 5]), (3, 3, 128, list(range(1000, 1064)))])
def test_attention_rows_over_one_cache(rt, heads, kv, head, positions, out_dtype):
    rng = np.random.default_rng(heads * 1000 + head + 1)
    layer = packed(rng, (), kv, max(positions) + 3, head)
    spoil(layer, positions, True)
    q = (rng.standard_normal((len(positions), heads, head)) * 1.5).astype(np.float32)
    got = attend(rt, q, layer, positions, out_dtype)
    check_attention(got, q, layer, positions, out_dtype, True)


@pytest.mark.parametrize("heads,kv,head,pos", [(32, 8, 128, 70000), (2, 2, 64, 30001)])
def test_attention_over_a_long_cache(rt, heads, kv, head, pos):
    rng = np.random.default_rng(pos)
    layer = packed(rng, (), kv, pos + 1, head)
    q = rng.standard_normal((1, heads, head)).astype(np.float32)
    check_attention(attend(rt, q, layer, [pos]), q, layer, [pos], ab.F32, True)


def test_attention_where_one_position_outweighs_all(rt):
    """Scores that differ by hundreds: the weights of all but one position vanish."""
    rng = np.random.default_rng(8)
    layer = packed(rng, (3,), 2, 200, 64)
    q = (rng.standard_normal((3, 4, 64)) * np.array([300, 1e4, 1e-6])[:, None, None]).astype(np.float32)
    got = attend(rt, q, layer, [199, 150, 77])
    # d of attention_bound is far above 1 here; what holds is that no weight is lost or NaN: the
    # result is the value at the largest score wherever that leads by more than 2 d
    for r, pos in enumerate((199, 150)):
        kc, ks, vc, vs = [a[r] for a in layer]
        k, v = ref.values(kc, ks, 64), ref.values(vc, vs, 64)
        for h in range(4):
            score = k[h // 2, :pos + 1] @ q[r, h].astype(np.float64) / 8
            best = np.argsort(score)[::-1][:2]
            s = ref.bf16_values((ks[h // 2, :pos + 1] & 0xFFFF).astype(np.uint16)).astype(np.float64)
            m = ref.bf16_values((ks[h // 2, :pos + 1] >> 16).astype(np.uint16)).astype(np.float64)
            d = 80 * 2.0 ** -23 * np.abs(q[r, h]).sum() * (np.abs(m) + 15 * s).max() / 8
            assert np.isfinite(got[r, h]).all()
            if score[best[0]] - score[best[1]] > 2 * d + 40:
                want = v[h // 2, best[0]]
                assert np.abs(got[r, h] - want).max() <= np.abs(v[h // 2]).max() * 2.0 ** -20
    check_attention(got[2:], q[2:], [a[2:] for a in layer], [77], ab.F32, False)


def test_attention_over_rows_that_are_not_finite(rt):
    """A NaN vector at a position a row attends over gives NaN to the heads of its kv head
    alone; past the row's position it is never met."""
    rng = np.random.default_rng(9)
    layer = packed(rng, (2,), 2, 90, 64)
    for which in (1, 3):
        layer[which][0, 1, 50] = NAN_WORD
        layer[which][1, 1, 50] = NAN_WORD
    q = rng.standard_normal((2, 4, 64)).astype(np.float32)
    got = attend(rt, q, layer, [60, 49])
    assert np.isnan(got[0, 2:]).all() and np.isfinite(got[0, :2]).all()
    clean = [a[1:] for a in layer]
    check_attention(got[1:], q[1:], clean, [49], ab.F32, False)
    q[1, 3, 5] = np.inf
    q[0, 0, 0] = np.nan
    got = attend(rt, q, layer, [40, 49])
    assert np.isnan(got[0, 0]).all() and np.isfinite(got[0, 1:]).all()
    assert np.isnan(got[1, 3]).all() and np.isfinite(got[1, :3]).all()


def test_attention_past_the_end_gives_a_zero_row_and_is_reported(rt):
    rng = np.random.default_rng(10)
    layer = packed(rng, (3,), 2, 20, 32)
    q = rng.standard_normal((3, 4, 32)).astype(np.float32)
    got = attend(rt, q, layer, [19, 20, 4], past_the_end=True)
    assert (got[1] == 0).all()
    check_attention(got[::2], q[::2], [a[::2] for a in layer], [19, 4], ab.F32, False)
    # the next call of the same shape is unharmed
    got = attend(rt, q, layer, [19, 3, 4])
    check_attention(got, q, layer, [19, 3, 4], ab.F32, False)
    rt.synchronize()


def test_attention_replays_give_the_same_bits_at_changing_positions(rt):
    """One recorded call over growing positions; each replay equals a fresh call bit for bit,
    and two recorded calls of one scheme do not disturb each other."""
    rng = np.random.default_rng(11)
    heads, kv, head, seq = 8, 2, 128, 2100
    layer = packed(rng, (2,), kv, seq, head)
    q = rng.standard_normal((2, heads, head)).astype(np.float32)
    up, qt = upload(rt, layer), ab.Tensor.from_array(rt, q)
    outs = [ab.Tensor.zeros(rt, (2, heads * head)) for _ in range(2)]
    parcels = [steps(rt, [0, 0]), steps(rt, [0, 0])]
    s = rt.scheme()
    for o, p in zip(outs, parcels):
        K.Kv4AttentionKernel.prepare(rt).record(s, "attend", qt, up, o, p)
    for a, b in ((0, 5), (700, 64), (2099, 1), (3, 2000)):
        rt.deposit(parcels[0], [ab.DecodeStep(0, a), ab.DecodeStep(0, b)])
        rt.deposit(parcels[1], [ab.DecodeStep(0, b), ab.DecodeStep(0, a)])
        s.submit()
        for o, pos in zip(outs, ([a, b], [b, a])):
            got = o.read().reshape(2, heads, head)
            assert np.array_equal(got, attend(rt, q, layer, pos))
            check_attention(got, q, layer, pos, ab.F32, False)


# ---- together ------------------------------------------------------------------------------
@pytest.mark.parametrize("heads,kv,head", [(8, 2, 128), (6, 6, 48)])
def test_prompt_then_steps_on_one_cache(rt, heads, kv, head):
    """A prompt stored in one call, then single tokens stored and attended over in one recorded
    scheme, then the whole cache read back: every stage against the 64-bit definition."""
    rng = np.random.default_rng(12)
    prompt, more, seq = 45, 6, 64
    n = prompt + more
    keys, vals = (rows_like(rng, (n, kv, head)) for _ in range(2))
    q = rng.standard_normal((n, heads, head)).astype(np.float32)
    cache = ab.Kv4Cache(rt, 1, seq, kv, head)
    layer = cache.layer(0)
    up = [ab.Tensor.from_array(rt, a[:prompt]) for a in (keys, vals, q)]
    out = ab.Tensor.zeros(rt, (prompt, heads * head))
    at = steps(rt, range(prompt))
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", up[0], up[1], layer, at)
    K.Kv4AttentionKernel.prepare(rt).record(s, "attend", up[2], layer, out, at)
    s.submit()
    packed_rows = []
    for a in (keys, vals):
        codes, scales = ref.quantise(a.transpose(1, 0, 2))
        packed_rows += [codes, scales]
    check_attention(out.read().reshape(prompt, heads, head), q[:prompt], packed_rows,
                    list(range(prompt)), ab.F32, True)
    one = [ab.Tensor.zeros(rt, (kv, head)), ab.Tensor.zeros(rt, (kv, head)),
           ab.Tensor.zeros(rt, (heads, head))]
    step, out1 = steps(rt, [0]), ab.Tensor.zeros(rt, (heads * head,))
    s1 = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s1, "store", one[0], one[1], layer, step)
    K.Kv4AttentionKernel.prepare(rt).record(s1, "attend", one[2], layer, out1, step)
    for t in range(prompt, n):
        for dst, src in zip(one, (keys, vals, q)):
            dst.write(src[t])
        rt.deposit(step, [ab.DecodeStep(0, t)])
        s1.submit()
        check_attention(out1.read().reshape(1, heads, head), q[t:t + 1], packed_rows, [t],
                        ab.F32, True)
    back = [ab.Tensor.zeros(rt, (n, kv, head)) for _ in range(2)]
    s2 = rt.scheme()
    K.Kv4LoadKernel.prepare(rt).record(s2, "load", layer, steps(rt, [0]), *back)
    s2.submit()
    for which in range(2):
        want = ref.values(packed_rows[2 * which], packed_rows[2 * which + 1], head)
        assert np.array_equal(back[which].read(), want.transpose(1, 0, 2).astype(np.float32))
    rt.synchronize()
