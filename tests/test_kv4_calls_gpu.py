"""The 4-bit key/value cache called in ways that its first tests leave out: many rows of unlike
lengths, odd alignments, more caches than rows, several schemes, no graph, far offsets."""
import numpy as np
import pytest

import ammon_b200 as ab
from ammon_b200 import kernels as K

import kv4_ref as ref
from test_kv4_gpu import (attend, check_attention, packed, rows_like, rt, steps,  # noqa: F401
                          upload)

pytestmark = pytest.mark.gpu


def shifted(rt, a, elements, dtype=None):
    """The array on the device, `elements` elements past an aligned address."""
    flat = np.concatenate([np.zeros(elements, a.dtype), np.ascontiguousarray(a).reshape(-1)])
    base = ab.Tensor.from_array(rt, flat, dtype)
    desc = ab.Tensor._desc(base.t.data + elements * a.dtype.itemsize, base.t.dtype, a.shape)
    return ab.Tensor(desc, rt, owner=base), base


@pytest.mark.parametrize("heads,kv,head,out_dtype", [(8, 4, 64, ab.F32), (16, 2, 32, ab.BF16)])
def test_attention_of_many_rows_of_unlike_lengths(rt, heads, kv, head, out_dtype):
    """More units than the device takes at once: most one position long, a few much longer, so
    that stretches begin and end in a unit, before one, and hold dozens."""
    rng = np.random.default_rng(20)
    rows, seq = 601, 1300
    positions = rng.integers(0, 3, rows)
    positions[[0, 7, 300, 301, 600]] = [1299, 255, 256, 1100, 511]
    layer = packed(rng, (rows,), kv, seq, head)
    q = rng.standard_normal((rows, heads, head)).astype(np.float32)
    got = attend(rt, q, layer, positions, out_dtype)
    check_attention(got, q, layer, positions, out_dtype, False)
    assert np.array_equal(got, attend(rt, q, layer, positions, out_dtype))
    rt.synchronize()


@pytest.mark.parametrize("rows", [100, 297, 1000])
def test_attention_of_a_step_for_many_sequences_of_one_length(rt, rows):
    rng = np.random.default_rng(rows)
    layer = packed(rng, (rows,), 1, 70, 16)
    q = rng.standard_normal((rows, 4, 16)).astype(np.float32)
    positions = [69] * rows
    check_attention(attend(rt, q, layer, positions), q, layer, positions, ab.F32, False)
    rt.synchronize()


@pytest.mark.parametrize("head,out_dtype", [(64, ab.F32), (128, ab.BF16), (30, ab.F32)])
def test_attention_at_odd_addresses(rt, head, out_dtype):
    """q, out and the scales aligned to their elements only; a cache of odd length."""
    rng = np.random.default_rng(21)
    rows, heads, kv, seq, positions = 3, 6, 2, 333, [332, 100, 31]
    layer = packed(rng, (rows,), kv, seq, head)
    q = rng.standard_normal((rows, heads, head)).astype(np.float32)
    keep = [shifted(rt, layer[i], 1, ab.U32) for i in (1, 3)]
    codes = [ab.Tensor.from_array(rt, layer[i], ab.U32) for i in (0, 2)]
    cache = ab.Kv4Layer(codes[0], keep[0][0], codes[1], keep[1][0])
    qt, qbase = shifted(rt, q, 1)
    empty = np.zeros((rows, heads * head), np.uint16 if out_dtype == ab.BF16 else np.float32)
    out, obase = shifted(rt, empty, 1, out_dtype)
    s = rt.scheme()
    K.Kv4AttentionKernel.prepare(rt).record(s, "attend", qt, cache, out, steps(rt, positions))
    s.submit()
    got = obase.read_f32()[1:].reshape(rows, heads, head)
    check_attention(got, q, layer, positions, out_dtype, False)
    rt.synchronize()


@pytest.mark.parametrize("dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("head", [128, 64, 40])
def test_store_and_load_at_odd_addresses(rt, head, dtype):
    rng = np.random.default_rng(22)
    rows, kv, seq = 9, 3, 11
    x = [rows_like(rng, (rows, kv, head)) for _ in range(2)]
    arrays = [ref.bf16_bits(a) if dtype == ab.BF16 else a for a in x]
    seen = [ref.bf16_values(a) if dtype == ab.BF16 else a for a in arrays]
    sources = [shifted(rt, a, 1, dtype) for a in arrays]
    shape = (kv, seq)
    zeros = np.zeros(shape + (ref.words_of(head),), np.uint32), np.zeros(shape, np.uint32)
    codes = [ab.Tensor.from_array(rt, zeros[0], ab.U32) for _ in range(2)]
    scales = [shifted(rt, zeros[1], 3, ab.U32) for _ in range(2)]
    cache = ab.Kv4Layer(codes[0], scales[0][0], codes[1], scales[1][0])
    backs = [shifted(rt, np.zeros((rows, kv, head), arrays[0].dtype), 1, dtype) for _ in range(2)]
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", sources[0][0], sources[1][0], cache,
                                        steps(rt, range(1, rows + 1)))
    K.Kv4LoadKernel.prepare(rt).record(s, "load", cache, steps(rt, [1]), backs[0][0], backs[1][0])
    s.submit()
    for which in range(2):
        want_c, want_s = ref.quantise(seen[which])
        got_s = scales[which][1].read()[3:].reshape(shape)
        assert np.array_equal(codes[which].read()[:, 1:rows + 1], want_c.transpose(1, 0, 2))
        assert np.array_equal(got_s[:, 1:rows + 1], want_s.T) and not got_s[:, [0, 10]].any()
        want = ref.values(want_c, want_s, head).astype(np.float32)
        got = backs[which][1].read_f32()
        assert got[0] == 0
        if dtype == ab.BF16:
            want = ref.bf16_values(ref.bf16_bits(want))
        assert np.array_equal(got[1:].reshape(want.shape), want)
    rt.synchronize()


def test_fewer_rows_than_caches(rt):
    rng = np.random.default_rng(23)
    layer = packed(rng, (5,), 2, 40, 64)
    q = rng.standard_normal((3, 4, 64)).astype(np.float32)
    check_attention(attend(rt, q, layer, [39, 0, 17]), q, layer, [39, 0, 17], ab.F32, False)
    x = rows_like(rng, (3, 2, 64))
    up = upload(rt, layer)
    before = up.key_scales.read()
    s = rt.scheme()
    xt = ab.Tensor.from_array(rt, x)
    K.Kv4StoreKernel.prepare(rt).record(s, "store", xt, xt, up, steps(rt, [3, 4, 5]))
    s.submit()
    want = before.copy()
    for r in range(3):
        want[r, :, 3 + r] = ref.quantise(x[r])[1]
    assert np.array_equal(up.key_scales.read(), want)
    rt.synchronize()


def test_schemes_with_calls_of_different_sizes_in_turn_and_without_a_graph(rt):
    """Two schemes of two calls each, the second call of a scheme larger than its first, both
    schemes in flight at once; then the same calls launched one by one."""
    rng = np.random.default_rng(24)
    small, large = packed(rng, (2,), 2, 600, 64), packed(rng, (40,), 4, 900, 128)
    qs = rng.standard_normal((2, 6, 64)).astype(np.float32)
    ql = rng.standard_normal((40, 16, 128)).astype(np.float32)
    ps, pl = [599, 3], list(rng.integers(0, 900, 40))
    ups, upl = upload(rt, small), upload(rt, large)
    qts, qtl = ab.Tensor.from_array(rt, qs), ab.Tensor.from_array(rt, ql)
    kernel = K.Kv4AttentionKernel.prepare(rt)
    made = []
    for graph in (True, True, False):
        s = rt.scheme()
        s.use_graph(graph)
        outs = [ab.Tensor.zeros(rt, (2, 6 * 64)), ab.Tensor.zeros(rt, (40, 16 * 128))]
        kernel.record(s, "small", qts, ups, outs[0], steps(rt, ps))
        kernel.record(s, "large", qtl, upl, outs[1], steps(rt, pl))
        made.append((s, outs))
    for _ in range(3):
        for s, _ in made:
            s.submit()
    first = [o.read() for o in made[0][1]]
    check_attention(first[0].reshape(2, 6, 64), qs, small, ps, ab.F32, False)
    check_attention(first[1].reshape(40, 16, 128), ql, large, pl, ab.F32, False)
    for _, outs in made[1:]:
        for a, b in zip(first, outs):
            assert np.array_equal(a, b.read())
    rt.synchronize()


def test_two_runtimes_over_one_cache(rt):
    """Caches written through one runtime's stream and read, after a synchronise, on another's."""
    other = ab.create_runtime(0)
    rng = np.random.default_rng(25)
    x = rows_like(rng, (30, 2, 96))
    cache = ab.Kv4Cache(rt, 1, 32, 2, 96)
    s = rt.scheme()
    xt = ab.Tensor.from_array(rt, x)
    K.Kv4StoreKernel.prepare(rt).record(s, "store", xt, xt, cache.layer(0), steps(rt, range(30)))
    s.submit()
    rt.synchronize()
    q = rng.standard_normal((1, 2, 96)).astype(np.float32)
    out = ab.Tensor.zeros(other, (2 * 96,))
    so = other.scheme()
    K.Kv4AttentionKernel.prepare(other).record(so, "attend", ab.Tensor.from_array(other, q),
                                               cache.layer(0), out, steps(other, [29]))
    so.submit()
    c, sc = ref.quantise(x.transpose(1, 0, 2))
    check_attention(out.read().reshape(1, 2, 96), q, [c, sc, c, sc], [29], ab.F32, True)
    other.synchronize()


def test_cache_too_large_to_count_is_refused(rt):
    out = ab._abi.C.c_void_p()
    top = 2 ** 32 - 1
    assert ab._abi.lib().ab_kv4cache_create(rt.handle, top, top, top, 128, top,
                                            ab._abi.C.byref(out)) == ab._abi.AB_ERR_ARGUMENT
    assert b"2^40" in ab._abi.lib().ab_last_error()


def test_offsets_past_32_bits(rt):
    """Row 2's cache begins 2^32 words into the codes; its second head's lies past that."""
    torch = pytest.importorskip("torch")
    kv, head, seq, rows = 2, 128, (1 << 26) + 3, 3
    words = ref.words_of(head)
    need = rows * kv * seq * (words + 1) * 4 * 2
    if torch.cuda.mem_get_info(0)[0] < need + (8 << 30):
        pytest.skip("needs %d GB of device memory" % (need >> 30))
    rng = np.random.default_rng(26)
    cache = ab.Kv4Cache(rt, 1, seq, kv, head, rows)
    n, at = 50, seq - 50
    x = [rows_like(rng, (n, kv, head)) for _ in range(2)]
    q = rng.standard_normal((rows, 4, head)).astype(np.float32)
    # the first positions and the last ones, of every row
    kt, vt = (ab.Tensor.zeros(rt, (rows, kv, head)) for _ in range(2))
    step, step0 = steps(rt, [0] * rows), steps(rt, [at] * rows)
    out = ab.Tensor.zeros(rt, (rows, 4 * head))
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", kt, vt, cache.layer(0), step)
    for base in (0, at):
        for t in range(n):
            for dst, src in ((kt, x[0]), (vt, x[1])):
                dst.write(np.stack([src[(t + r) % n] for r in range(rows)]))
            rt.deposit(step, [ab.DecodeStep(0, base + t)] * rows)
            s.submit()
            rt.synchronize()
    layers = [[], [], [], []]
    for r in range(rows):
        for i, a in enumerate(x):
            c, sc = ref.quantise(np.roll(a, -r, 0).transpose(1, 0, 2))
            layers[2 * i].append(c)
            layers[2 * i + 1].append(sc)
    layers = [np.stack(a) for a in layers]
    s1 = rt.scheme()
    K.Kv4AttentionKernel.prepare(rt).record(s1, "attend", ab.Tensor.from_array(rt, q),
                                            cache.layer(0), out, steps(rt, [n - 1] * rows))
    back = [ab.Tensor.zeros(rt, (rows, n, kv, head)) for _ in range(2)]
    K.Kv4LoadKernel.prepare(rt).record(s1, "load", cache.layer(0), step0, *back)
    s1.submit()
    check_attention(out.read().reshape(rows, 4, head), q, layers, [n - 1] * rows, ab.F32, False)
    for i in range(2):
        want = ref.values(layers[2 * i], layers[2 * i + 1], head).transpose(0, 2, 1, 3)
        assert np.array_equal(back[i].read(), want.astype(np.float32))
    rt.synchronize()
    cache.close()


@pytest.mark.parametrize("heads,kv,head,out_dtype", [(4, 1, 128, ab.BF16), (4, 2, 33, ab.F32),
                                                     (8, 1, 128, ab.F32), (6, 1, 90, ab.BF16),
                                                     (3, 1, 96, ab.F32), (2, 2, 20, ab.BF16)])
def test_attention_of_many_short_rows(rt, heads, kv, head, out_dtype):
    """More units of up to four query heads than the device holds small blocks; lengths about the
    tiles' and turns' ends, rows that fill several tiles among them, one past the end."""
    rng = np.random.default_rng(heads * 1000 + head)
    rows, seq = 650, 400
    positions = rng.integers(0, 40, rows)
    positions[::50] = [0, 31, 32, 127, 128, 129, 255, 256, 383, 384, 399, 63, 1]
    positions[1::50] = 399
    layer = packed(rng, (rows,), kv, seq, head)
    q = rng.standard_normal((rows, heads, head)).astype(np.float32)
    got = attend(rt, q, layer, positions, out_dtype)
    check_attention(got, q, layer, positions, out_dtype, False)
    assert np.array_equal(got, attend(rt, q, layer, positions, out_dtype))
    bad = positions.copy()
    bad[333] = seq
    other = attend(rt, q, layer, bad, out_dtype, past_the_end=True)
    assert (other[333] == 0).all()
    # where the line's stretches end moves with the lengths, and with them the order of sums
    keep = np.arange(rows) != 333
    check_attention(other[keep], q[keep], [a[keep] for a in layer], positions[keep], out_dtype,
                    False)
    rt.synchronize()
