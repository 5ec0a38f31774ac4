"""The 4-bit key/value cache on CPU: the packed format's own definition, and what the record
calls refuse (errors name the parameter; a refused call adds no node)."""
import numpy as np
import pytest

import ammon_b200 as ab
from ammon_b200 import _abi, kernels as K

import kv4_ref as ref

FAKE = 0x10000  # never dereferenced at record time


def fake(shape, dtype=ab.F32, ptr=FAKE):
    return ab.Tensor(ab.Tensor._desc(ptr, dtype, shape))


def layer(lead=(), kv=2, seq=16, words=8, **change):
    t = {"key_codes": fake(lead + (kv, seq, words), ab.U32),
         "key_scales": fake(lead + (kv, seq), ab.U32),
         "value_codes": fake(lead + (kv, seq, words), ab.U32),
         "value_scales": fake(lead + (kv, seq), ab.U32)}
    t.update(change)
    return ab.Kv4Layer(**t)


def step(n=1):
    return fake((n, 2), ab.U32)


@pytest.fixture()
def scheme():
    s = ab.Scheme(None)
    yield s
    s.close()


def refused(scheme, fn, *needles, cls=ab.ValidationError):
    before = scheme.ir_node_count()
    with pytest.raises(cls) as e:
        fn()
    for n in needles:
        assert n in str(e.value), str(e.value)
    assert scheme.ir_node_count() == before


def test_values_are_within_half_a_step_of_what_was_quantised():
    rng = np.random.default_rng(0)
    x = (rng.standard_normal((50, 3, 77)) * 3 + rng.standard_normal(77)).astype(np.float32)
    codes, scales = ref.quantise(x)
    back = ref.values(codes, scales, 77)
    s = ref.bf16_values((scales & 0xFFFF).astype(np.uint16)).astype(np.float64)
    m = ref.bf16_values((scales >> 16).astype(np.uint16)).astype(np.float64)
    # half a step, and at the ends what rounding m (2^-8 of it) and s (2^-8 of 15 s) moves them
    bound = s / 2 * (1 + 1e-9) + np.abs(m) * 2.0 ** -8 + 15 * s * 2.0 ** -8
    assert (np.abs(back - x) <= bound[..., None]).all()
    assert codes.shape[-1] == 12 and not (codes[..., 10:] >> 0).any()


def test_store_refusals(scheme):
    k = K.Kv4StoreKernel.prepare(None)
    rec = lambda key, value, cache, st: (lambda: k.record(scheme, "s", key, value, cache, st))
    x = fake((3, 2, 64))
    refused(scheme, rec(fake((64,)), fake((64,)), layer(), step()), "parameter `key`", "rank")
    refused(scheme, rec(x, fake((3, 2, 63)), layer(), step(3)), "parameter `value`")
    refused(scheme, rec(x, fake((3, 2, 64), ab.BF16), layer(), step(3)), "parameter `value`")
    refused(scheme, rec(fake((3, 2, 64), ab.U32), x, layer(), step(3)), "parameter `key`")
    refused(scheme, rec(x, x, layer(words=4), step(3)), "`cache.key_codes`", "`words`")
    refused(scheme, rec(x, x, layer(kv=3), step(3)), "`cache.key_codes`", "`kv_heads`")
    refused(scheme, rec(x, x, layer(lead=(2,)), step(3)), "`cache.key_codes`", "`batch`")
    refused(scheme, rec(x, x, layer(), step(2)), "parameter `step`", "batch needs 3")
    refused(scheme, rec(x, x, layer(key_scales=fake((2, 15), ab.U32)), step(3)),
            "`cache.key_scales`")
    refused(scheme, rec(x, x, layer(value_codes=fake((2, 15, 8), ab.U32)), step(3)),
            "`cache.value_codes`")
    refused(scheme, rec(x, x, layer(value_scales=fake((2, 16))), step(3)),
            "`cache.value_scales`", "u32")
    refused(scheme, rec(x, x, layer(key_codes=fake((2, 16, 8), ab.U32, FAKE + 4)), step(3)),
            "`cache.key_codes`", "16-byte aligned")
    refused(scheme, rec(x, x, layer(value_scales=fake((2, 16), ab.U32, FAKE + 2)), step(3)),
            "`cache.value_scales`", "4-byte aligned")
    refused(scheme, rec(fake((3, 2, 129)), fake((3, 2, 129)), layer(words=20), step(3)), "1..128")
    k.record(scheme, "s", x, x, layer(), step(3))
    k.record(scheme, "s", fake((2, 64)), fake((2, 64)), layer(lead=(1,)), step())
    assert scheme.ir_node_count() == 2


def test_load_refusals(scheme):
    k = K.Kv4LoadKernel.prepare(None)
    x = fake((5, 2, 64))
    refused(scheme, lambda: k.record(scheme, "l", layer(), step(), fake((2, 64)), fake((2, 64))),
            "parameter `key`", "rank")
    refused(scheme, lambda: k.record(scheme, "l", layer(), step(), fake((17, 2, 64)),
                                     fake((17, 2, 64))), "17 positions")
    refused(scheme, lambda: k.record(scheme, "l", layer(lead=(2,)), step(3), fake((3, 5, 2, 64)),
                                     fake((3, 5, 2, 64))), "`batch`")
    refused(scheme, lambda: k.record(scheme, "l", layer(lead=(3,)), step(2), fake((3, 5, 2, 64)),
                                     fake((3, 5, 2, 64))), "parameter `step`")
    refused(scheme, lambda: k.record(scheme, "l", layer(), step(), x, fake((5, 2, 64), ab.BF16)),
            "parameter `value`")
    k.record(scheme, "l", layer(), step(), x, x)
    assert scheme.ir_node_count() == 1


def test_attention_refusals():
    scheme = ab.Scheme(None)
    k = K.Kv4AttentionKernel.prepare(None)
    q, out = fake((3, 8, 64)), fake((3, 512))
    rec = lambda *a: (lambda: k.record(scheme, "a", *a))
    refused(scheme, rec(fake((3, 8, 64), ab.BF16), layer(), out, step(3)), "parameter `q`", "f32")
    refused(scheme, rec(fake((64,)), layer(), out, step(3)), "parameter `q`", "rank")
    refused(scheme, rec(fake((3, 7, 64)), layer(), out, step(3)), "must divide")
    refused(scheme, rec(q, layer(words=4), out, step(3)), "`words`")
    refused(scheme, rec(q, layer(lead=(2,)), out, step(3)), "`batch`")
    refused(scheme, rec(q, layer(), fake((3, 511)), step(3)), "parameter `out`", "1536")
    refused(scheme, rec(q, layer(), fake((3, 512), ab.U32), step(3)), "parameter `out`")
    refused(scheme, rec(q, layer(), out, step(2)), "parameter `step`")
    refused(scheme, rec(q, layer(), out, fake((3, 3), ab.U32)), "parameter `step`")
    scheme.close()


def test_cache_handle_refusals():
    out = _abi.C.c_void_p()
    assert _abi.lib().ab_kv4cache_create(None, 1, 1, 1, 1, 1, _abi.C.byref(out)) == _abi.AB_ERR_ARGUMENT
    assert _abi.lib().ab_kv4cache_layer(None, 0, None) == _abi.AB_ERR_ARGUMENT
    assert _abi.lib().ab_kv4cache_zero(None) == _abi.AB_ERR_ARGUMENT
    assert _abi.lib().ab_kv4cache_destroy(None) == _abi.AB_OK


def test_rows_not_aligned_to_their_elements_are_refused(scheme):
    for dtype, off in ((ab.F32, 2), (ab.BF16, 1)):
        good, bad = fake((3, 2, 64), dtype), fake((3, 2, 64), dtype, FAKE + off)
        for key, value in ((bad, good), (good, bad)):
            refused(scheme, lambda: K.Kv4StoreKernel.prepare(None).record(
                scheme, "s", key, value, layer(), step(3)), "not aligned")
            refused(scheme, lambda: K.Kv4LoadKernel.prepare(None).record(
                scheme, "l", layer(), step(), key, value), "not aligned")


def test_more_vectors_than_a_call_takes_are_refused(scheme):
    many = fake((1 << 28, 8, 16))
    refused(scheme, lambda: K.Kv4StoreKernel.prepare(None).record(
        scheme, "s", many, many, layer(kv=8, words=4), step(1 << 28)), "too many vectors")
    refused(scheme, lambda: K.Kv4LoadKernel.prepare(None).record(
        scheme, "l", layer(kv=8, seq=1 << 28, words=4), step(), many, many), "too many vectors")


def test_attention_onto_its_own_queries_is_refused(scheme):
    k = K.Kv4AttentionKernel.prepare(None)
    q = fake((3, 8, 64))
    for out in (fake((3, 512)), fake((3, 512), ab.BF16, FAKE + 3 * 512 * 4 - 2),
                fake((3, 512), ab.F32, FAKE - 4)):
        refused(scheme, lambda: k.record(scheme, "a", q, layer(), out, step(3)), "overlaps q")
    # beside them: refused for the runtime that a scheme of no device lacks, not for this
    for ptr in (FAKE - 3 * 512 * 4, FAKE + 3 * 512 * 4):
        refused(scheme, lambda: k.record(scheme, "a", q, layer(), fake((3, 512), ab.F32, ptr),
                                         step(3)), "runtime", cls=ab.AmmonError)
