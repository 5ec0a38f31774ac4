"""CausalAttentionBlock and LlamaModel over the 4-bit key/value cache: the block against 64 bits
(with the values that the cache holds), the model against the same modules recorded by hand, and
its prefill and device loop against single steps."""
import numpy as np
import pytest

import ammon_b200 as ab
from ammon_b200 import kernels as K

import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def rt():
    r = ab.create_runtime(0)
    yield r
    r.synchronize()


def steps(rt, pairs):
    p = ab.DecodeStep.parcel(rt, len(pairs))
    rt.deposit(p, [ab.DecodeStep(int(t), int(x)) for t, x in pairs])
    return p


def rope64(x, pos, theta):
    """Rotates pairs of the last axis; the angles as the kernels round them, in float32."""
    head = x.shape[-1]
    i = np.arange(0, head, 2)
    freq = (np.float32(1) / np.float32(theta) ** (i.astype(np.float32) / np.float32(head)))
    a = (np.float32(pos) * freq.astype(np.float32)).astype(np.float64)
    out = np.empty_like(x)
    out[..., 0::2] = x[..., 0::2] * np.cos(a) - x[..., 1::2] * np.sin(a)
    out[..., 1::2] = x[..., 0::2] * np.sin(a) + x[..., 1::2] * np.cos(a)
    return out


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("heads,kv,head,rows", [(8, 2, 64, 3), (6, 6, 48, 2), (6, 2, 32, 12),
                                                (5, 1, 64, 1)])
def test_block_matches_64_bits(rt, heads, kv, head, rows, shared):
    rng = np.random.default_rng(heads * 10 + rows)
    hidden, seq, theta = heads * head, 40, 10000.0
    positions = list(range(3, 3 + rows)) if shared else [int(p) for p in rng.integers(0, 12, rows)]
    w = {n: (rng.standard_normal(s) / np.sqrt(hidden)).astype(np.float32) for n, s in
         (("q", (hidden, hidden)), ("k", (kv * head, hidden)), ("v", (kv * head, hidden)),
          ("o", (hidden, hidden)))}
    norm = rng.uniform(0.5, 1.5, hidden).astype(np.float32)
    x = rng.standard_normal((rows, hidden)).astype(np.float32)
    cache = ab.Kv4Cache(rt, 1, seq, kv, head, batch=1 if shared or rows == 1 else rows)
    layer = cache.layer(0)
    # earlier positions of the cache
    lead = (kv, seq) if len(layer.key_scales.shape) == 2 else (rows, kv, seq)
    for codes, scales in ((layer.key_codes, layer.key_scales),
                          (layer.value_codes, layer.value_scales)):
        c, s = ref.quantise(rng.standard_normal(lead + (head,)).astype(np.float32))
        codes.write(c)
        scales.write(s)
    block = ab.CausalAttentionBlock(rt, hidden, heads, seq, max_batch=rows)
    xt = ab.Tensor.from_array(rt, x if rows > 1 else x[0])
    weights = ab.CausalAttentionBlockWeights(*[ab.Tensor.from_array(rt, a) for a in
                                               (norm, w["q"], w["k"], w["v"], w["o"])])
    s = rt.scheme()
    block.record(s, xt, weights, layer, steps(rt, [(0, p) for p in positions]))
    assert s.node_labels()[1:3] == ["attn_kv4_store", "attn_kv4"] or "attn_kv4" in s.node_labels()
    s.submit()
    got = xt.read().reshape(rows, hidden)
    held = [t.read() for t in (layer.key_codes, layer.key_scales, layer.value_codes,
                               layer.value_scales)]
    x64 = x.astype(np.float64)
    xn = x64 / np.sqrt((x64 ** 2).mean(-1, keepdims=True) + 1e-5) * norm
    for r, pos in enumerate(positions):
        kc, ks, vc, vs = held if held[1].ndim == 2 else [a[r] for a in held]
        q, k, v = (xn[r] @ w[n].astype(np.float64).T for n in "qkv")
        q = rope64(q.reshape(heads, head), pos, theta)
        k = rope64(k.reshape(kv, head), pos, theta)
        for new, codes, scales in ((k, kc, ks), (v.reshape(kv, head), vc, vs)):
            back = ref.values(codes[:, pos], scales[:, pos], head)
            st = ref.bf16_values((scales[:, pos] & 0xFFFF).astype(np.uint16)).astype(np.float64)
            m = ref.bf16_values((scales[:, pos] >> 16).astype(np.uint16)).astype(np.float64)
            # half a step; what rounding m and s moves the ends by; the f32 projection
            bound = st / 2 + np.abs(m) * 2.0 ** -8 + 15 * st * 2.0 ** -8 + 1e-5 * np.abs(new).max()
            assert (np.abs(back - new) <= bound[:, None]).all()
        kk = ref.values(kc, ks, head)
        vv = ref.values(vc, vs, head)
        att = ref.attention(q, kk, vv, pos).reshape(hidden)
        want = x64[r] + att @ w["o"].astype(np.float64).T
        # three f32 products of `hidden` terms, the scores' own part far below them
        assert np.abs(got[r] - want).max() <= 1e-5 * (np.abs(want).max() + np.abs(att).max() * 4)
    rt.synchronize()


def test_block_bf16_weights(rt):
    """bf16 weights and activations: within 2e-2 of 64 bits, as the block over a bf16 cache."""
    rng = np.random.default_rng(5)
    heads, kv, head, rows, seq = 8, 2, 128, 6, 64
    hidden = heads * head
    cache = ab.Kv4Cache(rt, 1, seq, kv, head, batch=rows)
    layer = cache.layer(0)
    w = [ref.bf16_bits((rng.standard_normal(s) / np.sqrt(hidden)).astype(np.float32)) for s in
         ((hidden, hidden), (kv * head, hidden), (kv * head, hidden), (hidden, hidden))]
    norm = ref.bf16_bits(np.ones(hidden, np.float32))
    x = rng.standard_normal((rows, hidden)).astype(np.float32)
    block = ab.CausalAttentionBlock(rt, hidden, heads, seq, max_batch=rows)
    xt = ab.Tensor.from_array(rt, x)
    weights = ab.CausalAttentionBlockWeights(*[ab.Tensor.from_array(rt, a, ab.BF16)
                                               for a in [norm] + w])
    st = steps(rt, [(0, 0)] * rows)
    s = rt.scheme()
    block.record(s, xt, weights, layer, st)
    s.submit()  # position 0: the output is Wo of the row's own value, as the cache holds it
    got = xt.read()
    vals = ref.values(layer.value_codes.read(), layer.value_scales.read(), head)[:, :, 0]
    att = np.repeat(vals, heads // kv, axis=1).reshape(rows, hidden)
    want = x + att @ ref.bf16_values(w[3]).astype(np.float64).T
    assert np.abs(got - want).max() <= 2e-2 * np.abs(want).max()
    rt.synchronize()


CFG = ab.LlamaConfig(dim=288, layers=3, heads=6, kv_heads=6, head_dim=48, hidden=768, vocab=512,
                     seq=64)


def model(rt, **change):
    cfg = ab.LlamaConfig(**{**CFG.__dict__, **change})
    m = ab.LlamaModel(rt, cfg, kv4=True)
    m.init_synthetic(3, 0.05)
    return m


@pytest.mark.parametrize("change", [{}, {"batch": 3}, {"kv_heads": 2},
                                    {"batch": 6, "dtype": ab.BF16, "dim": 256, "heads": 4,
                                     "kv_heads": 2, "head_dim": 64}])
def test_model_step_equals_its_modules(rt, change):
    m = model(rt, **change)
    c = m.cfg
    n = c.batch
    cache = ab.Kv4Cache(rt, c.layers, c.seq, c.kv_heads, c.head_dim, batch=n)
    att = ab.CausalAttentionBlock(rt, c.dim, c.heads, c.seq, max_batch=n, rope_theta=c.rope_theta)
    ffn = ab.SwiGluBlock(rt, c.dim, c.hidden, max_batch=n)
    x = ab.Tensor.zeros(rt, (n, c.dim))
    st = ab.DecodeStep.parcel(rt, n)
    s = rt.scheme()
    ab.Embedding(rt).record(s, m.weight("embed"), st, x)
    for l in range(c.layers):
        w = ab.CausalAttentionBlockWeights(*[m.weight(k, l) for k in
                                             ("rms_att", "wq", "wk", "wv", "wo")])
        att.record(s, x, w, cache.layer(l), st)
        ffn.record(s, x, ab.SwiGluBlockWeights(m.weight("rms_ffn", l), m.weight("w1", l),
                                               m.weight("w3", l), m.weight("w2", l)))
    for turn in range(4):
        toks = [(7 * turn + 3 * b) % c.vocab for b in range(n)]
        pos = [turn + (b % 2) * 5 for b in range(n)]
        m.step_batch(toks, pos)
        rt.deposit(st, [ab.DecodeStep(t, p) for t, p in zip(toks, pos)])
        s.submit()
        rt.synchronize()
        for l in range(c.layers):
            a, b = m.kv4_cache().layer(l), cache.layer(l)
            for u, v in ((a.key_codes, b.key_codes), (a.value_scales, b.value_scales)):
                assert np.array_equal(u.read(), v.read()), (turn, l)


def test_model_device_loop_equals_steps_and_prefill_follows(rt):
    m = model(rt)
    c = m.cfg
    prompt = [5, 91, 17, 300, 2, 44, 8]
    m.reset()
    for i, t in enumerate(prompt):
        logits = m.step(t, i).copy()
    first = int(logits.argmax())
    ids, tok = [], first
    for i in range(12):
        _, am = m.step_batch([tok], [len(prompt) + i], logits=False, argmax=True)
        tok = int(am[0])
        ids.append(tok)
    m.reset()
    for i, t in enumerate(prompt):
        m.step(t, i)
    assert m.decode_device([first], [len(prompt)], 12)[:, 0].tolist() == ids
    # A prefill pass rounds its projections in another order: a value next to the middle of two
    # codes may take the other one, which moves a value by one step of fifteen in its range.
    m.reset()
    pre, _ = m.prefill(prompt)
    assert np.abs(pre - logits).max() <= 5e-2 * np.abs(logits).max()
    rt.synchronize()


def test_model_prefill_fills_its_stream_alone(rt):
    m = model(rt, batch=2)
    m.prefill([4, 9, 2, 7, 7], stream=1)
    layer = m.kv4_cache().layer(1)
    scales = layer.key_scales.read()
    assert not scales[0].any()
    assert scales[1][:, :5].all() and not scales[1][:, 5:].any()


def test_cache_of_the_other_kind_is_refused(rt):
    m = model(rt)
    with pytest.raises(ab.AmmonError, match="4-bit"):
        m.cache()
    plain = ab.LlamaModel(rt, ab.LlamaConfig(**CFG.__dict__))
    with pytest.raises(ab.AmmonError, match="4-bit"):
        plain.kv4_cache()


def test_refused_block_records_add_no_node(rt):
    block = ab.CausalAttentionBlock(rt, 256, 4, 32, max_batch=2)
    t = lambda *s: ab.Tensor.zeros(rt, s)
    w = ab.CausalAttentionBlockWeights(t(256), t(256, 256), t(128, 256), t(128, 256), t(256, 256))
    s = rt.scheme()
    x, st = t(2, 256), steps(rt, [(0, 0), (0, 1)])
    for cache, why in ((ab.Kv4Cache(rt, 1, 32, 4, 64), "kv_heads"),
                       (ab.Kv4Cache(rt, 1, 31, 2, 64), "seq"),
                       (ab.Kv4Cache(rt, 1, 32, 2, 32), "words")):
        with pytest.raises(ab.ValidationError, match=why):
            block.record(s, x, w, cache.layer(0), st)
        assert s.ir_node_count() == 0
    block.record(s, x, w, ab.Kv4Cache(rt, 1, 32, 2, 64, batch=2).layer(0), st)
    assert s.ir_node_count() == 4
