"""A model over the 4-bit cache along its paths: the order of the block's nodes, a step against the
same modules down to the logits, and the prefill of a bf16 model in several passes, whose attention
runs on tcgen05, against its single steps."""
import numpy as np
import pytest

import ammon_b200 as ab

import kv4_ref as ref
from test_kv4_model_gpu import model, rt  # noqa: F401

pytestmark = pytest.mark.gpu

ARRAYS = ("key_codes", "key_scales", "value_codes", "value_scales")
BF16 = {"batch": 6, "dtype": ab.BF16, "dim": 256, "heads": 4, "kv_heads": 2, "head_dim": 64}


def record_by_hand(rt, m, cache, x, st, s):
    c = m.cfg
    att = ab.CausalAttentionBlock(rt, c.dim, c.heads, c.seq, max_batch=c.batch, rope_theta=c.rope_theta)
    ffn = ab.SwiGluBlock(rt, c.dim, c.hidden, max_batch=c.batch)
    ab.Embedding(rt).record(s, m.weight("embed"), st, x)
    for l in range(c.layers):
        w = ab.CausalAttentionBlockWeights(*[m.weight(k, l) for k in
                                             ("rms_att", "wq", "wk", "wv", "wo")])
        att.record(s, x, w, cache.layer(l), st)
        ffn.record(s, x, ab.SwiGluBlockWeights(m.weight("rms_ffn", l), m.weight("w1", l),
                                               m.weight("w3", l), m.weight("w2", l)))


@pytest.mark.parametrize("change", [{}, {"batch": 3}, {"kv_heads": 2}, BF16])
def test_block_nodes_are_in_order(rt, change):
    """Once a layer, the store directly before the attention, both between the projections."""
    m = model(rt, **change)
    c = m.cfg
    s = rt.scheme()
    cache = ab.Kv4Cache(rt, c.layers, c.seq, c.kv_heads, c.head_dim, batch=c.batch)
    record_by_hand(rt, m, cache, ab.Tensor.zeros(rt, (c.batch, c.dim)),
                   ab.DecodeStep.parcel(rt, c.batch), s)
    labels = s.node_labels()
    order = [l for l in labels if l in ("attn_kv4_store", "attn_kv4")]
    assert order == ["attn_kv4_store", "attn_kv4"] * c.layers
    for i, l in enumerate(labels):
        if l == "attn_kv4_store":
            assert labels[i + 1] == "attn_kv4"
            assert any("attn_qkv" in x for x in labels[:i])
            assert any("attn_wo" in x for x in labels[i + 2:])


@pytest.mark.parametrize("change", [{}, {"batch": 3}, {"kv_heads": 2}, BF16])
def test_model_step_equals_its_modules_down_to_the_logits(rt, change):
    m = model(rt, **change)
    c = m.cfg
    n = c.batch
    cache = ab.Kv4Cache(rt, c.layers, c.seq, c.kv_heads, c.head_dim, batch=n)
    x, st, s = ab.Tensor.zeros(rt, (n, c.dim)), ab.DecodeStep.parcel(rt, n), rt.scheme()
    record_by_hand(rt, m, cache, x, st, s)
    norm, cls = (m.weight(k).read_f32().astype(np.float64) for k in ("rms_final", "wcls"))
    for turn in range(4):
        toks = [(7 * turn + 3 * b) % c.vocab for b in range(n)]
        pos = [turn + (b % 2) * 5 for b in range(n)]
        logits = m.step_batch(toks, pos)[0].copy()
        rt.deposit(st, [ab.DecodeStep(t, p) for t, p in zip(toks, pos)])
        s.submit()
        h = x.read().astype(np.float64)
        for l in range(c.layers):
            a, b = m.kv4_cache().layer(l), cache.layer(l)
            for name in ARRAYS:
                assert np.array_equal(getattr(a, name).read(), getattr(b, name).read()), (turn, l)
        h = h / np.sqrt((h ** 2).mean(-1, keepdims=True) + c.norm_eps) * norm
        want = h @ cls.T
        # f32: a product of dim terms; bf16: its normed rows are rounded to bf16 as operands
        bound = np.abs(h) @ np.abs(cls).T * (2.0 ** -8 if c.dtype == ab.BF16 else 2.0 ** -18)
        assert (np.abs(logits.reshape(n, -1) - want) <= bound).all(), turn
    rt.synchronize()


def cached(m, layer, n):
    """Values of the first n positions of a layer's keys and values, stream 0."""
    a = [getattr(m.kv4_cache().layer(layer), k).read() for k in ARRAYS]
    if a[1].ndim == 3:
        a = [x[0] for x in a]
    return [ref.values(a[i][:, :n], a[i + 1][:, :n], m.cfg.head_dim) for i in (0, 2)]


@pytest.mark.parametrize("rows", [256, 131])
def test_bf16_prefill_in_several_passes_follows_its_single_steps(rt, rows):
    """600 tokens in passes of `rows`: more than 256 query slots of a kv head a pass, from position
    0 and from later ones on. What differs is the order of the bf16 projections' sums, some 2^-8 a
    projection, and the codes that it moves to their neighbour: values a few percent of their norm
    off, logits less."""
    change = {"dtype": ab.BF16, "dim": 512, "heads": 8, "kv_heads": 2, "head_dim": 64, "seq": 700}
    m = model(rt, **change)
    prompt = [(i * i * 7 + 3 * i) % m.cfg.vocab for i in range(600)]
    for i, t in enumerate(prompt):
        logits = m.step(t, i)
    logits = logits.copy()
    steps = [cached(m, l, 600) for l in range(m.cfg.layers)]
    follow = m.step(11, 600).copy()
    m.reset()
    m.set_prefill_rows(rows)
    got, first = m.prefill(prompt)
    assert first == int(got.argmax())
    for l, want in enumerate(steps):
        for a, b in zip(cached(m, l, 600), want):
            # every position by itself: a pass at the wrong place would be off by its whole norm
            off = np.linalg.norm(a - b, axis=(0, 2)) / np.linalg.norm(b, axis=(0, 2))
            assert off.max() <= 0.3 and np.sqrt((off ** 2).mean()) <= 0.1, (l, off.max(), off.argmax())
    assert np.abs(got - logits).max() <= 5e-2 * np.abs(logits).max()
    assert np.abs(m.step(11, 600) - follow).max() <= 5e-2 * np.abs(follow).max()
    rt.synchronize()
