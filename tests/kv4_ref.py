"""The 4-bit key/value cache in numpy, 64 bits: the packed format, its values, and attention."""
import numpy as np


def words_of(head):
    return 4 * ((head + 31) // 32)


def bf16_bits(x):
    """Nearest bf16 (halves to even) of finite float32 values, as uint16 bits."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32).astype(np.uint64)
    return ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)


def bf16_values(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def quantise(x):
    """codes [..., words] and scales [...] (uint32) of float32 vectors [..., head]."""
    x = np.ascontiguousarray(x, np.float32)
    head, words = x.shape[-1], words_of(x.shape[-1])
    fine = np.isfinite(x).all(-1)
    safe = np.where(fine[..., None], x, 0)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        m_bits = bf16_bits(safe.min(-1))
        m = bf16_values(m_bits)
        span = np.maximum(safe.max(-1) - m, np.float32(0))  # float32 throughout
        s_bits = bf16_bits(span / np.float32(15))
        s = bf16_values(s_bits)
        fine &= np.isfinite(m) & np.isfinite(span) & np.isfinite(s)
        level = (safe.astype(np.float64) - m[..., None].astype(np.float64)) / s[..., None].astype(np.float64)
        level = np.where((s > 0)[..., None] & fine[..., None], level, 0)
    c = np.clip(np.rint(level), 0, 15).astype(np.uint32)
    padded = np.zeros(x.shape[:-1] + (words * 8,), np.uint32)
    padded[..., :head] = c
    nib = padded.reshape(x.shape[:-1] + (words, 8))
    codes = np.zeros(x.shape[:-1] + (words,), np.uint32)
    for i in range(8):
        codes |= nib[..., i] << np.uint32(4 * i)
    scales = s_bits.astype(np.uint32) | (m_bits.astype(np.uint32) << 16)
    return codes, np.where(fine, scales, np.uint32(0x7FFF7FFF))


def values(codes, scales, head):
    """float64 values [..., head] that packed vectors stand for."""
    shifts = np.arange(0, 32, 4, dtype=np.uint32)
    c = ((codes[..., None] >> shifts) & 15).reshape(codes.shape[:-1] + (-1,))[..., :head]
    s = bf16_values((scales & 0xFFFF).astype(np.uint16)).astype(np.float64)
    m = bf16_values((scales >> 16).astype(np.uint16)).astype(np.float64)
    return c * s[..., None] + m[..., None]


def attention(q, k, v, pos):
    """q [heads, head], k and v [kv_heads, seq, head] (64 bits): [heads, head] over 0..pos."""
    heads, head = q.shape
    group = heads // k.shape[0]
    out = np.zeros((heads, head))
    for h in range(heads):
        kk, vv = k[h // group, :pos + 1], v[h // group, :pos + 1]
        score = kk @ q[h].astype(np.float64) / np.sqrt(head)
        p = np.exp(score - score.max())
        out[h] = p @ vv / p.sum()
    return out


def attention_bound(q, k_codes, k_scales, v, pos):
    """How far 32-bit attention may be from attention(), per head: [heads, 1].

    A score is a sum of head + 1 products. Rounding q (held to 22 bits or better), the products
    and the sums costs at most (head + 16) 2^-23 of sum |q_i| (|m| + 15 s) / sqrt(head); call
    that d. Weights change by a factor within e^(+-2d) after the division, the exponential and
    the weights' own 22 bits add 2^-21, and the sums over n positions run as partial sums of
    random sign: 6 sqrt(n) 2^-24, six standard deviations."""
    heads, head = q.shape
    group = heads // k_scales.shape[0]
    out = np.zeros((heads, 1))
    for h in range(heads):
        sc = k_scales[h // group, :pos + 1]
        s = bf16_values((sc & 0xFFFF).astype(np.uint16)).astype(np.float64)
        m = bf16_values((sc >> 16).astype(np.uint16)).astype(np.float64)
        d = (head + 16) * 2.0 ** -23 * np.abs(q[h]).sum() * (np.abs(m) + 15 * s).max() / np.sqrt(head)
        top = np.abs(v[h // group, :pos + 1]).max()
        out[h] = top * (np.expm1(2 * d) + 2.0 ** -21 + 6 * np.sqrt(pos + 1) * 2.0 ** -24)
    return out
