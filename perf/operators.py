"""Operators of the 4-bit key/value cache: rows quantised as they are written, rows read back,
and attention over the packed cache. Plain torch forms beside the framework's kernels, with the
cases that both are timed and compared on.

The packed cache. One vector is the `head` values that one kv head keeps for one position. It is
held as 4-bit codes and one 32-bit word of scales:
    m = bf16(min x)                 the offset
    s = bf16(max(max x - m, 0) / 15)  the step
    c_i = the whole number nearest to (x_i - m) / s, halves to even, kept within 0..15
    (all c_i = 0 where s = 0; m, s and with them every value NaN where x is not finite throughout)
and stands for the values m + s c_i. Codes are int32 words [batch, kv_heads, seq, 4 ceil(head/32)]
(element i in word i // 8, bits 4 (i % 8) and up; the elements past `head` are 0), scales are
int32 words [batch, kv_heads, seq] with s in the low and m in the high half. Rows that share one
cache use the same arrays without the batch axis.
"""
import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
_runtime = None


def words_of(head):
    """32-bit words of codes a vector of `head` elements takes (rows are padded to 16 bytes)."""
    return 4 * ((head + 31) // 32)


# ---- the cases ---------------------------------------------------------------------------
def _write(name, rows, kv, head, shared, src, out, seq):
    return {"name": name, "op": "write", "rows": rows, "kv": kv, "head": head, "shared": shared,
            "src": src, "out": out, "seq": seq}


def _read(name, batch, n, kv, head, out, seq):
    return {"name": name, "op": "read", "batch": batch, "n": n, "kv": kv, "head": head,
            "out": out, "seq": seq}


def _attend(name, rows, heads, kv, head, shared, out, seq, last, ragged):
    return {"name": name, "op": "attend", "rows": rows, "heads": heads, "kv": kv, "head": head,
            "shared": shared, "out": out, "seq": seq, "last": last, "ragged": ragged}


def listed():
    return [
        # one new token of one stream of an 8B-shaped model (32/8 heads of 128): pure latency
        _write("write_token", 1, 8, 128, False, "f32", "f32", 8192),
        # a decode step of 64 such streams, each into its own cache
        _write("write_tokens_64", 64, 8, 128, False, "f32", "f32", 2048),
        # a small model (6 heads of 48) taking an odd-sized prompt
        _write("write_small_prompt", 37, 6, 48, True, "f32", "f32", 256),
        # a long prompt whose keys and values another stage computed in bf16
        _write("write_long_prompt", 32768, 8, 128, True, "bf16", "bf16", 32768),
        # 16 streams of a 12-head model read back for a further prompt pass
        _read("read_streams", 16, 1000, 12, 64, "f32", 1024),
        # one whole 128k-token cache read back
        _read("read_whole", 1, 131072, 8, 128, "bf16", 131072),
        # a decode step of the small model
        _attend("attend_small", 1, 6, 6, 48, False, "f32", 256, 100, False),
        # a decode step of the 8B shape, 8k tokens in
        _attend("attend_8k", 1, 32, 8, 128, False, "bf16", 8192, 8000, False),
        # the same 128k tokens in: the cache is the whole cost
        _attend("attend_128k", 1, 32, 8, 128, False, "f32", 131072, 131071, False),
        # 64 streams of unlike lengths in one step
        _attend("attend_64_ragged", 64, 32, 8, 128, False, "bf16", 8192, 8191, True),
        # 256 streams of a 12-head model without shared heads
        _attend("attend_256_streams", 256, 12, 12, 64, False, "f32", 1024, 1023, True),
        # a prompt pass: 256 rows over one cache, each attending up to its own position
        _attend("attend_prompt", 256, 32, 8, 128, True, "bf16", 8192, 2047, False),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["write", "read", "attend", "attend"])
    head = rng.choice([32, 48, 64, 64, 80, 96, 112, 128, 128, rng.randint(1, 128)])
    kv = rng.choice([1, 2, 3, 4, 5, 6, 8, 8, 12, 16])
    out = rng.choice(["f32", "bf16"])
    vector = kv * head
    if op == "write":
        shared = rng.random() < 0.5
        rows = _log_int(rng, 1, 16384 if shared else 256)
        rows = max(1, min(rows, (32 << 20) // vector))
        seq = (rows + rng.randint(0, 500) if shared
               else rng.randint(1, max(1, min(4096, (64 << 20) // (rows * vector)))))
        return {"op": op, "rows": rows, "kv": kv, "head": head, "shared": shared,
                "src": rng.choice(["f32", "bf16"]), "out": out, "seq": seq}
    if op == "read":
        batch = _log_int(rng, 1, 64)
        n = max(1, min(_log_int(rng, 1, 65536), (64 << 20) // (batch * vector)))
        return {"op": op, "batch": batch, "n": n, "kv": kv, "head": head, "out": out,
                "seq": n + rng.randint(0, 300)}
    group = rng.choice([1, 1, 2, 3, 4, 4, 5, 6, 7, 8, 8, 12, 16])
    shared = rng.random() < 0.35
    rows = _log_int(rng, 1, 256)
    if shared:
        last = rng.randint(rows - 1, max(rows - 1, _log_int(rng, rows, 4096)))
        while rows > 1 and rows * group * vector * (last + 1) > 1 << 31:
            rows = rows // 2
    else:
        last = max(0, min(_log_int(rng, 1, 131072) - 1, (100 << 20) // (rows * vector)))
    return {"op": op, "rows": rows, "heads": kv * group, "kv": kv, "head": head,
            "shared": shared, "out": out, "seq": last + 1 + rng.randint(0, 100), "last": last,
            "ragged": not shared and rng.random() < 0.6}


def work(case):
    size = {"f32": 4, "bf16": 2}
    kv, head = case["kv"], case["head"]
    packed = 2 * kv * (math.ceil(head / 2) + 4)  # bytes of one position's keys and values
    if case["op"] == "write":
        plain = 2 * kv * head * (size[case["src"]] + size[case["out"]])
        return {"bytes": case["rows"] * (plain + packed), "flops": case["rows"] * 2 * kv * head * 6}
    if case["op"] == "read":
        n = case["batch"] * case["n"]
        return {"bytes": n * (packed + 2 * kv * head * size[case["out"]]),
                "flops": n * 4 * kv * head}
    rows, last = case["rows"], case["last"]
    q = rows * case["heads"] * head * (4 + size[case["out"]])
    if case["shared"]:
        seen = rows * (last + 1) - rows * (rows - 1) // 2
        return {"bytes": (last + 1) * packed + q, "flops": seen * case["heads"] * head * 4}
    seen = sum(p + 1 for p in _positions(case))
    return {"bytes": seen * packed + q, "flops": seen * case["heads"] * head * 4}


def _positions(case):
    """The position every row of an attention case stands at."""
    rows, last = case["rows"], case["last"]
    if case["shared"]:
        return [last - rows + 1 + i for i in range(rows)]
    if not case["ragged"]:
        return [last] * rows
    # spread over the whole range in no order, the longest first
    return [last - (i * 2654435761 % 1000003) * (last + 1) // 1000003 for i in range(rows)]


# ---- inputs --------------------------------------------------------------------------------
def _values(shape, gen):
    """Keys or values as a trained model gives them: about normal, with some channels of each
    head off centre or wide, and a scale of its own for every position."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    channel = torch.randn(shape[-2:], generator=gen, device=DEVICE)
    wide = 1 + 4 * (torch.rand(shape[-2:], generator=gen, device=DEVICE) > 0.95)
    token = torch.rand(shape[:-2], generator=gen, device=DEVICE) + 0.5
    return (x + channel) * wide * token[..., None, None]


def _parcel(pairs):
    return torch.tensor(pairs, dtype=torch.int32, device=DEVICE)


def _empty_cache(lead, kv, seq, head):
    codes = torch.zeros(lead + (kv, seq, words_of(head)), dtype=torch.int32, device=DEVICE)
    scales = torch.zeros(lead + (kv, seq), dtype=torch.int32, device=DEVICE)
    return codes, scales


def prepare(case, seed):
    if own:
        _on_the_runtimes_stream()
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    kv, head, seq = case["kv"], case["head"], case["seq"]
    state = {"case": dict(case)}
    if case["op"] == "write":
        rows, shared = case["rows"], case["shared"]
        for name in ("key", "value"):
            state[name] = _values((rows, kv, head), gen).to(TYPES[case["src"]])
            state[name + "_codes"], state[name + "_scales"] = _empty_cache(
                () if shared else (rows,), kv, seq, head)
        if shared:  # consecutive positions, ending with the cache
            places = list(range(seq - rows, seq))
        else:
            places = torch.randint(0, seq, (rows,), generator=gen, device=DEVICE).tolist()
        state["step"] = _parcel([[0, p] for p in places])
        state["start"] = _parcel([[0, places[0]]]) if shared else state["step"]
        lead = (rows,) if shared else (rows, 1)
    elif case["op"] == "read":
        batch, n = case["batch"], case["n"]
        first = torch.randint(0, seq - n + 1, (batch,), generator=gen, device=DEVICE).tolist()
        state["start"] = _parcel([[0, p] for p in first])
        lead = (n,) if batch == 1 else (batch, n)
        _fill_caches(state, () if batch == 1 else (batch,), seq, gen)
    else:
        rows, heads = case["rows"], case["heads"]
        state["q"] = torch.randn((rows, heads, head), generator=gen, device=DEVICE) * 1.5
        state["step"] = _parcel([[0, p] for p in _positions(case)])
        _fill_caches(state, () if case["shared"] or rows == 1 else (rows,), seq, gen)
    if case["op"] == "attend":
        state["out"] = torch.zeros((case["rows"], case["heads"] * head), dtype=TYPES[case["out"]],
                                   device=DEVICE)
    else:
        for name in ("key", "value"):
            state["out_" + name] = torch.zeros(lead + (kv, head), dtype=TYPES[case["out"]],
                                               device=DEVICE)
    if own:
        state["scheme"] = _record(state)  # the recorded plan such a program keeps
    return state


def _fill_caches(state, lead, seq, gen):
    case = state["case"]
    kv, head = case["kv"], case["head"]
    for name in ("key", "value"):
        codes, scales = _empty_cache(lead, kv, seq, head)
        flat_codes = codes.view((-1,) + codes.shape[-3:])
        flat_scales = scales.view((-1,) + scales.shape[-2:])
        for b in range(flat_codes.shape[0]):
            for at in range(0, seq, 32768):
                part = slice(at, min(seq, at + 32768))
                x = _values((part.stop - at, kv, head), gen).transpose(0, 1)
                flat_codes[b][:, part], flat_scales[b][:, part] = _quantise(x)
        state[name + "_codes"], state[name + "_scales"] = codes, scales


# ---- the plain forms -----------------------------------------------------------------------
def _quantise(x):
    """Packs vectors [..., head] into codes [..., words] and scales [...]."""
    x = x.float()
    head = x.shape[-1]
    m = x.amin(-1).bfloat16()
    fifteen = x.new_full((), 15.0)  # a tensor: torch multiplies by the reciprocal of a number
    s = ((x.amax(-1) - m.float()).clamp_min(0) / fifteen).bfloat16()
    bad = ~(torch.isfinite(m) & torch.isfinite(s) & torch.isfinite(x).all(-1))
    m, s = m.masked_fill(bad, math.nan), s.masked_fill(bad, math.nan)
    # 64 bits: a quotient next to a half has to fall on its own side
    c = ((x.double() - m.double()[..., None]) / s.double()[..., None]).round().clamp(0, 15)
    c = torch.where((s > 0)[..., None], c, 0).to(torch.int32)
    c = torch.nn.functional.pad(c, (0, words_of(head) * 8 - head))
    c = c.view(c.shape[:-1] + (words_of(head), 8))
    codes = (c << torch.arange(0, 32, 4, device=c.device, dtype=torch.int32)).sum(-1, dtype=torch.int32)
    low = s.view(torch.int16).to(torch.int32) & 0xFFFF
    high = m.view(torch.int16).to(torch.int32) << 16
    return codes, high | low


def _dequantise(codes, scales, head):
    """The 32-bit values [..., head] that codes [..., words] and scales [...] stand for."""
    shifts = torch.arange(0, 32, 4, device=codes.device, dtype=torch.int32)
    c = ((codes[..., None] >> shifts) & 15).flatten(-2)[..., :head].float()
    s = (scales << 16).view(torch.float32)
    m = (scales & -65536).view(torch.float32)
    return c * s[..., None] + m[..., None]


def _places(state):
    """Positions to read: [batch, n]."""
    case = state["case"]
    if case["op"] == "write":
        n = case["rows"] if case["shared"] else 1
    else:
        n = case["n"]
    at = state["start"][:, 1].long()
    return at[:, None] + torch.arange(n, device=DEVICE)


def _plain_write(state):
    case = state["case"]
    at = state["step"][:, 1].long()
    for name in ("key", "value"):
        codes, scales = _quantise(state[name])
        if case["shared"]:
            state[name + "_codes"][:, at] = codes.transpose(0, 1)
            state[name + "_scales"][:, at] = scales.transpose(0, 1)
        else:
            row = torch.arange(case["rows"], device=DEVICE)
            state[name + "_codes"][row, :, at] = codes
            state[name + "_scales"][row, :, at] = scales


def _plain_read(state, name):
    case = state["case"]
    kv, head = case["kv"], case["head"]
    codes = state[name + "_codes"].view(-1, kv, case["seq"], words_of(head))
    scales = state[name + "_scales"].view(-1, kv, case["seq"])
    places = _places(state)
    row = torch.arange(places.shape[0], device=DEVICE)[:, None, None]
    head_at = torch.arange(kv, device=DEVICE)
    codes = codes[row, head_at, places[:, :, None]]  # [batch, n, kv, words]
    scales = scales[row, head_at, places[:, :, None]]
    values = _dequantise(codes, scales, head).to(TYPES[case["out"]])
    return values.view(state["out_" + name].shape)


def _plain_attend(state):
    case = state["case"]
    rows, heads, kv, head = case["rows"], case["heads"], case["kv"], case["head"]
    group, end = heads // kv, case["last"] + 1
    at = state["step"][:, 1].long()
    k, v = (_dequantise(state[n + "_codes"].view(-1, kv, case["seq"], words_of(head))[:, :, :end],
                        state[n + "_scales"].view(-1, kv, case["seq"])[:, :, :end], head)
            for n in ("key", "value"))
    q = state["q"] / math.sqrt(head)
    if case["shared"]:  # every row of the one cache: [1, kv, rows * group, head]
        q = q.view(rows, kv, group, head).permute(1, 0, 2, 3).reshape(1, kv, rows * group, head)
        limit = at.repeat_interleave(group).view(1, 1, rows * group, 1)
    else:
        q = q.view(rows, kv, group, head)
        limit = at.view(rows, 1, 1, 1)
    scores = q @ k.transpose(-1, -2)
    scores = scores.masked_fill(torch.arange(end, device=DEVICE) > limit, -math.inf)
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    out = (p @ v) / p.sum(-1, keepdim=True)
    if case["shared"]:
        out = out.view(kv, rows, group, head).permute(1, 0, 2, 3)
    return out.reshape(rows, heads * head).to(TYPES[case["out"]])


# ---- the framework's calls --------------------------------------------------------------------
def _on_the_runtimes_stream():
    """The runtime works on a stream of its own, with which nothing orders torch's: a program that
    mixes the two has torch work there too."""
    import ammon_b200 as ab

    global _runtime
    if _runtime is None:
        _runtime = ab.create_runtime(torch.cuda.current_device())
    before = torch.cuda.current_stream()
    if before.cuda_stream != _runtime.stream:
        stream = torch.cuda.ExternalStream(_runtime.stream)
        stream.wait_stream(before)
        torch.cuda.set_stream(stream)


def _record(state):
    import ammon_b200 as ab
    from ammon_b200 import kernels as K

    rt, case = _runtime, state["case"]
    scheme = rt.scheme()
    t = {n: ab.Tensor.from_torch(x, rt) for n, x in state.items() if isinstance(x, torch.Tensor)}
    cache = ab.Kv4Layer(t["key_codes"], t["key_scales"], t["value_codes"], t["value_scales"])
    if case["op"] == "write":
        K.Kv4StoreKernel.prepare(rt).record(scheme, "write", t["key"], t["value"], cache, t["step"])
    if case["op"] == "attend":
        K.Kv4AttentionKernel.prepare(rt).record(scheme, "attend", t["q"], cache, t["out"], t["step"])
    else:
        K.Kv4LoadKernel.prepare(rt).record(scheme, "read", cache, t["start"], t["out_key"],
                                           t["out_value"])
    return scheme


def run(state):
    op = state["case"]["op"]
    if own:
        state["scheme"].submit()
        if op == "attend":
            return state["out"]
        return {"key": state["out_key"], "value": state["out_value"]}
    if op == "attend":
        return _plain_attend(state)
    if op == "write":
        _plain_write(state)
    return {"key": _plain_read(state, "key"), "value": _plain_read(state, "value")}


# ---- 64 bits, from the definition ----------------------------------------------------------
def _exact_vectors(codes, scales, head):
    """[n, head] doubles of packed vectors: codes [n, words], scales [n], by bytes."""
    b = codes.contiguous().view(torch.uint8)
    c = torch.stack([b % 16, b // 16], -1).reshape(b.shape[0], -1)[:, :head].double()
    half = scales.contiguous().view(torch.bfloat16).view(-1, 2).double()
    return half[:, 1:] + half[:, :1] * c


def _exact_round_trip(x):
    """What a vector's values read back as: x [n, head] of any type."""
    x = x.double()
    m = x.min(1, keepdim=True).values.bfloat16().double()
    s = ((x.max(1, keepdim=True).values - m).clamp(min=0) / 15).bfloat16().double()
    level = torch.where(s > 0, (x - m) / torch.where(s > 0, s, 1.0), 0.0)
    return m + s * torch.round(level).clamp(0, 15)


def exact(case, seed):
    global own
    before, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = before
    kv, head, seq = case["kv"], case["head"], case["seq"]
    if case["op"] == "write":
        return {n: _exact_round_trip(state[n].reshape(-1, head)).view(state["out_" + n].shape)
                for n in ("key", "value")}
    if case["op"] == "read":
        got = {}
        for n in ("key", "value"):
            codes = state[n + "_codes"].view(-1, kv, seq, words_of(head))
            scales = state[n + "_scales"].view(-1, kv, seq)
            out = torch.empty((case["batch"], case["n"], kv, head), dtype=torch.float64, device=DEVICE)
            for b, first in enumerate(state["start"][:, 1].tolist()):
                for h in range(kv):
                    out[b, :, h] = _exact_vectors(codes[b, h, first:first + case["n"]],
                                                  scales[b, h, first:first + case["n"]], head)
            got[n] = out.view(state["out_" + n].shape)
        return got
    rows, heads = case["rows"], case["heads"]
    group = heads // kv
    codes = {n: state[n + "_codes"].view(-1, kv, seq, words_of(head)) for n in ("key", "value")}
    scales = {n: state[n + "_scales"].view(-1, kv, seq) for n in ("key", "value")}
    places = state["step"][:, 1].tolist()
    out = torch.empty((rows, heads, head), dtype=torch.float64, device=DEVICE)
    for h in range(kv):
        for r in range(rows):
            b = 0 if codes["key"].shape[0] == 1 else r
            if b == r or r == 0:
                end = max(places) + 1 if codes["key"].shape[0] == 1 else places[r] + 1
                k, v = (_exact_vectors(codes[n][b, h, :end], scales[n][b, h, :end], head)
                        for n in ("key", "value"))
            seen = places[r] + 1
            mine = slice(h * group, (h + 1) * group)
            weight = torch.softmax(state["q"][r, mine].double() @ k[:seen].T / math.sqrt(head), -1)
            out[r, mine] = weight @ v[:seen]
    return out.view(rows, heads * head)
