"""Attention of prompts over very long 4-bit caches: sums of codes in the tensor unit, whose additions
cut off, run over at most 131072 positions."""
import pytest

import ammon_b200 as ab
from ammon_b200 import kernels as K

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv,capacity,lasts", [(48, 1000000, (999999, 131071, 131072, 5, 262143)),
                                               (1, 300000, (299999,)), (48, 140000, (100,))])
def test_sums_over_long_prompts(kv, capacity, lasts):
    """Value vectors of codes 15, step 1 and offset -14.875: the output is 0.125 whatever the
    weights, which random keys make unlike. A chain of 131072 positions is 2^14 additions; the
    partial sums are half the last one on average and lose at most 2^-23 each: 15 x 2^-10. (One
    chain of a million positions was 0.044 low.)"""
    torch = pytest.importorskip("torch")
    rt = ab.create_runtime(0)
    rows, head = 300, 32
    with torch.cuda.stream(rt.torch_stream()):
        gen = torch.Generator(device="cuda").manual_seed(1)
        dev = dict(dtype=torch.int32, device="cuda")
        codes = [torch.randint(-2 ** 31, 2 ** 31 - 1, (kv, capacity, 4), generator=gen, **dev),
                 torch.full((kv, capacity, 4), -1, **dev)]
        minus = torch.tensor([-14.875]).bfloat16().view(torch.int16).item() << 16
        scales = [torch.full((kv, capacity), 0x3F80, **dev),
                  torch.full((kv, capacity), minus | 0x3F80, **dev)]
        q = torch.randn((rows, kv, head), generator=gen, device="cuda") * 0.05
        out = torch.zeros((rows, kv * head), dtype=torch.bfloat16, device="cuda")
        step = torch.zeros((rows, 2), **dev)
        t = [ab.Tensor.from_torch(x, rt) for x in (codes[0], scales[0], codes[1], scales[1], q, out, step)]
        s = rt.scheme()
        K.Kv4AttentionKernel.prepare(rt).record(s, "a", t[4], ab.Kv4Layer(*t[:4]), t[5], t[6])
        for last in lasts:
            first = max(0, last + 1 - rows)
            step[:, 1] = torch.clamp(first + torch.arange(rows, **dev), max=last)
            out.fill_(9)
            s.submit()
            off = (out.double() - 0.125).abs().max().item()
            assert off <= 15 * 2.0 ** -10 + 0.125 * 2.0 ** -8, (last, off)
    rt.synchronize()
