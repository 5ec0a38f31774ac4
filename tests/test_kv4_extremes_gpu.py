"""The quantising store of a 4-bit cache at the ends of the f32 range: codes equal the 64-bit
definition's bit for bit wherever the range of a vector is finite."""
import numpy as np
import pytest

import ammon_b200 as ab
from ammon_b200 import kernels as K

import kv4_ref as ref
from test_kv4_gpu import download, rt, steps, tensor, upload  # noqa: F401

pytestmark = pytest.mark.gpu

LARGEST = np.finfo(np.float32).max


def rows_of(rng, head):
    ramp = np.arange(head) / (head - 1.0)
    rows = []
    for top in (LARGEST, 3.3895313892515355e38, 3.4e38, 3.402e38, 15 * 2.0 ** 124, 3.2e38, 2.0 ** 127,
                2.0 ** 126, 15 * 2.0 ** 120, 2.0 ** 122):
        rows += [top * ramp, -top * ramp[::-1], top * (ramp - 0.5), top * rng.permutation(ramp),
                 top * np.r_[0, 1, rng.random(head - 2)], top * np.r_[0, 1, 1e38 / LARGEST * np.ones(head - 2)]]
    for step in (2.0 ** 124, 2.0 ** 123, 2.0 ** 120, 1.5 * 2.0 ** 119, 2.0 ** -100, 2.0 ** -101,
                 1.5 * 2.0 ** -126, 2.0 ** -133):  # halves of the step, and next to them
        half = (np.arange(head) % 16).astype(np.float64)
        half[1:15] += 0.5
        rows += [half * step, np.nextafter((half * step).astype(np.float32), np.float32(0)),
                 (half - 8) * step]
    # both ends just short of half the range each, and unlike
    rows += [np.linspace(-1.7014e38, 1.7014e38, head), np.linspace(-1e38, 2.4e38, head),
             np.linspace(-3.38e38, 1e36, head)]
    return np.stack(rows).astype(np.float32)


@pytest.mark.parametrize("dtype", [ab.F32, ab.BF16])
@pytest.mark.parametrize("head", [128, 33, 16])
def test_store_of_the_widest_rows(rt, head, dtype):
    rng = np.random.default_rng(head)
    x = rows_of(rng, head)
    if dtype == ab.BF16:  # the next finite bf16 numbers
        limit = ref.bf16_values(np.array([0x7F7F], np.uint16))[0]
        x = np.clip(x, -limit, limit)
    n = len(x)
    t, seen = tensor(rt, x[:, None], dtype)
    w = ref.words_of(head)
    layer = upload(rt, [np.full((1, n, w), 5, np.uint32), np.full((1, n), 6, np.uint32)] * 2)
    s = rt.scheme()
    K.Kv4StoreKernel.prepare(rt).record(s, "store", t, t, layer, steps(rt, range(n)))
    s.submit()
    codes, scales = ref.quantise(seen)
    got = download(layer)
    wide = scales[:, 0] != 0x7FFF7FFF
    assert wide.sum() > 0.8 * n
    for r in range(n):
        for i in (0, 2):
            assert got[i + 1][0, r] == scales[r, 0], (r, seen[r])
            assert np.array_equal(got[i][0, r], codes[r, 0]), (r, seen[r])
    rt.synchronize()
