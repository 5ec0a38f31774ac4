"""The runtime's stream: allocations do not wait for what is queued on it."""
import numpy as np
import pytest

import ammon_b200 as ab

pytestmark = pytest.mark.gpu


@pytest.fixture()
def rt():
    r = ab.create_runtime(0)
    yield r
    r.synchronize()


def test_zeros_do_not_wait_for_queued_work(rt):
    """A tensor made while half a second of work is queued is zero, and the work still runs."""
    torch = pytest.importorskip("torch")
    stream = torch.cuda.ExternalStream(rt.stream)
    ab.Tensor.zeros(rt, (64,)).read()  # first use
    with torch.cuda.stream(stream):
        torch.cuda._sleep(1)
        stream.synchronize()
        torch.cuda._sleep(10 ** 9)
    made = [ab.Tensor.zeros(rt, (64,)), ab.Tensor.zeros(rt, (3, 5), ab.BF16),
            ab.DecodeStep.parcel(rt, 4)]
    busy = not stream.query()
    assert all((t.read() == 0).all() for t in made)
    assert busy
