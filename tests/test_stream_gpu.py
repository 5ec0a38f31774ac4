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


def test_torch_on_the_runtimes_stream_is_ordered_with_it(rt):
    """Inputs that torch is still busy with when the scheme is submitted, outputs that torch reads
    right after, without a wait of the host's."""
    torch = pytest.importorskip("torch")
    s = rt.scheme()
    with torch.cuda.stream(rt.torch_stream()):
        a, b, out = (torch.zeros(4096, device="cuda") for _ in range(3))
        ab.kernels.TensorKernels.prepare(rt).add_into(
            s, "add", *[ab.Tensor.from_torch(x, rt) for x in (a, b, out)])
        for turn in range(1, 4):
            torch.cuda._sleep(10 ** 8)
            a.fill_(turn)
            b.fill_(10)
            s.submit()
            twice = out * 2
            torch.cuda.current_stream().synchronize()
            assert (twice == 2 * (turn + 10)).all()
    assert rt.torch_stream().cuda_stream == rt.stream
