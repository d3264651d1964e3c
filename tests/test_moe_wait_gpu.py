"""The mixture of experts' bounded wait on a counter in global memory, through its diagnostics entry
point: it ends by itself, reports, and leaves the context usable."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def _wait(counters, want, limit_ns=1_000_000):
    from nanovllm_b200 import _lib
    reached = torch.full((32,), -1, dtype=torch.int32, device="cuda")
    error = torch.zeros(1, dtype=torch.int32, device="cuda")
    a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    a.record()
    _lib.check(_lib.lib.fp8attn_diag_counter_wait(
        counters.data_ptr(), want, limit_ns, reached.data_ptr(), error.data_ptr(),
        torch.cuda.current_stream().cuda_stream))
    b.record()
    torch.cuda.synchronize()
    return reached.tolist(), int(error), a.elapsed_time(b)


@pytest.mark.parametrize("value", [7, 8, 2 ** 31 - 1])
def test_counter_that_has_the_value(value):
    reached, error, _ = _wait(torch.full((32,), value, dtype=torch.int32, device="cuda"), 7)
    assert reached == [1] * 32 and error == 0


@pytest.mark.parametrize("value", [6, 0, -5])
def test_counter_that_never_gets_there(value):
    """Gives up after its limit, in every lane, and says so; the context stays usable."""
    reached, error, ms = _wait(torch.full((32,), value, dtype=torch.int32, device="cuda"), 7)
    assert reached == [0] * 32 and error == 1
    assert ms >= 1.0
    assert int(torch.ones(5, device="cuda").sum()) == 5


def test_refusals():
    from nanovllm_b200 import _lib
    wait = _lib.lib.fp8attn_diag_counter_wait
    assert wait(None, 1, 10, 4096, 0, None) == _lib.EINVAL
    assert wait(4096, 1, 10, None, 0, None) == _lib.EINVAL
    assert wait(4096, 1, -1, 4096, 0, None) == _lib.EINVAL


@pytest.mark.parametrize("lane", [0, 1, 5, 31])
def test_every_lane_decides_by_the_value_that_it_read_itself(lane):
    """What a lane reads after the wait is ordered by its own reading of the counter, so one lane that
    has not seen the value keeps the warp waiting."""
    counters = torch.full((32,), 9, dtype=torch.int32, device="cuda")
    counters[lane] = 6
    reached, error, _ = _wait(counters, 7)
    assert reached == [0] * 32 and error == 1
