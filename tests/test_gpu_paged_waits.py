"""The bounded waits of attn_paged under the smallest limit, one poll (about 4 us), while copies on another stream hold up its loads, so that
some of them run out: every launch returns, the status word says so (the outputs are undefined then), and the next ordinary call gives the
bits that it gave before."""
import pytest
import torch

from tests.test_gpu_paged import run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture()
def tb():
    import tokenrush_b200 as tb
    yield tb
    tb._lib.lib().trb_set_wait_limits(0, 0, 0)                          # defaults again
    tb._lib.lib().trb_set_paged_prefix_bytes(-1)
    tb._lib.device_status()


@pytest.mark.parametrize("way", [0, 1 << 60], ids=["prefix kernel", "scan"])
@pytest.mark.parametrize("case", [
    (1, [300, 20, 64, 700, 5], 3000, 24, 4, 256, True, 64),
    (1, [300, 20, 64, 700, 5] * 20, 30000, 24, 4, 256, True, 64),
    (1, [300, 20, 64, 700, 5] * 20, 30000, 24, 4, 256, False, 64),
    (5, [300, -1, 64, 700, 5], 3000, 32, 8, 128, True, 32),
    (5, [3000, 200, 64, 700, -1] * 10, 20000, 32, 8, 128, False, 64),
    (1, [60000], 0, 24, 4, 256, False, 16),
])
def test_waits_that_run_out(tb, case, way):
    lib = tb._lib.lib()
    lib.trb_set_paged_prefix_bytes(way)
    call, *_ = run_attention(tb, case)
    want = call()
    assert tb._lib.device_status() == 0
    a = torch.zeros(1 << 28, device="cuda", dtype=torch.uint8)
    b, other = torch.empty_like(a), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        assert lib.trb_set_wait_limits(1, 0, 0) == 0
        with torch.cuda.stream(other):
            for _ in range(8):
                b.copy_(a)
        for _ in range(5):
            call()
        torch.cuda.synchronize()                                        # the launches returned
        assert tb._lib.device_status() in (0, tb._lib.ST_WAIT_TIMEOUT)
        assert lib.trb_set_wait_limits(0, 0, 0) == 0
        assert torch.equal(call(), want) and tb._lib.device_status() == 0
