"""The gate of attn_paged as a view of the projection that q, k and v come from: one row per sequence, one sequence, several of both."""
import pytest
import torch

from tests.test_gpu_paged import run_attention

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tb():
    import tokenrush_b200 as tb
    return tb


def views(b, m, hq, hkv, d):
    """[B, M, HQ, D] views of [q | gate] of each head, in rows that hold k and v too."""
    g = torch.Generator(device="cuda").manual_seed(3)
    w = hq * 2 * d
    qkv = torch.randn(b * m, w + 2 * hkv * d, device="cuda", generator=g).bfloat16()
    yield qkv[:, :w].view(b, m, hq, 2 * d)[..., d:]
    yield qkv.view(b, m, -1)[..., :w].unflatten(-1, (hq, 2 * d))[..., d:]
    if m == 1:
        yield qkv[:, :w].unflatten(-1, (hq, 2 * d))[..., d:].unsqueeze(1)
        yield qkv[:, :w].unflatten(-1, (hq, 2 * d))[..., d:][:, None].expand(b, 1, hq, d)
    if b == 1:
        yield qkv[:, :w].unflatten(-1, (hq, 2 * d))[..., d:].unsqueeze(0)
        yield torch.randn(2, 7, hq, d, device="cuda", generator=g).bfloat16()[1:, 2:2 + m]


@pytest.mark.parametrize("b,m", [(3, 1), (1, 1), (1, 4), (3, 2)])
@pytest.mark.parametrize("hq,hkv,d,fp8", [(24, 4, 256, True), (32, 8, 128, False)])
def test_gate_views(tb, b, m, hq, hkv, d, fp8):
    call, q, lens, _, _ = run_attention(tb, (m, [m + 30 * i for i in range(b)], 40, hq, hkv, d, fp8, 16))
    n = 0
    for gate in views(b, m, hq, hkv, d):
        assert gate.shape == q.shape
        assert torch.equal(call(gate=gate), call(gate=gate.contiguous()))
        n += 1
    assert n >= 2 and tb._lib.device_status() == 0


def test_gates_that_cannot_be_served(tb):
    b, m, hq, d = 3, 2, 24, 256
    call, q, lens, _, _ = run_attention(tb, (m, [2, 30, 60], 40, hq, 4, d, True, 16))
    for bad in (torch.zeros(b, 2 * m, hq, d, device="cuda").bfloat16()[:, :m],          # rows not equally spaced
                torch.zeros(b, m, hq, 2 * d, device="cuda").bfloat16()[..., ::2], torch.zeros(b, m, hq, d, device="cuda"),
                torch.zeros(b, m, hq - 1, d, device="cuda").bfloat16()):
        with pytest.raises(ValueError):
            call(gate=bad)
