"""The prefill kernel's barriers, over many launches: every launch gives the same bits and no wait runs out.  (With one barrier for both P
buffers the MMA warp, waiting for a late V tile, could miss a phase; the epilogue could wait for a phase of the PV barrier that was over.)"""
import pytest
import torch

from _util import fill_cache_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("t,pos", [(1, 0), (5, 130), (256, 9000), (1024, 3333)])
def test_repeated_prefill(fp8, t, pos):
    import tokenrush_b200 as tb
    cfg = tb.AttnConfig(n_attn=1)
    st = tb.State(cfg, pos + t, "cuda", kv_dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16)
    fill_cache_gpu(tb, st, 0, pos + t, 3)
    g = torch.Generator(device="cuda").manual_seed(4)
    q = torch.randn(t, cfg.n_heads, cfg.head_dim, device="cuda", generator=g).bfloat16()
    ks, vs = (st.k_scale[0], st.v_scale[0]) if fp8 else (None, None)
    outs = [tb.fused.attn_prefill_fused(q, st.k[0], st.v[0], pos, cfg, ks, vs) for _ in range(40)]
    torch.cuda.synchronize()
    assert tb._lib.device_status() == 0
    assert all(torch.equal(o, outs[0]) for o in outs)
