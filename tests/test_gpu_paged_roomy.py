"""A prefix table with room for more rows than the prefix has: how the prefix is read goes by its rows where the host knows them."""
import pytest
import torch

from tests.test_gpu_paged import check_attention, make_pool, make_table, rows_of

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tb():
    import tokenrush_b200 as tb
    return tb


@pytest.mark.parametrize("rows,kernels", [(0, 2), (50, 2), (1024, 2), (8192, 3)])
def test_a_short_prefix_in_a_long_table(tb, rows, kernels):
    """16 sequences, 128 pages of 64: 272 MB of scans over 8192 rows, 34 MB over 1024."""
    b, hq, hkv, d, page = 16, 24, 4, 256, 64
    own = [1 + 9 * i for i in range(b)]
    table, pages = make_table(own + [8192], page, 2)
    k, v, ks, vs = make_pool(pages, hkv, page, d, True, 3)
    q = torch.randn(b, 1, hq, d, device="cuda", generator=torch.Generator(device="cuda").manual_seed(4)).bfloat16()
    own_table, pt, lens = table[:b, :3].contiguous().cuda(), table[-1].cuda(), torch.tensor(own, device="cuda") - 1
    lib = tb._lib.lib()
    call = lambda t, n: tb.fused.attn_paged(q, k, v, own_table, lens, ks, vs, prefix_table=t, prefix_len=n)      # noqa: E731
    at = lib.trb_launch_count()
    got = call(pt, rows)
    assert lib.trb_launch_count() - at == kernels
    assert torch.equal(got, call(pt[:-(-rows // page)], rows))           # the same as with the pages in use alone
    at = lib.trb_launch_count()
    device = call(pt, torch.tensor([rows], device="cuda"))              # the host knows the room alone
    assert lib.trb_launch_count() - at == 3
    assert tb._lib.device_status() == 0
    kp, vp = (rows_of(x, s, table[-1], rows, page) for x, s in ((k, ks), (v, vs)))
    for i in (0, 15):
        ko, vo = (rows_of(x, s, table[i], own[i], page) for x, s in ((k, ks), (v, vs)))
        for o in (got, device):
            check_attention(o[i], q[i].double().cpu(), kp, vp, ko, vo, d ** -0.5, (rows, i))
