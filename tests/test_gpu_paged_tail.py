"""attn_paged over a long prefix whose mass lies mostly in many small weights: a sink far above a flat or uneven tail.  Both ways of reading
the prefix against 64 bits, with a tolerance that does not grow with the number of keys."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E16 = 2.0 ** -8                 # half a step of bf16
N, PAGE = 65536, 64


@pytest.fixture(scope="module")
def tb():
    import tokenrush_b200 as tb
    return tb


@pytest.fixture(params=[0, 1 << 60], ids=["prefix kernel", "scan"])
def prefix_bytes(request, tb):
    tb._lib.lib().trb_set_paged_prefix_bytes(request.param)
    yield request.param
    tb._lib.lib().trb_set_paged_prefix_bytes(-1)


def pool(d, hkv, scores, fp8, g, bare=None):
    """N prefix rows and one own page; row i's score with the query 1, 0, 0, .. is scores[i] (natural log units); V of nonzero mean,
    the scales of V spread over a factor of four; V of row `bare` has one dim."""
    pages = N // PAGE + 1
    k = torch.zeros(pages * PAGE, d, device="cuda", dtype=torch.float64)
    k[:N, 0] = scores * math.sqrt(d)
    k[N:, 0] = scores.median() * math.sqrt(d)
    v = 1 + 0.25 * torch.randn(pages * PAGE, d, device="cuda", generator=g, dtype=torch.float64)
    v *= torch.exp2(2 * torch.rand(pages * PAGE, 1, device="cuda", generator=g, dtype=torch.float64) - 1)
    if bare is not None:
        v[bare, 1:] = 0
    out = []
    for x in (k, v):
        if fp8:
            s = x.abs().amax(-1).clamp_min(1e-6).float() / 448
            c = (x / s.double().unsqueeze(-1)).float().to(torch.float8_e4m3fn)
            real = c.double() * s.double().unsqueeze(-1)
        else:
            c, s = x.bfloat16(), None
            real = c.double()
        # every kv head holds the same rows
        shape = lambda y, *t: y.view(pages, 1, PAGE, *t).expand(pages, hkv, PAGE, *t).contiguous()      # noqa: E731
        c = shape(c.view(torch.uint8), d).view(torch.float8_e4m3fn) if fp8 else shape(c, d)
        out.append((c, None if s is None else shape(s), real))
    return out


TAILS = {
    # bits below the sink
    "flat 17.5": lambda g: torch.full((N,), 17.5, device="cuda", dtype=torch.float64),
    "flat 18.5": lambda g: torch.full((N,), 18.5, device="cuda", dtype=torch.float64),
    "flat 19.7": lambda g: torch.full((N,), 19.7, device="cuda", dtype=torch.float64),
    "flat 22.6": lambda g: torch.full((N,), 22.6, device="cuda", dtype=torch.float64),
    "uneven": lambda g: 18.5 + 2 * torch.randn(N, device="cuda", generator=g, dtype=torch.float64),
    # in every run of 128 keys one stands out above the others
    "ridges": lambda g: torch.where(torch.arange(N, device="cuda") % 128 == 77, 8.0, 18.5 + torch.rand(N, device="cuda", generator=g, dtype=torch.float64)),
    # falls slowly through the whole range
    "slope": lambda g: 30.0 * torch.arange(N, device="cuda", dtype=torch.float64) / N,
    "climb": lambda g: 30.0 - 30.0 * torch.arange(N, device="cuda", dtype=torch.float64) / N,
    # a few keys, then nothing near them
    "far": lambda g: torch.full((N,), 60.0, device="cuda", dtype=torch.float64),
}


def weight_error(w, v, vs, own_kernel):
    """What weights over an e4m3 pool may be off by beyond 8 bits, weights with the scale of V in them.  Prefix kernel: half of 2^-17 of a reference
    that lies at most 2 bits above the tile's largest weight.  Scan: half of f16's smallest step, 2^-25 of the largest weight."""
    ws, c = w * vs, v.abs() / vs.unsqueeze(-1)
    if not own_kernel:
        return 2.0 ** -25 * ws.amax() * c.sum(0)
    n = len(w) // 128 * 128
    tiles = 2.0 ** -16 * (ws[:n].view(-1, 128).amax(1, keepdim=True) * c[:n].view(n // 128, 128, -1).sum(1)).sum(0)
    return tiles + (2.0 ** -16 * ws[n:].amax() * c[n:].sum(0) if n < len(w) else 0)


# many query rows: a piece of the prefix kernel then goes over all keys, and a warp of the scan over a quarter of them
@pytest.mark.parametrize("b,m,hq,hkv,d,fp8", [(38, 21, 24, 4, 256, True), (19, 32, 32, 8, 128, True), (3, 1, 24, 4, 256, True), (38, 21, 24, 4, 256, False)])
@pytest.mark.parametrize("sink,sink_v", [(0, "alike"), (40000, "alike"), (N - 1, "alike"), (0, "one dim"), (40000, "one dim")])
@pytest.mark.parametrize("tail", TAILS)
def test_sink_and_tail(tb, b, m, hq, hkv, d, fp8, sink, sink_v, tail, prefix_bytes):
    g = torch.Generator(device="cuda").manual_seed(5)
    scores = -TAILS[tail](g) * math.log(2.0)
    scores[sink] = 0.0
    (k, ks, kr), (v, vs, vr) = pool(d, hkv, scores, fp8, g, sink if sink_v == "one dim" else None)
    q = torch.zeros(b, m, hq, d, device="cuda", dtype=torch.bfloat16)
    some = [1.0, 0.9375, 1.0625]                                         # (the last two: tails a little nearer, a little farther)
    q[..., 0] = torch.tensor(some, device="cuda")[torch.arange(b, device="cuda") % 3].view(b, 1, 1)
    order = torch.randperm(N // PAGE + 1, generator=torch.Generator().manual_seed(3))
    at = torch.empty_like(order)
    at[order] = torch.arange(len(order))                                 # page i of the plain order lies at at[i]
    move = lambda x: None if x is None else (x.view(torch.uint8)[order.cuda()].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x[order.cuda()])      # noqa: E731
    table = at.to(torch.int32).cuda()
    own = table[-1:].view(1, 1).expand(b, 1).contiguous()
    lens = torch.zeros(b, dtype=torch.long, device="cuda")
    got = tb.fused.attn_paged(q, move(k), move(v), own, lens, move(ks), move(vs), prefix_table=table[:-1].contiguous(), prefix_len=N)
    torch.cuda.synchronize()
    assert tb._lib.device_status() == 0
    for x in range(3):
        for i in sorted({0, m - 1}):
            n = N + i + 1
            w = torch.softmax(kr[:n, 0] * some[x] / math.sqrt(d), 0)
            o, a = w @ vr[:n], w @ vr[:n].abs()
            # half a bf16 step of o; weights rounded to 8 bits: 2^-8 (a + |o|); scores of up to 60 bits in fp32 with five roundings,
            # 2 * 60 ln 2 * 5 * 2^-24; 2^-20 for exp2 and the joins
            tol = E16 * o.abs() + (E16 + 600 * math.log(2.0) * 2.0 ** -24 + 2.0 ** -20) * (a + o.abs()) * (1 + E16)
            if fp8 and sink_v == "one dim":                              # (elsewhere the strict bound has to hold as it is)
                tol += weight_error(w, vr[:n], vs[:, 0].flatten()[:n].double(), prefix_bytes == 0)
            err = (got[x::3, i].double() - o).abs()
            assert (err <= tol).all(), (x, i, float((err / a).max()), float((err / tol).max()))
