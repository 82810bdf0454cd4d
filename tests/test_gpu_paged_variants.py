"""The variants of the batched kernels that only larger calls or odder geometries reach: the append with two tokens per CTA and four rounds of
heads, rotations of more than half a head, the verification with every cluster size, and the launch modes."""
import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests._util import bits_of
from tests.test_gpu_paged import E16, E32, TURN, make_pool, make_table, norm_ref, rotate_ref
from tests.test_gpu_verify import compare, inputs

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tb():
    import tokenrush_b200 as tb
    return tb


def check_append(tb, counts, starts, hq, hkv, d, rd, inter, norm, fp8, page, base, pad=0):
    """paged_append of sequences of unequal length against the plain form in 64 bits, with the bounds of test_append, all rows at once."""
    g, t = torch.Generator(device="cuda").manual_seed(sum(counts) + rd), sum(counts)
    table, pages = make_table([max(s, 0) + c for s, c in zip(starts, counts)], page, 3)
    k0, v0, ks0, vs0 = make_pool(pages, hkv, page, d, fp8, 4)
    k, v = k0.clone(), v0.clone()
    ks, vs = (ks0.clone(), vs0.clone()) if fp8 else (None, None)
    qkv = torch.randn(t + pad, (2 * hq + 2 * hkv) * d, device="cuda", generator=g).mul_(3).bfloat16()
    q = qkv[:, :2 * hq * d].view(t + pad, hq, 2 * d)[..., :d]
    kx, vx = qkv[:, 2 * hq * d:(2 * hq + hkv) * d].view(-1, hkv, d), qkv[:, (2 * hq + hkv) * d:].view(-1, hkv, d)
    qw, kw = ((torch.randn(d, device="cuda", generator=g) * 0.3).bfloat16() for _ in range(2)) if norm else (None, None)
    f, amp = tb.rope.frequencies(rd, 1e6, "yarn", 8.0, trained=4096)
    cu = torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device="cuda")
    lens = torch.tensor(starts, device="cuda")
    call = lambda: tb.fused.paged_append(kx, vx, k, v, table.cuda(), lens, ks, vs, q=q, cu=cu, base=base, q_norm_w=qw, k_norm_w=kw, inv_freq=f,     # noqa: E731
                                         interleaved=inter, amplitude=amp)
    out = call()
    kept = [x.clone() for x in (k, v, ks, vs) if x is not None]
    again = call()
    torch.cuda.synchronize()
    assert tb._lib.device_status() == 0
    same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))      # noqa: E731
    assert same(out, again) and all(same(a, b) for a, b in zip(kept, [x for x in (k, v, ks, vs) if x is not None]))
    seq = torch.tensor(np.repeat(np.arange(len(counts)), counts))
    row = torch.cat([torch.arange(c) + s for s, c in zip(starts, counts)])
    live = torch.tensor(starts)[seq] >= 0
    want, mag = rotate_ref(norm_ref(q[:t].cpu().double(), qw), row + base, f.cpu(), inter, amp)
    assert ((out[:t].double().cpu() - want).abs() <= E16 * want.abs() + (1 + E16) * TURN * mag)[live].all()
    assert (out[:t].cpu()[~live] == 0).all() and (out[t:] == 0).all()
    want, mag = rotate_ref(norm_ref(kx[:t].cpu().double(), kw), row + base, f.cpu(), inter, amp)
    want, mag, vl = want[live], mag[live], vx[:t].cpu()[live]
    pg, at = table[seq, (row // page).clamp_min(0)][live].long(), (row % page)[live]
    got = lambda x: x.cpu().view(torch.uint8)[pg, :, at].view(x.dtype) if x.dtype == torch.float8_e4m3fn else x.cpu()[pg, :, at]      # noqa: E731
    if fp8:
        s, top = got(ks).double(), want.abs().amax(-1)
        assert ((s - top.clamp_min(1e-6) / 448).abs() <= (TURN * mag.amax(-1) + 2 * E32 * top) / 448).all()
        err = (got(k).float().double() * s.unsqueeze(-1) - want).abs()
        assert (err <= 2.0 ** -4 * want.abs() + s.unsqueeze(-1) * 2.0 ** -10 + 2 * TURN * mag).all()
        codes, scales = O.quantize_rows(O.bf16_bits_to_f32(bits_of(vl.contiguous())))
        assert np.array_equal(got(v).view(torch.uint8).numpy(), codes) and np.array_equal(got(vs).numpy(), scales)
    else:
        assert ((got(k).double() - want).abs() <= E16 * want.abs() + (1 + E16) * TURN * mag).all()
        assert torch.equal(got(v), vl)
    rest = torch.ones(pages, page, dtype=torch.bool)
    rest[pg, at] = False
    for new, old in ((k, k0), (v, v0)):
        w = torch.uint8 if fp8 else torch.int16
        assert torch.equal(new.cpu().view(w).transpose(1, 2)[rest], old.cpu().view(w).transpose(1, 2)[rest])
    if fp8:
        assert all(torch.equal(a.cpu().transpose(1, 2)[rest], b.cpu().transpose(1, 2)[rest]) for a, b in ((ks, ks0), (vs, vs0)))


# two tokens per CTA: borders of sequences inside a CTA, an odd number of rows, empty slots, rows behind the last sequence; heads that fill the
# rounds (32 of 32, 56 of 64), leave some of a second block of them empty (56 = 32 + 24) or end inside a warp (36 = 32 + 4)
LARGE = [
    ([1, 1200, 3, 0, 1197, 1], [7, 0, -1, 5, 63, 2], 24, 4, 256, 64, False, True, True, 64, 0, 2),
    ([2500], [0], 24, 4, 256, 256, True, True, False, 64, 100000, 1),
    ([801, 799, 2, 799], [5, -1, 0, 31], 40, 8, 128, 128, False, True, True, 16, 1 << 20, 0),
    ([1] * 300 + [2100], [3 * i for i in range(300)] + [9], 32, 8, 128, 64, True, False, False, 32, 0, 3),
    ([600, 601], [1, 2], 40, 8, 256, 192, False, False, True, 128, 12345, 0),
    ([1300], [17], 20, 8, 256, 32, False, True, False, 16, 0, 1),
]


@pytest.mark.parametrize("case", LARGE)
def test_append_of_many_rows(tb, case):
    check_append(tb, *case)


@pytest.mark.parametrize("d,rd,inter", [(256, r, False) for r in (16, 112, 128, 144, 160, 192, 208, 240, 256)] + [(128, r, False) for r in (48, 64, 80, 96, 112, 128)] +
                         [(256, r, True) for r in (2, 126, 128, 130, 200, 254, 256)] + [(128, r, True) for r in (62, 64, 66, 100, 126)])
@pytest.mark.parametrize("fp8", [True, False])
def test_rotations_of_every_width(tb, d, rd, inter, fp8):
    check_append(tb, [3, 1, 20], [0, 40, 7], 6, 2, d, rd, inter, True, fp8, 16, 777, 1)


# 444 / n CTAs per row on 148 SMs: 1, 2, 3, 4, 5, 6, 7, 8
@pytest.mark.parametrize("b", [444, 222, 148, 111, 88, 74, 64, 63, 55])
@pytest.mark.parametrize("v", [4100, 20011])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verify_with_every_cluster_size(tb, b, v, dtype):
    p, drafts, u, q = inputs(b, 2, v, dtype, b + v)
    compare(tb, p, drafts, u, draft_probs=q)
    compare(tb, p, drafts, u)


@pytest.fixture()
def launch_mode(tb):
    yield tb.fused.set_launch_mode
    tb.fused.set_launch_mode(1)
    tb._lib.lib().trb_set_paged_prefix_bytes(-1)


@pytest.mark.parametrize("way", [0, 1 << 60], ids=["prefix kernel", "scan"])
def test_launch_modes_give_the_same_bits(tb, launch_mode, way):
    """A step of append, attention and verification three times over, ordinary, dependent and chained, beside contiguous appends and decodes."""
    hq, hkv, d, m, b, page = 24, 4, 256, 3, 9, 32
    cfg = tb.AttnConfig(n_attn=1)
    f, amp = tb.rope.frequencies(cfg.rotary_dim, cfg.rope_theta)
    tb._lib.lib().trb_set_paged_prefix_bytes(way)
    table, pages = make_table([60 + 40 * i for i in range(b)] + [1000], page, 3)
    k0, v0, ks0, vs0 = make_pool(pages, hkv, page, d, True, 4)
    g = torch.Generator(device="cuda").manual_seed(9)
    x = torch.randn(3, b * m, hq + 2 * hkv, d, device="cuda", generator=g).bfloat16()
    p = torch.rand(3, b, m, 500, device="cuda", generator=g)
    drafts, u = torch.randint(0, 500, (b, m - 1), device="cuda", generator=g), torch.rand(b, m, device="cuda", generator=g)
    own, pt, one = table[:b].cuda(), table[-1].cuda()[:32].contiguous(), torch.tensor([5], device="cuda")
    results = []
    for mode in (0, 1, 2):
        launch_mode(mode)
        for _ in range(2):
            k, v, ks, vs = (y.clone() for y in (k0, v0, ks0, vs0))
            st = tb.State(cfg, 64, "cuda", kv_dtype=torch.float8_e4m3fn)
            lens = torch.arange(b, device="cuda") * 40 + 10
            out = []
            torch.cuda.synchronize()
            for i in range(3):
                q = tb.fused.paged_append(x[i, :, hq:hq + hkv], x[i, :, hq + hkv:], k, v, own, lens, ks, vs, q=x[i, :, :hq], base=1000, inv_freq=f, amplitude=amp)
                out.append(tb.fused.attn_paged(q.view(b, m, hq, d), k, v, own, lens, ks, vs, prefix_table=pt, prefix_len=1000))
                tb.fused.kv_append(x[i, :1, :hkv].transpose(0, 1), x[i, :1, hkv:2 * hkv].transpose(0, 1), st.k[0], st.v[0], one, st.k_scale[0], st.v_scale[0])
                out.append(tb.fused.attn_decode_fused(q[:1].view(1, -1), None, st.k[0], st.v[0], one, cfg, st.k_scale[0], st.v_scale[0]))
                out += list(tb.fused.spec_verify(p[i], drafts, u, lens=lens))
            torch.cuda.synchronize()
            assert tb._lib.device_status() == 0
            results.append(out + [k.view(torch.uint8), v.view(torch.uint8), ks, vs, lens])
    for n, other in enumerate(results[1:], 1):
        for i, (a, c) in enumerate(zip(results[0], other)):
            # (a chained decode takes its new row from the append's source, as a partial of its own: its bits are not compared)
            assert torch.equal(a, c) or (i < 12 and i % 4 == 1), (n, i)
