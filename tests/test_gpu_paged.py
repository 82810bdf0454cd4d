"""Batched path over a paged cache against plain implementations in 64 bits: paged_append, attn_paged, and a run of them with
spec_verify as a server would use them."""
import math

import numpy as np
import pytest
import torch

from oracle import kv_oracle as O
from tests._util import bits_of

pytestmark = pytest.mark.gpu

E32 = 2.0 ** -24                # half a step of fp32, of bf16
E16 = 2.0 ** -8


@pytest.fixture(scope="module")
def tb():
    import tokenrush_b200 as tb
    return tb


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def make_table(rows, page, seed, spare=3, most=None):
    """A shuffled page table for sequences of that many rows; entries behind a sequence's last page point outside the pool."""
    counts = [-(-max(r, 0) // page) for r in rows]
    pages = sum(counts) + spare
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((len(rows), most or max(1, max(counts))), -7, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        table[i, :c] = order[at:at + c]
        at += c
    return table, pages


def make_pool(pages, hkv, page, d, fp8, seed, poison=False):
    """A pool whose every row holds N(0, 1) values; poison: NaN and infinities instead (for rows that nobody may read)."""
    g = gen(seed)
    out = []
    for _ in range(2):
        x = torch.randn(pages, hkv, page, d, device="cuda", generator=g).bfloat16()
        if poison:
            x[..., 0::2], x[..., 1::2] = math.nan, math.inf
        if fp8:
            s = x.float().abs().amax(-1).clamp_min(1e-6) / 448
            c = (x.float() / s.unsqueeze(-1)).to(torch.float8_e4m3fn)
            out.append((c, s))
        else:
            out.append((x, None))
    (k, ks), (v, vs) = out
    return k, v, ks, vs


def rows_of(pool, scales, table, n, page):
    """Rows 0..n-1 of a table as float64 [hkv, n, d] on the CPU."""
    x = pool.cpu()
    parts = [x[int(t)].float().double() * (1.0 if scales is None else scales.cpu()[int(t)].double().unsqueeze(-1)) for t in table[:-(-n // page)]]
    return torch.cat(parts, 1)[:, :n] if parts else torch.zeros(pool.shape[1], 0, pool.shape[3], dtype=torch.float64)


def attend_ref(q, kp, vp, ko, vo, scale):
    """q [m, hq, d], keys [hkv, n, d]: (o, mean |v| under the weights, bound on a score's error), row i sees ko[: n - m + i + 1]."""
    m, hq, d = q.shape
    hkv = ko.shape[0]
    o, a, e = torch.zeros(m, hq, d, dtype=torch.float64), torch.zeros(m, hq, d, dtype=torch.float64), torch.zeros(m, hq, 1, dtype=torch.float64)
    for i in range(m):
        n = ko.shape[1] - m + i + 1
        for h in range(hq):
            j = h // (hq // hkv)
            k = torch.cat((kp[j], ko[j, :max(n, 0)]))
            v = torch.cat((vp[j], vo[j, :max(n, 0)]))
            if not len(k):
                continue
            s = (k @ q[i, h]) * scale
            w = torch.softmax(s, 0)
            o[i, h], a[i, h] = w @ v, w @ v.abs()
            # fp32 accumulation of d products (d roundings of the running sum), plus the f16 form of q: 2^-25 of its largest element
            e[i, h] = scale * ((k.abs() @ q[i, h].abs()).max() * d * E32 + d * 2.0 ** -25 * q[i, h].abs().max() * k.abs().max())
    return o, a, e


def check_attention(got, q, kp, vp, ko, vo, scale, what=""):
    """|got - o| <= half a bf16 step of o, + the weights' rounding to 8 bits (f16 weights have 11): each weight off by 2^-8 moves o by at
    most 2^-8 sum p |v - o| <= 2^-8 (a + |o|), + scores off by e: weights off by 2 e; 2^-20 for exp2 and the joins of partials."""
    o, a, e = attend_ref(q, kp, vp, ko, vo, scale)
    got = got.double().cpu()
    tol = E16 * o.abs() + (E16 + 2 * e + 2.0 ** -20) * (a + o.abs()) * (1 + E16)
    err = (got - o).abs()
    assert torch.isfinite(got).all(), what
    assert (err <= tol).all(), (what, float((err - tol).max()), float(err.max()))


# ------------------------------------------------------------------------------ append

def rotate_ref(x, pos, f, inter, amp):
    """(rotated, |a| + |b| of each element's pair) in float64."""
    rd = 2 * len(f)
    ang = pos.double().view(-1, 1, 1) * f
    c, s = ang.cos() * amp, ang.sin() * amp
    y, mag = x.clone(), x.abs()
    one, two = (slice(0, rd, 2), slice(1, rd, 2)) if inter else (slice(0, rd // 2), slice(rd // 2, rd))
    a, b = x[..., one], x[..., two]
    y[..., one], y[..., two] = a * c - b * s, b * c + a * s
    mag[..., one] = mag[..., two] = (a.abs() + b.abs()) * amp
    return y, mag


def norm_ref(x, w, eps=1e-6):
    return x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * (1 + w.double().cpu())


# relative to |a| + |b| of the pair: the sum of squares (13 roundings, halved by the root), root, two products: 10 * 2^-24; cos and sin: the
# fraction of a turn rounded to fp32 (2^-25 of half a turn = pi 2^-25), 2 ulp of sincospi, the amplitude, two products and a sum: 12 * 2^-24
TURN = 24 * E32

APPENDS = [
    # counts, starts, hq, hkv, d, rd, interleaved, norm, gated layout, fp8, page, base, lens type
    ([1], [0], 24, 4, 256, 64, False, True, True, True, 64, 0, torch.int64),
    ([1], [63], 24, 4, 256, 64, False, True, True, False, 64, 12345, torch.int32),
    ([1, 1, 1], [5, -1, 64], 8, 1, 256, 256, False, False, False, True, 64, 7, torch.int64),
    ([5, 0, 17, 1], [0, 3, 30, 15], 32, 8, 128, 128, True, False, False, False, 16, 1999999, torch.int64),
    ([33, 2], [100, 0], 16, 16, 128, 32, False, True, True, True, 32, 0, torch.int32),
    ([3, 40, 9], [1, 15, -1], 6, 2, 128, 2, True, True, False, True, 16, 0, torch.int64),
    ([7], [2], 4, 4, 256, 16, False, False, True, False, 128, 1 << 20, torch.int64),
    ([4, 4], [2, 9], 0, 4, 256, 0, False, True, False, True, 16, 0, torch.int64),
    ([300], [1000], 40, 8, 128, 64, True, True, False, True, 256, 0, torch.int64),
]


@pytest.mark.parametrize("case", APPENDS)
@pytest.mark.parametrize("device_base", [False, True])
def test_append(tb, case, device_base):
    counts, starts, hq, hkv, d, rd, inter, norm, gated, fp8, page, base, lens_t = case
    g, b, t = gen(11), len(counts), sum(counts)
    uniform = len(set(counts)) == 1
    pad = 0 if uniform else 2                                            # rows behind the last sequence
    table, pages = make_table([max(s, 0) + c for s, c in zip(starts, counts)], page, 3)
    k0, v0, ks0, vs0 = make_pool(pages, hkv, page, d, fp8, 4)
    k, v = k0.clone(), v0.clone()
    ks, vs = (ks0.clone(), vs0.clone()) if fp8 else (None, None)
    wide = hq * (2 if gated else 1)
    qkv = torch.randn(t + pad, (wide + 2 * hkv) * d, device="cuda", generator=g).mul_(3).bfloat16()
    qs = qkv[:, :wide * d].view(t + pad, hq, -1)[..., :d] if hq else None
    kx, vx = qkv[:, wide * d:(wide + hkv) * d].view(-1, hkv, d), qkv[:, (wide + hkv) * d:].view(-1, hkv, d)
    vx[0, 0] = 0                                                         # a zero row: the scale's floor
    qw, kw = ((torch.randn(d, device="cuda", generator=g) * 0.3).bfloat16() for _ in range(2)) if norm else (None, None)
    f, amp = tb.rope.frequencies(rd, 1e6, "yarn", 8.0, trained=4096) if rd else (None, 1.0)
    cu = None if uniform else torch.tensor(np.concatenate(([0], np.cumsum(counts))), dtype=torch.int32, device="cuda")
    lens = torch.tensor(starts, dtype=lens_t, device="cuda")
    out = tb.fused.paged_append(kx, vx, k, v, table.cuda(), lens, ks, vs, q=qs, cu=cu, base=torch.tensor([base], device="cuda") if device_base else base,
                                q_norm_w=qw, k_norm_w=kw, inv_freq=f, interleaved=inter, amplitude=amp)
    torch.cuda.synchronize()
    assert tb._lib.device_status() == 0
    assert lens.tolist() == starts
    # the plain form
    seq = np.repeat(np.arange(b), counts)
    row = torch.tensor([starts[s] + i for s, c in enumerate(counts) for i in range(c)])
    live = torch.tensor([starts[s] >= 0 for s in seq], dtype=torch.bool)
    freq = f.cpu() if rd else torch.zeros(0, dtype=torch.float64)
    if hq:
        want, mag = rotate_ref(norm_ref(qs[:t].cpu().double(), qw), row + base, freq, inter, amp)
        got = out[:t].double().cpu()
        assert ((got - want).abs() <= E16 * want.abs() + (1 + E16) * TURN * mag)[live].all()
        assert (got[~live] == 0).all() and (out[t:] == 0).all()
    else:
        assert out is None
    kw_ref, kmag = rotate_ref(norm_ref(kx[:t].cpu().double(), kw), row + base, freq, inter, amp)
    touched = torch.zeros(pages, page, dtype=torch.bool)
    for n in range(t):
        if not live[n]:
            continue
        pg, at = int(table[seq[n], int(row[n]) // page]), int(row[n]) % page
        touched[pg, at] = True
        if fp8:
            s = ks[pg, :, at].cpu().double()
            top = kw_ref[n].abs().amax(-1)
            slack = TURN * kmag[n].amax(-1)
            assert ((s - top.clamp_min(1e-6) / 448).abs() <= (slack + 2 * E32 * top) / 448).all()
            # half an e4m3 step of the value (2^-4), or of the smallest step (2^-10)
            err = (k[pg, :, at].cpu().float().double() * s.unsqueeze(-1) - kw_ref[n]).abs()
            assert (err <= 2.0 ** -4 * kw_ref[n].abs() + s.unsqueeze(-1) * 2.0 ** -10 + 2 * TURN * kmag[n]).all()
            codes, scales = O.quantize_rows(O.bf16_bits_to_f32(bits_of(vx[n].contiguous())))
            assert np.array_equal(v[pg, :, at].view(torch.uint8).cpu().numpy(), codes) and np.array_equal(vs[pg, :, at].cpu().numpy(), scales)
        else:
            assert ((k[pg, :, at].cpu().double() - kw_ref[n]).abs() <= E16 * kw_ref[n].abs() + (1 + E16) * TURN * kmag[n]).all()
            assert torch.equal(v[pg, :, at].cpu(), vx[n].cpu())
    rest = (~touched).cuda()
    for new, old in ((k, k0), (v, v0)):                                  # every other row as it was, bit for bit
        w = torch.uint8 if fp8 else torch.int16
        assert torch.equal(new.view(w).transpose(1, 2)[rest], old.view(w).transpose(1, 2)[rest])
    if fp8:
        assert torch.equal(ks.transpose(1, 2)[rest], ks0.transpose(1, 2)[rest]) and torch.equal(vs.transpose(1, 2)[rest], vs0.transpose(1, 2)[rest])


def test_append_outside_the_table_writes_nothing(tb):
    table = torch.tensor([[0, 1], [99, -1]], dtype=torch.int32, device="cuda")
    k, v, _, _ = make_pool(3, 2, 16, 128, False, 1)
    k0, v0 = k.clone(), v.clone()
    x = torch.randn(2, 2, 128, device="cuda").bfloat16()
    tb.fused.paged_append(x, x, k, v, table, torch.tensor([32, 3], device="cuda"))
    assert tb._lib.device_status() == tb._lib.ST_CURSOR_RANGE
    assert torch.equal(k, k0) and torch.equal(v, v0)


# ------------------------------------------------------------------------------ attention

ATTENDS = [
    # m, own rows (with the m new ones; -1: empty slot), prefix, hq, hkv, d, fp8, page
    (1, [1], 0, 24, 4, 256, True, 64),
    (1, [0 + 1, 17, 64, 65], 0, 24, 4, 256, True, 16),
    (1, [1, 2, 15, 16, 17, 700], 0, 24, 4, 256, False, 64),
    (1, [1], 1, 24, 4, 256, True, 64),
    (1, [5, -1, 130, 33], 129, 24, 4, 256, True, 64),
    (1, [5, 70, 130, 33, 1], 640, 24, 4, 256, False, 32),
    (1, [20, 300, 31], 1111, 32, 8, 128, True, 16),
    (1, [20, 300, 31], 1111, 32, 8, 128, False, 128),
    (1, [7, 100], 200, 8, 8, 128, True, 32),
    (1, [7, 100], 200, 16, 1, 256, False, 64),
    (2, [2, 50], 100, 24, 4, 256, True, 64),
    (5, [5, 77, -1, 260], 300, 24, 4, 256, True, 32),
    (8, [8, 9, 129], 77, 24, 4, 256, False, 16),
    (7, [7, 200], 0, 40, 8, 128, True, 64),
    (16, [16, 150], 65, 32, 4, 128, False, 64),
    (1, [3] * 40, 513, 24, 4, 256, True, 64),
    (3, [3 + 11 * i for i in range(30)], 900, 24, 4, 256, True, 64),
    (1, [1 + 13 * i for i in range(50)], 385, 40, 8, 128, False, 256),
]


def run_attention(tb, case, seed=5, peaked=False, gate=False, dev_prefix=False, lens_t=torch.int64):
    m, own, prefix, hq, hkv, d, fp8, page = case
    g, b = gen(seed), len(own)
    table, pages = make_table(own + [prefix], page, seed)
    k, v, ks, vs = make_pool(pages, hkv, page, d, fp8, seed + 1)
    bad = make_pool(pages, hkv, page, d, False, 0, poison=True)[0]
    # rows that nobody sees hold NaN and infinities
    seen = torch.zeros(pages, page, dtype=torch.bool)
    for i, n in enumerate(own + [prefix]):
        for r in range(max(n, 0)):
            seen[int(table[i, r // page]), r % page] = True
    hide = (~seen).cuda().unsqueeze(1).expand(pages, hkv, page)
    for x in (k, v):
        if fp8:
            x.view(torch.uint8)[hide] = 0x7f                             # the e4m3 NaN
        else:
            x[hide] = bad[hide]
    if fp8:
        ks[hide], vs[hide] = math.nan, math.inf
    q = torch.randn(b, m, hq, d, device="cuda", generator=g).mul_(6.0 if peaked else 1.5).bfloat16()
    lens = torch.tensor([n - m if n >= 0 else -1 for n in own], dtype=lens_t, device="cuda")
    gt = torch.randn(b * m, hq * 2 * d, device="cuda", generator=g).bfloat16().view(b, m, hq, 2 * d)[..., d:] if gate else None
    kw = {}
    if prefix:
        kw = dict(prefix_table=table[-1].cuda()[:-(-prefix // page)].contiguous(), prefix_len=torch.tensor([prefix], dtype=torch.int32, device="cuda") if dev_prefix else prefix)
    own_table = table[:b].cuda()
    call = lambda **x: tb.fused.attn_paged(q, k, v, own_table, lens, ks, vs, **kw, **x)      # noqa: E731
    return call, q, lens, gt, (k, v, ks, vs, table)


@pytest.fixture(params=[0, -1], ids=["prefix kernel", "scan"])
def prefix_bytes(request, tb):
    """A prefix read by its own kernel whatever its size, or (at these sizes) by the scan of every sequence."""
    tb._lib.lib().trb_set_paged_prefix_bytes(request.param)
    yield request.param
    tb._lib.lib().trb_set_paged_prefix_bytes(-1)


@pytest.mark.parametrize("case", ATTENDS)
@pytest.mark.parametrize("peaked", [False, True])
def test_attention(tb, case, peaked, prefix_bytes):
    m, own, prefix, hq, hkv, d, fp8, page = case
    call, q, lens, _, (k, v, ks, vs, table) = run_attention(tb, case, peaked=peaked, dev_prefix=peaked, lens_t=torch.int32 if peaked else torch.int64)
    got = call()
    torch.cuda.synchronize()
    assert tb._lib.device_status() == 0
    kp, vp = (rows_of(x, s, table[-1], prefix, page) for x, s in ((k, ks), (v, vs)))
    for i, n in enumerate(own):
        if n < 0:
            assert (got[i] == 0).all()
            continue
        ko, vo = (rows_of(x, s, table[i], n, page) for x, s in ((k, ks), (v, vs)))
        check_attention(got[i], q[i].double().cpu(), kp, vp, ko, vo, d ** -0.5, (i, n))
    assert torch.equal(call(), got)                                      # the same again, bit for bit


@pytest.mark.parametrize("hq,hkv,d,fp8", [(24, 4, 256, True), (24, 4, 256, False), (32, 8, 128, True), (16, 16, 128, False)])
def test_attention_long(tb, hq, hkv, d, fp8):
    """Hundreds of tiles per CTA, repeated (a wait that is missed shows as a timeout in the status word); 64 bits on the GPU."""
    b, prefix, page, g = 30, 20011, 64, gen(9)
    own = [1 + 173 * i % 2500 for i in range(b)]
    table, pages = make_table(own + [prefix], page, 8)
    k, v, ks, vs = make_pool(pages, hkv, page, d, fp8, 10)
    q = torch.randn(b, 1, hq, d, device="cuda", generator=g).mul_(2).bfloat16()
    own_table, pt = table[:b].cuda(), table[-1].cuda()
    lens = torch.tensor(own, device="cuda") - 1
    call = lambda: tb.fused.attn_paged(q, k, v, own_table, lens, ks, vs, prefix_table=pt, prefix_len=prefix)      # noqa: E731
    got = call()
    for _ in range(20):
        assert torch.equal(call(), got)
    assert tb._lib.device_status() == 0

    def rows(x, s, t, n, j):
        y = x[t[:-(-n // page)].long(), j].double() if not fp8 else x.view(torch.uint8)[t[:-(-n // page)].long(), j].view(x.dtype).double()
        y = y if s is None else y * s[t[:-(-n // page)].long(), j].double().unsqueeze(-1)
        return y.flatten(0, 1)[:n]
    for j in range(0, hkv, max(1, hkv - 1)):
        h = slice(j * hq // hkv, (j + 1) * hq // hkv)
        kp, vp = rows(k, ks, pt, prefix, j), rows(v, vs, pt, prefix, j)
        for i in range(0, b, 7):
            kk, vv = torch.cat((kp, rows(k, ks, own_table[i], own[i], j))), torch.cat((vp, rows(v, vs, own_table[i], own[i], j)))
            x = q[i, 0, h].double()
            w = torch.softmax(x @ kk.T * d ** -0.5, 1)
            o, a = w @ vv, w @ vv.abs()
            e = d ** -0.5 * ((x.abs() @ kk.abs().T).amax(1, keepdim=True) * d * E32)
            # as check_attention; e4m3 weights of the prefix kernel are off by at most 2^-18 of the row's largest weight where they are small
            floor = 2.0 ** -18 * w.amax(1, keepdim=True) * vv.abs().sum(0) if fp8 else 0.0
            assert ((got[i, 0, h].double() - o).abs() <= E16 * o.abs() + (E16 + 2 * e + 2.0 ** -20) * (a + o.abs()) * (1 + E16) + floor).all()


def test_attention_gate_and_out(tb, prefix_bytes):
    case = (2, [40, 3], 70, 24, 4, 256, True, 64)
    call, q, lens, gt, _ = run_attention(tb, case, gate=True)
    plain = call()
    out = torch.full_like(q, 9.0)
    assert call(gate=gt, out=out) is out
    want = plain.float() * torch.sigmoid(gt.float()).bfloat16().float()
    # the sigmoid's own fp32 error can move its rounding by one bf16 step (2^-7 relative), the product is rounded once
    assert ((out.float() - want).abs() <= (2 * E16 + E16 + 2.0 ** -16) * want.abs()).all()


def test_attention_scale_and_large_values(tb, prefix_bytes):
    """q far outside f16's range, and a scale that brings the scores back."""
    case = (1, [33, 2], 20, 24, 4, 256, True, 16)
    call, q, lens, _, (k, v, ks, vs, table) = run_attention(tb, case)
    want = call()
    q.mul_(2.0 ** 40)
    assert torch.equal(call(scale=256 ** -0.5 * 2.0 ** -40), want)


def test_attention_empty_rows(tb, prefix_bytes):
    """No prefix rows and no own rows: zeros, whatever the pages hold."""
    case = (2, [2, 18], 0, 24, 4, 256, False, 16)
    call, q, lens, _, _ = run_attention(tb, case)
    lens.fill_(-1)
    assert (call() == 0).all()
    assert tb._lib.device_status() == 0


def test_attention_reports_lengths_beyond_the_table(tb):
    case = (1, [16, 32], 16, 24, 4, 256, True, 16)
    call, q, lens, _, _ = run_attention(tb, case)
    lens[1] = 40
    call()
    assert tb._lib.device_status() == tb._lib.ST_CURSOR_RANGE


def test_absurd_lengths_read_and_write_nothing_outside(tb, prefix_bytes):
    case = (2, [16, 32, 20], 40, 24, 4, 256, True, 16)
    call, q, lens, _, (k, v, ks, vs, table) = run_attention(tb, case)
    kp, vp = (rows_of(y, z, table[-1], 40, 16) for y, z in ((k, ks), (v, vs)))
    k0 = k.clone()
    x = torch.zeros(6, 4, 256, device="cuda", dtype=torch.bfloat16)
    for n in (2 ** 63 - 1, 2 ** 62, 2 ** 31, 2 ** 31 - 1, -2 ** 63):
        lens[1] = n
        got = call()
        assert tb._lib.device_status() == (0 if n < 0 else tb._lib.ST_CURSOR_RANGE)
        for i, own in ((0, 16), (2, 20)):                                # (not the same bits: the cut of the line depends on every length)
            check_attention(got[i], q[i].double().cpu(), kp, vp, *(rows_of(y, z, table[i], own, 16) for y, z in ((k, ks), (v, vs))), 256 ** -0.5, (n, i))
        others = lens.clone()
        others[0] = others[2] = -1
        tb.fused.paged_append(x, x, k, v, table[:3].cuda(), others, ks, vs)
        tb._lib.device_status()
        assert torch.equal(k.view(torch.uint8), k0.view(torch.uint8))


def test_on_another_stream(tb, prefix_bytes):
    """Calls run on the current stream: their inputs are made there and their outputs are ready there."""
    case = (1, [300, 20, 64], 200, 24, 4, 256, False, 32)
    call, q, lens, _, _ = run_attention(tb, case)
    want = call()
    torch.cuda.synchronize()
    q0 = q.clone()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        for _ in range(5):
            q.zero_()
            torch.cuda._sleep(200000)
            q.copy_(q0)
            got = call() + 0
    s.synchronize()
    assert torch.equal(got, want)


def test_captured_attention_follows_the_lengths(tb, prefix_bytes):
    """One graph for all lengths, two graphs replayed on two streams at once, and the eager call beside them."""
    case = (2, [90, 300, 257], 400, 24, 4, 256, True, 64)
    call, q, lens, _, _ = run_attention(tb, case)
    call()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, out))
    for n in ([10, 200, 255], [-1, 0, 100], [88, 298, 255]):
        lens.copy_(torch.tensor(n))
        want = call()
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for (g, _), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for _ in range(20):
                    g.replay()
        beside = [call() for _ in range(10)]
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out, want)
        for out in beside:
            assert torch.equal(out, want)


def test_refusals_on_the_gpu(tb):
    case = (1, [5, 6], 10, 24, 4, 256, True, 16)
    call, q, lens, _, (k, v, ks, vs, table) = run_attention(tb, case)
    f, t = tb.fused, table[:2].cuda()
    for bad in (lambda: f.attn_paged(q[:1], k, v, t, lens, ks, vs), lambda: f.attn_paged(q.float(), k, v, t, lens, ks, vs),
                lambda: f.attn_paged(q, k, v, t, lens), lambda: f.attn_paged(q, k, v, t.long(), lens, ks, vs), lambda: f.attn_paged(q, k, v, t, lens.float(), ks, vs),
                lambda: f.attn_paged(q, k, v, t, lens, ks, vs, prefix_len=3), lambda: f.attn_paged(q, k[:, :, ::2], v[:, :, ::2], t, lens, ks, vs),
                lambda: f.attn_paged(q, k, v, t, lens, ks, vs, prefix_table=t[0], prefix_len=16 * t.shape[1] + 1),
                lambda: f.attn_paged(q[:, :, :22], k, v, t, lens, ks, vs), lambda: f.attn_paged(q.transpose(0, 1), k, v, t, lens, ks, vs)):
        with pytest.raises(ValueError):
            bad()
    x = torch.zeros(3, 4, 256, device="cuda", dtype=torch.bfloat16)
    for bad in (lambda: f.paged_append(x, x, k, v, t, lens, ks, vs), lambda: f.paged_append(x[:2], x[:1], k, v, t, lens, ks, vs),
                lambda: f.paged_append(x[:2].float(), x[:2], k, v, t, lens, ks, vs), lambda: f.paged_append(x[:2, :3], x[:2, :3], k, v, t, lens, ks, vs),
                lambda: f.paged_append(x[:2], x[:2], k, v, t, lens, ks, vs, inv_freq=torch.ones(32, device="cuda")),
                lambda: f.paged_append(x[:2], x[:2], k, v, t, lens, ks, vs, cu=torch.zeros(2, device="cuda", dtype=torch.int32))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(TypeError):
        f.attn_paged(q, k, v.view(torch.uint8), t, lens, ks, vs)
    assert f.paged_append(x[:0], x[:0], k, v, t, lens, ks, vs) is None


# ------------------------------------------------------------------------------ together

@pytest.mark.parametrize("kv", ["fp8", "bf16"])
def test_a_server_s_steps(tb, kv, prefix_bytes):
    """Shared prefix, prompts of unequal length, verify steps that advance the lengths on the device, a sequence that leaves and one that
    comes: attention after every step against 64-bit attention over the pool's rows."""
    cfg = tb.AttnConfig(n_attn=1)
    hq, hkv, d, m, page = cfg.n_heads, cfg.n_kv_heads, cfg.head_dim, 4, 32
    st = tb.PagedState(cfg, num_pages=64, max_seqs=4, max_pages=12, page_size=page, kv_dtype=torch.float8_e4m3fn if kv == "fp8" else torch.bfloat16, max_prefix_pages=8)
    pool, g = st.layer(0), gen(77)
    f, amp = tb.rope.frequencies(cfg.rotary_dim, cfg.rope_theta)
    rope = dict(inv_freq=f, amplitude=amp, eps=cfg.eps, q_norm_w=torch.zeros(d, device="cuda").bfloat16(), k_norm_w=torch.zeros(d, device="cuda").bfloat16())
    draw = lambda n: torch.randn(n, hq + 2 * hkv, d, device="cuda", generator=g).bfloat16()      # noqa: E731

    def append(rows, table, lens, base, cu=None):
        return tb.fused.paged_append(rows[:, hq:hq + hkv], rows[:, hq + hkv:], pool[0], pool[1], table, lens, pool[2], pool[3], q=rows[:, :hq], cu=cu, base=base, **rope)

    st.set_prefix(200)
    append(draw(200), st.prefix_table[None], torch.zeros(1, device="cuda", dtype=torch.long), 0)
    prompts = [50, 1, 0, 33]
    for i, n in enumerate(prompts):
        if n:
            st.open(i, n + m)
    cu = torch.tensor(np.concatenate(([0], np.cumsum(prompts))), dtype=torch.int32, device="cuda")
    append(draw(sum(prompts)), st.table, st.lens, st.prefix_len, cu)
    st.lens += torch.tensor(prompts, device="cuda")                      # slot 2: still empty (-1)
    kept = list(prompts)
    for step in range(6):
        if step == 3:
            st.close(0)
            st.open(2, m)
            kept[0], kept[2] = None, 0
        lens = st.lens.tolist()
        for i, n in enumerate(lens):
            if n >= 0:
                st.reserve(i, n + m)
        q = append(draw(4 * m), st.table, st.lens, st.prefix_len).view(4, m, hq, d)
        o = tb.fused.attn_paged(q, pool[0], pool[1], st.table, st.lens, pool[2], pool[3], prefix_table=st.prefix_table, prefix_len=st.prefix_len)
        p = torch.rand(4, m, 97, device="cuda", generator=g)
        p /= p.sum(-1, keepdim=True)
        drafts = torch.randint(0, 97, (4, m - 1), device="cuda", generator=g)
        live = torch.tensor([m - 1 if n >= 0 else -1 for n in lens], dtype=torch.int32, device="cuda")
        u = torch.rand(4, m, device="cuda", generator=g) * 0.02
        _, n_acc = tb.fused.spec_verify(p, drafts, u, n_drafts=live, lens=st.lens)
        torch.cuda.synchronize()
        assert tb._lib.device_status() == 0
        kp, vp = (rows_of(x, s, st.prefix_table.cpu(), 200, page) for x, s in ((pool[0], pool[2]), (pool[1], pool[3])))
        for i, n in enumerate(lens):
            if n < 0:
                assert (o[i] == 0).all() and int(st.lens[i]) == -1
                continue
            ko, vo = (rows_of(x, s, st.table[i].cpu(), n + m, page) for x, s in ((pool[0], pool[2]), (pool[1], pool[3])))
            check_attention(o[i], q[i].double().cpu(), kp, vp, ko, vo, d ** -0.5, (step, i))
            assert int(st.lens[i]) == n + int(n_acc[i]) + 1
