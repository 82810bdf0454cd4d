"""spec_verify against the definition in 64 bits on the CPU: tokens and counts have to be equal."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def tb():
    import tokenrush_b200 as tb
    return tb


def clean(x):
    return np.where((x > 0) & np.isfinite(x), x, 0.0)


def reference(p, drafts, u, q=None, n_drafts=None):
    p, u = p.double().cpu().numpy(), u.double().cpu().numpy()
    q = None if q is None else q.double().cpu().numpy()
    drafts = drafts.cpu().numpy()
    b, k = drafts.shape
    v = p.shape[2]
    tokens, counts = np.full((b, k + 1), -1, np.int64), np.zeros(b, np.int64)
    for i in range(b):
        nd = k if n_drafts is None else min(int(n_drafts[i]), k)
        if nd < 0:
            continue
        n = 0
        while n < nd:
            x = drafts[i, n]
            if not (0 <= x < v):
                break
            pv, qv = clean(p[i, n, x]), 1.0 if q is None else clean(q[i, n, x])
            if not u[i, n] * qv < pv:
                break
            n += 1
        w = clean(p[i, n])
        if n < nd:
            less = np.zeros(v)
            if q is not None:
                less = clean(q[i, n])
            elif 0 <= drafts[i, n] < v:
                less[drafts[i, n]] = np.inf
            left = np.maximum(w - less, 0)
            if left.sum() > 0:
                w = left
        c = np.cumsum(w)
        token = -1
        if c[-1] > 0:
            border = u[i, k] * c[-1]
            hit = np.nonzero(c > border)[0]
            token = hit[0] if len(hit) else np.nonzero(w)[0][-1]
            # sums in another order differ by at most v 2^-53 of the total: the inputs must not put a border that near
            near = np.abs(c - border)[w > 0].min()
            assert near > v * 2.0 ** -53 * c[-1] or c[-1] == c[np.nonzero(w)[0][0]], "choose other inputs"
        tokens[i, :n], tokens[i, n], counts[i] = drafts[i, :n], token, n
    return tokens, counts


def compare(tb, p, drafts, u, **kw):
    tokens, n = tb.fused.spec_verify(p, drafts, u, **kw)
    want_t, want_n = reference(p, drafts, u, kw.get("draft_probs"), kw.get("n_drafts"))
    assert np.array_equal(n.cpu().numpy(), want_n) and np.array_equal(tokens.cpu().numpy(), want_t)
    return tokens, n


def inputs(b, k, v, dtype, seed, sparse=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    p = torch.randn(b, k + 1, v, device="cuda", generator=g).mul_(3).softmax(-1)
    q = (p[:, :k] * 0.6 + 0.4 * torch.randn(b, k, v, device="cuda", generator=g).mul_(3).softmax(-1))
    if sparse:                                                           # what top-k leaves: most entries zero
        keep = torch.rand(b, k + 1, v, device="cuda", generator=g) < 0.02
        keep[..., v // 2] = True
        p = p * keep
    drafts = torch.multinomial(q.reshape(b * k, v), 1, generator=g).view(b, k) if k else torch.zeros(b, 0, device="cuda", dtype=torch.long)
    u = torch.rand(b, k + 1, device="cuda", generator=g)
    return p.to(dtype), drafts, u, q.to(dtype)


@pytest.mark.parametrize("v", [1, 2, 31, 128, 1000, 1025, 50021, 131072])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("certain", [False, True])
def test_verify(tb, v, dtype, certain):
    p, drafts, u, q = inputs(9, 3, v, dtype, v)
    compare(tb, p, drafts, u, draft_probs=None if certain else q)


@pytest.mark.parametrize("b,k", [(1, 0), (1, 1), (3, 7), (2, 33), (2, 64), (200, 2), (17, 5)])
def test_shapes(tb, b, k):
    p, drafts, u, q = inputs(b, k, 777, torch.float32, b * 100 + k, sparse=True)
    u[0, :k] *= 1e-3                                                     # long runs of accepted drafts
    compare(tb, p, drafts, u, draft_probs=q if k else None)


def test_strides_and_alignment(tb):
    """Rows of a wider buffer, rows that start off a 16-byte boundary, sequences interleaved."""
    p, drafts, u, q = inputs(4, 3, 1000, torch.float32, 8)
    wide = torch.zeros(4, 4, 1013, device="cuda")
    wide[..., 5:1005] = p
    compare(tb, wide[..., 5:1005], drafts, u, draft_probs=q)
    turned = p.transpose(0, 1).contiguous().transpose(0, 1)
    compare(tb, turned, drafts, u, draft_probs=q)
    compare(tb, p.half(), drafts, u, draft_probs=torch.cat((q, q), -1).half()[..., :1000])


def test_borders(tb):
    """Exactly representable sums: a number on a border takes the next token; tokens without mass are never drawn."""
    p = torch.zeros(7, 1, 4096, device="cuda")
    at = [7, 1000, 1001, 4000]
    p[:, 0, at] = 0.25
    # (0.5 - 2^-26 lies half-way between two fp32 numbers and is 0.5; 0.5 - 2^-25 is the number below)
    u = torch.tensor([[0.0], [0.25], [0.5 - 2.0 ** -26], [0.75], [1.0 - 2.0 ** -24], [1.0], [0.5 - 2.0 ** -25]], device="cuda")
    assert float(u[2]) == 0.5 and float(u[6]) < 0.5
    tokens, n = tb.fused.spec_verify(p, torch.zeros(7, 0, dtype=torch.long, device="cuda"), u)
    assert tokens.view(-1).tolist() == [7, 1000, 1001, 4000, 4000, 4000, 1000] and n.tolist() == [0] * 7
    # acceptance is strict, and its product exact (0.125 - 2^-28 is 0.125, as above)
    p = torch.full((3, 2, 8), 0.125, device="cuda")
    tokens, n = tb.fused.spec_verify(p, torch.zeros(3, 1, dtype=torch.long, device="cuda"),
                                     torch.tensor([[0.125, 0.0], [0.125 - 2.0 ** -28, 0.0], [0.125 - 2.0 ** -27, 0.0]], device="cuda"))
    assert n.tolist() == [0, 0, 1] and tokens.tolist() == [[1, -1], [1, -1], [0, 0]]


def test_rows_without_mass(tb):
    v = 300
    u = torch.full((4, 2), 0.5, device="cuda")
    drafts = torch.full((4, 1), 3, dtype=torch.long, device="cuda")
    p, q = torch.zeros(4, 2, v, device="cuda"), torch.zeros(4, 1, v, device="cuda")
    p[0, 0, 5] = 1.0; q[0, 0, 5] = 1.0                                   # the residual is empty: drawn from p
    p[1, 0, 3] = 1.0; q[1, 0, 3] = 1.0                                   # accepted, nothing behind it
    q[2, 0, 9] = 1.0                                                     # nothing at all
    p[3, 0] = float("nan"); p[3, 0, 8] = float("inf"); p[3, 0, 9] = -1.0; p[3, 0, 250] = 0.5; q[3, 0] = float("nan")
    tokens, n = tb.fused.spec_verify(p, drafts, u, draft_probs=q)
    assert tokens.tolist() == [[5, -1], [3, -1], [-1, -1], [250, -1]] and n.tolist() == [0, 1, 0, 0]


def test_drafts_outside_the_vocabulary_and_odd_numbers(tb):
    p, drafts, u, q = inputs(6, 3, 500, torch.float32, 3)
    drafts[0, 0], drafts[1, 1], drafts[2, 0] = 500, -1, 1 << 40
    u[:3, :3] = 0.0
    u[3, 0] = float("nan")
    compare(tb, p, drafts, u, draft_probs=q)
    compare(tb, p, drafts, u)


@pytest.mark.parametrize("width", [torch.int32, torch.int64])
def test_counts_and_lengths(tb, width):
    p, drafts, u, q = inputs(6, 4, 600, torch.bfloat16, 21)
    u[:, :4] *= 0.3
    n_drafts = torch.tensor([4, 0, -1, 2, 9, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor([10, 20, -1, 0, 7, -1], dtype=width, device="cuda")
    tokens, n = compare(tb, p, drafts, u, draft_probs=q, n_drafts=n_drafts, lens=lens)
    assert tokens[2].tolist() == [-1] * 5
    want = [10 + int(n[0]) + 1, 21, -1, int(n[3]) + 1, 7 + int(n[4]) + 1, -1]
    assert lens.tolist() == want


def test_greedy_agrees_with_spec_commit(tb):
    """One-hot targets: the same tokens, counts and positions as the greedy commit."""
    k, v = 5, 1000
    pred = torch.tensor([4, 900, 17, 17, 3, 8], device="cuda")
    for wrong in range(k + 1):
        drafts = pred[:k].clone()
        if wrong < k:
            drafts[wrong] = 5
        p = torch.nn.functional.one_hot(pred, v).float().unsqueeze(0)
        pos = torch.tensor([50], device="cuda")
        lens, n0, tok = pos.clone(), torch.zeros(1, dtype=torch.long, device="cuda"), torch.zeros(1, dtype=torch.long, device="cuda")
        tb.fused.spec_commit(pred, drafts, n0, tok, pos)
        tokens, n = tb.fused.spec_verify(p, drafts.unsqueeze(0), torch.full((1, k + 1), 0.7, device="cuda"), lens=lens)
        assert int(n) == int(n0) and int(tokens[0, int(n)]) == int(tok) and int(lens) == int(pos)


def test_capture_and_streams(tb):
    p, drafts, u, q = inputs(20, 3, 4099, torch.float32, 5)
    tb.fused.spec_verify(p, drafts, u, draft_probs=q)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        tokens, n = tb.fused.spec_verify(p, drafts, u, draft_probs=q)
    for seed in range(3):
        p2, d2, u2, q2 = inputs(20, 3, 4099, torch.float32, 50 + seed)
        for a, b in ((p, p2), (drafts, d2), (u, u2), (q, q2)):
            a.copy_(b)
        torch.cuda.synchronize()
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            g.replay()
            t2, n2 = tb.fused.spec_verify(p, drafts, u, draft_probs=q)
        torch.cuda.synchronize()
        want_t, want_n = reference(p, drafts, u, q)
        for a, b in ((tokens, n), (t2, n2)):
            assert np.array_equal(a.cpu().numpy(), want_t) and np.array_equal(b.cpu().numpy(), want_n)


def test_refusals(tb):
    p, drafts, u, q = inputs(2, 3, 64, torch.float32, 1)
    f = tb.fused.spec_verify
    for bad in (lambda: f(p.double(), drafts, u), lambda: f(p, drafts.int(), u), lambda: f(p, drafts, u[:, :3]), lambda: f(p, drafts, u.double()),
                lambda: f(p, drafts[:, :2], u), lambda: f(p, drafts, u, draft_probs=q.half()), lambda: f(p, drafts, u, draft_probs=p),
                lambda: f(p.transpose(1, 2), drafts, u), lambda: f(p, drafts, u, n_drafts=torch.zeros(2, device="cuda")),
                lambda: f(p, drafts, u, lens=torch.zeros(3, device="cuda", dtype=torch.long))):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        f(p, drafts.cpu(), u)
    tokens, n = f(p[:0], drafts[:0], u[:0])
    assert tokens.shape == (0, 4) and n.shape == (0,)
