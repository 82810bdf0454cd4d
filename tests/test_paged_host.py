"""CPU-side checks of the batched path: the page bookkeeping, the rotation frequencies, and the refusals of the entry
points that need no GPU."""
import ctypes as C
import math

import pytest
import torch

from tokenrush_b200 import PagedState, _lib as L, fused, rope


class Cfg:
    n_kv_heads, head_dim, attn_layers = 2, 128, (3, 7)


@pytest.fixture(scope="module")
def lib():
    from tokenrush_b200 import build
    build.build()
    return L.lib()


def state(**kw):
    return PagedState(Cfg, num_pages=10, max_seqs=3, max_pages=4, page_size=16, device="cpu", max_prefix_pages=3, **kw)


def test_pages_are_handed_out_once_and_come_back():
    st = state(kv_dtype=torch.float8_e4m3fn)
    assert st.k.shape == (2, 10, 2, 16, 128) and st.layer(1)[2].shape == (10, 2, 16)
    st.set_prefix(17)                                   # two pages
    st.open(0, 1)
    st.open(2)
    st.reserve(0, 33)
    st.reserve(2, 64)
    used = st.prefix_table[:2].tolist() + st.table[0, :3].tolist() + st.table[2, :4].tolist()
    assert len(set(used)) == 9 and st.free_pages == 1
    assert st.lens.tolist() == [0, -1, 0] and int(st.prefix_len) == 17
    st.reserve(0, 20)                                   # already there
    assert st.free_pages == 1
    st.open(1, 16)
    with pytest.raises(RuntimeError):
        st.reserve(1, 17)                               # the pool is full
    st.close(2)
    assert st.free_pages == 4 and st.lens.tolist() == [0, 0, -1]
    st.reserve(1, 17)


def test_page_bookkeeping_refuses():
    st = state()
    with pytest.raises(ValueError):
        st.open(0, 65)                                  # beyond the table
    st.open(0, 1)
    for call in (lambda: st.open(0), lambda: st.close(1), lambda: st.reserve(1, 1), lambda: st.set_prefix(1)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(ValueError):
        PagedState(Cfg, 4, 2, 2, page_size=24, device="cpu")
    assert st.free_pages == 9                           # the refused calls took nothing


def test_frequencies():
    f, a = rope.frequencies(64, 1e7, device="cpu")
    assert f.dtype == torch.float64 and a == 1.0 and f[0] == 1.0 and abs(float(f[-1]) - 1e7 ** (-62 / 64)) < 1e-20
    assert torch.equal(rope.frequencies(64, 1e7, "linear", 4.0, device="cpu")[0], f / 4)
    n, _ = rope.frequencies(64, 1e7, "ntk", 4.0, device="cpu")
    assert n[0] == 1.0 and abs(float(n[-1] * 4 / f[-1]) - 1) < 1e-12        # the slowest pair stretched by the factor
    y, a = rope.frequencies(64, 1e4, "yarn", 8.0, trained=4096, device="cpu")
    g, _ = rope.frequencies(64, 1e4, device="cpu")
    turns = 4096 * g / (2 * math.pi)
    assert torch.equal(y[turns > 40], g[turns > 40]) and torch.allclose(y[turns < 0.8], g[turns < 0.8] / 8, rtol=1e-15)
    assert ((y <= g) & (y >= g / 8)).all() and abs(a - (0.1 * math.log(8) + 1)) < 1e-15
    for bad in (dict(rotary_dim=7, theta=1e4), dict(rotary_dim=8, theta=1e4, scaling="other"), dict(rotary_dim=8, theta=1e4, factor=0.5),
                dict(rotary_dim=2, theta=1e4, scaling="ntk", factor=2.0)):
        with pytest.raises(ValueError):
            rope.frequencies(device="cpu", **bad)


def test_wrappers_refuse_cpu_tensors():
    st = state()
    k = torch.zeros(3, 2, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError):
        fused.paged_append(k, k, *st.layer(0)[:2], st.table, st.lens)
    with pytest.raises(RuntimeError):
        fused.attn_paged(k.view(3, 1, 2, 128), *st.layer(0)[:2], st.table, st.lens)
    with pytest.raises(RuntimeError):
        fused.spec_verify(torch.zeros(1, 2, 8), torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1, 2))


X = 4096          # an address that is never read: every call below is refused before anything is launched


def pool(**kw):
    f = dict(k=X, v=X, k_scale=X, v_scale=X, hkv=4, d=256, kv_dtype=1, page_size=64, num_pages=8)
    f.update(kw)
    return L.Paged(**f)


def batch(**kw):
    f = dict(table=X, table_stride=4, lens=X, lens_width=8, n_seqs=2, table_pages=4, reserved=0)
    f.update(kw)
    return L.Batch(**f)


BAD_POOLS = [(dict(k=None), -1), (dict(d=96), -5), (dict(d=64), -5), (dict(page_size=48), -5), (dict(page_size=8), -5), (dict(num_pages=0), -1),
             (dict(k_scale=None), -1), (dict(kv_dtype=2), -1), (dict(v=X + 8), -2), (dict(hkv=65), -5), (dict(num_pages=1 << 31), -5),
             (dict(page_size=1 << 17), -5), (dict(v_scale=X + 2), -2)]
BAD_BATCHES = [(dict(table=None), -1), (dict(lens=None), -1), (dict(lens_width=2), -1), (dict(n_seqs=0), -1), (dict(n_seqs=1025), -5),
               (dict(table_stride=3), -1), (dict(table_pages=0), -1), (dict(lens=X + 4), -2), (dict(table=X + 2), -2)]


def append(lib, p, b, **kw):
    f = dict(q=X, k=X, v=X, q_out=X, q_row_stride=6144, q_head_stride=256, k_row_stride=1024, k_head_stride=256, v_row_stride=1024,
             v_head_stride=256, inv_freq=X, n_rows=2, rows_per_seq=1, hq=24, rotary_dim=64, eps=1e-6, amplitude=1.0, base=L.Cursor(None, 8, 0, 0))
    f.update(kw)
    return lib.trb_paged_append(C.byref(p), C.byref(b), C.byref(L.PagedAppendArgs(**f)), None)


def attend(lib, p, b, **kw):
    f = dict(q=X, out=X, m=1, hq=24, scale=1.0, workspace=X, workspace_bytes=1 << 40, prefix_len=L.Cursor(None, 8, 0, 0))
    f.update(kw)
    return lib.trb_attn_paged(C.byref(p), C.byref(b), C.byref(L.AttnPagedArgs(**f)), None)


@pytest.mark.parametrize("bad,code", BAD_POOLS)
def test_bad_pools(lib, bad, code):
    assert append(lib, pool(**bad), batch()) == code
    assert attend(lib, pool(**bad), batch()) == code
    assert lib.trb_attn_paged_workspace_bytes(C.byref(pool(**bad)), 2, 1, 24, 0) == 0


@pytest.mark.parametrize("bad,code", BAD_BATCHES)
def test_bad_batches(lib, bad, code):
    assert append(lib, pool(), batch(**bad)) == code
    assert attend(lib, pool(), batch(**bad)) == code


@pytest.mark.parametrize("bad,code", [
    (dict(k=None), -1), (dict(q_out=None), -1), (dict(hq=0), -1), (dict(n_rows=-1), -1), (dict(n_rows=3), -1), (dict(rows_per_seq=0), -1),
    (dict(rotary_dim=7), -5), (dict(rotary_dim=258), -5), (dict(rotary_dim=24), -5), (dict(inv_freq=None), -1), (dict(k=X + 2), -2),
    (dict(k_row_stride=1020), -2), (dict(cu=X + 1), -2), (dict(q_norm_w=X + 8), -2), (dict(base=L.Cursor(X, 3, 0, 0)), -1),
    (dict(base=L.Cursor(X + 4, 8, 0, 0)), -2)])
def test_append_refuses(lib, bad, code):
    assert append(lib, pool(), batch(), **bad) == code


def test_append_of_nothing(lib):
    assert append(lib, pool(), batch(), n_rows=0, cu=X) == 0


@pytest.mark.parametrize("bad,code", [
    (dict(q=None), -1), (dict(out=None), -1), (dict(workspace=None), -1), (dict(workspace_bytes=16), -3), (dict(m=0), -1), (dict(hq=22), -1),
    (dict(hq=0), -1), (dict(m=22), -5), (dict(prefix_pages=1), -1), (dict(prefix_pages=-1), -1), (dict(q=X + 8), -2), (dict(workspace=X + 64), -2),
    (dict(prefix_pages=1, prefix_table=X, prefix_len=L.Cursor(X, 5, 0, 0)), -1), (dict(prefix_pages=1 << 26, prefix_table=X), -5)])
def test_attention_refuses(lib, bad, code):
    assert attend(lib, pool(), batch(), **bad) == code


def test_attention_refuses_more_rows_than_it_counts(lib):
    assert attend(lib, pool(), batch(n_seqs=1024, table_pages=1 << 20, table_stride=1 << 20)) == -5


@pytest.mark.parametrize("bad,code", [
    (dict(probs=None), -1), (dict(drafts=None), -1), (dict(u=None), -1), (dict(tokens=None), -1), (dict(n_seqs=0), -1), (dict(vocab=0), -1),
    (dict(k=-1), -1), (dict(k=65), -5), (dict(dtype=3), -1), (dict(lens=X, lens_width=2), -1), (dict(probs=X + 2), -2), (dict(drafts=X + 4), -2),
    (dict(lens=X + 4, lens_width=8), -2)])
def test_verify_refuses(lib, bad, code):
    f = dict(probs=X, draft_probs=X, probs_seq_stride=32, probs_row_stride=8, draft_seq_stride=24, draft_row_stride=8, drafts=X, u=X, tokens=X,
             n_accepted=X, n_seqs=2, k=3, vocab=8, dtype=0)
    f.update(bad)
    assert lib.trb_spec_verify(C.byref(L.SpecVerifyArgs(**f)), None) == code
