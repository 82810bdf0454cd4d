"""PagedState's tables name only pages that a sequence or the prefix holds: a step past the reservation is reported, it writes nothing."""
import pytest
import torch

from tokenrush_b200 import PagedState


class Cfg:
    n_kv_heads, head_dim, attn_layers = 2, 128, (3,)


def state(device):
    return PagedState(Cfg, num_pages=10, max_seqs=3, max_pages=4, page_size=16, device=device, max_prefix_pages=3)


def holds(st):
    """The tables hold each page in use once, in order, and -1 elsewhere."""
    used = []
    for row, pages in list(zip(st.table.tolist(), st._own)) + ([(st.prefix_table.tolist(), st._prefix)]):
        pages = pages or []
        assert row == pages + [-1] * (len(row) - len(pages))
        used += pages
    assert len(set(used)) == len(used) and not set(used) & set(st._free) and len(used) + st.free_pages == 10


def test_tables_follow_the_pages():
    st = state("cpu")
    holds(st)
    st.set_prefix(40)
    st.open(0, 48)
    st.open(1, 16)
    holds(st)
    st.close(0)
    st.open(2, 32)
    st.open(0, 16)                                      # (fewer pages than the slot had before)
    holds(st)
    st.reserve(0, 33)
    holds(st)
    for i in range(3):
        st.close(i)
    st.set_prefix(16)
    holds(st)
    st.set_prefix(0)
    holds(st)


@pytest.mark.gpu
def test_a_step_past_the_reservation_is_reported_and_writes_nothing():
    import tokenrush_b200 as tb
    st = state("cuda")
    k, v, _, _ = st.layer(0)
    g = torch.Generator(device="cuda").manual_seed(1)
    for x in (k, v):
        x.copy_(torch.randn(x.shape, device="cuda", generator=g))
    st.set_prefix(16)
    st.open(0, 48)
    st.open(1, 16)
    st.close(0)
    st.open(2, 32)
    st.open(0, 16)
    before = [x.clone() for x in (k, v)]
    st.lens[0], st.lens[1], st.lens[2] = 15, -1, -1
    rows = torch.randn(6, 2, 128, device="cuda", generator=g).bfloat16()      # rows 15 and 16 of slot 0: the second has no page
    tb.fused.paged_append(rows, rows, k, v, st.table, st.lens)
    assert tb._lib.device_status() == tb._lib.ST_CURSOR_RANGE
    mine = int(st.table[0, 0])
    for new, old, src in ((k, before[0], rows), (v, before[1], rows)):
        assert torch.equal(new[mine, :, 15], src[0])
        keep = torch.ones(10, 16, dtype=torch.bool, device="cuda")
        keep[mine, 15] = False
        assert torch.equal(new.transpose(1, 2)[keep], old.transpose(1, 2)[keep])
    q = torch.randn(3, 2, 4, 128, device="cuda", generator=g).bfloat16()
    tb.fused.attn_paged(q, k, v, st.table, st.lens)
    assert tb._lib.device_status() == tb._lib.ST_CURSOR_RANGE


def test_prefix_pages_are_those_in_use():
    st = state("cpu")
    assert st.prefix_pages.tolist() == []
    for rows, n in ((40, 3), (17, 2), (0, 0), (1, 1)):
        st.set_prefix(rows)
        assert st.prefix_pages.tolist() == st.prefix_table[:n].tolist() and len(st.prefix_pages) == n and -1 not in st.prefix_pages.tolist()


@pytest.mark.gpu
def test_a_state_without_room_for_a_prefix_serves_the_same_calls():
    import tokenrush_b200 as tb
    st = PagedState(Cfg, num_pages=4, max_seqs=2, max_pages=2, page_size=16, device="cuda")
    k, v, _, _ = st.layer(0)
    st.open(0, 5)
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(10, 2, 128, device="cuda", generator=g).bfloat16()
    tb.fused.paged_append(rows, rows, k, v, st.table, st.lens, base=st.prefix_len)
    q = torch.randn(2, 5, 4, 128, device="cuda", generator=g).bfloat16()
    got = tb.fused.attn_paged(q, k, v, st.table, st.lens, prefix_table=st.prefix_table, prefix_len=st.prefix_len)
    assert torch.equal(got, tb.fused.attn_paged(q, k, v, st.table, st.lens)) and tb._lib.device_status() == 0


def test_a_state_without_room_for_a_prefix_refuses_one():
    st = PagedState(Cfg, num_pages=4, max_seqs=2, max_pages=2, page_size=16, device="cpu")
    for rows in (0, 1):
        with pytest.raises(ValueError):
            st.set_prefix(rows)


def test_a_negative_prefix_is_refused():
    st = state("cpu")
    st.set_prefix(40)
    for rows in (-1, -40):
        with pytest.raises(ValueError):
            st.set_prefix(rows)
        holds(st)
        assert int(st.prefix_len) == 40 and len(st._prefix) == 3
