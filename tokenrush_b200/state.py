"""Preallocated KV state, the attention half of the reference's `State`
(tokenrush/state.py:13-75): one contiguous cache `[layer, kv_head, position, head_dim]` in
bf16 or e4m3 with fp32 per-(head, position) scales, and the position as a device tensor with
a host mirror.  The GDN fields of the reference's State belong to other layers and are not
kept here."""
from __future__ import annotations

import torch


class State:
    def __init__(self, cfg, max_len: int, device="cuda", kv_dtype=torch.bfloat16, n_slots: int = 1,
                 shard_lo=None, pos_dtype=torch.long):
        """cfg: anything with n_kv_heads, head_dim and attn_layers (the reference's ModelConfig
        or tokenrush_b200.config.AttnConfig).  shard_lo: first position held by this cache
        when the sequence is sharded over several GPUs (None: a whole cache)."""
        layers = list(cfg.attn_layers)
        n_attn = len(layers)
        self.max_len = max_len
        self.kv_dtype = kv_dtype
        self.fp8 = kv_dtype == torch.float8_e4m3fn
        self.shard_lo = shard_lo
        self.k = torch.zeros(n_attn, cfg.n_kv_heads, max_len, cfg.head_dim, device=device, dtype=kv_dtype)
        self.v = torch.zeros_like(self.k)
        if self.fp8:
            self.k_scale = torch.ones(n_attn, cfg.n_kv_heads, max_len, device=device, dtype=torch.float32)
            self.v_scale = torch.ones_like(self.k_scale)
        else:
            self.k_scale = self.v_scale = None
        self.n_slots = n_slots
        self.pos = 0
        self.pos_t = torch.zeros(1, device=device, dtype=pos_dtype)
        self.attn_slot = {l: i for i, l in enumerate(layers)}

    def reset(self):
        self.pos = 0
        self.pos_t.zero_()

    def advance(self, T: int):
        self.pos += T
        self.pos_t += T

    def set_pos(self, pos: int):
        """Rewind / resume at `pos`: rows beyond it stay in the cache as dead data and are
        overwritten by the next append (tokenrush/mtp.py:84-87, tokenrush/session.py:94-95)."""
        self.pos = pos
        self.pos_t.fill_(pos)

    @property
    def nbytes(self):
        ts = [self.k, self.v] + ([self.k_scale, self.v_scale] if self.fp8 else [])
        return sum(t.numel() * t.element_size() for t in ts)

    @property
    def kv_bytes_per_token(self):
        n_attn = self.k.shape[0]
        b = 2 * n_attn * self.k.shape[1] * self.k.shape[3] * self.k.element_size()
        if self.fp8:
            b += 2 * n_attn * self.k.shape[1] * 4
        return b


class PagedState:
    """Preallocated paged KV state of a batch: one pool of pages for every layer, `[layer, page, kv_head, row, head_dim]` in bf16 or
    e4m3 with fp32 scales, a page table and lengths on the device, and the pages of a prefix that all sequences share.
    Pages are handed out on the host, and table entries that name none are -1 (a step that goes past a sequence's pages is reported as
    ST_CURSOR_RANGE and writes nothing there); lengths live on the device (`fused.spec_verify` advances them there), so a
    captured step keeps working while sequences come, grow and leave.  Counterpart of `State` for `fused.paged_append`
    and `fused.attn_paged`."""

    def __init__(self, cfg, num_pages: int, max_seqs: int, max_pages: int, page_size: int = 64, device="cuda", kv_dtype=torch.bfloat16,
                 max_prefix_pages: int = 0):
        """max_pages: the longest own page list of a sequence; max_prefix_pages: the longest shared prefix."""
        if page_size < 16 or page_size & (page_size - 1):
            raise ValueError("page_size must be a power of two, 16 or more")
        if min(num_pages, max_seqs, max_pages) < 1:
            raise ValueError("num_pages, max_seqs and max_pages must be positive")
        layers = list(cfg.attn_layers)
        self.page_size, self.kv_dtype, self.fp8 = page_size, kv_dtype, kv_dtype == torch.float8_e4m3fn
        self.k = torch.zeros(len(layers), num_pages, cfg.n_kv_heads, page_size, cfg.head_dim, device=device, dtype=kv_dtype)
        self.v = torch.zeros_like(self.k)
        self.k_scale = torch.ones(self.k.shape[:4], device=device, dtype=torch.float32) if self.fp8 else None
        self.v_scale = torch.ones_like(self.k_scale) if self.fp8 else None
        self.table = torch.full((max_seqs, max_pages), -1, device=device, dtype=torch.int32)
        self.lens = torch.full((max_seqs,), -1, device=device, dtype=torch.long)      # -1: an empty slot
        self.prefix_table = torch.full((max_prefix_pages,), -1, device=device, dtype=torch.int32)     # (no entries: no room for a prefix)
        self.prefix_len = torch.zeros(1, device=device, dtype=torch.long)
        self.attn_slot = {l: i for i, l in enumerate(layers)}
        self._free = list(range(num_pages - 1, -1, -1))
        self._own = [None] * max_seqs            # pages of each open slot
        self._prefix = []

    def layer(self, slot: int):
        """(k_pages, v_pages, k_scale, v_scale) of attention layer number `slot`."""
        if not self.fp8:
            return self.k[slot], self.v[slot], None, None
        return self.k[slot], self.v[slot], self.k_scale[slot], self.v_scale[slot]

    @property
    def free_pages(self) -> int:
        return len(self._free)

    @property
    def prefix_pages(self):
        """The entries of prefix_table in use, the form for `fused.attn_paged`, which reads a long prefix otherwise than a short one.  A captured
        step keeps the number of entries that it was captured with."""
        return self.prefix_table[:len(self._prefix)]

    def _grow(self, pages: list, table: torch.Tensor, rows: int):
        want = -(-rows // self.page_size)
        if want > table.shape[0]:
            raise ValueError(f"{rows} rows need {want} pages, the table holds {table.shape[0]}")
        more = want - len(pages)
        if more <= 0:
            return
        if more > len(self._free):
            raise RuntimeError(f"the pool is full: {more} pages wanted, {len(self._free)} free")
        new = [self._free.pop() for _ in range(more)]
        table[len(pages):want] = torch.tensor(new, dtype=torch.int32)
        pages += new

    def open(self, seq: int, rows: int = 0):
        """Start an empty sequence in slot `seq`, with pages for `rows` rows."""
        if self._own[seq] is not None:
            raise ValueError(f"slot {seq} is in use")
        pages = []
        self._grow(pages, self.table[seq], rows)
        self._own[seq] = pages
        self.lens[seq] = 0

    def reserve(self, seq: int, rows: int):
        """Pages for `rows` own rows of an open sequence in all: before the append that writes them."""
        if self._own[seq] is None:
            raise ValueError(f"slot {seq} is empty")
        self._grow(self._own[seq], self.table[seq], rows)

    def close(self, seq: int):
        """End the sequence of slot `seq`: its pages are free again."""
        if self._own[seq] is None:
            raise ValueError(f"slot {seq} is empty")
        self._free += reversed(self._own[seq])
        self._own[seq] = None
        self.table[seq] = -1
        self.lens[seq] = -1

    def set_prefix(self, rows: int):
        """Pages for a shared prefix of `rows` rows, appended as one sequence with `table=prefix_table[None]`.  Only while no
        sequence is open: their positions count from its end."""
        if any(p is not None for p in self._own):
            raise ValueError("the prefix can only change while every slot is empty")
        if not len(self.prefix_table):
            raise ValueError("made without room for a prefix (max_prefix_pages)")
        if rows < 0:
            raise ValueError("a prefix has no negative number of rows")
        want = -(-rows // self.page_size)
        if want < len(self._prefix):
            self._free += reversed(self._prefix[want:])
            del self._prefix[want:]
            self.prefix_table[want:] = -1
        self._grow(self._prefix, self.prefix_table, rows)
        self.prefix_len.fill_(rows)
