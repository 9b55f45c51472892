"""A paged KV cache in 16 or 4 bits: append with the position rotation on the way, attention, rows back.

The operators (csrc/paged_append.cu, csrc/paged_attention.cu) work on `Pages`: a page holds page_size rows of one slot
(one KV head of one sequence; slot = sequence * heads + head), so the heads of a sequence can hold different numbers of
rows, as evictions leave them.  Row r of a slot lies in page table[slot, r // page_size], place r % page_size.  In 4 bits
a row is a code per channel and a float16 (scale, offset) pair per group of channels; a channel's value is
offset + scale * (code - 8).

    paged_append      new tokens' keys and values into their slots, rotated by position on the way; the queries too
    paged_attention   queries over their slots, causal at the end of each slot; single tokens, a few, or long chunks
    paged_read        rows of slots in the packed layout, as the values they stand for

PagedCache keeps the pages, tables and lengths of every layer, and moves a request between the packed layout, which
audits and evictions work on (kvcache.PackedCache), and pages, which decode reads: `load` after an audit, `to_packed`
before the next one.  They have no gradient (a KV cache has no backward pass): inputs that require one are refused outside of torch.no_grad().
No counterpart in the reference, whose attention is FlashAttention over the packed layer
(attention.py:15-35) and whose cache is 16-bit (cache.py:16-265).
"""
from __future__ import annotations

from dataclasses import dataclass
from typing import List, Optional, Sequence

import numpy as np

from . import operators, upload

_module = None


def _operators():
    """operators(), looked up once: a decode step's host time counts here."""
    global _module
    if _module is None:
        _module = operators()
    return _module


#: Bytes of an attention workspace (lrk_paged_attention_workspace_bytes), and how many of them, from the first, must be
#: zero before its first call (every call leaves them so).
WORKSPACE_BYTES = 64 << 20
WORKSPACE_COUNTER_BYTES = 16 << 10


@dataclass
class Pages:
    """The page memory of the operators.  16-bit: keys, values [pages, page_size, D] of float16 or bfloat16.  4-bit:
    uint8 codes [pages, page_size, D / 2] (channel 2j in the low half of byte j) with key_scales, value_scales float16
    [pages, page_size, D / group, 2].  positions: float32 [pages, page_size], each row's logical position."""

    keys: "object"
    values: "object"
    positions: "object"
    key_scales: "Optional[object]" = None
    value_scales: "Optional[object]" = None

    @classmethod
    def empty(cls, pages: int, page_size: int, dim: int, device, dtype=None, bits: int = 16, group: int = 64) -> "Pages":
        """Page memory for `pages` pages; `dtype` is the 16-bit rows' type, `group` the channels of a 4-bit scale."""
        import torch

        if bits not in (4, 16):
            raise ValueError(f"rows are held in 16 or 4 bits, not {bits}")
        if page_size not in (16, 32, 64, 128):
            raise ValueError(f"page size must be 16, 32, 64 or 128, not {page_size}")
        if dim not in (64, 128):
            raise ValueError(f"head dimension must be 64 or 128, not {dim}")
        positions = torch.zeros(pages, page_size, dtype=torch.float32, device=device)
        if bits == 16:
            keys = torch.empty(pages, page_size, dim, dtype=dtype or torch.bfloat16, device=device)
            return cls(keys, torch.empty_like(keys), positions)
        if group not in (32, 64, 128) or group > dim:
            raise ValueError(f"a scale's group must be 32, 64 or 128 channels, at most the head dimension, not {group}")
        codes = torch.empty(pages, page_size, dim // 2, dtype=torch.uint8, device=device)
        scales = torch.empty(pages, page_size, dim // group, 2, dtype=torch.float16, device=device)
        return cls(codes, torch.empty_like(codes), positions, scales, torch.empty_like(scales))

    @property
    def dim(self) -> int:
        return self.keys.shape[2] * (1 if self.key_scales is None else 2)


def rotary_table(positions: int, rotary_dim: int, theta: float, device):
    """float32 [positions, rotary_dim]: per position rotary_dim / 2 cosines, then as many sines, of
    position * theta ** (-2 j / rotary_dim), formed in float64."""
    import torch

    rate = theta ** (-torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / rotary_dim)
    angle = torch.arange(positions, dtype=torch.float64, device=device)[:, None] * rate
    return torch.cat((angle.cos(), angle.sin()), 1).float()


def attention_workspace(device):
    """A workspace for paged_attention: zeroed once, kept between calls.  Calls that may overlap (on two streams, or in
    two graphs that are replayed at a time) need one each.  Make it outside of a graph's capture: inside, the zeroing
    belongs to the graph."""
    import torch

    return torch.zeros(WORKSPACE_BYTES, dtype=torch.uint8, device=device)


def paged_append(pages: Pages, table, lengths, new_keys, new_values, new_positions, token_starts, flag, rotary=None,
                 interleaved: bool = False, queries=None):
    """Write new tokens' rows into the pages.  table int32 [slots, pages of a slot]; lengths int32 [slots], the lengths
    AFTER the append (left as they are); new_keys, new_values [tokens, heads, D] (any strides); new_positions int64
    [tokens]; token_starts int32 [sequences + 1]: token i of sequence s, of n_s, becomes row lengths - n_s + i of its
    slots.  `rotary` (rotary_table) rotates keys and `queries` [tokens, query heads, D]; the rotated queries are
    returned.  Rows without a place, and positions outside the table, are left out (such a token's queries are NaN) and
    set bits of `flag` (int32 [1])."""
    return _operators().paged_append(pages.keys, pages.values, pages.positions, pages.key_scales, pages.value_scales,
                                    table, lengths, new_keys, new_values, new_positions, token_starts, flag, rotary,
                                    interleaved, queries)


def paged_attention(pages: Pages, table, lengths, queries, token_starts, workspace, flag,
                    scale: Optional[float] = None, causal: bool = True):
    """(out [tokens, query heads, D] of the queries' type, lse float32 [tokens, query heads]) of queries [tokens, query
    heads, D] over their slots; query head h reads KV head h // (query heads / heads).  Token i of n_s sees rows
    r <= lengths - n_s + i, or all of them where not `causal`; one that sees none gives 0 and -inf.  `scale` defaults
    to D ** -0.5; workspace: attention_workspace."""
    if scale is None:
        scale = queries.shape[2] ** -0.5
    return _operators().paged_attention(pages.keys, pages.values, pages.positions, pages.key_scales, pages.value_scales,
                                       table, lengths, queries, token_starts, workspace, flag, scale, causal)


def paged_read(pages: Pages, table, first_rows, row_starts, rows: int, dtype, flag):
    """(keys, values [rows, D] of `dtype`, positions float32 [rows]): of each slot s, row_starts[s + 1] - row_starts[s]
    rows from first_rows[s] on (both int32; `rows` is row_starts[-1]), back to back.  Rows without a place are NaN and set
    a bit of `flag`."""
    return _operators().paged_read(pages.keys, pages.values, pages.positions, pages.key_scales, pages.value_scales,
                                  table, first_rows, row_starts, rows, dtype, flag)


class PagedCache:
    """Pages, page tables and lengths of every layer of a batch of sequences; page allocation is on the host.

    A step: `advance(counts)` once, then per layer `append` and `attend`.  The step's token_starts and the page tables
    are shared by every launch of the step, and keep their places: a graph captured of a step's appends and attentions
    serves later steps of as many tokens, `advance` called before each replay."""

    def __init__(self, layers: int, sequences: int, heads: int, dim: int, pages: int, device, dtype=None, bits: int = 16,
                 group: int = 64, page_size: int = 64, max_rows: int = 1 << 17):
        import torch

        self.layers, self.sequences, self.heads, self.dim = int(layers), int(sequences), int(heads), int(dim)
        self.device, self.dtype = torch.device(device), dtype or torch.bfloat16
        self.page_size = int(page_size)
        self.pages = Pages.empty(pages, page_size, dim, self.device, self.dtype, bits, group)
        slots, width = self.sequences * self.heads, -(-int(max_rows) // self.page_size)
        self.tables = torch.zeros(self.layers, slots, width, dtype=torch.int32, device=self.device)
        self.lengths = torch.zeros(self.layers, slots, dtype=torch.int32, device=self.device)
        self.flag = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.rows = np.zeros((self.layers, slots), dtype=np.int64)  # host mirror of the lengths
        self.prompt_rows = np.zeros((self.layers, slots), dtype=np.int64)
        self.seen_tokens = np.zeros(self.sequences, dtype=np.int64)  # as PackedCache.seen_tokens, a step's tokens added
        self._free: List[int] = list(range(int(pages) - 1, -1, -1))
        self._held: List[List[List[int]]] = [[[] for _ in range(slots)] for _ in range(self.layers)]
        self._workspaces = {}
        # The step's token starts and new rows a slot, in place: a captured step finds the next step's there.
        self._step = torch.zeros(self.sequences + 1 + slots, dtype=torch.int32, device=self.device)
        self.token_starts = None

    # ------------------------------------------------------------ allocation

    def free_pages(self) -> int:
        return len(self._free)

    def _hold(self, rows: np.ndarray) -> None:
        """Give every slot pages for `rows` [layers, slots] rows; raises MemoryError, with nothing changed, when the
        pages do not suffice."""
        need = -(-rows // self.page_size)
        if int(need.max(initial=0)) > self.tables.shape[2]:
            raise MemoryError(f"a slot would pass {self.tables.shape[2] * self.page_size} rows")
        held = np.asarray([[len(p) for p in layer] for layer in self._held], dtype=np.int64).reshape(need.shape)
        short = np.argwhere(need > held)
        total = int((need - held)[need > held].sum())
        if total > len(self._free):
            raise MemoryError(f"{total} pages needed, {len(self._free)} free")
        entries = []
        for layer, slot in short.tolist():
            pages = self._held[layer][slot]
            while len(pages) < need[layer, slot]:
                page = self._free.pop()
                entries.append((layer, slot, len(pages), page))
                pages.append(page)
        if entries:
            import torch

            at = upload(np.asarray(entries, dtype=np.int64).T.copy(), self.device)
            self.tables.index_put_((at[0], at[1], at[2]), at[3].to(torch.int32))

    def _slots(self, sequence: int) -> slice:
        if not 0 <= sequence < self.sequences:
            raise ValueError(f"the cache has sequences 0 to {self.sequences - 1}, not {sequence}")
        return slice(sequence * self.heads, (sequence + 1) * self.heads)

    def release(self, sequence: int) -> None:
        """Return a sequence's pages; its slots become empty."""
        slots = self._slots(sequence)
        for layer in self._held:
            for slot in range(slots.start, slots.stop):
                self._free.extend(reversed(layer[slot]))
                layer[slot] = []
        self.rows[:, slots] = 0
        self.prompt_rows[:, slots] = 0
        self.seen_tokens[sequence] = 0
        self.lengths[:, slots] = 0

    def check_flags(self) -> None:
        """Raise if an operator set a bit of the flag (a synchronisation)."""
        state = int(self.flag.item())
        if state:
            self.flag.zero_()
            raise RuntimeError(f"paged cache flagged: {state} (1: row outside its pages or token of no sequence, "
                               "2: position outside the rotary table, 4: a kernel's bounded wait ran out, "
                               "8: a kernel's shared memory was not aligned)")

    # ------------------------------------------------------------------ steps

    def advance(self, counts: Sequence[int]) -> None:
        """Begin a step of counts[s] new tokens for each sequence: every layer's slots get their pages and their new
        lengths, and the step's token_starts."""
        import torch

        counts = np.asarray(counts, dtype=np.int64).reshape(-1)
        if counts.shape != (self.sequences,) or (counts < 0).any():
            raise ValueError(f"one count per sequence expected, none negative, got {counts.tolist()}")
        per_slot = np.repeat(counts, self.heads)
        self._hold(self.rows + per_slot)
        self.rows += per_slot
        self.seen_tokens += counts
        starts = np.concatenate(([0], np.cumsum(counts)))
        staged = torch.from_numpy(np.concatenate((starts, per_slot)).astype(np.int32)).pin_memory()
        self._step.copy_(staged, non_blocking=True)
        self.token_starts = self._step[:self.sequences + 1]
        self.lengths.add_(self._step[self.sequences + 1:])

    def append(self, layer: int, new_keys, new_values, positions, rotary=None, interleaved: bool = False, queries=None):
        """The step's rows of one layer (paged_append); returns the rotated queries, if any."""
        return paged_append(self.pages, self.tables[layer], self.lengths[layer], new_keys, new_values, positions,
                            self.token_starts, self.flag, rotary, interleaved, queries)

    def attend(self, layer: int, queries, scale: Optional[float] = None, causal: bool = True, workspace=None):
        """(out, lse) of the step's queries over one layer (paged_attention).  Without a `workspace` the cache takes one
        that it keeps for the current stream; in a graph's capture, where neither that stream nor what a call left
        behind says what the replays will find, memory of the graph whose counters the graph zeroes each time."""
        import torch

        if workspace is None and torch.cuda.is_current_stream_capturing():
            workspace = torch.empty(WORKSPACE_BYTES, dtype=torch.uint8, device=self.device)
            workspace[:WORKSPACE_COUNTER_BYTES].zero_()
        elif workspace is None:
            stream = torch.cuda.current_stream(self.device).cuda_stream
            workspace = self._workspaces.get(stream)
            if workspace is None:
                workspace = self._workspaces[stream] = attention_workspace(self.device)
        return paged_attention(self.pages, self.tables[layer], self.lengths[layer], queries, self.token_starts,
                               workspace, self.flag, scale, causal)

    # ------------------------------------------------- to and from the packed layout

    def load(self, sequence: int, packed) -> None:
        """Put a request (kvcache.PackedCache) into a sequence, in place of what it held: the rows are already
        rotated, so they are only stored (quantised where the pages are 4-bit).  Raises, with nothing changed, ValueError
        for a request of another shape or type and MemoryError for one that the pages do not hold."""
        import torch

        slots = self._slots(sequence)
        if len(packed.layers) != self.layers or any(len(layer.head_lens) != self.heads for layer in packed.layers):
            raise ValueError("packed cache has another number of layers or heads")
        types = (torch.float16, torch.bfloat16) if self.pages.key_scales is not None else (self.pages.keys.dtype,)
        for layer in packed.layers:
            if layer.keys.dtype not in types or layer.values.dtype != layer.keys.dtype:
                raise ValueError(f"rows of {layer.keys.dtype} and {layer.values.dtype} into pages of {self.pages.keys.dtype}")
            if layer.keys.shape != (sum(layer.head_lens), self.dim) or layer.values.shape != layer.keys.shape or (
                    layer.positions.numel() != layer.keys.shape[0]):
                raise ValueError("packed rows do not fit the head lengths or the cache's head dimension")
            if any(t.device != self.lengths.device for t in (layer.keys, layer.values, layer.positions, layer.cumulative)):
                raise ValueError("packed rows are on another device")
        rows = self.rows.copy()
        rows[:, slots] = [layer.head_lens for layer in packed.layers]
        need = -(-rows[:, slots] // self.page_size)
        free = len(self._free) + sum(len(pages) for layer in self._held for pages in layer[slots])
        if int(need.max(initial=0)) > self.tables.shape[2]:
            raise MemoryError(f"a slot would pass {self.tables.shape[2] * self.page_size} rows")
        if int(need.sum()) > free:
            raise MemoryError(f"{int(need.sum())} pages needed, {free} free without what the sequence holds")
        self.release(sequence)
        self._hold(rows)
        self.rows[:] = rows
        self.prompt_rows[:, slots] = [layer.prompt_lens for layer in packed.layers]
        self.seen_tokens[sequence] = packed.seen_tokens
        self.lengths[:, slots] = upload(rows[:, slots].astype(np.int32), self.device)
        for index, layer in enumerate(packed.layers):
            # Each head's rows are the new tokens of a one-head sequence of their own.
            paged_append(self.pages, self.tables[index, slots], self.lengths[index, slots], layer.keys[:, None],
                         layer.values[:, None], layer.positions.reshape(-1).to(torch.int64), layer.cumulative,
                         self.flag)

    def to_packed(self, sequence: int, dtype=None):
        """A sequence's rows (and its count of seen tokens) as a kvcache.PackedCache of `dtype` (the cache's by default)."""
        from .kvcache import PackedCache

        slots = self._slots(sequence)
        packed = PackedCache(seen_tokens=int(self.seen_tokens[sequence]))
        first = self.lengths.new_zeros(self.heads)
        for index in range(self.layers):
            lens = self.rows[index, slots]
            starts = upload(np.concatenate(([0], np.cumsum(lens))).astype(np.int32), self.device)
            keys, values, positions = paged_read(self.pages, self.tables[index, slots], first, starts, int(lens.sum()),
                                                 dtype or self.dtype, self.flag)
            packed.add_layer(keys, values, positions, lens.tolist(), self.prompt_rows[index, slots].tolist())
        return packed
