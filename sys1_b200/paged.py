"""One new token at a time: the paged key-value cache and the recurrent states that let the decoder go on from where a
prompt ended (`s1_block_tables`, `s1_release_blocks`, `s1_cache_write`, `s1_attention_paged`, and the states of
`s1_gated_delta_rule_prefill` / `s1_gated_delta_rule_step`).

The reference keeps no cache (`Decoder::forward`, src/archs/qwen35_text.rs:942-1005, runs whole prompts). `PagedCache` holds the
memory of a fixed number of rows (requests in flight); `qwen35.Decoder.prefill` enters prompts into it and
`qwen35.Decoder.step` moves every row one token further. The functions are the calls of the C ABI on tensors.
"""
from __future__ import annotations

from typing import List, NamedTuple, Optional, Sequence

import numpy as np
import torch

from . import _lib, device


class BlockTables(NamedTuple):
    """What `block_tables` returns (int32 CUDA tensors): tokens a row holds now `[rows]`, first token of every row
    `[rows + 1]`, position and slot of every token `[max_tokens]` and the pages left `[1]`."""
    lengths: torch.Tensor
    cu_seqlens: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    free_count: torch.Tensor


def _ints(t: torch.Tensor, dev: int, n: int, name: str) -> int:
    if t.dtype is not torch.int32 or t.get_device() != dev or dev < 0 or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous int32 CUDA tensor on the call's GPU (no CPU fallback)")
    if t.shape != (n,):
        raise ValueError(f"{name} must have shape [{n}], not {list(t.shape)}")
    return t.data_ptr()


def _table(t: torch.Tensor, dev: int, rows: int):
    """Address, row stride and width of the block tables."""
    if t.dtype is not torch.int32 or t.get_device() != dev or dev < 0 or t.dim() != 2 or t.shape[0] != rows or (t.stride(1) != 1 and t.shape[1] != 1):
        raise ValueError(f"block tables must be an int32 CUDA tensor [{rows}, pages] with contiguous rows")
    return t.data_ptr(), t.shape[1] if rows == 1 else t.stride(0), t.shape[1]


def _context(dev: int, ctx: Optional[device.Context]):
    """The context of a call on tensors of GPU `dev` (-1: none - the call will refuse them) and its address."""
    if ctx is None:
        if dev < 0:
            return None, None
        ctx = device.load(dev)
    elif ctx.ordinal != dev:
        raise ValueError(f"the tensors are on GPU {dev}, the context on GPU {ctx.ordinal}")
    return ctx, ctx.handle.value


def block_tables(cached: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor, page_size: int,
                 added: Optional[torch.Tensor] = None, max_tokens: Optional[int] = None, lengths: Optional[torch.Tensor] = None,
                 free_count_out: Optional[torch.Tensor] = None, ctx: Optional[device.Context] = None) -> BlockTables:
    """Pages, positions and slots for the tokens that a step adds (`s1_block_tables`): `cached` int32 `[rows]` tokens each row holds
    (negative: idle), `added` int32 `[rows]` tokens it gets (None: one each), `free_pages` / `free_count` `[1]` the stack that new
    pages are taken from, `tables` int32 `[rows, width]` updated in place. `max_tokens`: tokens of the packed batch, with those
    behind the last row (needed with `added`). `lengths` may be `cached` and `free_count_out` may be `free_count`: both are then
    advanced in place."""
    ctx, handle = _context(cached.get_device(), ctx)
    r = (_lib.binding or _lib.load_binding()).block_tables(handle, cached, tables, free_pages, free_count, page_size, added, max_tokens, lengths, free_count_out)
    if r.__class__ is int:
        ctx.check(r)
    return BlockTables._make(r)


def release_blocks(ended: torch.Tensor, lengths: torch.Tensor, tables: torch.Tensor, free_pages: torch.Tensor, free_count: torch.Tensor,
                   page_size: int, ctx: Optional[device.Context] = None) -> None:
    """Puts the pages of every row with `ended[row] != 0` back on the stack and makes the row idle (`s1_release_blocks`)."""
    dev, rows, pool = lengths.get_device(), lengths.numel(), free_pages.numel()
    ep, lp, fp, np_ = (_ints(ended, dev, rows, "ended"), _ints(lengths, dev, rows, "lengths"), _ints(free_pages, dev, pool, "free_pages"),
                       _ints(free_count, dev, 1, "free_count"))
    tp, ldt, width = _table(tables, dev, rows)
    ctx, handle = _context(dev, ctx)
    ctx.check(ctx._lib.s1_release_blocks(handle, ep, rows, page_size, lp, tp, ldt, width, fp, pool, np_))


def cache_write(k: torch.Tensor, v: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, slots: torch.Tensor,
                norm_weight: Optional[torch.Tensor] = None, eps: float = 1e-6, cos: Optional[torch.Tensor] = None, sin: Optional[torch.Tensor] = None,
                positions: Optional[torch.Tensor] = None, rotary_dim: int = 0, bf16_ops: bool = True, ctx: Optional[device.Context] = None) -> None:
    """Keys and values `[T, kv_heads, head_dim]` (rows may be strided) into the slots of `k_cache`, `v_cache` `[pages, page_size,
    kv_heads, head_dim]` (`s1_cache_write`); a token with slot -1 is left out. With `norm_weight` `[head_dim]` the keys are normed and
    rotated on the way, as `norm.head_norm_rope_` would do in place (`cos`, `sin` f32 `[positions, rotary_dim / 2]`)."""
    ctx, handle = _context(k.get_device(), ctx)
    rc = (_lib.binding or _lib.load_binding()).cache_write(handle, k, v, k_cache, v_cache, slots, norm_weight, eps, cos, sin, positions, rotary_dim, bf16_ops)
    if rc:
        ctx.check(rc)


def attention_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, tables: torch.Tensor, lengths: torch.Tensor,
                    gate: Optional[torch.Tensor] = None, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                    workspace: Optional[torch.Tensor] = None, ctx: Optional[device.Context] = None) -> torch.Tensor:
    """Attention of one new token per row over the first `lengths[row]` tokens of its block table (`s1_attention_paged`): q `[rows,
    heads, head_dim]` (rows may be strided), optional gate of the same shape (pre-sigmoid). Rows of length <= 0 get zeros. Returns
    `[rows, heads * head_dim]`. `workspace`: uint8 CUDA tensor of `attention_paged_workspace(head_dim)` bytes; by default
    the context's own, which the calls of one stream share. Graphs that may run at the same time need one each."""
    ctx, handle = _context(q.get_device(), ctx)
    if workspace is None and ctx is not None:
        workspace = ctx.attention_workspace()
    r = (_lib.binding or _lib.load_binding()).attention_paged(handle, q, k_cache, v_cache, tables, lengths, gate, scale, out, workspace)
    if r.__class__ is int:
        ctx.check(r)
    return r


def attention_paged_workspace(head_dim: int) -> int:
    """Bytes of workspace that `attention_paged` needs, whatever the batch."""
    return int(_lib.load_library().s1_attention_paged_workspace(int(head_dim)))


# ------------------------------------------------------------------------------------------------ the decoder's cache
class KvPages(NamedTuple):
    """A full-attention layer's cache: `[pages, page_size, kv_heads, head_dim]` bf16 each."""
    k: torch.Tensor
    v: torch.Tensor


class DeltaState(NamedTuple):
    """A linear-attention layer's states: `[rows, 4, channels]` bf16 (the conv's last inputs) and `[rows, value_heads, 128, 128]` f32."""
    conv: torch.Tensor
    state: torch.Tensor


def layout(cfg) -> tuple:
    """What a decoder of configuration `cfg` keeps of a request in each layer: KV heads and head dim, or key and value heads."""
    return tuple(("pages", cfg.num_key_value_heads, cfg.head_dim) if cfg.layer_type(i) == "full_attention" else
                 ("state", cfg.linear_num_key_heads, cfg.linear_num_value_heads) for i in range(cfg.num_hidden_layers))


class PagedCache:
    """The memory of up to `rows` requests in flight for a decoder of configuration `cfg` (see `qwen35.Decoder`): `num_pages` pages of
    `page_size` tokens that the rows share, at most `max_length` tokens a row, and one recurrent state a row and layer.

    `admit(n)` picks idle rows, `Decoder.prefill` fills them, `Decoder.step` adds a token to every active row, `release(rows)`
    gives their pages back. The bookkeeping lives on the GPU (`lengths`, `tables`, `free_pages`, `free_count`), so that a captured
    step can be replayed; `held` and `pages_left` mirror it on the host, where a request that does not fit is refused before
    anything is launched. After replaying a captured step, tell the mirror with `advanced(steps)`.

    A step that raises between its layers has moved the states of some and not of others. Its rows are then `unfinished`: no step is
    taken until they have been released."""

    def __init__(self, cfg, rows: int, num_pages: int, page_size: int = 64, max_length: int = 8192, dev="cuda"):
        if rows < 1 or num_pages < 1 or max_length < 1 or page_size < 1 or page_size & (page_size - 1):
            raise ValueError("rows, num_pages and max_length must be positive, page_size a power of two")
        if rows > 8192 or page_size > 65536 or num_pages >= 1 << 30 or num_pages * page_size > 1 << 31 or max_length > 1 << 30:
            raise ValueError("at most 8192 rows, pages of 65536 tokens, 2^31 tokens in all pages and 2^30 in a row")
        if cfg.head_dim not in (64, 128, 256):
            raise ValueError(f"the paged attention has head dim 64, 128 or 256, not {cfg.head_dim}")
        self.rows, self.num_pages, self.page_size, self.max_length = int(rows), int(num_pages), int(page_size), int(max_length)
        dev = torch.device(dev)
        if dev.type != "cuda":
            raise ValueError("the cache lives on a GPU (no CPU fallback)")
        if dev.index is None:
            dev = torch.device("cuda", torch.cuda.current_device())
        self.device = dev
        i32 = dict(dtype=torch.int32, device=dev)
        width = -(-max_length // page_size)
        group = cfg.num_attention_heads // cfg.num_key_value_heads
        spans = rows * cfg.num_key_value_heads * (1 if group <= 8 else -(-group // 16))  # s1_attention_paged's limit
        if (spans + 1) * (width * page_size // 64 + 5) > 1 << 31:
            raise ValueError("rows x KV heads x max_length / 64 must be below 2^31")
        self.tables = torch.zeros((rows, width), **i32)
        self.lengths = torch.full((rows,), -1, **i32)
        self.free_pages = torch.arange(num_pages - 1, -1, -1, **i32)
        self.free_count = torch.full((1,), num_pages, **i32)
        self.state_index = torch.full((rows,), -1, **i32)
        self.held = np.full(rows, -1, dtype=np.int64)
        self.unfinished = np.zeros(rows, dtype=bool)
        self.positions = self.max_length  # up to which rows may grow: those of a decoder whose step was captured, if it has fewer
        self.pages_left = int(num_pages)
        channels = (2 * cfg.linear_num_key_heads + cfg.linear_num_value_heads) * 128
        self.layers: List = []
        self.layout = layout(cfg)
        for i in range(cfg.num_hidden_layers):
            if cfg.layer_type(i) == "full_attention":
                shape = (num_pages, page_size, cfg.num_key_value_heads, cfg.head_dim)
                self.layers.append(KvPages(*(torch.empty(shape, dtype=torch.bfloat16, device=dev) for _ in range(2))))
            else:
                self.layers.append(DeltaState(torch.empty((rows, 4, channels), dtype=torch.bfloat16, device=dev),
                                              torch.empty((rows, cfg.linear_num_value_heads, 128, 128), dtype=torch.float32, device=dev)))
        self.workspace = torch.empty(attention_paged_workspace(cfg.head_dim), dtype=torch.uint8, device=dev)

    def _pages(self, tokens) -> int:
        return -(-int(tokens) // self.page_size)

    @property
    def active(self) -> List[int]:
        return [int(r) for r in np.flatnonzero(self.held >= 0)]

    def admit(self, lengths: Sequence[int]) -> List[int]:
        """Idle rows for prompts of these lengths, in ascending order (the order of the packed batch); refuses what does not fit."""
        idle = np.flatnonzero(self.held < 0)
        if len(lengths) > len(idle):
            raise ValueError(f"{len(lengths)} prompts, {len(idle)} idle rows")
        if any(n < 1 or n > self.max_length for n in lengths):
            raise ValueError(f"prompts must have 1 to {self.max_length} tokens")
        need = sum(self._pages(n) for n in lengths)
        if need > self.pages_left:
            raise ValueError(f"the prompts need {need} pages, {self.pages_left} are left")
        return [int(r) for r in idle[:len(lengths)]]

    def enter(self, rows: Sequence[int], lengths: Sequence[int]) -> BlockTables:
        """Takes pages for the prompts of `rows` (from `admit`); the tokens of the packed batch follow one another in that order."""
        if len(rows) != len(lengths) or list(rows) != sorted(set(rows)) or any(not 0 <= r < self.rows or self.held[r] >= 0 for r in rows):
            raise ValueError("rows must be different idle rows in ascending order, one for each length")
        if any(n < 1 or n > self.max_length for n in lengths) or sum(self._pages(n) for n in lengths) > self.pages_left:
            raise ValueError("the prompts do not fit the cache")
        added, index = np.zeros(self.rows, np.int32), self.held >= 0
        added[list(rows)], index[list(rows)] = lengths, True
        start = np.where(added > 0, 0, -1).astype(np.int32)  # lengths that change: the new rows' only
        state = np.where(index, np.arange(self.rows), -1).astype(np.int32)
        added_dev, start_dev, state_dev = torch.from_numpy(np.stack([added, start, state])).to(self.device)
        # nothing of the cache changes before this call, and nothing fails after it
        plan = block_tables(torch.maximum(self.lengths, start_dev), self.tables, self.free_pages, self.free_count, self.page_size, added=added_dev,
                            max_tokens=int(sum(lengths)), lengths=self.lengths, free_count_out=self.free_count)
        self.state_index.copy_(state_dev)
        for r, n in zip(rows, lengths):
            self.held[r] = n
            self.pages_left -= self._pages(n)
        return plan

    def extend(self) -> BlockTables:
        """One more token for every active row. Token r of the step belongs to row r; idle rows have slot -1."""
        eager = not torch.cuda.is_current_stream_capturing()
        if eager:
            self._refuse(1)
        plan = block_tables(self.lengths, self.tables, self.free_pages, self.free_count, self.page_size, lengths=self.lengths,
                            free_count_out=self.free_count)
        if eager:
            self._advance(1)
        return plan

    def fits(self, steps: int = 1) -> bool:
        """Whether every active row can grow by `steps` tokens."""
        live = self.held[self.held >= 0]
        need = sum(self._pages(n + steps) - self._pages(n) for n in live)
        return not self.unfinished.any() and need <= self.pages_left and (len(live) == 0 or int(live.max()) + steps <= self.positions)

    def advanced(self, steps: int = 1) -> None:
        """Notes on the host that every active row has `steps` more tokens; refuses steps that do not fit. (`Decoder.step` does as much;
        call it yourself before replaying a captured step.)"""
        self._refuse(steps)
        self._advance(steps)

    def _refuse(self, steps: int) -> None:
        if self.unfinished.any():
            raise ValueError(f"a call failed half-way and left rows {np.flatnonzero(self.unfinished).tolist()} with part of a token: release them")
        if not self.fits(steps):
            raise ValueError(f"{steps} more token(s) do not fit: {self.pages_left} pages left, rows of up to {self.positions} tokens")

    def _advance(self, steps: int) -> None:
        live = self.held >= 0
        self.pages_left -= sum(self._pages(n + steps) - self._pages(n) for n in self.held[live])
        self.held[live] += steps

    def release(self, rows: Sequence[int]) -> None:
        """Ends the requests of `rows`: their pages go back, the rows are idle."""
        rows = sorted(set(int(r) for r in rows))
        if any(not 0 <= r < self.rows or self.held[r] < 0 for r in rows):
            raise ValueError("only active rows can be released")
        ended = np.zeros(self.rows, np.int32)
        ended[rows] = 1
        index = np.where((self.held >= 0) & (ended == 0), np.arange(self.rows), -1).astype(np.int32)
        ended_dev, index_dev = torch.from_numpy(np.stack([ended, index])).to(self.device)
        release_blocks(ended_dev, self.lengths, self.tables, self.free_pages, self.free_count, self.page_size)
        self.state_index.copy_(index_dev)
        self.unfinished[rows] = False
        for r in rows:
            self.pages_left += self._pages(self.held[r])
            self.held[r] = -1
