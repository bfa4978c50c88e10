"""Decode attention of rows that share the leading pages of their cache (kernels in attention_shared.cu and
attention_shared_f32.cu): the beams of a search, which have one prompt.  Shared pages are read once for all rows of a group."""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from functools import lru_cache
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import build
from .ops import KernelError, _check, _here, _stream_on, register_error_word

HEAD_DIMS = (64, 128)
PAGE = build.PAGE_TOKENS
MAX_GROUPS = 256               # groups of one call
MAX_HEADS = {torch.bfloat16: 16, torch.float32: 32}     # query heads per key/value head
BLOCK_ROWS = {torch.bfloat16: 64, torch.float32: 32}    # rows of a unit (rows of a group, times query heads)
TILE_PAGES = {torch.bfloat16: 2, torch.float32: 1}      # pages that a block takes at a time
PER_SM = {torch.bfloat16: 1, torch.float32: 2}          # resident blocks
MAX_PARTS = 160                # pieces of a unit that the merge takes
# When shared pages are worth the kernel: (bytes, share).  It takes some 4 us more than the per-row kernels (two launches, units whose tiles
# differ, one block for all beams' own pages), which read what rows share from the L2 cache at up to 9 TB/s; so the bytes of keys and values
# that rows need not read again have to exceed `bytes` and `share` of those that rows hold alone.  Measured over 1296 shapes (1 to 16
# groups of 2 to 8 rows, 64 to 4096 common and 20 to 1000 own tokens, six head layouts, cold cache), per row / shared: bfloat16, 32 over
# 8 heads of 128, 4 groups of 4: 256 + 200 tokens 9.9 / 14.0 us, 1024 + 20 14.4 / 14.1, 4096 + 20 38 / 20; 16 groups of 8 with 4096 +
# 20 239 / 63; 32-bit, 1 group of 8, 256 + 20 14.1 / 14.9, 1024 + 20 31 / 21; 4 groups of 4, 64 + 20 8.7 / 14.5.  The rule is 0.4 % (bfloat16)
# and 3 % (32-bit) above the better of both in the geometric mean; always per row 12 % and 49 %, always shared 37 % and 5 %.  At its worst it
# takes 25 % longer than the other kernel would (bfloat16, 32 over 4 heads of 64, 16 groups of 8, 1024 + 1000: 39.6 / 49.5; more than 10 % on
# 10 of 648 shapes) and 84 % (32-bit, the same heads, 16 groups of 2, 64 + 1000: 54.4 / 29.6, where the per-row kernel is slow; 69 of 648).
WORTH = {torch.bfloat16: (50e6, 0.5), torch.float32: (7.5e6, 0.0)}

for _hd in HEAD_DIMS:
    build.register_library(f"attn_shared_bf16_hd{_hd}", ("attention_shared.cu",), (f"-DHEAD_DIM={_hd}",))
build.register_library("attn_shared_f32", ("attention_shared_f32.cu",), ())


@lru_cache(maxsize=4096)
def shared_plan(lens: Tuple[int, ...], shared: Tuple[int, ...], group_rows: int, nkv: int, group: int, window: int,
                dtype: torch.dtype, blocks: int, bound: int = 0) -> Tuple[int, int]:
    """(row_blocks, parts): units that the rows of a group are split into, and the pieces of a unit that there is room for.  The
    kernel cuts the line of all units' tiles into equal stretches, one per block; `parts` is what the longest unit then falls into with
    two to spare (were there less room, the kernel would make the stretches longer).  `lens` and `shared` per group; `bound`: columns that
    the common pages may come to fill while a recorded call is replayed."""
    row_blocks = -(-group_rows // (BLOCK_ROWS[dtype] // group))
    beams = -(-group_rows // row_blocks)
    tile = TILE_PAGES[dtype]
    total, longest = 0, 1
    for n, c in zip(lens, shared):
        first = max(0, n - window) // PAGE if window else 0
        end = -(-n // PAGE)
        border = min(max(c, first), end)
        tiles = -(-(border - first + (end - border) * beams) // tile)
        total += tiles * row_blocks * nkv
        longest = max(longest, tiles, -(-(max(bound, border - first) + (end - border) * beams) // tile) if bound else 0)
    share = max(1, -(-total // blocks))
    return row_blocks, max(2, min(MAX_PARTS, -(-longest // share) + 3))


def worth_sharing(rows: Sequence[int], lens: Sequence[int], shared: Sequence[int], nkv: int, head_dim: int,
                  window: Optional[int], dtype: torch.dtype) -> bool:
    """Whether reading common pages once saves more than the kernel costs; per group its rows, length and common pages."""
    saved = own = 0
    for b, n, c in zip(rows, lens, shared):
        first = max(0, n - window) if window else 0
        border = min(max(c * PAGE, first), n)
        saved += (b - 1) * (border - first)
        own += b * (n - border)
    token = 2 * nkv * head_dim * dtype.itemsize
    least, share = WORTH[dtype]
    return saved * token > least + share * own * token


_sms: Dict[int, int] = {}


def _sm_count(device: int) -> int:
    if device not in _sms:
        _sms[device] = torch.cuda.get_device_properties(device).multi_processor_count
    return _sms[device]


class SharedAttention:
    _known: Dict[tuple, "SharedAttention"] = {}

    @classmethod
    def get(cls, dtype: torch.dtype, head_dim: int) -> Optional["SharedAttention"]:
        """The kernels for this type and head size, or None where there are none (the per-row kernels then read the same
        pages through the same tables)."""
        if dtype not in MAX_HEADS or head_dim not in HEAD_DIMS:
            return None
        key = (dtype, head_dim)
        if key not in cls._known:
            cls._known[key] = cls(dtype, head_dim)
        return cls._known[key]

    def __init__(self, dtype: torch.dtype, head_dim: int):
        self.dtype, self.head_dim = dtype, head_dim
        self._call = None        # loaded with the first call (a model can be put together without a device)

    def _load(self) -> None:
        P, I, L = c_void_p, c_int, c_longlong
        head = [P, P, P, L, P, P, P, P, P, P, I, P, P, I, I, I, I, I]
        rest = [I, c_float, I, I, I, P]
        if self.dtype == torch.bfloat16:
            name = f"attn_shared_bf16_hd{self.head_dim}"
            lib = build.load_library(name)
            call, take = getattr(lib, f"tl_attn_shared_hd{self.head_dim}"), getattr(lib, f"tl_attn_shared_take_error_hd{self.head_dim}")
            call.argtypes = head + rest
        else:
            name = "attn_shared_f32"
            lib = build.load_library(name)
            call, take = lib.tl_attn_shared_f32, lib.tl_attn_shared_f32_take_error
            call.argtypes = head + [I] + rest
        call.restype = take.restype = c_int
        register_error_word(name, lambda: int(take()))
        self._call = call        # last: another thread calls as soon as it is there

    def takes(self, nh: int, nkv: int) -> bool:
        return nkv > 0 and nh % nkv == 0 and nh // nkv <= MAX_HEADS[self.dtype]

    def decode(self, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, out: torch.Tensor, seq_len: torch.Tensor,
               seq_slot: torch.Tensor, page_table: torch.Tensor, group_start: torch.Tensor, group_pages: torch.Tensor, nh: int,
               nkv: int, window: Optional[int], scale: float, workspace, lens: Sequence[int], shared: Sequence[int],
               group_rows: int, bound: int = 0) -> None:
        """One new token per row: `q` and `out` [rows, nh * head_dim], keys and values in the cache's pages already (`k_pages`
        [pages, nkv, PAGE, head_dim], `v_pages` [pages, nkv, head_dim, PAGE]).  Row r's pages are page_table[seq_slot[r]], its
        length seq_len[r].  Group g is the rows group_start[g] to group_start[g + 1] - 1, at most `group_rows` of them; they have one
        length, lens[g], and their page tables agree in the first shared[g] = group_pages[g] columns.  All of these int32 on the
        device, `lens` and `shared` lists on the host.  `q`, `out` and the pages begin on 16-byte boundaries.  `bound`: columns that
        common pages may come to fill while a recorded graph of this call is replayed."""
        hd, rows, groups = self.head_dim, q.shape[0], len(lens)
        if not self.takes(nh, nkv):
            raise KernelError(f"shared attention: {nh} query heads over {nkv} are not taken")
        dev = _here(q, "shared attention q")
        pages = k_pages.shape[0]
        if q.shape != (rows, nh * hd) or out.shape != q.shape or k_pages.shape != (pages, nkv, PAGE, hd) or \
                v_pages.shape != (pages, nkv, hd, PAGE):
            raise KernelError(f"shared attention: shapes do not fit: q {tuple(q.shape)}, out {tuple(out.shape)}, k pages "
                              f"{tuple(k_pages.shape)}, v pages {tuple(v_pages.shape)}, {nh} heads over {nkv} of {hd}")
        for t in (q, k_pages, v_pages, out):
            if t.dtype != self.dtype or not t.is_contiguous() or t.get_device() != dev:
                raise KernelError(f"shared attention: q, out, k pages and v pages must be contiguous {self.dtype} tensors on one device")
        for t, count in ((seq_len, rows), (seq_slot, rows), (group_start, groups + 1), (group_pages, groups)):
            if t.dtype != torch.int32 or t.numel() != count or not t.is_contiguous() or t.get_device() != dev:
                raise KernelError(f"shared attention: {rows} lengths and slots, {groups + 1} group starts and {groups} group pages are "
                                  f"needed, contiguous int32 on {q.device}")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1 or page_table.get_device() != dev:
            raise KernelError(f"shared attention: the page table must be int32 [slots, columns] on {q.device}")
        if rows == 0:
            return
        if len(shared) != groups or not 1 <= groups <= MAX_GROUPS or not 1 <= group_rows <= rows:
            raise KernelError(f"shared attention: one length and one number of common pages per group are needed, at most {MAX_GROUPS} "
                              "groups of at least one row")
        if min(lens) < 0 or max(lens) > page_table.shape[1] * PAGE or min(shared) < 0:
            raise KernelError(f"shared attention: lengths must lie in 0 to {page_table.shape[1] * PAGE}, numbers of pages be positive")
        if window is not None and window < 1:
            raise KernelError(f"shared attention: a window of {window}")
        if self._call is None:
            self._load()
        blocks = _sm_count(dev) * PER_SM[self.dtype]
        row_blocks, parts = shared_plan(tuple(lens), tuple(shared), group_rows, nkv, nh // nkv, window or 0, self.dtype, blocks, bound)
        part = workspace.get("attn_shared_part", (rows * nh * parts * (hd + 2),), torch.float32)
        pieces = workspace.get("attn_shared_pieces", (groups * row_blocks * nkv,), torch.int32)
        head = (q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), pages, out.data_ptr(), part.data_ptr(), pieces.data_ptr(),
                seq_len.data_ptr(), seq_slot.data_ptr(), page_table.data_ptr(), page_table.stride(0), group_start.data_ptr(),
                group_pages.data_ptr(), groups, rows, group_rows, nh, nkv)
        rest = (window or 0, scale, row_blocks, parts, blocks, _stream_on(dev))
        _check(self._call(*head, *rest) if self.dtype == torch.bfloat16 else self._call(*head, hd, *rest), "attn_shared")
        _check(0, "attn_shared_merge")


def run_shared(q, cache_view, out, batch, nh: int, nkv: int, window, scale: float, workspace) -> bool:
    """A decode step whose rows hold leading pages together (`batch.groups`).  False where no kernel takes it or too little is shared:
    the caller then uses one that reads every row's pages for itself.  (A recorded step keeps what it was recorded with: steps of one
    graph have lengths in one bucket, and either kernel is right for all of them.)"""
    g, c, hd = batch.groups, cache_view, q.shape[1] // nh
    kernel = SharedAttention.get(q.dtype, hd)
    if kernel is None or not kernel.takes(nh, nkv) or len(g.rows) > MAX_GROUPS:
        return False
    key = ("attn_shared", nkv, hd, window, q.dtype)
    if key not in batch.plans:
        batch.plans[key] = worth_sharing(g.rows, g.lens, g.shared, nkv, hd, window, q.dtype)
    if not batch.plans[key]:
        return False
    seen = min(batch.len_bucket, window + PAGE) if window else batch.len_bucket
    kernel.decode(q, c.k_pages, c.v_pages, out, batch.seq_len, batch.seq_slot, c.page_table, g.start, g.pages, nh, nkv, window, scale,
                  workspace, lens=g.lens, shared=g.shared, group_rows=max(g.rows), bound=-(-seen // PAGE))
    return True
