"""Decode attention of rows that share the leading pages of their cache (kernels in attention_shared.cu and
attention_shared_f32.cu): the beams of a search, which have one prompt.  Shared pages are read once for all rows of a group."""
from __future__ import annotations

from ctypes import c_float, c_int, c_longlong, c_void_p
from functools import lru_cache
from typing import Dict, Optional, Sequence, Tuple

import torch

from . import build
from .ops import KernelError, _check, _here, _need, _sm_count, _stream, register_error_word

HEAD_DIMS = (64, 128)
PAGE = build.PAGE_TOKENS
MAX_PARTS = 64                 # partial results of a row and head that the merge takes
BLOCK_ROWS = 32                # rows (of a group, times query heads) that one block holds
MAX_GROUP = {torch.bfloat16: 16, torch.float32: 32}     # query heads per key/value head

for _hd in HEAD_DIMS:
    build.register_library(f"attn_shared_bf16_hd{_hd}", ("attention_shared.cu",), (f"-DHEAD_DIM={_hd}",))
build.register_library("attn_shared_f32", ("attention_shared_f32.cu",), ())

# What the plan knows about the kernels (measured on a B200, head size 128)
PAGE_US = {torch.bfloat16: 1.0, torch.float32: 2.8}     # a block alone, a page
SETUP_US = 1.5                                          # a block's start and the write of its partial results
MERGE_US, PART_US = 2.5, 0.03                           # the second kernel, and what every part adds to it
HBM_GBS = 6500.0
PER_SM = {torch.bfloat16: 2, torch.float32: 1}          # resident blocks


@lru_cache(maxsize=4096)
def shared_plan(lens: Tuple[int, ...], shared: Tuple[int, ...], group_rows: int, nkv: int, group: int, head_dim: int,
                window: int, dtype: torch.dtype, sms: int, bound: int = 0) -> Tuple[int, int, int]:
    """(splits, quantum, tails): blocks that share a group's common pages of one kv head and the pages of each, and blocks that
    share a row's own pages.  `lens` and `shared` per group: length and pages in common; `bound`: columns that the common pages may
    come to fill (0: as they are), of which `splits` is a function.  The quantum with the least estimated time: blocks run
    on sms * PER_SM places, a page takes a block PAGE_US unless all together ask more of the memory than HBM_GBS."""
    size = 2 if dtype == torch.bfloat16 else 4
    common, own = [], []
    for n, c in zip(lens, shared):
        first = max(0, n - window) // PAGE if window else 0
        end = -(-n // PAGE)
        border = min(max(c, first), end)
        common.append(border - first)
        own.append(end - border)
    row_blocks = -(-group_rows // (BLOCK_ROWS // group))
    page_us = PAGE_US[dtype] * head_dim / 128
    places = sms * PER_SM[dtype]
    pages = nkv * (sum(common) * row_blocks + sum(own) * group_rows)
    floor = nkv * (sum(common) + sum(own) * group_rows) * PAGE * head_dim * 2 * size / (HBM_GBS * 1e3)
    longest, most = max(common), max(own)
    widest = max(longest, most, 1)
    best = None
    for q in [k for k in (1, 2, 3, 4, 5, 6, 7, 8, 10, 12, 14, 16, 20, 24, 28, 32, 40, 48, 64, 96, 128, 192, 256) if k < widest] + [widest]:
        tails = max(1, -(-most // q))
        splits = max(1, -(-max(longest, bound) // q))
        if splits + tails > MAX_PARTS:
            continue
        blocks = nkv * (sum(-(-c // q) for c in common) * row_blocks + sum(min(o, tails) for o in own) * group_rows)
        work = pages * page_us + blocks * SETUP_US
        t = max(floor + SETUP_US, work / places + 0.5 * (min(q, widest) * page_us + SETUP_US), min(q, widest) * page_us + SETUP_US)
        t += MERGE_US + PART_US * (splits + tails)
        if best is None or t < 0.99 * best[0]:
            best = (t, splits, q, tails)
    if best is None:             # very long: as many parts as the merge takes
        tails = max(1, min(MAX_PARTS // 2, -(-most // 256)))
        splits = MAX_PARTS - tails
        return splits, max(1, -(-max(longest, bound) // splits)), tails
    return best[1:]


class SharedAttention:
    _known: Dict[tuple, "SharedAttention"] = {}

    @classmethod
    def get(cls, dtype: torch.dtype, head_dim: int) -> Optional["SharedAttention"]:
        """The kernels for this type and head size, or None where there are none (the per-row kernels then read the same
        pages through the same tables)."""
        if dtype not in MAX_GROUP or head_dim not in HEAD_DIMS:
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
        head = [P, P, P, L, P, P, P, P, P, I, P, P, I, I, I, I, I]
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
        return nkv > 0 and nh % nkv == 0 and nh // nkv <= MAX_GROUP[self.dtype]

    def decode(self, q: torch.Tensor, k_pages: torch.Tensor, v_pages: torch.Tensor, out: torch.Tensor, seq_len: torch.Tensor,
               seq_slot: torch.Tensor, page_table: torch.Tensor, group_start: torch.Tensor, group_pages: torch.Tensor, nh: int,
               nkv: int, window: Optional[int], scale: float, workspace, lens: Sequence[int], shared: Sequence[int],
               group_rows: int, bound: int = 0) -> None:
        """One new token per row: `q` and `out` [rows, nh * head_dim], keys and values in the cache's pages already (`k_pages`
        [pages, nkv, PAGE, head_dim], `v_pages` [pages, nkv, head_dim, PAGE]).  Row r's pages are page_table[seq_slot[r]], its
        length seq_len[r].  Group g is the rows group_start[g] to group_start[g + 1] - 1, at most `group_rows` of them; they have one
        length, lens[g], and their page tables agree in the first shared[g] = group_pages[g] columns.  All of these int32 on the
        device, `lens` and `shared` lists on the host.  `bound`: columns that common pages may come to fill while a recorded
        graph of this call is replayed."""
        hd, rows, groups = self.head_dim, q.shape[0], len(lens)
        if not self.takes(nh, nkv):
            raise KernelError(f"shared attention: {nh} query heads over {nkv} are not taken")
        _here(q, "shared attention q")
        for t, n in ((q, "q"), (k_pages, "k pages"), (v_pages, "v pages"), (out, "out")):
            _need(t, self.dtype, f"shared attention {n}")
        pages = k_pages.shape[0]
        if q.shape != (rows, nh * hd) or out.shape != q.shape or k_pages.shape != (pages, nkv, PAGE, hd) or \
                v_pages.shape != (pages, nkv, hd, PAGE):
            raise KernelError(f"shared attention: shapes do not fit: q {tuple(q.shape)}, out {tuple(out.shape)}, k pages "
                              f"{tuple(k_pages.shape)}, v pages {tuple(v_pages.shape)}, {nh} heads over {nkv} of {hd}")
        for t, n, count in ((seq_len, "lengths", rows), (seq_slot, "slots", rows), (group_start, "group starts", groups + 1),
                            (group_pages, "group pages", groups)):
            _need(t, torch.int32, f"shared attention {n}")
            if t.numel() != count:
                raise KernelError(f"shared attention: {count} {n} are needed, got {t.numel()}")
        if page_table.dtype != torch.int32 or page_table.dim() != 2 or page_table.stride(1) != 1:
            raise KernelError("shared attention: the page table must be int32 [slots, columns]")
        for t, n in ((k_pages, "k pages"), (v_pages, "v pages"), (out, "out"), (seq_len, "lengths"), (seq_slot, "slots"),
                     (page_table, "page table"), (group_start, "group starts"), (group_pages, "group pages")):
            if t.device != q.device:
                raise KernelError(f"shared attention: {n} lie on {t.device}, q on {q.device}")
        if rows == 0:
            return
        if len(shared) != groups or groups == 0 or not 1 <= group_rows <= rows:
            raise KernelError("shared attention: one length and one number of common pages per group are needed")
        if min(lens) < 0 or max(lens) > page_table.shape[1] * PAGE or min(shared) < 0:
            raise KernelError(f"shared attention: lengths must lie in 0 to {page_table.shape[1] * PAGE}, numbers of pages be positive")
        if window is not None and window < 1:
            raise KernelError(f"shared attention: a window of {window}")
        if self._call is None:
            self._load()
        splits, quantum, tails = shared_plan(tuple(lens), tuple(shared), group_rows, nkv, nh // nkv, hd, window or 0, self.dtype,
                                             _sm_count(q.device), bound)
        part = workspace.get("attn_shared_part", (rows * nh * (splits + tails) * (hd + 2),), torch.float32)
        head = (q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), pages, out.data_ptr(), part.data_ptr(), seq_len.data_ptr(),
                seq_slot.data_ptr(), page_table.data_ptr(), page_table.stride(0), group_start.data_ptr(), group_pages.data_ptr(),
                groups, rows, group_rows, nh, nkv)
        rest = (window or 0, scale, splits, quantum, tails, _stream())
        _check(self._call(*head, *rest) if self.dtype == torch.bfloat16 else self._call(*head, hd, *rest), "attn_shared")
        _check(0, "attn_shared_merge")


def run_shared(q, cache_view, out, batch, nh: int, nkv: int, window, scale: float, workspace) -> bool:
    """A decode step whose rows hold leading pages together (`batch.groups`).  False where no kernel takes it: the caller
    then uses one that reads every row's pages for itself."""
    kernel = SharedAttention.get(q.dtype, q.shape[1] // nh)
    if kernel is None or not kernel.takes(nh, nkv):
        return False
    g, c = batch.groups, cache_view
    seen = min(batch.len_bucket, window + PAGE) if window else batch.len_bucket
    kernel.decode(q, c.k_pages, c.v_pages, out, batch.seq_len, batch.seq_slot, c.page_table, g.start, g.pages, nh, nkv, window, scale,
                  workspace, lens=g.lens, shared=g.shared, group_rows=max(g.rows), bound=-(-seen // PAGE))
    return True
