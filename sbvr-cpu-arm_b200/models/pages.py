"""A KV cache in pages, for sequences that come and go and that begin alike (`PagedCache`).

Sequences live in slots.  A page holds `page_size` consecutive tokens of a sequence, K and V of all layers; a slot's row of `table` names its
pages, and slots that begin with the same tokens hold the same pages (`fork`).  Which page goes where is decided on the GPU: no call waits for
it, and all but those that are given lists can be captured into a graph.  What cannot be done (no free page, a sequence beyond `max_pages`, a slot
named twice) changes nothing and is reported by `check()`.

The reference keeps the Hugging Face cache of its vendored Llama (models/sbvr_llama.py:330-336), one tensor per sequence batch and layer, and has
no counterpart of these calls.
"""
from __future__ import annotations

import ctypes
import math
from typing import List, Optional, Union

import torch

from sbvr import _lib

Slots = Union[torch.Tensor, List[int], None]


class PagedCache:
    """`pool` fp16 [layers, 2 (K, V), pages, n_kv, page_size, 128]; `table` int32 [max_seqs, max_pages], -1 where there is no page; `lengths`
    int32 [max_seqs]; `refs` int32 [pages], how many slots hold a page.  The last three and `status` lie in `book`, so that a copy of that tensor
    keeps who holds what (not what the pages hold).

    `reserve`, `free`, `fork`, `copy`, `compact` and `rope_append` change the cache: the caller orders them with every other call on it (other streams).
    `attention` and `common` only read it and may overlap one another.
    """

    FORK_PAIRS = 1024                              # of one fork or copy, which does all of them at once

    def __init__(self, layers: int, n_kv: int, pages: int, page_size: int = 64, max_seqs: int = 64, max_pages: Optional[int] = None,
                 head_dim: int = 128, device="cuda"):
        if head_dim != 128:
            raise ValueError("the attention kernels serve head_dim 128")
        if page_size not in (16, 32, 64, 128, 256):
            raise ValueError(f"page_size must be 16, 32, 64, 128 or 256, not {page_size}")
        max_pages = pages if max_pages is None else max_pages
        if min(layers, n_kv, pages, max_seqs, max_pages) < 1:
            raise ValueError("layers, n_kv, pages, max_seqs and max_pages must be positive")
        if max_seqs > 65536:
            raise ValueError("at most 65536 slots")
        if max(pages * n_kv * page_size, max_pages * page_size, max_pages * max_seqs) >= 2 ** 30:
            raise ValueError("rows of a layer's pages, tokens of a slot and entries of the table must each be fewer than 2^30")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError(f"SBVR kernels run on CUDA tensors only (there is no CPU path); got device {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.layers, self.n_kv, self.pages, self.page_size, self.head_dim = layers, n_kv, pages, page_size, head_dim
        self.max_seqs, self.max_pages = max_seqs, max_pages
        i32 = dict(dtype=torch.int32, device=self.device)
        self.pool = torch.zeros((layers, 2, pages, n_kv, page_size, head_dim), dtype=torch.float16, device=self.device)
        seqs4, pages4 = (max_seqs + 3) // 4 * 4, (pages + 3) // 4 * 4
        self.book = torch.zeros(4 + seqs4 + pages4 + max_seqs * max_pages, **i32)
        self.status, self.lengths = self.book[:1], self.book[4:4 + max_seqs]
        self.refs = self.book[4 + seqs4:4 + seqs4 + pages]
        self.table = self.book[4 + seqs4 + pages4:].view(max_seqs, max_pages)
        self.table.fill_(-1)
        self._c = _lib.Pages(pool=self.pool.data_ptr(), table=self.table.data_ptr(), lengths=self.lengths.data_ptr(), refs=self.refs.data_ptr(),
                             status=self.status.data_ptr(), scratch=None, layers=layers, pages=pages, page=page_size, n_kv=n_kv, head_dim=head_dim,
                             max_seqs=max_seqs, max_pages=max_pages)
        need = ctypes.c_size_t(0)
        _lib.check(_lib.lib.sbvr_pages_scratch_bytes(ctypes.byref(self._c), ctypes.byref(need)), "sbvr_pages_scratch_bytes")
        self._scratch = torch.empty((need.value + 3) // 4, **i32)
        self._c.scratch = self._scratch.data_ptr()
        self._at = ctypes.addressof(self._c)

    # ------------------------------------------------------------------ who holds what
    def _slots(self, slots: Slots, what: str = "slots", twice: bool = False) -> torch.Tensor:
        """A list of slots as the device tensor that the kernels read; lists are checked here, tensors on the GPU."""
        if isinstance(slots, torch.Tensor):
            return slots
        slots = [int(s) for s in slots]
        if not slots or min(slots) < 0 or max(slots) >= self.max_seqs:
            raise ValueError(f"{what} must name some of the cache's {self.max_seqs} slots")
        if not twice and len(set(slots)) < len(slots):
            raise ValueError(f"{what} names a slot twice")
        return torch.tensor(slots, dtype=torch.int32, device=self.device)

    def _tokens(self, tokens):
        if isinstance(tokens, (torch.Tensor, int)):
            return tokens
        return torch.tensor([int(t) for t in tokens], dtype=torch.int32, device=self.device)

    def reserve(self, slots: Slots, tokens, tokens_per_seq: int = 0) -> Optional[torch.Tensor]:
        """Room for `tokens` (one number, or one per slot) more tokens in every slot (None: in all).  With `tokens_per_seq`: their positions, int32
        [slots * tokens_per_seq], -1 behind a slot's last."""
        if isinstance(tokens, int) and tokens < 0:
            raise ValueError("tokens must not be negative")
        return _lib.native.pages_reserve(self._at, self.device.index, None if slots is None else self._slots(slots), self.max_seqs,
                                         self._tokens(tokens), tokens_per_seq)

    def free(self, slots: Slots) -> None:
        """The slots hold nothing afterwards."""
        _lib.native.pages_free(self._at, self.device.index, self._slots(slots))

    def fork(self, src: Slots, dst: Slots) -> None:
        """Slot dst[i] becomes what slot src[i] is, all at once (at most FORK_PAIRS): whole pages in common, the tokens of a part-filled last page
        copied."""
        _lib.native.pages_fork(self._at, self.device.index, self._slots(src, "src", True), self._slots(dst, "dst"), 1)

    def copy(self, src: Slots, dst: Slots) -> None:
        """The same with pages of its own for every dst."""
        _lib.native.pages_fork(self._at, self.device.index, self._slots(src, "src", True), self._slots(dst, "dst"), 0)

    def compact(self) -> None:
        """Moves pages so that the U pages in use are pages 0 .. U - 1."""
        _lib.native.pages_compact(self._at, self.device.index)

    def common(self, slots: Slots, group_starts: torch.Tensor) -> torch.Tensor:
        """Tokens that the sequences slots[group_starts[g] : group_starts[g + 1]] hold in the same pages, int32 [groups]: `shared` of `attention`."""
        return _lib.native.pages_common(self._at, self.device.index, None if slots is None else self._slots(slots, twice=True), self.max_seqs, group_starts)

    def check(self) -> None:
        """Raises for what earlier calls could not do, once.  Waits for the GPU."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            said = [text for bit, text in ((_lib.PAGES_NO_PAGE, "fewer free pages than a call needed"),
                                           (_lib.PAGES_TOO_LONG, f"a sequence beyond {self.max_pages} pages"),
                                           (_lib.PAGES_BAD_SLOT, "a slot out of range or named twice, or a negative number of tokens"),
                                           (_lib.PAGES_NO_ENTRY, "a token where its slot has no page")) if bits & bit]
            raise RuntimeError("paged cache: " + "; ".join(said or [f"status {bits}"]))

    # ------------------------------------------------------------------ a layer's tokens
    def rope_append(self, layer: int, qkv: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor, slots: Slots = None, scaling: float = 1.0,
                    q_out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """qkv [tokens, (n_heads + 2 n_kv) * 128], as many tokens for every slot of `slots` (None: of all, in order), at `positions` (below 0: a place of the batch that holds no
        token).  Returns the rotated queries; k and v go to the slots' pages."""
        return _lib.native.pages_rope_append(self._at, self.device.index, layer, qkv, positions, inv_freq, scaling,
                                             None if slots is None else self._slots(slots, twice=True), self.max_seqs, q_out)

    def attention(self, layer: int, q: torch.Tensor, positions: torch.Tensor, slots: Slots = None, scale: Optional[float] = None,
                  group_starts: Optional[torch.Tensor] = None, shared: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Causal attention of q [tokens, n_heads * 128] (rows may lie apart) over the slots' tokens 0 .. positions[token].  `group_starts` [groups
        + 1] and `shared` [groups] (from `common`): sequences group_starts[g] .. of the batch hold their first shared[g] tokens in the same pages, so
        the first one's may be read once for all of them (they are for fewer than 64 rows per sequence, tokens times heads per KV head, where that
        saves enough; else every sequence's own).  Scores and sums are fp32, weights are rounded to fp16 once for their product with V (2^-11 of each;
        the dense cache's attention keeps 2^-22 and more).  A row whose scores are all -inf is NaN, one at a position below 0 zeros."""
        return _lib.native.pages_attention(self._at, self.device.index, layer, q, positions, None if slots is None else self._slots(slots, twice=True),
                                           self.max_seqs, 1.0 / math.sqrt(self.head_dim) if scale is None else scale, group_starts, shared, out)
