"""An uncompressed KV cache of pages, for batches that the Fourier cache does not take: sequences of different lengths,
prompts that never reach the compressed span, requests that share a long prefix.

No counterpart in the reference, whose uncompressed sequences are dense tensors grown by ``torch.cat``
(cache_utils_fourier.py:681-686) behind a library attention (modeling_llama_fourier.py:627-633).  Keys and values of
every layer live in ``(num_pages, kv_heads, page_size, head_dim)`` tensors; one page table serves all layers.
``LlamaSdpaAttention`` hands its projections to :meth:`PagedCache.attend`: one launch norms, rotates and stores, the
next ones attend.
"""
from typing import List, Optional, Sequence, Union

import torch

from . import ops
from .cache_utils_fourier import Cache

__all__ = ["PagedCache"]


class PagedCache(Cache):
    """``batch`` sequences of up to ``max_tokens`` keys each (a shared prefix not counted), in ``num_pages`` pages of
    ``page_size`` keys per layer (default: as many as all sequences need at their longest, and a prefix of
    ``max_tokens``)."""

    def __init__(self, num_layers: int, num_kv_heads: int, head_dim: int, batch: int, max_tokens: int,
                 num_pages: Optional[int] = None, page_size: int = 64, dtype=torch.bfloat16, device=None):
        super().__init__()
        if min(num_layers, num_kv_heads, batch, max_tokens) < 1:
            raise ValueError("PagedCache: sizes must be positive")
        if page_size < 16 or page_size % 16:
            raise ValueError(f"PagedCache: the page size must be a multiple of 16 (got {page_size})")
        if head_dim not in (64, 128):
            raise ValueError(f"PagedCache: the head dimension must be 64 or 128 (got {head_dim})")
        if dtype not in (torch.float16, torch.bfloat16):
            raise ValueError(f"PagedCache: unsupported dtype {dtype}")
        if device is None:
            if not torch.cuda.is_available():
                raise RuntimeError("fourierattention_b200.PagedCache needs a CUDA device (there is no CPU path)")
            device = torch.device("cuda", torch.cuda.current_device())
        self.batch, self.max_tokens, self.page_size = batch, max_tokens, page_size
        self.max_pages = -(-max_tokens // page_size)
        self.num_pages = num_pages if num_pages is not None else (batch + 1) * self.max_pages
        if self.num_pages < 1:
            raise ValueError("PagedCache: num_pages must be positive")
        shape = (self.num_pages, num_kv_heads, page_size, head_dim)
        self.k_pages = [torch.empty(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.v_pages = [torch.empty(shape, dtype=dtype, device=device) for _ in range(num_layers)]
        self.device = self.k_pages[0].device
        self.page_table = torch.zeros((batch, self.max_pages), dtype=torch.int32, device=self.device)
        self.kv_lens = torch.zeros((batch,), dtype=torch.int32, device=self.device)
        self.cu_seqlens: Optional[torch.Tensor] = None      # of the current step; None: one token per sequence
        self._cu_seqlens = torch.zeros((batch + 1,), dtype=torch.int32, device=self.device)   # in one place: captured steps read it
        self.prefix_pages: Optional[torch.Tensor] = None
        self.prefix_len = 0
        self.lengths: List[int] = [0] * batch               # host copy of kv_lens
        self._pages: List[List[int]] = [[] for _ in range(batch)]
        self._free: List[int] = list(range(self.num_pages - 1, -1, -1))
        self._plan: Optional[List[int]] = None              # new tokens of the next step, where given
        self._prefix_ids: List[int] = []
        self._before = None                                 # lengths and plan before the step begun last

    # -------------------------------------------------------------------------------------------- steps
    def plan(self, new_tokens: Sequence[int]):
        """New tokens of every sequence in the next step; the model is then called on all of them packed in one row,
        ``(1, sum(new_tokens))``.  Without a plan every sequence gets the same number, ``(batch, n)``."""
        new_tokens = [int(n) for n in new_tokens]
        if len(new_tokens) != self.batch or min(new_tokens) < 0 or sum(new_tokens) == 0:
            raise ValueError(f"plan: {self.batch} numbers of new tokens are wanted, not all of them 0")
        self._plan = new_tokens

    @property
    def planned(self) -> Optional[List[int]]:
        """New tokens of every sequence in the next step, where :meth:`plan` gave them."""
        return self._plan

    def begin_step(self, rows: int, tokens: int):
        """Makes room for the new tokens of a model call on ``(rows, tokens)`` input ids.  Host work, not to be captured: a
        captured step is that of the layers, and this call comes before each of its replays."""
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedCache.begin_step cannot be captured: a replay would move on the lengths, not the pages; "
                               "capture the layers and call begin_step before each replay")
        new = self._plan
        if new is None:
            if rows != self.batch:
                raise ValueError(f"{rows} rows of tokens for {self.batch} sequences: call plan() for packed tokens")
            new = [tokens] * self.batch
        elif (rows, tokens) != (1, sum(new)):
            raise ValueError(f"the plan is of (1, {sum(new)}) tokens, got ({rows}, {tokens})")
        lengths = [a + b for a, b in zip(self.lengths, new)]
        if max(lengths) > self.max_tokens:
            raise ValueError(f"a sequence of {max(lengths)} tokens, the cache holds {self.max_tokens}")
        grow = [-(-n // self.page_size) - len(p) for n, p in zip(lengths, self._pages)]
        if sum(grow) > len(self._free):
            raise RuntimeError(f"PagedCache: {sum(grow)} pages wanted, {len(self._free)} of {self.num_pages} are free")
        self._before = self.lengths, self._plan
        self._plan = None
        for b, n in enumerate(grow):
            for _ in range(n):
                self._pages[b].append(self._free.pop())
        if sum(grow):
            self._upload_table()
        self.lengths = lengths
        if all(n == 1 for n in new):
            self.kv_lens.add_(1)
            self.cu_seqlens = None
        else:
            at = [0]
            for n in new:
                at.append(at[-1] + n)
            self.kv_lens.copy_(torch.tensor(lengths, dtype=torch.int32))
            self._cu_seqlens.copy_(torch.tensor(at, dtype=torch.int32))
            self.cu_seqlens = self._cu_seqlens

    def cancel_step(self):
        """Takes back the step begun last, for one whose layers failed: the cache and its plan are as before."""
        if self._before is None:
            raise RuntimeError("cancel_step: no step has been begun")
        lengths, self._plan = self._before
        self._before = None
        for b, n in enumerate(lengths):
            self.truncate(b, n)

    def _upload_table(self):
        self.page_table.copy_(torch.tensor([p + [0] * (self.max_pages - len(p)) for p in self._pages], dtype=torch.int32))

    def attend(self, q, k, v, layer_idx: int, inv_freq, positions=None, q_weight=None, k_weight=None, eps: float = 1e-6,
               sm_scale: Optional[float] = None):
        """Stores the new tokens of the step in layer ``layer_idx`` and attends them.  q: (tokens, Hq, D), k, v:
        (tokens, Hkv, D), not yet rotated; returns (tokens, Hq, D)."""
        kp, vp = self.k_pages[layer_idx], self.v_pages[layer_idx]
        q = ops.paged_append(k, v, kp, vp, self.page_table, self.kv_lens, inv_freq, cu_seqlens=self.cu_seqlens,
                             positions=positions, pos_offset=self.prefix_len, q=q, q_weight=q_weight, k_weight=k_weight,
                             eps=eps)
        return ops.paged_attention(q, kp, vp, self.page_table, self.kv_lens, cu_seqlens=self.cu_seqlens,
                                   prefix_pages=self.prefix_pages, prefix_len=self.prefix_len, sm_scale=sm_scale)

    def last_rows(self, hidden):
        """The hidden state of the last new token of every sequence, (batch, 1, hidden); zeros for one without new tokens in
        the step."""
        if self.cu_seqlens is None:
            return hidden.reshape(self.batch, 1, -1)
        rows = hidden.reshape(-1, hidden.shape[-1])
        end, idle = self.cu_seqlens[1:].long(), self.cu_seqlens[1:] == self.cu_seqlens[:-1]
        return rows[(end - 1).clamp(min=0)].masked_fill(idle[:, None], 0)[:, None]

    # -------------------------------------------------------------------------------------------- sequences
    def share_prefix(self, sequence: int = 0):
        """Makes the tokens of ``sequence`` the prefix of every sequence of the batch: its pages are read once for all of
        them.  The sequence itself starts anew behind the prefix; every other one must be empty."""
        if self.prefix_len:
            raise RuntimeError("the cache has a prefix already")
        if any(n for b, n in enumerate(self.lengths) if b != sequence):
            raise RuntimeError("share_prefix: the other sequences must be empty")
        if not self.lengths[sequence]:
            raise RuntimeError("share_prefix: the sequence is empty")
        self._before = None
        self._prefix_ids, self.prefix_len = self._pages[sequence], self.lengths[sequence]
        self.prefix_pages = torch.tensor(self._prefix_ids, dtype=torch.int32, device=self.device)
        self._pages[sequence], self.lengths[sequence] = [], 0
        self.kv_lens.zero_()

    def truncate(self, sequence: int, length: int = 0):
        """Drops the tokens of ``sequence`` from ``length`` on and frees the pages behind them (0: the sequence has ended,
        its place takes another)."""
        if not 0 <= length <= self.lengths[sequence]:
            raise ValueError(f"truncate: {length} of {self.lengths[sequence]} tokens")
        self._before = None
        keep = -(-length // self.page_size)
        self._free.extend(reversed(self._pages[sequence][keep:]))
        self._pages[sequence] = self._pages[sequence][:keep]
        self.lengths[sequence] = length
        self.kv_lens[sequence] = length

    def reset(self):
        """Drops every sequence and the prefix."""
        for b in range(self.batch):
            self.truncate(b)
        self._free.extend(reversed(self._prefix_ids))
        self._prefix_ids, self.prefix_pages, self.prefix_len = [], None, 0
        self.cu_seqlens = self._plan = None

    def get_seq_length(self, layer_idx: Optional[int] = 0) -> int:
        """Length of the longest sequence, the prefix included."""
        return self.prefix_len + max(self.lengths)

    def get_max_cache_shape(self) -> Optional[int]:
        return self.max_tokens

    def update(self, key_states, value_states, layer_idx, cache_kwargs: Union[dict, None] = None):
        raise NotImplementedError("PagedCache stores keys before they are rotated: use attend()")
