"""Paged quantized KV cache: many sequences of different lengths in one pool of pages, for serving.

``VAR_Q.quant.VAR_Q`` holds one batch whose samples all have the same length.  A server holds sequences that come, grow and go one by one: it
keeps fixed-size pages, a block table that says which pages hold a sequence, and three operators:

* ``PagedCache.append``  quantise the K and V of new tokens and write them to their slots (one launch);
* ``PagedCache.read``    the values that slots stand for;
* ``PagedCache.attend``  attention of the last tokens of every sequence over its pages: a chunk of a prompt, one token, or one scale of an
  image schedule; causal or not, with a sliding window and first tokens that stay visible; query heads may share a head of the cache.

The quantization is the reference's symmetric per-token-per-head mode (VAR_Q/quant.py:92-95, 112-121) with a scale of its own for every
token and head; 2, 4 or 8 bits, for K and V separately.  ``PageTable`` is the bookkeeping on the host: which pages are free, which
belong to whom, and the slots of a sequence's next tokens.

Inference only: outputs have no gradient, whether or not the inputs require one.
"""
from typing import List, Optional, Sequence, Tuple

import torch

from . import _cabi
from .quant import _host


def _native():
    return _host if _host is not None else _cabi.lib()                    # which says what to build


class PagedCache:
    """Pools of quantized K and V: ``k_codes`` / ``v_codes`` int32 ``[num_pages, num_heads, page_size, head_dim * bits / 32]``, ``k_scale`` /
    ``v_scale`` fp32 ``[num_pages, num_heads, page_size]``.  ``page_size`` is a power of two from 16 to 1024, ``head_dim`` 64 or 128.  A slot is
    ``page * page_size + offset``; what is not written is never looked at, so the pools start uninitialised."""

    def __init__(self, num_pages: int, page_size: int, num_heads: int, head_dim: int, k_bits: int = 8, v_bits: int = 8, device="cuda"):
        for bits in (k_bits, v_bits):
            if bits not in (2, 4, 8):
                raise ValueError(f"[VAR-Q]: bits must be 2, 4 or 8 (got {bits})")
        if head_dim not in (64, 128):
            raise ValueError(f"[VAR-Q]: head_dim {head_dim} is not 64 or 128")
        if page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
            raise ValueError(f"[VAR-Q]: page_size must be a power of two from 16 to 1024 (got {page_size})")
        if num_pages < 1 or num_heads < 1:
            raise ValueError(f"[VAR-Q]: {num_pages} pages, {num_heads} heads")
        shape = (num_pages, num_heads, page_size)
        self._set(*(torch.empty((*shape, head_dim * b // 32), dtype=torch.int32, device=device) for b in (k_bits, v_bits)),
                  *(torch.empty(shape, dtype=torch.float32, device=device) for _ in range(2)), head_dim)

    @classmethod
    def over(cls, k_codes: torch.Tensor, v_codes: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor, head_dim: int) -> "PagedCache":
        """A cache over pools that are there already.  Scales may be 0 (``attend`` takes V scales below 2^-100 for 2^-100); they are not negative."""
        cache = cls.__new__(cls)
        cache._set(k_codes, v_codes, k_scale, v_scale, head_dim)
        return cache

    def _set(self, k_codes, v_codes, k_scale, v_scale, head_dim):
        self.k_codes, self.v_codes, self.k_scale, self.v_scale, self.head_dim = k_codes, v_codes, k_scale, v_scale, head_dim
        self._pools = (k_codes, v_codes, k_scale, v_scale, head_dim)
        self.num_pages, self.num_heads, self.page_size = k_codes.shape[:3]
        self.eps = 1e-12

    @property
    def k_bits(self) -> int:
        return self.k_codes.size(3) * 32 // self.head_dim

    @property
    def v_bits(self) -> int:
        return self.v_codes.size(3) * 32 // self.head_dim

    def append(self, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor) -> None:
        """Quantise ``k`` and ``v`` ``[tokens, heads, head_dim]`` (float32, float16 or bfloat16; strided views are fine) into ``slots`` (int64
        ``[tokens]``, all different).  Slot -1 writes nothing: a padding token.  A row that holds a NaN or an infinity reads as NaN throughout."""
        _native().paged_append(*self._pools, k, v, slots, self.eps)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """K and V ``[tokens, heads, head_dim]`` that ``slots`` (int64 ``[tokens]``) stand for; zeros for slot -1."""
        return _native().paged_read(*self._pools, slots, dtype)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor, max_q: int, max_kv: int,
               softmax_scale: float, *, causal: bool = True, window: Optional[int] = None, sinks: int = 0, return_lse: bool = False):
        """softmax(q k^T * softmax_scale) v over the pages of every sequence.

        ``q`` ``[tokens, query heads, head_dim]`` (float16 or bfloat16) holds the queries of all sequences one after another, those of sequence
        b in rows ``q_starts[b]`` .. ``q_starts[b + 1] - 1`` (int32, one entry more than sequences).  They are its last tokens: with n queries and
        ``kv_lens[b]`` tokens in the cache (int32, the chunk's own tokens included) query i stands at position ``kv_lens[b] - n + i``.
        ``block_table`` (int32 ``[sequences, pages]``): the pages of a sequence in order; what stands for pages behind its last token, or for pages in
        which no query sees a key any more, does not matter.
        ``max_q`` / ``max_kv``: bounds of a sequence's queries and tokens, so that nothing has to come back from the device.

        Rows of ``q`` in front of ``q_starts[0]`` and behind ``q_starts[-1]`` belong to no sequence (a batch padded to a fixed size): zeros, and -inf.

        ``causal=False``: every query sees the whole sequence.  ``causal=True``: a query at position p sees the keys up to p, with ``window`` only
        the last ``window`` of them and the first ``sinks`` keys of the sequence.  A query that sees nothing gets zeros.
        Returns the output in q's type and shape (contiguous); with ``return_lse`` also the float32 log of the sum of exponentials ``[tokens, query heads]``
        (-inf where nothing is seen), with which results over disjoint parts of a context can be merged."""
        return _native().paged_attend(*self._pools, q, block_table, kv_lens, q_starts, max_q, max_kv, softmax_scale, causal, window, sinks, return_lse)


class PageTable:
    """Which pages belong to which sequence (host memory)."""

    def __init__(self, num_pages: int, page_size: int):
        self.page_size = page_size
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages = {}
        self._lens = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def __contains__(self, seq) -> bool:
        return seq in self._pages

    def add(self, seq) -> None:
        """A new, empty sequence."""
        if seq in self._pages:
            raise ValueError(f"[VAR-Q]: sequence {seq!r} is there already")
        self._pages[seq], self._lens[seq] = [], 0

    def remove(self, seq) -> None:
        """The sequence's pages are free again."""
        self._free.extend(reversed(self._pages.pop(seq)))
        del self._lens[seq]

    def length(self, seq) -> int:
        return self._lens[seq]

    def extend(self, seqs: Sequence, counts: Sequence[int], device="cuda") -> torch.Tensor:
        """Room for ``counts[i]`` more tokens of ``seqs[i]``; their slots, one sequence after another.  Nothing is taken if the pages do not
        suffice for all of them."""
        if len(seqs) != len(counts) or len(set(seqs)) != len(seqs) or any(c < 0 for c in counts):
            raise ValueError("[VAR-Q]: a count per sequence, each sequence once")
        size = self.page_size
        lacking = [max(0, -(-(self._lens[s] + c) // size) - len(self._pages[s])) for s, c in zip(seqs, counts)]
        if sum(lacking) > len(self._free):
            raise RuntimeError(f"[VAR-Q] {sum(lacking)} pages needed, {len(self._free)} are free")
        slots: List[int] = []
        for s, c, n in zip(seqs, counts, lacking):
            pages = self._pages[s]
            pages.extend(self._free.pop() for _ in range(n))
            slots.extend(pages[i // size] * size + i % size for i in range(self._lens[s], self._lens[s] + c))
            self._lens[s] += c
        return torch.tensor(slots, dtype=torch.int64, device=device)

    def slots(self, seq, device="cuda") -> torch.Tensor:
        """The slots of all tokens of a sequence, in order."""
        size, pages = self.page_size, self._pages[seq]
        return torch.tensor([pages[i // size] * size + i % size for i in range(self._lens[seq])], dtype=torch.int64, device=device)

    def batch(self, seqs: Sequence, counts: Sequence[int], device="cuda"):
        """``block_table, kv_lens, q_starts, max_q, max_kv`` for ``attend`` with the last ``counts[i]`` tokens of ``seqs[i]`` as queries."""
        if len(seqs) != len(counts):
            raise ValueError("[VAR-Q]: a count per sequence")
        width = max((len(self._pages[s]) for s in seqs), default=0)
        table = [self._pages[s] + [-1] * (width - len(self._pages[s])) for s in seqs]
        lens, starts = [self._lens[s] for s in seqs], [0]
        for c in counts:
            starts.append(starts[-1] + c)
        ints = dict(dtype=torch.int32, device=device)
        return (torch.tensor(table, **ints).view(len(table), width), torch.tensor(lens, **ints), torch.tensor(starts, **ints), max(counts, default=0),
                max(lens, default=0))
