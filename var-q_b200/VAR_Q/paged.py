"""Paged quantized KV cache: many sequences of different lengths in one pool of pages, for serving.

``VAR_Q.quant.VAR_Q`` holds one batch whose samples all have the same length.  A server holds sequences that come, grow and go one by one: it
keeps fixed-size pages, a block table that says which pages hold a sequence, and these operators:

* ``PagedCache.append``  quantise the K and V of new tokens and write them to their slots (one launch);
* ``PagedCache.read``    the values that slots stand for;
* ``PagedCache.attend``  attention of the last tokens of every sequence over its pages: a chunk of a prompt, one token, or one scale of an
  image schedule; causal or not, with a sliding window and first tokens that stay visible; query heads may share a head of the cache; or the tokens of
  a tree that a drafting model proposes, each of which sees its ancestors;
* ``PagedCache.append_rotated``  norms and rotary positions (``VAR_Q.rotary``) of Q and K in front of ``append``, in its launch;
* ``draft_tree``  the masks and positions of drafted tokens from their parents;
* ``copy_pages``, ``move_tokens``  pages and tokens of all layers to other places: forked sequences, compacted pools, accepted drafts.

The quantization is the reference's symmetric per-token-per-head mode (VAR_Q/quant.py:92-95, 112-121) with a scale of its own for every
token and head; 2, 4 or 8 bits, for K and V separately.  ``PageTable`` is the bookkeeping on the host: which pages are free, which
belong to whom (forked sequences share full pages), and the slots of a sequence's next tokens.

Inference only: outputs have no gradient, whether or not the inputs require one.
"""
from typing import List, Optional, Sequence, Tuple

import torch

from .rotary import Rotary, _native, _norm


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

    def append_rotated(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, rotary: Rotary, positions: torch.Tensor, *,
                       norm: Optional[str] = None, q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                       eps: Optional[float] = None) -> torch.Tensor:
        """``q`` after norm and rotation (contiguous, in its type), and ``k``, after the same in fp32, and ``v`` quantised into ``slots`` as by ``append``:
        one launch, and K is rounded once, to its codes.  ``q`` ``[tokens, query heads, head_dim]``, ``k`` and ``v`` ``[tokens, heads, head_dim]``, all of one
        type; ``positions`` ``[axes, tokens]`` (or ``[tokens]``); ``norm``, the weights and ``eps`` as in ``Rotary.rotate``."""
        code, eps = _norm(norm, eps)
        return _native().paged_append_rotated(*self._pools, *rotary._handle, q, k, v, slots, positions, code, eps, q_weight, k_weight, self.eps)

    def read(self, slots: torch.Tensor, dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
        """K and V ``[tokens, heads, head_dim]`` that ``slots`` (int64 ``[tokens]``) stand for; zeros for slot -1."""
        return _native().paged_read(*self._pools, slots, dtype)

    def attend(self, q: torch.Tensor, block_table: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor, max_q: int, max_kv: int,
               softmax_scale: float, *, causal: bool = True, window: Optional[int] = None, sinks: int = 0, return_lse: bool = False,
               tree: Optional[torch.Tensor] = None):
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

        ``tree`` (with ``causal=True``): the queries are drafted tokens, not a chain.  int32 ``[tokens, words]`` of at least ``max_q`` bits a row, as
        ``draft_tree`` makes it: bit i % 32 of word i / 32 says whether the query sees drafted token i of its sequence (its own bit included).  It also sees the
        tokens in front of the drafted ones; with ``window`` (at least ``max_q``) those of the window that ends at its own position, the number of
        bits in its row behind them, and the ``sinks``.

        Returns the output in q's type and shape (contiguous); with ``return_lse`` also the float32 log of the sum of exponentials ``[tokens, query heads]``
        (-inf where nothing is seen), with which results over disjoint parts of a context can be merged."""
        return _native().paged_attend(*self._pools, q, block_table, kv_lens, q_starts, max_q, max_kv, softmax_scale, causal, window, sinks, return_lse, tree)


def draft_tree(parents: torch.Tensor, kv_lens: torch.Tensor, q_starts: torch.Tensor, max_q: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """Masks ``[tokens, ceil(max_q / 32)]`` (of no more than ``tokens`` bits a row) for ``attend(tree=...)`` and positions ``[tokens]`` of drafted tokens, both int32.

    ``parents`` (int32 ``[tokens]``): the number of a token's parent among the drafted tokens of its sequence, smaller than its own, or -1 for a child of the
    sequence's last token before them.  ``kv_lens``, ``q_starts``, ``max_q`` as for ``attend``.  A mask has the bits of a token's ancestors and its own;
    its position is that of a chain of them.  Zeros for rows that belong to no sequence.  Made once per step, for all layers."""
    return _native().paged_tree(parents, kv_lens, q_starts, max_q)


def copy_pages(caches: Sequence[PagedCache], src: torch.Tensor, dst: torch.Tensor) -> None:
    """Page ``dst[i]`` of every cache becomes a copy of its page ``src[i]`` (int64 vectors), in one launch for up to 64 caches.  The ``dst`` are all
    different and none of them is a ``src``; a pair with a page that a cache does not have (-1) copies nothing there."""
    _native().paged_copy_pages([c._pools for c in caches], src, dst)


def move_tokens(caches: Sequence[PagedCache], src: torch.Tensor, dst: torch.Tensor, starts: torch.Tensor, most: int) -> None:
    """The tokens in slots ``src[i]`` of every cache go to slots ``dst[i]`` (int64 vectors), in one launch for up to 64 caches.

    Moves ``starts[g]`` .. ``starts[g + 1] - 1`` (int32) are those of one sequence, ``most`` of them at most (a hint).  A sequence's moves go towards its front, in
    order: its ``dst`` may be the ``src`` of an earlier move, never of a later one.  All ``dst`` are different, and no other sequence has them.  A move with a slot
    that a cache does not have (-1) does nothing.  No cache may be there twice."""
    _native().paged_move_tokens([c._pools for c in caches], src, dst, starts, most)


class PageTable:
    """Which pages belong to which sequence (host memory).  A page may belong to several sequences (``fork``): then it is full, and nobody writes to it."""

    def __init__(self, num_pages: int, page_size: int):
        self.num_pages, self.page_size = num_pages, page_size
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages = {}
        self._lens = {}
        self._owners = [0] * num_pages                                   # sequences that a page belongs to

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
        """The sequence's pages are free again, but for those that others share."""
        self._give_back(self._pages.pop(seq))
        del self._lens[seq]

    def length(self, seq) -> int:
        return self._lens[seq]

    def _take(self) -> int:
        page = self._free.pop()
        self._owners[page] = 1
        return page

    def _give_back(self, pages) -> None:
        for page in reversed(pages):
            self._owners[page] -= 1
            if not self._owners[page]:
                self._free.append(page)

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
            pages.extend(self._take() for _ in range(n))
            slots.extend(pages[i // size] * size + i % size for i in range(self._lens[s], self._lens[s] + c))
            self._lens[s] += c
        return torch.tensor(slots, dtype=torch.int64, device=device)

    def fork(self, seqs: Sequence, children: Sequence, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
        """New sequences ``children[i]`` that begin as ``seqs[i]`` (which may be there several times) stands now.  They share its full pages; a last page
        that is not full gets a copy: returns pages ``src``, ``dst`` for ``copy_pages`` over the caches of all layers, before anything else is written.
        Nothing is taken if the pages do not suffice."""
        if len(seqs) != len(children) or len(set(children)) != len(children):
            raise ValueError("[VAR-Q]: a child per sequence, each child once")
        for c in children:
            if c in self._pages:
                raise ValueError(f"[VAR-Q]: sequence {c!r} is there already")
        size = self.page_size
        parted = [self._lens[s] % size != 0 for s in seqs]
        if sum(parted) > len(self._free):
            raise RuntimeError(f"[VAR-Q] {sum(parted)} pages needed, {len(self._free)} are free")
        src: List[int] = []
        dst: List[int] = []
        for s, c, part in zip(seqs, children, parted):
            full = self._lens[s] // size
            pages = self._pages[s][:full]
            for page in pages:
                self._owners[page] += 1
            if part:
                src.append(self._pages[s][full])
                dst.append(self._take())
                pages.append(dst[-1])
            self._pages[c], self._lens[c] = pages, self._lens[s]
        return torch.tensor(src, dtype=torch.int64, device=device), torch.tensor(dst, dtype=torch.int64, device=device)

    def accept(self, seqs: Sequence, counts: Sequence[int], kept: Sequence[Sequence[int]], device="cuda"):
        """Of the last ``counts[i]`` tokens of ``seqs[i]`` (a draft) those with the numbers ``kept[i]`` stay (increasing; none: all go), one behind another; what
        is behind them is given back.  Returns ``src, dst, starts, most`` for ``move_tokens`` over the caches of all layers, before anything else is
        written.  Tokens in pages that a forked sequence shares can not be taken back."""
        if not (len(seqs) == len(counts) == len(kept)) or len(set(seqs)) != len(seqs):
            raise ValueError("[VAR-Q]: a count and the numbers kept per sequence, each sequence once")
        size = self.page_size
        lists = [list(k) for k in kept]
        for s, c, k in zip(seqs, counts, lists):
            if c < 0 or c > self._lens[s] or any(a >= b for a, b in zip(k, k[1:])) or (k and (k[0] < 0 or k[-1] >= c)):
                raise ValueError(f"[VAR-Q]: sequence {s!r} of {self._lens[s]} tokens: the numbers kept must increase from 0 to {c - 1} at most")
            base = self._lens[s] - c
            first = next((base + j for j, i in enumerate(k) if i != j), base + len(k))       # from here on something is written, now or by the next tokens
            if base + len(k) < self._lens[s] or first < base + len(k):
                if any(self._owners[p] > 1 for p in self._pages[s][first // size:-(-(base + len(k)) // size)]):
                    raise ValueError(f"[VAR-Q]: the draft of sequence {s!r} lies in pages that another sequence shares")
        src: List[int] = []
        dst: List[int] = []
        starts = [0]
        for s, c, k in zip(seqs, counts, lists):
            pages, base = self._pages[s], self._lens[s] - c
            for j, i in enumerate(k):
                if i != j:
                    src.append(pages[(base + i) // size] * size + (base + i) % size)
                    dst.append(pages[(base + j) // size] * size + (base + j) % size)
            starts.append(len(src))
            self._lens[s] = base + len(k)
            n = -(-self._lens[s] // size)
            self._give_back(pages[n:])
            del pages[n:]
        longs = dict(dtype=torch.int64, device=device)
        return (torch.tensor(src, **longs), torch.tensor(dst, **longs), torch.tensor(starts, dtype=torch.int32, device=device),
                max((b - a for a, b in zip(starts, starts[1:])), default=0))

    def compact(self, device="cuda") -> Tuple[torch.Tensor, torch.Tensor]:
        """Sequences move to the first pages of the pool: afterwards the last ``free_pages`` pages are free.  Returns pages ``src``, ``dst`` for ``copy_pages``
        over the caches of all layers, before anything else is written.  Block tables and slots from before name the old pages."""
        used = self.num_pages - len(self._free)
        src = [p for p in range(used, self.num_pages) if self._owners[p]]
        dst = [p for p in range(used) if not self._owners[p]]
        place = dict(zip(src, dst))
        for s, pages in self._pages.items():
            self._pages[s] = [place.get(p, p) for p in pages]
        for a, b in place.items():
            self._owners[b], self._owners[a] = self._owners[a], 0
        self._free = list(range(self.num_pages - 1, used - 1, -1))
        return torch.tensor(src, dtype=torch.int64, device=device), torch.tensor(dst, dtype=torch.int64, device=device)

    def slots(self, seq, device="cuda") -> torch.Tensor:
        """The slots of all tokens of a sequence, in order."""
        size, pages = self.page_size, self._pages[seq]
        return torch.tensor([pages[i // size] * size + i % size for i in range(self._lens[seq])], dtype=torch.int64, device=device)

    def positions(self, seqs: Sequence, counts: Sequence[int], device="cuda") -> torch.Tensor:
        """The positions (int32) of the last ``counts[i]`` tokens of ``seqs[i]``, one sequence after another."""
        if len(seqs) != len(counts):
            raise ValueError("[VAR-Q]: a count per sequence")
        return torch.tensor([i for s, c in zip(seqs, counts) for i in range(self._lens[s] - c, self._lens[s])], dtype=torch.int32, device=device)

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
