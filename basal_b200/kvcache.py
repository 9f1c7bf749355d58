"""A paged key / value cache: the pages of every attention layer, which sequence holds which of them, and forks that
share them. The reference answers from one prefill pass and keeps whole key / value buffers; a model that goes on from
there token by token (hybrid.HybridClassifier.open / step / answer) keeps its keys and values here.

  PagedKVCache(layers, pages, kv_heads, head_dim, page_size, dtype, fp8, device)
      .add()                  a new, empty sequence -> its number
      .fork(seq)              a new sequence with seq's tokens, its pages shared and counted (nothing is copied). What
                              seq last grew by is appended before: a batch made after the fork brings nothing of it
      .grow(seqs, n)          room for n more tokens in each of seqs: new pages, and a copy of a shared page before it
                              is written (one basal::kv_copy_pages over every layer); raises MemoryError, with nothing
                              changed, when the free pages do not suffice
      .batch(seqs)            -> Batch: the sequences' table and lengths on the device, for append and attend
      .append(layer, batch, k, v), .attend(layer, batch, q, scale, window)
                              basal::kv_append of the tokens that grow() made room for, basal::paged_attention
      .free(seq)              gives its pages back
      .compact()              moves the live pages to the lowest numbers (one kv_copy_pages) -> how many pages are live

The bookkeeping is on the host; the device sees the pages, and tables and lengths as int32 tensors. A Batch says how things
were when it was made: after grow, free or compact, make another (outside of a captured graph). The copies run on the
current stream: use the cache from one stream, or order the streams.
"""
import dataclasses

import numpy as np
import torch

from . import ops

E4M3 = torch.float8_e4m3fn


@dataclasses.dataclass
class Batch:
    """Some sequences, in order, as the kernels see them: table [rows, width], the lengths [rows] with the tokens that
    the last grow() made room for, where those begin and how many they are (0 for a sequence that it did not name, or
    that was forked since: an append leaves it as it is)."""
    seqs: list
    table: torch.Tensor
    lengths: torch.Tensor
    start: torch.Tensor
    count: torch.Tensor
    most: int = 0  # the largest count


class PagedKVCache:
    def __init__(self, layers, pages, kv_heads, head_dim, page_size=64, dtype=torch.bfloat16, fp8=False,
                 device="cuda"):
        if head_dim not in (64, 128, 256):
            raise ValueError(f"PagedKVCache: heads of 64, 128 or 256, not {head_dim}")
        if dtype not in (torch.bfloat16, torch.float16):
            raise ValueError(f"PagedKVCache: keys and values of bfloat16 or float16, not {dtype}")
        if min(layers, pages, kv_heads, page_size) <= 0:
            raise ValueError("PagedKVCache: layers, pages, kv_heads and page_size must be positive")
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.device = torch.device(device)
        self.page_size, self.pages, self.dtype = page_size, pages, dtype
        self.k = torch.empty(shape, dtype=E4M3 if fp8 else dtype, device=self.device)
        self.v = torch.empty_like(self.k)
        self.k_scale = torch.empty(shape[:4], dtype=torch.float32, device=self.device) if fp8 else None
        self.v_scale = torch.empty_like(self.k_scale) if fp8 else None
        self._free = list(range(pages - 1, -1, -1))
        self._shares = [0] * pages   # sequences that hold a page
        self._of = {}                # sequence -> its pages, in order
        self._row = {}               # the same as an array, made again after a change: a long cache's table is not built
                                     # page by page at every step
        self._length = {}
        self._new = {}               # sequence -> tokens that the last grow() made room for, where it named the sequence
        self._next = 0

    @property
    def pools(self):
        return [p for p in (self.k, self.v, self.k_scale, self.v_scale) if p is not None]

    @property
    def free_pages(self):
        return len(self._free)

    def _known(self, seq):
        if seq not in self._of:
            raise KeyError(f"PagedKVCache: no sequence {seq}")
        return self._of[seq]

    def length(self, seq):
        self._known(seq)
        return self._length[seq]

    def pages_of(self, seq):
        return list(self._known(seq))

    def add(self):
        seq, self._next = self._next, self._next + 1
        self._of[seq], self._length[seq] = [], 0
        return seq

    def fork(self, seq):
        pages = self._known(seq)
        new = self.add()
        self._of[new], self._length[new] = list(pages), self._length[seq]
        for p in pages:
            self._shares[p] += 1
        self._new.pop(seq, None)  # its last page is shared now
        return new

    def free(self, seq):
        for p in self._known(seq):
            self._shares[p] -= 1
            if not self._shares[p]:
                self._free.append(p)
        del self._of[seq], self._length[seq]
        self._new.pop(seq, None)
        self._row.pop(seq, None)

    def grow(self, seqs, n=1):
        """n: tokens for each sequence, a number or a list."""
        seqs = list(seqs)
        n = [n] * len(seqs) if isinstance(n, int) else list(n)
        if len(n) != len(seqs) or len(set(seqs)) != len(seqs) or min(n, default=0) < 0:
            raise ValueError("PagedKVCache: grow takes each sequence once, with its number of tokens")
        # the shared page that a sequence writes into next is replaced by a copy; of the sequences that share a page
        # and all write it, the last keeps it
        left, copies, need = {}, [], 0
        for s, m in zip(seqs, n):
            pages, length = self._known(s), self._length[s]
            if m and length % self.page_size:
                p = pages[length // self.page_size]
                if left.get(p, self._shares[p]) > 1:
                    left[p] = left.get(p, self._shares[p]) - 1
                    copies.append(s)
                    need += 1
            need += max(0, -(-(length + m) // self.page_size) - len(pages))
        if need > len(self._free):
            raise MemoryError(f"PagedKVCache: {need} pages are needed, {len(self._free)} are free")
        # the copies come first: where they are refused, nothing has changed
        where = [self._length[s] // self.page_size for s in copies]
        src = [self._of[s][at] for s, at in zip(copies, where)]
        dst = [self._free[-1 - i] for i in range(len(copies))]
        if src:
            ops.kv_copy_pages(self.pools, src, dst)
        for s, at, old, new in zip(copies, where, src, dst):
            self._free.pop()
            self._shares[old] -= 1
            self._shares[new] = 1
            self._of[s][at] = new
            self._row.pop(s, None)
        self._new = dict(zip(seqs, n))
        for s, m in zip(seqs, n):
            pages = self._of[s]
            while len(pages) * self.page_size < self._length[s] + m:
                self._row.pop(s, None)
                pages.append(self._free.pop())
                self._shares[pages[-1]] = 1
            self._length[s] += m

    def batch(self, seqs):
        seqs = list(seqs)
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("PagedKVCache: a graph would keep the host memory that a batch is copied from: make the "
                               "batch before the capture, and copy later ones over its tensors")
        width = max([len(self._known(s)) for s in seqs], default=0) or 1
        host = torch.empty((len(seqs), width + 3), dtype=torch.int32, pin_memory=self.device.type == "cuda")
        rows = host.numpy()
        for i, s in enumerate(seqs):
            pages = self._row.get(s)
            if pages is None:
                pages = self._row[s] = np.asarray(self._of[s], np.int32)
            rows[i, :len(pages)] = pages
            rows[i, len(pages):width] = -1
            new = self._new.get(s, 0)
            rows[i, width:] = self._length[s], self._length[s] - new, new
        t = host.to(self.device, non_blocking=True)
        lengths, start, count = t[:, width:].t().contiguous()
        return Batch(seqs, t[:, :width], lengths, start, count, max([self._new.get(s, 0) for s in seqs], default=0))

    def _layer(self, i):
        return (self.k[i], self.v[i]), (None, None) if self.k_scale is None else (self.k_scale[i], self.v_scale[i])

    def append(self, layer, batch, k, v):
        if k.dim() > 1 and k.shape[1] < batch.most:
            raise ValueError(f"PagedKVCache: {k.shape[1]} tokens, where grow made room for {batch.most}")
        (pk, pv), (ks, vs) = self._layer(layer)
        ops.kv_append(k, v, pk, pv, batch.table, batch.start, batch.count, ks, vs)

    def attend(self, layer, batch, q, scale, window=0):
        (pk, pv), (ks, vs) = self._layer(layer)
        return ops.paged_attention(q, pk, pv, batch.table, batch.lengths, scale, window, ks, vs)

    def compact(self):
        live = [p for p in range(self.pages) if self._shares[p]]
        n = len(live)
        holes = [p for p in range(n) if not self._shares[p]]
        movers = [p for p in live if p >= n]  # as many as there are holes below n
        if movers:
            ops.kv_copy_pages(self.pools, movers, holes)
            to = dict(zip(movers, holes))
            for pages in self._of.values():
                pages[:] = [to.get(p, p) for p in pages]
            self._row.clear()
            for a, b in to.items():
                self._shares[b], self._shares[a] = self._shares[a], 0
        self._free = list(range(self.pages - 1, n - 1, -1))
        return n
