"""A paged key/value cache for RACLlamaBlock: sequences, their pages, and steps over them.

The keys and values of every layer lie in pages of ``page_size`` rows,
``k`` and ``v`` [layers, pages, kv_heads, page_size, dim]; a sequence owns a list of
pages, the same in every layer.  Which page belongs to whom is kept on the
host (a free list and reference counts); the rows are moved by kernels.

    cache = RACPagedCache(n_layers, n_pages, n_kv_heads, dim)
    a = cache.add()
    step = cache.step([a], len(prompt))          # reserves rows for the prompt
    for i, block in enumerate(blocks):
        x = block(x, is_causal=True, cache=step, layer=i)
    b = cache.fork(a)                            # shares a's full pages
    step = cache.step([a, b], 1)                 # one token each
    step = cache.step([a], 5, parents=[-1, 0, 0, 1, 1])   # a tree of drafted tokens
    cache.accept(step, [[0, 2]])                 # keeps nodes 0 and 2
    cache.free(b)
"""
from __future__ import annotations

import torch

from . import ext


class RACCacheStep:
    """The new rows of some sequences: where they go and what they see.  Made by RACPagedCache.step,
    handed to every layer's forward in turn."""

    def __init__(self, cache, ids, starts, counts, parents, table):
        self.cache, self.ids, self.starts_host, self.counts_host = cache, ids, starts, counts
        self.parents = parents
        self._turns = [cache._turns[i] for i in ids]
        self.tokens = sum(counts)
        self.width = max(counts)
        self.longest = max(s + n for s, n in zip(starts, counts))
        self.uniform = all(n == self.width for n in counts)
        # A prompt: nothing but new rows, each seeing those before it.
        self.is_prompt = parents is None and not any(starts)
        b, pw = len(ids), max(len(t) for t in table)
        depth = [None if parents is None else _depths(p) for p in (parents or [None] * b)]
        cu = [0]
        for n in counts:
            cu.append(cu[-1] + n)
        pos = [s + (i if d is None else d[i]) for s, n, d in zip(starts, counts, depth) for i in range(n)]
        flat = [p for t in table for p in t + [0] * (pw - len(t))]
        ints = flat + starts + [s + n for s, n in zip(starts, counts)] + counts + cu + pos
        dev = cache.k.device
        ints = torch.tensor(ints, dtype=torch.int32).to(dev)
        sizes = [b * pw, b, b, b, b + 1, self.tokens]
        table_, self.starts, self.lengths, self.counts, self.cu_seqlens, self.positions = ints.split(sizes)
        self.page_table = table_.view(b, pw)
        self.tree = None
        if parents is not None:
            rows = []
            for p in parents:
                m = _masks(p)
                rows += m + [0] * (self.width - len(m))
            self.tree = torch.tensor(rows, dtype=torch.int64).view(b, self.width).to(dev)
        self._pad = None
        if not self.uniform:
            at = [i * self.width + j for i, n in enumerate(counts) for j in range(n)]
            self._pad = torch.tensor(at, dtype=torch.int64).to(dev)

    def attend(self, layer: int, q, k, v, scale: float | None = None) -> torch.Tensor:
        """Writes k, v [tokens, kv_heads, dim] into layer's pages and returns the attention of
        q [tokens, heads, dim] over the cache, [tokens, heads, dim]."""
        c = self.cache
        if self.stale():
            raise ValueError("the sequences of this step have moved on: take a new step")
        if any(c._forked.get(i) == t for i, t in zip(self.ids, self._turns)):
            raise ValueError("a sequence of this step was forked before all layers had run: take a new step")
        kp, vp = c.k[layer], c.v[layer]
        k, v = k.to(c.dtype), v.to(c.dtype)
        ext.cache_append_(kp, vp, k, v, self.page_table, self.starts, self.cu_seqlens)
        if self.is_prompt:
            return ext.attention_packed(q.to(c.dtype), k, v, self.cu_seqlens, True, scale).to(q.dtype)
        b, (t, h, hd) = len(self.ids), q.shape
        if self.uniform:
            qb = q.to(c.dtype).reshape(b, self.width, h, hd)
        else:
            qb = q.new_zeros((b * self.width, h, hd), dtype=c.dtype)
            qb[self._pad] = q.to(c.dtype)
            qb = qb.view(b, self.width, h, hd)
        o = ext.attention_cached(qb, kp, vp, self.page_table, self.lengths, None if self.uniform else self.counts,
                                 self.tree, scale)
        o = o.view(b * self.width, h, hd)
        return (o if self.uniform else o[self._pad]).to(q.dtype)

    def stale(self) -> bool:
        """Whether one of the sequences has taken another step, been cut back or freed since."""
        return any(self.cache._turns.get(i) != t for i, t in zip(self.ids, self._turns))


def _depths(parents: list[int]) -> list[int]:
    d = []
    for p in parents:
        d.append(0 if p < 0 else d[p] + 1)
    return d


def _masks(parents: list[int]) -> list[int]:
    """For each node the bits of itself and of the nodes above it, as signed 64-bit values."""
    m = []
    for i, p in enumerate(parents):
        m.append((1 << i) | (m[p] if p >= 0 else 0))
    return [x - (1 << 64) if x >> 63 else x for x in m]


class RACPagedCache:
    """Keys and values of n_layers layers in n_pages pages of page_size rows."""

    def __init__(self, n_layers: int, n_pages: int, n_kv_heads: int, head_dim: int, page_size: int = 64,
                 dtype: torch.dtype = torch.float32, device="cuda"):
        if min(n_layers, n_pages, n_kv_heads, page_size) < 1:
            raise ValueError("n_layers, n_pages, n_kv_heads and page_size must be at least 1")
        ext._check_heads(n_kv_heads, n_kv_heads, head_dim)
        if dtype not in ext._ELEM:
            raise ValueError(f"float32, float16 or bfloat16 required, got {dtype}")
        shape = (n_layers, n_pages, n_kv_heads, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.page_size, self.dtype = page_size, dtype
        self._free = list(range(n_pages - 1, -1, -1))
        self._uses = [0] * n_pages                 # sequences that hold the page
        self._seqs: dict[int, tuple[list[int], int]] = {}
        self._turns: dict[int, int] = {}           # of each sequence, how often its rows have changed
        self._forked: dict[int, int] = {}          # the count at which it was last forked
        self._next = 0

    # ── sequences ──
    def add(self) -> int:
        """A new, empty sequence."""
        self._next += 1
        self._seqs[self._next - 1] = ([], 0)
        self._turns[self._next - 1] = 0
        return self._next - 1

    def length(self, seq: int) -> int:
        return self._get(seq)[1]

    def pages(self, seq: int) -> list[int]:
        return list(self._get(seq)[0])

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _get(self, seq: int):
        if seq not in self._seqs:
            raise ValueError(f"no sequence {seq} in the cache")
        return self._seqs[seq]

    def _take(self, n: int) -> list[int]:
        if n > len(self._free):
            raise RuntimeError(f"{n} pages needed, {len(self._free)} free")
        got = [self._free.pop() for _ in range(n)]
        for p in got:
            self._uses[p] = 1
        return got

    def _drop(self, pages: list[int]) -> None:
        for p in pages:
            self._uses[p] -= 1
            if self._uses[p] == 0:
                self._free.append(p)

    def _copy(self, src: list[int], dst: list[int]) -> None:
        if src:
            at = torch.tensor([src, dst], dtype=torch.int32).to(self.k.device)
            ext.cache_copy_pages_(self.k, self.v, at[0], at[1])

    def _shared(self, places: list[tuple[list[int], int]]) -> list[tuple[list[int], int]]:
        """Of places (a sequence's pages, index) that are to be written to, those whose page another sequence keeps."""
        uses, got = list(self._uses), []
        for pages, at in places:
            if uses[pages[at]] > 1:
                uses[pages[at]] -= 1
                got.append((pages, at))
        return got

    def _replace(self, places: list[tuple[list[int], int]], new: list[int]) -> None:
        """Puts copies, on the pages `new`, in these places."""
        src = [pages[at] for pages, at in places]
        for (pages, at), p in zip(places, new):
            pages[at] = p
        self._drop(src)
        self._copy(src, new)

    def fork(self, seq: int) -> int:
        """A new sequence with seq's rows.  Full pages are shared; a page that is partly filled is copied.  The rows
        of seq's last step have to be there, in every layer: none of its layers runs after the fork."""
        pages, n = self._get(seq)
        whole = n // self.page_size
        last = self._take(len(pages) - whole)
        self._copy(pages[whole:], last)
        for p in pages[:whole]:
            self._uses[p] += 1
        new = self.add()
        self._seqs[new] = (pages[:whole] + last, n)
        self._forked[seq] = self._turns[seq]
        return new

    def free(self, seq: int) -> None:
        """Gives up a sequence; pages that nobody else holds are free again."""
        pages, _ = self._get(seq)
        del self._seqs[seq], self._turns[seq]
        self._forked.pop(seq, None)
        self._drop(pages)

    def truncate(self, seq: int, length: int) -> None:
        """Forgets seq's rows from `length` on."""
        pages, n = self._get(seq)
        if not 0 <= length <= n:
            raise ValueError(f"length must be between 0 and {n}, got {length}")
        if length == n:
            return
        self._turns[seq] += 1
        keep = -(-length // self.page_size)
        self._seqs[seq] = (pages[:keep], length)
        self._drop(pages[keep:])

    # ── steps ──
    def step(self, seqs: list[int], n_new, parents=None) -> RACCacheStep:
        """Reserves n_new new rows (one number, or one a sequence) for each sequence.  parents: the tree of
        the new rows, node i's parent or -1, one list for all sequences or one each; without it each new row
        sees the ones before it.  Rows that see a cache, or a tree, are at most 64 a sequence."""
        seqs = list(seqs)
        if not seqs or len(set(seqs)) != len(seqs):
            raise ValueError("a step takes at least one sequence, each of them once")
        counts = [n_new] * len(seqs) if isinstance(n_new, int) else list(n_new)
        if len(counts) != len(seqs) or any(n < 1 for n in counts):
            raise ValueError(f"n_new must give each of the {len(seqs)} sequences at least one row")
        have = [self._get(s) for s in seqs]
        if parents is not None:
            parents = [list(p) for p in parents] if parents and not isinstance(parents[0], int) \
                else [list(parents)] * len(seqs)
            if len(parents) != len(seqs) or any(len(p) != n for p, n in zip(parents, counts)):
                raise ValueError("parents must name one parent for each new row")
            if any(not -1 <= q < i for p in parents for i, q in enumerate(p)):
                raise ValueError("a node's parent must be -1 or a node before it")
        if (parents is not None or any(n for _, n in have)) and max(counts) > ext.MAX_NEW_ROWS:
            raise ValueError(f"at most {ext.MAX_NEW_ROWS} new rows over a cache or in a tree, got {max(counts)}")
        ps = self.page_size
        # A page that new rows are written to and that others hold too is copied first.  Counted before
        # anything is taken: a step that does not fit changes nothing.
        lists = [list(pages) for pages, _ in have]
        shared = self._shared([(p, n // ps) for p, (_, n) in zip(lists, have) if n % ps])
        grow = [-(-(n + c) // ps) - len(p) for p, (_, n), c in zip(lists, have, counts)]
        new = self._take(len(shared) + sum(grow))
        at = len(shared)
        self._replace(shared, new[:at])
        for i, g in enumerate(grow):
            lists[i] += new[at:at + g]
            at += g
        starts = [n for _, n in have]
        for s, p, n, c in zip(seqs, lists, starts, counts):
            self._seqs[s] = (p, n + c)
            self._turns[s] += 1
        return RACCacheStep(self, seqs, starts, counts, parents, lists)

    def accept(self, step: RACCacheStep, accepted: list[list[int]]) -> None:
        """Keeps the given new rows of a step (rising node numbers, one list a sequence) and forgets the
        others: the kept rows move together in every layer, the sequences shorten to them.  Pages that others
        hold too, forks of these sequences, are copied before a row moves into them."""
        if step.cache is not self or step.stale():
            raise ValueError("not the latest step of these sequences")
        if len(accepted) != len(step.ids):
            raise ValueError(f"accepted must have one list for each of {len(step.ids)} sequences")
        for a, n in zip(accepted, step.counts_host):
            if any(not 0 <= x < n for x in a) or any(x >= y for x, y in zip(a, a[1:])):
                raise ValueError("accepted nodes must be rising numbers of the step's new rows")
        if any(a != list(range(len(a))) for a in accepted):
            if step.width > ext.MAX_NEW_ROWS:
                raise ValueError(f"at most {ext.MAX_NEW_ROWS} new rows can be moved together")
            w, b, ps = step.width, len(accepted), self.page_size
            lists = [list(self._get(i)[0]) for i in step.ids]
            into = [sorted({(s + i) // ps for i, x in enumerate(a) if x != i})
                    for s, a in zip(step.starts_host, accepted)]
            shared = self._shared([(p, at) for p, ats in zip(lists, into) for at in ats])
            table = step.page_table
            if shared:
                self._replace(shared, self._take(len(shared)))
                for i, p in zip(step.ids, lists):
                    self._seqs[i] = (p, self.length(i))
                flat = [x for p in lists for x in p + [0] * (table.shape[1] - len(p))]
                table = torch.tensor(flat, dtype=torch.int32).view(table.shape).to(self.k.device)
            flat = [x for a in accepted for x in list(a) + [0] * (w - len(a))] + [len(a) for a in accepted]
            t = torch.tensor(flat, dtype=torch.int32).to(self.k.device)
            ext.cache_compact_(self.k, self.v, table, step.starts, t[:b * w].view(b, w), t[b * w:])
        for i, s, a in zip(step.ids, step.starts_host, accepted):
            self.truncate(i, s + len(a))
