"""Decode loops with several continuations of a sequence, over one paged cache.

``PagedKv`` owns the page pools of every layer with their block table, lengths
and reference counts, and drives the page operations of include/strata_b200.h
(``kv_fork``, ``kv_compact``, ``kv_accept``) on the plugin's stream.
``BeamDecoder`` runs beam-search steps: a fork of the cache by the parents chosen
before, then one decoder graph with the beam head.  ``TreeDecoder`` runs drafted-tree
steps: one graph that scores every node, the longest branch the argmax agrees
with, then the accepted rows kept in place.

No counterpart in the reference, whose runtime has no decode loop
(crates/ferrite-strata-runtime/src/session.rs runs one compiled graph).
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import abi
from .blocks import DecoderShape, decoder_graph
from .ir import BF16, F32, I32
from .plugin import Buffer, Device, Plugin, StrataError

_P, _I64 = C.c_void_p, C.c_int64
_FORK = [_P] + [_I64] * 5 + [_P] * 4 + [_I64] * 3 + [_P] * 6
_COMPACT = [_P] + [_I64] * 5 + [_P] * 2 + [_I64] * 2 + [_P] * 6
_ACCEPT = [_P] + [_I64] * 2 + [_P] * 4 + [_I64] * 6 + [_P] * 2
_FAULTS = {2: "a length, parent or path is out of range", 3: "a page's count is below its references",
           5: "the pool has too few free pages", 6: "a block-table entry names no page of the pool"}


def _entry(plugin: Plugin, name: str, argtypes, restype=C.c_int32):
    f = getattr(plugin.lib, "strata_b200_" + name)
    f.argtypes, f.restype = argtypes, restype
    return f


def ancestor_masks(parents) -> np.ndarray:
    """Mask words I32 [B, T, ceil(T / 32)] of drafted trees: ``parents`` [B, T] gives each node's
    parent among the nodes before it, -1 for a node that follows the cached tokens directly."""
    parents = np.asarray(parents)
    B, T = parents.shape
    sees = np.zeros((B, T, -(-T // 32) * 32), bool)
    for b in range(B):
        for t in range(T):
            p = int(parents[b, t])
            if not -1 <= p < t:
                raise ValueError(f"node {t}'s parent {p} is not one of the nodes before it")
            if p >= 0:
                sees[b, t] = sees[b, p]
            sees[b, t, t] = True
    return np.packbits(sees, axis=-1, bitorder="little").view("<u4").astype(np.uint32).view(np.int32)


class PagedKv:
    """Page pools of ``pools`` caches (every layer's k and v), ``rows`` rows of a block table of
    ``pages_per_row`` pages, and who holds which page.

    The table, lengths and counts have two buffers each and a page operation writes the ones
    that are not current, so ``side`` flips with every fork or compaction; a prepared run that
    names the table is made for either side."""

    def __init__(self, plugin: Plugin, *, pools: int, pages: int, kv_heads: int, page_size: int, head_dim: int,
                 rows: int, pages_per_row: int):
        self.plugin, self.kv_heads, self.page_size, self.pages = plugin, kv_heads, page_size, pages
        self.rows, self.pages_per_row, self.row_bytes = rows, pages_per_row, 2 * head_dim
        if not 0 < pools <= 256:
            raise ValueError("one cache has at most 256 pools")
        self._bufs: list[Buffer] = []

        def alloc(dtype, dims):
            b = plugin.alloc(dtype, dims)
            self._bufs.append(b)
            return b

        try:
            self.pools = [alloc(BF16, (pages, kv_heads, page_size, head_dim)) for _ in range(pools)]
            self._table = [alloc(I32, (rows, pages_per_row)) for _ in range(2)]
            self._lens = [alloc(I32, (rows,)) for _ in range(2)]
            self._refs = [alloc(I32, (pages,)) for _ in range(2)]
            self._parents, self._report, self._remap = alloc(I32, (rows,)), alloc(I32, (4,)), alloc(I32, (pages,))
            ws = max(_entry(plugin, "kv_fork_workspace_bytes", [_I64] * 3, C.c_uint64)(rows, pages_per_row, pages),
                     _entry(plugin, "kv_compact_workspace_bytes", [_I64], C.c_uint64)(pages))
            self._ws = alloc(I32, (max(-(-ws // 4), 1),))
            self._path = alloc(I32, (rows, 1024))
            self._n, self._base = alloc(I32, (rows,)), alloc(I32, (rows,))
            self._ptrs = (_P * pools)(*[b.device_ptr() for b in self.pools])
            self.side = 0
            self.lens = np.zeros(rows, np.int32)  # the host's copy of the rows' lengths
            self.held = np.zeros(rows, np.int64)  # positions that each row has pages for
            self._table[0].write(np.full((rows, pages_per_row), -1, np.int32))
            self._refs[0].write(np.zeros(pages, np.int32))
        except Exception:
            self.release()
            raise
        self._fork = _entry(plugin, "kv_fork", _FORK)
        self._compact = _entry(plugin, "kv_compact", _COMPACT)
        self._accept = _entry(plugin, "kv_accept", _ACCEPT)

    @property
    def table(self) -> Buffer:
        return self._table[self.side]

    def tables(self) -> list[Buffer]:
        """Both block tables, by side."""
        return list(self._table)

    def _pool_args(self):
        return self._ptrs, len(self.pools), self.row_bytes, self.kv_heads, self.page_size, self.pages

    def _check(self, rc: int, what: str) -> np.ndarray:
        if rc:
            raise StrataError(rc, f"{what} was refused")
        report = np.frombuffer(self._report.read(), np.int32)
        if report[0]:
            code = abi.RESOURCE_EXHAUSTED if report[0] == 5 else abi.INVALID_ARGUMENT
            more = f" ({report[3]} more are needed)" if report[0] == 5 else ""
            raise StrataError(code, f"{what}: {_FAULTS.get(int(report[0]), 'error')}{more}")
        return report

    def fork(self, parents, reserve: int = 1) -> np.ndarray:
        """Row r continues row ``parents[r]`` (-1: becomes empty) and gets pages for ``reserve`` more
        positions; returns [0, pages copied, pages reserved, pages left free].  On an error the
        cache stays as it was."""
        parents = np.ascontiguousarray(parents, np.int32)
        if parents.shape != (self.rows,):
            raise ValueError("one parent per row")
        a, b = self.side, 1 - self.side
        self._parents.write(parents)
        self._lens[a].write(self.lens)
        rc = self._fork(*self._pool_args(), self._table[a].device_ptr(), self._lens[a].device_ptr(),
                        self._refs[a].device_ptr(), self._parents.device_ptr(), self.rows, self.pages_per_row, reserve,
                        self._table[b].device_ptr(), self._lens[b].device_ptr(), self._refs[b].device_ptr(),
                        self._report.device_ptr(), self._ws.device_ptr(), self.plugin.stream())
        report = self._check(rc, "kv_fork")
        self.side = b
        self.lens = np.where(parents >= 0, self.lens[np.maximum(parents, 0)], 0).astype(np.int32)
        pages = -(-(self.lens.astype(np.int64) + reserve) // self.page_size)
        self.held = np.where(parents >= 0, pages * self.page_size, 0)
        return report

    def reserve(self, need) -> None:
        """Gives each row free pages for ``need[r]`` positions past its length, the lowest ids first, to
        rows in ascending order; a row that has them keeps its pages.  A row's partly filled page has
        to be its own, as a fork leaves it.  On an error the rows stay as they were."""
        need = np.asarray(need, np.int64)
        if need.shape != (self.rows,) or (need < 0).any():
            raise ValueError("one number of positions per row")
        want = -(-(self.lens + need) // self.page_size)
        if (want > self.pages_per_row).any():
            raise StrataError(abi.INVALID_ARGUMENT, "reserve: a row would pass its last page")
        for attempt in range(2):
            have = self.held // self.page_size
            more = np.maximum(want - have, 0)
            if not more.any():
                return
            refs = np.frombuffer(self._refs[self.side].read(), np.int32).copy()
            free = np.flatnonzero(refs == 0)
            if more.sum() <= free.size:
                break
            if attempt:
                raise StrataError(abi.RESOURCE_EXHAUSTED, "reserve: the pool has too few free pages "
                                                          f"({more.sum() - free.size} more are needed)")
            self.fork(np.arange(self.rows), reserve=0)  # what rows hold past their lengths goes back
        table = np.frombuffer(self.table.read(), np.int32).reshape(self.rows, self.pages_per_row).copy()
        at = 0
        for r in np.flatnonzero(more):
            table[r, have[r]:want[r]] = free[at:at + more[r]]
            at += more[r]
        refs[free[:at]] = 1
        self.table.write(table)
        self._refs[self.side].write(refs)
        self.held = np.maximum(self.held, want * self.page_size)

    def compact(self) -> np.ndarray:
        """Moves the used pages to the lowest ids; returns [0, pages used, pages moved, pages free]."""
        a, b = self.side, 1 - self.side
        rc = self._compact(*self._pool_args(), self._table[a].device_ptr(), self._refs[a].device_ptr(), self.rows,
                           self.pages_per_row, self._table[b].device_ptr(), self._refs[b].device_ptr(),
                           self._remap.device_ptr(), self._report.device_ptr(), self._ws.device_ptr(),
                           self.plugin.stream())
        report = self._check(rc, "kv_compact")
        self.side = b
        return report

    def accept(self, paths) -> None:
        """Keeps, of each row's drafted rows from its length on, those of ``paths[r]`` (strictly
        increasing node numbers, within the positions the row has pages for) and moves the length
        past them."""
        width = max([len(p) for p in paths] + [1])
        if len(paths) != self.rows or width > 1024:
            raise ValueError("one path per row, of at most 1024 nodes")
        path, n = np.zeros((self.rows, width), np.int32), np.array([len(p) for p in paths], np.int32)
        for r, p in enumerate(paths):
            if any(y <= x for x, y in zip([-1, *p], p)):
                raise ValueError("a path is strictly increasing from 0 on")
            if len(p) and self.lens[r] + p[-1] >= self.held[r]:
                raise ValueError("a path ends past the row's pages")
            path[r, :len(p)] = p
        self._path.write(path)
        self._n.write(n)
        self._base.write(self.lens)
        self._report.write(np.zeros(4, np.int32))
        rc = self._accept(self._ptrs, len(self.pools), self.row_bytes, self.table.device_ptr(), self._base.device_ptr(),
                          self._path.device_ptr(), self._n.device_ptr(), self.rows, self.kv_heads,
                          self.pages_per_row * self.page_size, width, self.page_size, self.pages,
                          self._report.device_ptr(), self.plugin.stream())
        self._check(rc, "kv_accept")
        self.lens = self.lens + n

    def release(self) -> None:
        for b in self._bufs:
            b.release()
        self._bufs.clear()


class _Decoder:
    """What the decode loops share: prefill of one row each, and the prepared runs of a step graph."""

    def __init__(self, plugin: Plugin, shape: DecoderShape, weights: dict, kv: PagedKv, fmt: str, layers: int):
        self.plugin, self.shape, self.weights, self.kv, self.fmt, self.layers = plugin, shape, weights, kv, fmt, layers
        self._bufs: list[Buffer] = []
        self._bound, self._exes = [], []

    def _alloc(self, dtype, dims) -> Buffer:
        b = self.plugin.alloc(dtype, dims)
        self._bufs.append(b)
        return b

    def _arena(self, g, hd, table: Buffer) -> dict:
        """Weights by name, the pools, and the given block table."""
        arena = {hd.block_table: Device(table)}
        for i, v in enumerate(g.values):
            if v.producer is None and v.name in self.weights:
                arena[i] = Device(self.weights[v.name])
        for li, layer in enumerate(hd.layers):
            arena[layer.ids["k_cache"]] = Device(self.kv.pools[2 * li])
            arena[layer.ids["v_cache"]] = Device(self.kv.pools[2 * li + 1])
        return arena

    def _graph(self, **kw):
        kv = self.kv
        return decoder_graph(self.shape, max_len=kv.pages_per_row * kv.page_size, fmt=self.fmt, layers=self.layers,
                             kv_page=kv.page_size, kv_pages=kv.pages, **kw)

    def _compile(self, g):
        exe = self.plugin.compile(g)
        if exe is None:
            raise StrataError(abi.DECLINED, "the plugin declined the decode step")
        self._exes.append(exe)
        return exe

    def prefill(self, prompts: dict) -> None:
        """Empties the cache and puts the tokens of ``prompts`` (row -> tokens) into it."""
        kv = self.kv
        prompts = {r: t for r, t in prompts.items() if len(t)}
        kv.fork(np.full(kv.rows, -1), reserve=0)
        if not prompts:
            return
        kv.reserve([len(prompts.get(r, ())) for r in range(kv.rows)])
        for row, tokens in prompts.items():
            n = len(tokens)
            g, hd = self._graph(batch=1, seq=n, head="none")
            bufs, exe = [], self.plugin.compile(g)
            if exe is None:
                raise StrataError(abi.DECLINED, "the plugin declined the prefill")
            try:
                table = kv.table.read(4 * kv.pages_per_row, 4 * kv.pages_per_row * row)
                for dims, data in (((1, kv.pages_per_row), table), ((n,), np.ascontiguousarray(tokens, np.int32)),
                                   ((n,), np.arange(n, dtype=np.int32))):
                    bufs.append(self.plugin.upload(I32, dims, data))
                arena = self._arena(g, hd, bufs[0])
                arena.update({hd.tokens: Device(bufs[1]), hd.pos: Device(bufs[2])})
                exe.run(arena, every_value=False)
            finally:
                exe.free()
                for b in bufs:
                    b.release()
            kv.lens[row] = n

    def release(self) -> None:
        for b in self._bound:
            b.release()
        for e in self._exes:
            e.free()
        for b in self._bufs:
            b.release()
        self._bound, self._exes, self._bufs = [], [], []


class BeamDecoder(_Decoder):
    """Beam search of ``sentences`` prompts with ``beams`` beams each: the kv cache has one row
    per beam, and sentence s's beams are rows s * beams, ...

    A step first gives every row the parent that the step before chose and room for its
    token, so the cache follows a choice when the next step starts, and a step that
    fills the rows still returns.  Ended beams take a position a step like the others."""

    def __init__(self, plugin: Plugin, shape: DecoderShape, weights: dict, kv: PagedKv, *, sentences: int, beams: int,
                 eos: int = -1, fmt: str = "w4g32", layers: int | None = None):
        super().__init__(plugin, shape, weights, kv, fmt, shape.layers if layers is None else layers)
        R = sentences * beams
        if kv.rows != R:
            raise ValueError("one cache row per beam")
        self.sentences, self.beams, self.eos = sentences, beams, eos
        self.g, self.hd = self._graph(batch=R, seq=1, head="beam", beams=beams, eos=eos)
        exe = self._compile(self.g)
        # Tokens, scores and flags ping-pong: a step's outputs are the next one's inputs.
        self._state = [(self._alloc(F32, (R,)), self._alloc(I32, (R,)), self._alloc(I32, (R,))) for _ in range(2)]
        self._pos, self._parents = self._alloc(I32, (R,)), self._alloc(I32, (R,))
        hd = self.hd
        self._runs = {}
        for side, table in enumerate(kv.tables()):
            for cur in range(2):
                arena = self._arena(self.g, hd, table)
                (s0, t0, d0), (s1, t1, d1) = self._state[cur], self._state[1 - cur]
                arena.update({hd.tokens: Device(t0), hd.scores: Device(s0), hd.done: Device(d0),
                              hd.pos: Device(self._pos)})
                for o, b in zip(hd.beam_outs, (s1, self._parents, t1, d1)):
                    arena[o] = Device(b)
                self._runs[side, cur] = exe.bind(arena)
        self._bound = list(self._runs.values())
        self._cur = 0
        self._next = np.arange(R)  # each row's parent at the next step
        self.tokens = self.parents = self.scores = self.done = None

    def start(self, prompts) -> None:
        """Prefills every sentence's prompt but its last token and spreads it over the beams."""
        W, kv = self.beams, self.kv
        if len(prompts) != self.sentences or not all(len(p) for p in prompts):
            raise ValueError("one prompt of at least one token per sentence")
        self.prefill({s * W: p[:-1] for s, p in enumerate(prompts)})
        last = [int(p[-1]) for p in prompts for _ in range(W)]
        self._next = np.repeat(np.arange(self.sentences) * W, W)
        scores = np.where(np.arange(kv.rows) % W == 0, 0.0, -np.inf).astype(np.float32)  # the beams are equal: one counts
        s, t, d = self._state[self._cur]
        s.write(scores)
        t.write(np.array(last, np.int32))
        d.write(np.zeros(kv.rows, np.int32))

    def step(self):
        """One step of every beam: (scores, parent rows, tokens, done), each [sentences, beams].
        Where the rows or the pool have no room for it, nothing changes; after another error the
        search has to start again."""
        kv = self.kv
        kv.fork(self._next, reserve=1)
        self._next = np.arange(kv.rows)
        self._pos.write(kv.lens)
        self._runs[kv.side, self._cur].run()
        self._cur = 1 - self._cur
        s, t, d = self._state[self._cur]
        shape = (self.sentences, self.beams)
        self.scores = np.frombuffer(s.read(), np.float32).reshape(shape)
        self.parents, self.tokens, self.done = (np.frombuffer(b.read(), np.int32).reshape(shape)
                                                for b in (self._parents, t, d))
        if (self.parents < 0).any():
            raise StrataError(abi.INVALID_ARGUMENT, "a sentence has fewer continuations than beams")
        kv.lens = kv.lens + 1
        self._next = self.parents.reshape(-1)
        return self.scores, self.parents, self.tokens, self.done

    def search(self, prompts, steps: int):
        """The beams after at most ``steps`` steps, best first: (tokens, scores) per sentence and beam."""
        self.start(prompts)
        W = self.beams
        hist = [[[] for _ in range(W)] for _ in range(self.sentences)]
        for _ in range(steps):
            _, parents, tokens, done = self.step()
            hist = [[hist[s][parents[s, w] - s * W] + [int(tokens[s, w])] for w in range(W)]
                    for s in range(self.sentences)]
            if done.all():
                break
        return hist, self.scores


class TreeDecoder(_Decoder):
    """Greedy decoding that checks drafted trees of ``nodes`` nodes per row.  Node 0 of every
    tree is the row's newest token, which is not in the cache yet."""

    def __init__(self, plugin: Plugin, shape: DecoderShape, weights: dict, kv: PagedKv, *, nodes: int,
                 fmt: str = "w4g32", layers: int | None = None):
        super().__init__(plugin, shape, weights, kv, fmt, shape.layers if layers is None else layers)
        self.nodes = nodes
        B = kv.rows
        self.g, self.hd = self._graph(batch=B, seq=nodes, head="argmax", tree=True)
        hd = self.hd
        exe = self._compile(self.g)
        self._ids, self._pos = self._alloc(I32, (B * nodes,)), self._alloc(I32, (B * nodes,))
        self._base, self._count = self._alloc(I32, (B,)), self._alloc(I32, (B,))
        self._mask = self._alloc(I32, (B * nodes, -(-nodes // 32)))
        self._out = self._alloc(I32, (B * nodes,))
        self._runs = []
        for table in kv.tables():
            arena = self._arena(self.g, hd, table)
            arena.update({hd.tokens: Device(self._ids), hd.pos: Device(self._pos), hd.base: Device(self._base),
                          hd.count: Device(self._count), hd.mask: Device(self._mask), hd.out: Device(self._out)})
            self._runs.append(exe.bind(arena))
        self._bound = list(self._runs)
        self.newest = np.zeros(B, np.int32)

    def start(self, prompts) -> None:
        if len(prompts) != self.kv.rows or not all(len(p) for p in prompts):
            raise ValueError("one prompt of at least one token per row")
        self.prefill({r: p[:-1] for r, p in enumerate(prompts)})
        self.newest = np.array([p[-1] for p in prompts], np.int32)

    def _make_room(self, count) -> None:
        """Pages for ``count[r]`` nodes of each row; a partly filled page becomes the row's own.  As many
        for every row as the largest tree takes, by one fork, where they fit; else each row's own."""
        kv, rows, most = self.kv, np.arange(self.kv.rows), int(count.max())
        if (kv.lens + most <= kv.pages_per_row * kv.page_size).all():
            try:
                kv.fork(rows, reserve=most)
                return
            except StrataError as e:
                if e.code != abi.RESOURCE_EXHAUSTED:
                    raise
        kv.fork(rows, reserve=0)
        kv.reserve(count)

    def step(self, drafts):
        """``drafts[r]``: (tokens, parents) of row r's drafted nodes, parents among the nodes before
        (0: the newest token), or None for a row that sits the step out.  Returns, per row, the tokens
        the model's argmax accepts and the one it adds: at least one, none for a row that sits out.
        Where a row or the pool has no room for its nodes, nothing changes."""
        kv, T, B = self.kv, self.nodes, self.kv.rows
        ids, parents = np.zeros((B, T), np.int32), np.zeros((B, T), np.int32)
        pos, count = np.zeros((B, T), np.int32), np.zeros(B, np.int32)
        if len(drafts) != B:
            raise ValueError("one draft, or None, per row")
        for r, draft in enumerate(drafts):
            if draft is None:
                parents[r, 0] = -1
                pos[r] = kv.lens[r]
                continue
            tokens, par = draft
            n = 1 + len(tokens)
            if n > T or len(par) != len(tokens):
                raise ValueError(f"a tree has at most {T} nodes, its first the newest token")
            ids[r, 0], parents[r, 0], count[r] = self.newest[r], -1, n
            ids[r, 1:n], parents[r, 1:n] = tokens, par
            if any(not 0 <= p < t + 1 for t, p in enumerate(par)):
                raise ValueError("a drafted node follows one of the nodes before it")
            for t in range(1, n):
                pos[r, t] = pos[r, parents[r, t]] + 1
            pos[r] += kv.lens[r]
        self._make_room(count)
        for b, x in ((self._ids, ids), (self._pos, pos), (self._base, kv.lens), (self._count, count),
                     (self._mask, ancestor_masks(parents))):
            b.write(np.ascontiguousarray(x))
        self._runs[kv.side].run()
        best = np.frombuffer(self._out.read(), np.int32).reshape(B, T)
        paths, found = [], []
        for r in range(B):
            if not count[r]:
                paths.append([])
                found.append([])
                continue
            path, got = [0], [int(best[r, 0])]
            while True:
                nxt = next((t for t in range(path[-1] + 1, count[r])
                            if parents[r, t] == path[-1] and ids[r, t] == got[-1]), None)
                if nxt is None:
                    break
                path.append(nxt)
                got.append(int(best[r, nxt]))
            paths.append(path)
            found.append(got)
            self.newest[r] = got[-1]
        kv.accept(paths)
        return found
