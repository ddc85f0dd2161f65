"""Decode steps with several continuations of a sequence, through the plugin:
the tree and beam graphs, and the page operations run together as the decode
loops of strata_host.decoding use them.

On the CPU the oracle's tree step must equal sequential decode steps along every
branch.  On the GPU the graphs are compared with the oracle, a speculative loop
with plain greedy decoding, and a beam search with one that re-reads every beam
from its prompt."""
import ctypes

import numpy as np
import pytest

from oracle import graph_eval, oracle as ora
from strata_host import (BF16, F32, I32, BeamDecoder, Device, GraphBuilder, Op, PagedKv, StrataError, TreeDecoder,
                         ancestor_masks)
from strata_host.blocks import DecoderShape, decoder_graph
from tests.helpers import TOL_BF16, assert_close, page_table, seeded_graph_inputs, to_device_bytes

SMALL = DecoderShape(256, 4, 2, 64, 512, 300, 2)


def _copy(d):
    return {k: (v.copy() if isinstance(v, np.ndarray) else v) for k, v in d.items()}


def _by_name(g):
    return {v.name: i for i, v in enumerate(g.values) if v.producer is None}


PARENTS = np.array([[-1, 0, 0, 1, 2, 2, 5], [-1, 0, 1, 2, 3, 1, 0]])


def tree_inputs(shape, base, max_len, page=0, parents=PARENTS, count=None, fmt="w4g32", head="logits"):
    B, T = parents.shape
    g, hd = decoder_graph(shape, batch=B, seq=T, max_len=max_len, fmt=fmt, head=head, tree=True, kv_page=page,
                          kv_pages=B * max_len // page + 3 if page else None)
    host = seeded_graph_inputs(g, cache_fill=max(base))
    depth = np.zeros((B, T), np.int32)
    for t in range(1, T):
        depth[:, t] = np.where(parents[:, t] >= 0, depth[np.arange(B), parents[:, t]] + 1, 0)
    host[hd.tokens] = ora.uniform_i32(2, B * T, 0, shape.vocab)
    host[hd.pos] = (np.array(base, np.int32)[:, None] + depth).reshape(-1)
    host[hd.base] = np.array(base, np.int32)
    host[hd.count] = np.full(B, T, np.int32) if count is None else np.array(count, np.int32)
    host[hd.mask] = ancestor_masks(parents).reshape(B * T, -1)
    if page:
        host[hd.block_table] = page_table(B, max_len // page, B * max_len // page + 3)
    return g, hd, host


def test_ancestor_masks():
    m = ancestor_masks(np.array([[-1, 0, 0, 2] + [3] * 31])).view(np.uint32)
    assert m.shape == (1, 35, 2)
    assert [int(x) for x in m[0, :4, 0]] == [1, 3, 5, 13] and int(m[0, 34, 1]) == 1 << 2
    assert int(m[0, 34, 0]) == 13
    for bad in ([[0]], [[-1, 1]], [[-1, -2]]):
        with pytest.raises(ValueError):
            ancestor_masks(np.array(bad))


def test_decoder_graph_refuses_what_the_heads_cannot_do():
    kw = dict(batch=4, seq=1, max_len=64)
    for bad in (dict(head="beam"), dict(head="beam", beams=3), dict(head="beam", beams=2, tp_world=2),
                dict(head="beam", beams=2, seq=2), dict(tree=True, fmt="f32"),
                dict(tree=True, seq=4, last_token=True)):
        with pytest.raises(ValueError):
            decoder_graph(SMALL, **{**kw, **bad})


@pytest.mark.parametrize("page", [0, 16])
def test_oracle_tree_step_equals_decoding_along_each_branch(page):
    """Each leaf's logits equal those of decoding its branch token by token."""
    base, max_len = [20, 9], 48
    g, hd, host = tree_inputs(SMALL, base, max_len, page=page)
    got = graph_eval.evaluate(g, _copy(host))[hd.out].reshape(2, 7, -1)
    gs, hs = decoder_graph(SMALL, batch=2, seq=1, max_len=max_len, fmt="w4g32", head="logits", kv_page=page,
                           kv_pages=2 * max_len // page + 3 if page else None)
    names, snames = _by_name(g), _by_name(gs)
    vals = {snames[n]: host[i].copy() for n, i in names.items() if n in snames and n not in ("ids", "pos")}
    for leaf in (3, 4, 6):
        chains = []
        for b in range(2):
            chain, t = [], leaf
            while t >= 0:
                chain.insert(0, t)
                t = int(PARENTS[b, t])
            chains.append(chain)
        run = _copy(vals)
        for step in range(max(map(len, chains))):
            ids = [host[hd.tokens].reshape(2, 7)[b, c[min(step, len(c) - 1)]] for b, c in enumerate(chains)]
            pos = [base[b] + min(step, len(c) - 1) for b, c in enumerate(chains)]
            run[hs.tokens], run[hs.pos] = np.array(ids, np.int32), np.array(pos, np.int32)
            vals_after = graph_eval.evaluate(gs, run)
            want = vals_after[hs.out]
            run.update({i: vals_after[i] for n, i in snames.items() if n.endswith(("cache", "pages"))})
            for b, c in enumerate(chains):
                if step >= len(c) - 1:
                    assert np.allclose(got[b, leaf], want[b], rtol=2e-2, atol=2e-2 * np.abs(want).max())


@pytest.mark.parametrize("change,status", [
    (dict(mask_words=2), "invalid"), (dict(heads=3), "invalid"), (dict(table=False), "invalid"),
    (dict(f32=True), "declined"), (dict(head_dim=32), "declined")])
def test_tree_node_is_checked(plugin, change, status):
    B, T, H, G, d = 2, 5, change.get("heads", 4), 2, change.get("head_dim", 64)
    act = F32 if change.get("f32") else BF16
    b = GraphBuilder("t")
    q, k, v = (b.input(act, (B * T, n * d), x) for n, x in ((H, "q"), (G, "k"), (G, "v")))
    page = "table" in change
    kc, vc = (b.input(act, (8, G, 16, d) if page else (B, G, 64, d), x) for x in ("kc", "vc"))
    ins = [q, k, v, kc, vc, b.input(I32, (B,), "base"), b.input(I32, (B,), "count"),
           b.input(I32, (B * T, change.get("mask_words", 1)), "mask")]
    attrs = {"num_heads": H, "num_kv_heads": G, "head_dim": d, **({"page_size": 16} if page else {})}
    b.output(b.node(Op.custom("fused::tree_attention"), ins, [(act, (B * T, H * d))], attrs, "n")[0])
    if status == "declined":
        assert plugin.compile(b.build()) is None
    else:
        with pytest.raises(StrataError):
            plugin.compile(b.build())


@pytest.mark.parametrize("change,status", [
    (dict(), "ok"), (dict(beams=3), "invalid"), (dict(eos=50), "invalid"), (dict(outs=3), "declined"),
    (dict(keep=65), "declined"), (dict(scores=5), "invalid")])
def test_beam_node_is_checked(plugin, change, status):
    rows, beams, keep = 8, change.get("beams", 4), change.get("keep", 4)
    b = GraphBuilder("t")
    ins = [b.input(BF16, (rows, 50), "x"), b.input(F32, (change.get("scores", rows),), "s"), b.input(I32, (rows,), "d")]
    n = rows // beams * keep
    outs = [(F32, (n,)), (I32, (n,)), (I32, (n,)), (I32, (n,))][:change.get("outs", 4)]
    for o in b.node(Op.custom("fused::beam_select"), ins, outs,
                    {"beams": beams, "keep": keep, "eos": change.get("eos", -1)}, "n"):
        b.output(o)
    if status == "invalid":
        with pytest.raises(StrataError):
            plugin.compile(b.build())
    else:
        exe = plugin.compile(b.build())
        assert (exe is None) == (status == "declined")
        if exe is not None:
            exe.free()


# ---------------------------------------------------------------------------
# GPU
# ---------------------------------------------------------------------------
def _run(plugin, g, host):
    arena, bufs = {}, []
    for i, v in enumerate(g.values):
        if v.producer is None and i in host:
            bufs.append(plugin.upload(v.dtype, v.dims, to_device_bytes(v, host[i])))
            arena[i] = Device(bufs[-1])
    exe = plugin.compile(g)
    assert exe is not None, "the plugin declined the graph"
    try:
        for _ in range(3):  # eager, captured, replayed
            exe.run(arena, every_value=False)
        out = {o: np.array(arena[o]) for o in g.outputs}
        caches = {v.name: np.frombuffer(arena[i].buffer.read(), np.uint16).reshape(v.dims)
                  for i, v in enumerate(g.values) if i in arena and v.name.endswith(("cache", "pages"))}
    finally:
        exe.free()
        for b in bufs:
            b.release()
    return out, caches


@pytest.mark.gpu
@pytest.mark.parametrize("page,count", [(0, None), (16, None), (16, [7, 3])])
def test_tree_step_matches_the_oracle(cuda, plugin, page, count):
    g, hd, host = tree_inputs(SMALL, [200, 37], 256, page=page, count=count)
    out, caches = _run(plugin, g, host)
    ref = graph_eval.evaluate(g, _copy(host))
    want = ref[hd.out]
    got = ora.from_bf16(np.asarray(out[hd.out]).view(np.uint16))
    live = (np.arange(7) < np.array(count or [7, 7])[:, None]).reshape(-1)
    assert_close(got[live], want[live], TOL_BF16, "tree logits")
    for i, v in enumerate(g.values):
        if v.name in caches and v.name.startswith("l0."):
            # the first layer's appended rows; later layers' depend on the outputs' rounding
            assert_close(ora.from_bf16(caches[v.name]), ref[i], TOL_BF16, v.name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_beam_node_matches_the_oracle(cuda, plugin, dtype):
    rng = np.random.default_rng(4)
    b = GraphBuilder("beam")
    x, s, d = b.input(dtype, (12, 1001), "x"), b.input(F32, (12,), "s"), b.input(I32, (12,), "d")
    outs = b.node(Op.custom("fused::beam_select"), [x, s, d], [(F32, (24,))] + [(I32, (24,))] * 3,
                  {"beams": 4, "keep": 8, "eos": 3}, "beam")
    for o in outs:
        b.output(o)
    g = b.build()
    host = {x: ora.round_bf16((rng.standard_normal((12, 1001)) * 3).astype(np.float32)),
            s: (-5 * rng.random(12)).astype(np.float32), d: (rng.random(12) < 0.3).astype(np.int32)}
    out, _ = _run(plugin, g, host)
    want = graph_eval.evaluate(g, host)
    for o in outs[1:]:
        assert np.array_equal(np.asarray(out[o]), want[o])
    assert np.allclose(out[outs[0]], want[outs[0]], rtol=0, atol=2.0 ** -19)


class Model:
    """A small decoder's weights on the device, and greedy / full-context evaluation on it."""

    def __init__(self, plugin, shape=SMALL, fmt="w4g32"):
        self.plugin, self.shape, self.fmt = plugin, shape, fmt
        g, hd = decoder_graph(shape, batch=1, seq=1, max_len=16, fmt=fmt, head="logits")
        host = seeded_graph_inputs(g)
        self.weights = {}
        for i, v in enumerate(g.values):
            if v.producer is None and i in host and not v.name.endswith("cache"):
                self.weights[v.name] = plugin.upload(v.dtype, v.dims, to_device_bytes(v, host[i]))

    def logits(self, tokens):
        """f32 logits after the last of `tokens`, by a prefill of all of them."""
        n, p = len(tokens), self.plugin
        g, hd = decoder_graph(self.shape, batch=1, seq=n, max_len=-(-n // 16) * 16, fmt=self.fmt, head="logits",
                              last_token=True)
        bufs, arena = [], {}
        for i, v in enumerate(g.values):
            if v.producer is not None:
                continue
            if v.name in self.weights:
                arena[i] = Device(self.weights[v.name])
                continue
            data = {"ids": np.array(tokens, np.int32), "pos": np.arange(n, dtype=np.int32)}.get(
                v.name, np.zeros(v.dims, np.uint16))
            bufs.append(p.upload(v.dtype, v.dims, data))
            arena[i] = Device(bufs[-1])
        exe = p.compile(g)
        exe.run(arena, every_value=False)
        out = ora.from_bf16(np.array(arena[hd.out]).view(np.uint16)).reshape(-1).astype(np.float64)
        exe.free()
        for b in bufs:
            b.release()
        return out

    def close(self):
        for b in self.weights.values():
            b.release()


@pytest.fixture(scope="module")
def model(cuda, plugin):
    m = Model(plugin)
    yield m
    m.close()


def _gap(x):
    y = np.sort(x)[::-1]
    return y[0] - y[1]


@pytest.mark.gpu
def test_tree_decoding_equals_greedy_decoding(cuda, plugin, model):
    """Drafts of the greedy continuation beside wrong branches: every step accepts
    the right branch up to the first wrong token, whatever the branch's place in
    the tree, and the cache stays exact over many steps."""
    rng = np.random.default_rng(1)
    prompts = [[int(x) for x in rng.integers(0, 300, n)] for n in (5, 40, 1)]
    total = 24
    greedy = []
    for p in prompts:
        seq = list(p)
        for _ in range(total + 8):
            x = model.logits(seq)
            seq.append(int(np.argmax(x)))
        greedy.append(seq[len(p):])
    kv = PagedKv(plugin, pools=2 * SMALL.layers, pages=48, kv_heads=2, page_size=16, head_dim=64, rows=3,
                 pages_per_row=8)
    dec = TreeDecoder(plugin, SMALL, model.weights, kv, nodes=9)
    try:
        dec.start(prompts)
        done = [[] for _ in prompts]
        step = 0
        while min(len(d) for d in done) < total:
            drafts = []
            for r, d in enumerate(done):
                ahead = greedy[r][len(d):len(d) + 4]
                k = (step + r) % 4  # so many right tokens, then a wrong one
                right = ahead[:k]
                # wrong siblings first, the right branch behind them
                tokens, parents = [(right[0] + 1) % 300 if right else 7, 11], [0, 1]
                at = 0
                for x in right:
                    tokens.append(x)
                    parents.append(at)
                    at = len(tokens)
                tokens.append((ahead[k] + 5) % 300 if k < len(ahead) else 3)
                parents.append(at)
                drafts.append((tokens, parents))
            for d, got in zip(done, dec.step(drafts)):
                d += got
            step += 1
        for r, d in enumerate(done):
            # a near tie of two logits may be decided either way by another rounding
            for i, t in enumerate(d[:total]):
                if t != greedy[r][i]:
                    assert _gap(model.logits(prompts[r] + greedy[r][:i])) < 0.02, (r, i)
                    break
        assert step < total  # several tokens a step
        assert kv.lens.tolist() == [len(p) - 1 + len(d) for p, d in zip(prompts, done)]
    finally:
        dec.release()
        kv.release()


@pytest.mark.gpu
def test_beam_decoding_equals_a_search_without_a_cache(cuda, plugin, model):
    """Beam search over the forked, shared, copied and compacted pages against one
    that re-reads every beam's tokens from the start."""
    rng = np.random.default_rng(2)
    W, steps, eos = 4, 14, 17
    prompts = [[int(x) for x in rng.integers(0, 300, n)] for n in (33, 6)]
    kv = PagedKv(plugin, pools=2 * SMALL.layers, pages=60, kv_heads=2, page_size=16, head_dim=64, rows=2 * W,
                 pages_per_row=5)
    dec = BeamDecoder(plugin, SMALL, model.weights, kv, sentences=2, beams=W, eos=eos)
    try:
        dec.start(prompts)
        hist = [[list() for _ in range(W)] for _ in prompts]
        ref = [[(0.0, [], False)] + [(-np.inf, [], False)] * (W - 1) for _ in prompts]
        for step in range(steps):
            scores, parents, tokens, done = dec.step()
            if step == 6:
                used = kv.compact()
                assert used[0] == 0 and used[1] <= 60
            for s in range(2):
                hist[s] = [hist[s][parents[s, w] - s * W] + [int(tokens[s, w])] for w in range(W)]
                cand = []
                for w, (sc, toks, end) in enumerate(ref[s]):
                    if sc == -np.inf:
                        continue
                    if end:
                        cand.append((sc, w * 300 + eos, toks + [eos], True))
                        continue
                    x = model.logits(prompts[s] + toks)
                    y = x - x.max()
                    y -= np.log(np.exp(y).sum())
                    cand += [(sc + y[v], w * 300 + v, toks + [v], v == eos) for v in np.argsort(-y)[:W + 1]]
                cand.sort(key=lambda c: (-c[0], c[1]))
                # Candidates nearer than the bf16 logits' rounding (2^-8 of a logit of a few units, on
                # either side) may come out in another order: then follow the decoder's choice.
                assert cand[W - 1][0] - scores[s].min() < 0.05 * (step + 1)
                mine = {tuple(h): float(x) for h, x in zip(hist[s], scores[s])}
                by = {tuple(c[2]): c for c in cand}
                nxt = []
                for h in hist[s]:
                    assert tuple(h) in by, "a beam that the search without a cache does not reach"
                    c = by[tuple(h)]
                    assert abs(c[0] - mine[tuple(h)]) < 0.05 * (step + 1)
                    nxt.append((c[0], c[2], c[3]))
                ref[s] = nxt
            assert (kv.lens == np.repeat([len(p) + step for p in prompts], W)).all()
    finally:
        dec.release()
        kv.release()


@pytest.mark.gpu
def test_a_cache_that_runs_out_of_pages_stays_as_it_was(cuda, plugin, model):
    kv = PagedKv(plugin, pools=2 * SMALL.layers, pages=5, kv_heads=2, page_size=16, head_dim=64, rows=4,
                 pages_per_row=6)
    try:
        kv.fork([0, -1, -1, -1], reserve=60)
        kv.lens[0] = 60  # of 64 positions
        before = kv.table.read()
        with pytest.raises(StrataError) as e:
            kv.fork([0, 0, 0, 0], reserve=1)
        assert e.value.code == -5 and "more are needed" in str(e.value)
        assert kv.table.read() == before and kv.lens.tolist() == [60, 0, 0, 0]
        with pytest.raises(StrataError) as e:
            kv.fork([0, 9, 0, 0])
        assert e.value.code == -3
        with pytest.raises(ValueError):
            kv.accept([[1, 1], [], [], []])
        with pytest.raises(ValueError):
            kv.accept([[0, 4], [], [], []])  # the row has pages for 64 positions
        kv.fork([0, 0, -1, -1], reserve=0)
        assert kv.lens.tolist() == [60, 60, 0, 0]
    finally:
        kv.release()


@pytest.mark.gpu
@pytest.mark.parametrize("op", ["fork", "fork of the table alone", "compact"])
def test_a_step_right_behind_a_page_operation(cuda, plugin, op):
    """A decode attention graph launched behind a fork or a compaction, without a wait in between,
    reads the new table, lengths and pages."""
    torch = cuda
    rng = np.random.default_rng(9)
    R, per, ps, G, H, d, pools = 96, 12, 16, 2, 8, 128, 16
    pages = R * per + 200
    lib, stream = plugin.lib, plugin.stream()
    dev = lambda x: torch.from_numpy(np.ascontiguousarray(x)).cuda()  # noqa: E731
    i32 = lambda *s: torch.full(s, -5, dtype=torch.int32, device="cuda")  # noqa: E731
    lens = rng.integers(1, (per - 1) * ps, R).astype(np.int32)
    ids, table, at = rng.permutation(pages).astype(np.int32), np.full((R, per), -1, np.int32), 0
    for r in range(R):
        n = -(-int(lens[r] + 1) // ps)
        table[r, :n] = ids[at:at + n]
        at += n
    refs = np.zeros(pages, np.int32)
    refs[ids[:at]] = 1
    init = torch.randn((pools, pages, G, ps, d), device="cuda", dtype=torch.bfloat16)
    pool = init.clone()
    ti, li, ri, pa = dev(table), dev(lens), dev(refs), i32(R)
    # two forks, or two placings of the same pages, in turn: what one left in a cache is wrong for the other
    parents = [dev(rng.integers(0, R, R).astype(np.int32)) for _ in range(2)]
    tables, counts = [ti.clone()], [ri.clone()]
    other = rng.permutation(pages).astype(np.int32)
    tables.append(dev(np.where(table >= 0, other[table], -1)))
    counts.append(dev(refs[np.argsort(other)]))
    to, lo, ro, remap, report = i32(R, per), i32(R), i32(pages), i32(pages), i32(4)
    n_pools = 0 if "alone" in op else pools
    ptrs = (ctypes.c_void_p * pools)(*[p.data_ptr() for p in pool])
    P, I64 = ctypes.c_void_p, ctypes.c_int64
    lib.strata_b200_kv_fork_workspace_bytes.restype = lib.strata_b200_kv_compact_workspace_bytes.restype = ctypes.c_uint64
    lib.strata_b200_kv_fork_workspace_bytes.argtypes = [I64] * 3
    lib.strata_b200_kv_compact_workspace_bytes.argtypes = [I64]
    ws = torch.empty(max(lib.strata_b200_kv_fork_workspace_bytes(R, per, pages),
                         lib.strata_b200_kv_compact_workspace_bytes(pages)), dtype=torch.uint8, device="cuda")
    lib.strata_b200_kv_fork.argtypes = [P] + [I64] * 5 + [P] * 4 + [I64] * 3 + [P] * 6
    lib.strata_b200_kv_compact.argtypes = [P] + [I64] * 5 + [P] * 2 + [I64] * 2 + [P] * 6

    def page_op(ti=ti, ri=ri, pa=pa):
        if op == "compact":
            return lib.strata_b200_kv_compact(ptrs, n_pools, 2 * d, G, ps, pages, ti.data_ptr(), ri.data_ptr(), R, per,
                                              to.data_ptr(), ro.data_ptr(), remap.data_ptr(), report.data_ptr(),
                                              ws.data_ptr(), stream)
        return lib.strata_b200_kv_fork(ptrs, n_pools, 2 * d, G, ps, pages, ti.data_ptr(), li.data_ptr(), ri.data_ptr(),
                                       pa.data_ptr(), R, per, 1, to.data_ptr(), lo.data_ptr(), ro.data_ptr(),
                                       report.data_ptr(), ws.data_ptr(), stream)

    b = GraphBuilder("t")
    q, k, v = (b.input(BF16, (R, n * d), x) for n, x in ((H, "q"), (G, "k"), (G, "v")))
    kc, vc = (b.input(BF16, (pages, G, ps, d), x) for x in ("kc", "vc"))
    pos, tab = b.input(I32, (R,), "pos"), b.input(I32, (R, per), "table")
    outs = b.node(Op.custom("fused::attention"), [q, k, v, kc, vc, pos, tab], [(BF16, (R, H * d))],
                  {"num_heads": H, "num_kv_heads": G, "head_dim": d, "page_size": ps}, "a")
    b.output(outs[0])
    g = b.build()
    new = [torch.randn((R, n * d), device="cuda", dtype=torch.bfloat16) for n in (H, G, G)]
    out = torch.empty((R, H * d), device="cuda", dtype=torch.bfloat16)
    where = {q: new[0], k: new[1], v: new[2], kc: pool[-2], vc: pool[-1], pos: li if op == "compact" else lo, tab: to,
             outs[0]: out}
    bufs = {i: plugin.wrap(t.data_ptr(), t.numel() * t.element_size()) for i, t in where.items()}

    def go(wait, which):
        pool.copy_(init)
        pa.copy_(parents[which])
        if op == "compact":
            ti.copy_(tables[which])
            ri.copy_(counts[which])
        torch.cuda.synchronize()
        exe = plugin.compile(g)  # a new one: its first run is not a captured one
        run = exe.bind({i: Device(x) for i, x in bufs.items()})
        try:
            assert page_op() == 0
            if wait:
                torch.cuda.synchronize()
            run.run_async()
            plugin.synchronize()
            assert report[0].item() == 0 and report[1].item() > 0
            return out.view(torch.int16).clone()
        finally:
            run.release()
            exe.free()

    want = [go(True, 0), go(True, 1)]
    assert not torch.equal(*want)
    for i in range(12):
        assert torch.equal(want[i % 2], go(False, i % 2))

    def chain(wait):  # operation, step, the other operation, step, ... with nothing else between
        pool.copy_(init)
        sinks = [torch.empty_like(out) for _ in range(6)]
        wrapped = [plugin.wrap(x.data_ptr(), x.numel() * 2) for x in sinks]
        exes = [plugin.compile(g) for _ in sinks]
        runs = [e.bind({**{i: Device(x) for i, x in bufs.items()}, outs[0]: Device(w)}) for e, w in zip(exes, wrapped)]
        torch.cuda.synchronize()
        try:
            for i, run in enumerate(runs):
                assert page_op(tables[i % 2], counts[i % 2], parents[i % 2]) == 0
                if wait:
                    torch.cuda.synchronize()
                run.run_async()
                if wait:
                    plugin.synchronize()
            plugin.synchronize()
            return torch.stack(sinks).view(torch.int16)
        finally:
            for x in (*runs, *wrapped):
                x.release()
            for e in exes:
                e.free()

    if op != "compact":  # the first page set serves both forks
        tables[1], counts[1] = tables[0], counts[0]
    steps = chain(True)
    for _ in range(4):
        assert torch.equal(steps, chain(False))
    for x in bufs.values():
        x.release()


@pytest.mark.gpu
def test_reserve_gives_each_row_its_pages(cuda, plugin):
    """Lowest free ids first, nothing for rows that have enough, and pages past a row's length
    taken back only when the pool is short."""
    kv = PagedKv(plugin, pools=2, pages=8, kv_heads=1, page_size=16, head_dim=64, rows=3, pages_per_row=4)

    def state():
        table = np.frombuffer(kv.table.read(), np.int32).reshape(3, 4).tolist()
        refs = np.frombuffer(kv._refs[kv.side].read(), np.int32).tolist()
        ids = [g for row in table for g in row if g >= 0]
        assert refs == [ids.count(g) for g in range(8)]
        assert kv.held.tolist() == [16 * sum(g >= 0 for g in row) for row in table]
        return [[g for g in row if g >= 0] for row in table]

    try:
        kv.reserve([17, 0, 1])
        assert state() == [[0, 1], [], [2]]
        kv.lens[:] = [5, 0, 16]
        kv.reserve([27, 0, 0])
        assert state() == [[0, 1], [], [2]]
        kv.reserve([0, 33, 1])
        assert state() == [[0, 1], [3, 4, 5], [2, 6]]
        with pytest.raises(StrataError) as e:
            kv.reserve([60, 0, 0])  # past the row
        assert e.value.code == -3 and state() == [[0, 1], [3, 4, 5], [2, 6]]
        kv.lens[1] = 33
        kv.reserve([0, 0, 32])
        assert state() == [[0, 1], [3, 4, 5], [2, 6, 7]]
        kv.reserve([43, 15, 0])  # no page is free: rows 0 and 2 let go of those they do not fill
        assert state() == [[0, 1, 6], [3, 4, 5], [2]]
        kv.reserve([43, 16, 0])
        assert state() == [[0, 1, 6], [3, 4, 5, 7], [2]]
        with pytest.raises(StrataError) as e:
            kv.reserve([59, 0, 17])
        assert e.value.code == -5 and "(2 more are needed)" in str(e.value)
        assert state() == [[0], [3, 4, 5], [2]] and kv.lens.tolist() == [5, 33, 16]
        for bad in ([1, 1], [1, -1, 0]):
            with pytest.raises(ValueError):
                kv.reserve(bad)
    finally:
        kv.release()


@pytest.mark.gpu
def test_a_ragged_prefill_needs_only_its_prompts_pages(cuda, plugin, model):
    """One long prompt beside short ones in a pool that holds them and one step, not the longest
    length for every row; the step then continues each prompt."""
    rng = np.random.default_rng(5)
    prompts = [[int(x) for x in rng.integers(0, 300, n)] for n in (7, 81, 3, 2)]  # 1 + 5 + 1 + 1 pages cached
    kv = PagedKv(plugin, pools=2 * SMALL.layers, pages=9, kv_heads=2, page_size=16, head_dim=64, rows=4,
                 pages_per_row=8)
    dec = TreeDecoder(plugin, SMALL, model.weights, kv, nodes=2)
    try:
        dec.start(prompts)
        assert kv.lens.tolist() == [6, 80, 2, 1]
        got = dec.step([([], [])] * 4)
        for p, g in zip(prompts, got):
            x = model.logits(p)
            assert len(g) == 1 and (g[0] == int(np.argmax(x)) or _gap(x) < 0.02)
        with pytest.raises(StrataError) as e:
            dec.start([prompts[1], prompts[1], [1], [1]])  # 5 + 5 pages of 9
        assert e.value.code == -5 and "1 more" in str(e.value)
        with pytest.raises(StrataError) as e:
            dec.start([[1] * 130, [1], [1], [1]])  # 129 of 128 positions
        assert e.value.code == -3
        dec.start(prompts)
        assert kv.lens.tolist() == [6, 80, 2, 1]
    finally:
        dec.release()
        kv.release()


@pytest.mark.gpu
def test_a_beam_search_goes_to_its_rows_end(cuda, plugin, model):
    """The step that fills the rows returns its results; the next one is refused and the
    cache and the beams stay as they were."""
    W = 3
    prompt = [int(x) for x in np.random.default_rng(6).integers(0, 300, 12)]
    long, short = (PagedKv(plugin, pools=2 * SMALL.layers, pages=40, kv_heads=2, page_size=16, head_dim=64, rows=W,
                           pages_per_row=n) for n in (4, 1))
    a, b = (BeamDecoder(plugin, SMALL, model.weights, kv, sentences=1, beams=W) for kv in (long, short))
    try:
        a.start([prompt])
        b.start([prompt])
        for step in range(5):  # positions 11 to 15
            for x, y in zip(a.step(), b.step()):
                assert np.array_equal(x, y)
        assert short.lens.tolist() == [16] * W
        before = b.tokens.copy(), b.scores.copy()
        with pytest.raises(StrataError) as e:
            b.step()
        assert e.value.code == -3 and short.lens.tolist() == [16] * W
        assert np.array_equal(b.tokens, before[0]) and np.array_equal(b.scores, before[1])
        a.step()
        b.start([prompt])  # the cache can be used again
        a.start([prompt])
        for x, y in zip(a.step(), b.step()):
            assert np.array_equal(x, y)
        hist, scores = b.search([prompt], 5)
        assert all(len(h) == 5 for h in hist[0])
    finally:
        a.release()
        b.release()
        long.release()
        short.release()


@pytest.mark.gpu
def test_tree_steps_near_a_rows_end_and_rows_that_sit_out(cuda, plugin, model):
    """A draft that fits its row is checked however many nodes the graph has; a row without a
    draft stays as it is, at any length, and goes on later."""
    rng = np.random.default_rng(7)
    prompts = [[int(x) for x in rng.integers(0, 300, n)] for n in (31, 5)]
    kv = PagedKv(plugin, pools=2 * SMALL.layers, pages=6, kv_heads=2, page_size=16, head_dim=64, rows=2,
                 pages_per_row=2)
    dec = TreeDecoder(plugin, SMALL, model.weights, kv, nodes=9)

    def right(seq, got):
        for t in got:
            x = model.logits(seq)
            assert t == int(np.argmax(x)) or _gap(x) < 0.02
            seq.append(t)

    try:
        dec.start(prompts)
        seqs = [list(p) for p in prompts]
        for drafts in ([([], []), ([1, 2, 3], [0, 1, 0])], [([], []), None], [None, ([], [])]):
            lens = kv.lens.copy()
            found = dec.step(drafts)
            for r, (d, got) in enumerate(zip(drafts, found)):
                assert kv.lens[r] == lens[r] + len(got) and (d is None) == (got == [])
                right(seqs[r], got)
        assert kv.lens[0] == 32
        with pytest.raises(StrataError) as e:
            dec.step([([], []), ([], [])])  # row 0 is full
        assert e.value.code == -3
        lens = kv.lens.copy()
        (none, got) = dec.step([None, ([4, 4], [0, 0])])
        assert none == [] and kv.lens[0] == 32 and kv.lens[1] == lens[1] + len(got)
        right(seqs[1], got)
        assert dec.step([None, None]) == [[], []]
    finally:
        dec.release()
        kv.release()


@pytest.mark.gpu
def test_a_tree_step_writes_no_page_that_another_row_shares(cuda, plugin, model):
    """A row that goes back into a page it shares gets a copy, also where only its own room fits."""
    prompt = [int(x) for x in np.random.default_rng(8).integers(0, 300, 33)]
    kv = PagedKv(plugin, pools=2 * SMALL.layers, pages=5, kv_heads=2, page_size=16, head_dim=64, rows=2,
                 pages_per_row=3)
    dec = TreeDecoder(plugin, SMALL, model.weights, kv, nodes=9)
    try:
        for sits_out in (False, True):
            dec.start([prompt, [1]])
            kv.fork([0, 0], reserve=0)  # two full pages, shared
            kv.lens[1] = 20
            dec.newest[1] = prompt[20]
            got = dec.step([None if sits_out else ([], []), ([7] * 8, [0] * 8)])
            x = model.logits(prompt[:21])
            assert got[1][0] == int(np.argmax(x)) or _gap(x) < 0.02
            if sits_out:
                got = dec.step([([], []), None])
            x = model.logits(prompt)
            assert got[0][0] == int(np.argmax(x)) or _gap(x) < 0.02
            table = np.frombuffer(kv.table.read(), np.int32).reshape(2, 3)
            assert table[0, 0] == table[1, 0] and table[0, 1] != table[1, 1]
    finally:
        dec.release()
        kv.release()
