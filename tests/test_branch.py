"""Kernels for several continuations of a sequence: tree attention, beam
selection, keeping an accepted branch, forking and compacting a paged cache,
through the C entry points of include/strata_b200.h.

Each is compared with its definition computed in 64 bits (numpy on the host);
page and row moves, ids, counts and parents must be equal."""
import ctypes as C

import numpy as np
import pytest

from oracle import oracle as ora
from tests.conftest import LIB

P, I64 = C.c_void_p, C.c_int64
INVALID = -3
SIG = {
    "strata_b200_tree_attention_bf16": [P] * 9 + [I64] * 8 + [P] * 4,
    "strata_b200_beam_select_bf16": [P] * 3 + [I64] * 5 + [P] * 6,
    "strata_b200_beam_select_f32": [P] * 3 + [I64] * 5 + [P] * 6,
    "strata_b200_kv_accept": [P] + [I64] * 2 + [P] * 4 + [I64] * 6 + [P] * 2,
    "strata_b200_kv_fork": [P] + [I64] * 5 + [P] * 4 + [I64] * 3 + [P] * 6,
    "strata_b200_kv_compact": [P] + [I64] * 5 + [P] * 2 + [I64] * 2 + [P] * 6,
}
SIZES = {
    "strata_b200_tree_attention_workspace_bytes": 4,
    "strata_b200_beam_select_workspace_bytes": 4,
    "strata_b200_kv_fork_workspace_bytes": 3,
    "strata_b200_kv_compact_workspace_bytes": 1,
}


def load():
    lib = C.CDLL(LIB)
    for name, args in SIG.items():
        getattr(lib, name).argtypes = args
        getattr(lib, name).restype = C.c_int32
    for name, n in SIZES.items():
        getattr(lib, name).argtypes = [I64] * n
        getattr(lib, name).restype = C.c_uint64
    return lib


@pytest.fixture(scope="module")
def hlib(plugin):  # the session's plugin fixture builds the library
    return load()


@pytest.fixture(scope="module")
def lib(cuda):
    return load()


class Dev:
    """Device copies of host arrays (bf16 as uint16 bit patterns) and back."""

    def __init__(self, torch):
        self.torch = torch
        self.keep = []

    def __call__(self, a):
        a = np.ascontiguousarray(a)
        if a.dtype == np.uint16:
            a = a.view(np.int16)
        elif a.dtype == np.uint32:
            a = a.view(np.int32)
        t = self.torch.from_numpy(a.copy()).cuda()
        self.keep.append(t)
        return t

    def empty(self, shape, dtype):
        t = self.torch.empty(shape, dtype=dtype, device="cuda")
        self.keep.append(t)
        return t


def ptr(t):
    return None if t is None else t.data_ptr()


def bf(x):
    return ora.to_bf16(np.asarray(x, np.float32))


# ---------------------------------------------------------------------------
# refusals (no GPU: a refused call launches nothing)
# ---------------------------------------------------------------------------
X = 1 << 20  # a stand-in address, 16-byte aligned; never read


def _tree_args(**kw):
    a = dict(q=X, k=X, v=X, kc=X, vc=X, table=None, base=X, count=None, mask=X, batch=1, tokens=4, heads=8, kv_heads=2,
             head_dim=128, max_len=64, page_size=0, num_pages=0, ws=X, out=X, status=None, stream=None)
    a.update(kw)
    return list(a.values())


@pytest.mark.parametrize("bad", [
    dict(tokens=0), dict(tokens=1025), dict(head_dim=96), dict(head_dim=32), dict(kv_heads=3), dict(kv_heads=0),
    dict(heads=258, kv_heads=2), dict(batch=-1), dict(batch=65536), dict(max_len=0), dict(q=X + 2), dict(q=None),
    dict(k=X + 8), dict(v=None), dict(kc=X + 8), dict(vc=None), dict(out=X + 2), dict(out=None), dict(ws=None),
    dict(base=None), dict(mask=None), dict(mask=X + 2), dict(count=X + 1), dict(status=X + 2),
    dict(max_len=1 << 30, batch=4), dict(table=X, page_size=24, num_pages=4, max_len=48),
    dict(table=X, page_size=16, num_pages=0), dict(table=X, page_size=64, num_pages=4, max_len=96),
    dict(table=X, page_size=8, num_pages=4), dict(table=X, page_size=4096, num_pages=1 << 19, max_len=4096)])
def test_tree_attention_refuses(hlib, bad):
    assert hlib.strata_b200_tree_attention_bf16(*_tree_args(**bad)) == INVALID


def test_empty_batches_and_sizes(hlib):
    assert hlib.strata_b200_tree_attention_bf16(*_tree_args(batch=0)) == 0
    assert hlib.strata_b200_tree_attention_workspace_bytes(0, 8, 2, 128) == 0
    assert hlib.strata_b200_tree_attention_workspace_bytes(4, 8, 2, 128) > 0
    assert hlib.strata_b200_beam_select_workspace_bytes(1, 4, 100, 65) == 0
    assert hlib.strata_b200_kv_fork_workspace_bytes(4, 8, 0) == 0
    assert hlib.strata_b200_kv_compact_workspace_bytes(0) == 0


@pytest.mark.parametrize("bad", [
    dict(beams=0), dict(beams=1025), dict(vocab=0), dict(keep=0), dict(keep=65), dict(eos=-2), dict(eos=100),
    dict(batch=-1), dict(batch=20000, beams=4), dict(logits=None), dict(logits=X + 1), dict(scores=None),
    dict(done=X + 2), dict(o0=None), dict(o1=None), dict(o2=None), dict(o3=X + 2), dict(ws=None), dict(ws=X + 4)])
@pytest.mark.parametrize("entry", ["strata_b200_beam_select_bf16", "strata_b200_beam_select_f32"])
def test_beam_select_refuses(hlib, bad, entry):
    a = dict(logits=X, scores=X, done=None, batch=1, beams=4, vocab=100, keep=4, eos=2, o0=X, o1=X, o2=X, o3=X, ws=X,
             stream=None)
    a.update(bad)
    assert getattr(hlib, entry)(*a.values()) == INVALID


@pytest.mark.parametrize("bad", [
    dict(n=257), dict(n=-1), dict(pools=None), dict(row=0), dict(row=24), dict(row=2 << 20), dict(batch=-1),
    dict(heads=0), dict(max_len=0), dict(max_path=1025), dict(max_path=-1), dict(base=None), dict(path=None),
    dict(n_path=X + 2), dict(status=X + 1), dict(table=X, page=48, pages=4), dict(table=X, page=16, pages=0)])
def test_kv_accept_refuses(hlib, bad):
    a = dict(pools=(P * 2)(X, X), n=2, row=256, table=None, base=X, path=X, n_path=X, batch=1, heads=2, max_len=64,
             max_path=4, page=0, pages=0, status=None, stream=None)
    a.update(bad)
    assert hlib.strata_b200_kv_accept(*a.values()) == INVALID
    assert hlib.strata_b200_kv_accept(*{**a, **dict(pools=(P * 2)(X, X + 8), n=2, row=256)}.values()) == INVALID


@pytest.mark.parametrize("bad", [
    dict(n=257), dict(pools=None), dict(row=8), dict(heads=0), dict(page=8), dict(page=48), dict(pages=0),
    dict(pages=1 << 29), dict(rows=-1), dict(rows=70000), dict(per=0), dict(reserve=-1), dict(t_in=None),
    dict(l_in=None), dict(r_in=X + 2), dict(par=None), dict(t_out=None), dict(l_out=None), dict(r_out=None),
    dict(rep=None), dict(ws=None), dict(t_out=X), dict(l_out=X), dict(r_out=X)])
def test_kv_fork_refuses(hlib, bad):
    a = dict(pools=(P * 2)(X, X), n=2, row=256, heads=2, page=16, pages=8, t_in=X, l_in=X, r_in=X, par=X, rows=2, per=4,
             reserve=1, t_out=2 * X, l_out=2 * X, r_out=2 * X, rep=2 * X, ws=X, stream=None)
    a.update(bad)
    assert hlib.strata_b200_kv_fork(*a.values()) == INVALID


@pytest.mark.parametrize("bad", [
    dict(n=300), dict(row=100), dict(heads=0), dict(page=12), dict(pages=0), dict(rows=-1), dict(per=0),
    dict(t_in=None), dict(r_in=None), dict(t_out=X), dict(r_out=X), dict(remap=None), dict(rep=None), dict(ws=X + 8)])
def test_kv_compact_refuses(hlib, bad):
    a = dict(pools=(P * 2)(X, X), n=2, row=256, heads=2, page=16, pages=8, t_in=X, r_in=X, rows=2, per=4, t_out=2 * X,
             r_out=2 * X, remap=3 * X, rep=2 * X, ws=X, stream=None)
    a.update(bad)
    assert hlib.strata_b200_kv_compact(*a.values()) == INVALID


@pytest.mark.parametrize("entry", ["strata_b200_kv_fork", "strata_b200_kv_compact"])
def test_tables_that_a_32_bit_index_cannot_step_over_are_refused(hlib, entry):
    """The planning kernels step through the table by up to 8192 entries, so a table that ends
    closer than that to 2^31 is refused; so is one past it."""
    tail = dict(l_in=X, r_in=X, par=X) if entry.endswith("fork") else dict(r_in=X)
    for rows, per in ((16, (1 << 27) - 1), (65536, 1 << 15), (32765, 65542)):
        a = dict(pools=(P * 2)(X, X), n=2, row=256, heads=2, page=16, pages=8, t_in=X, **tail, rows=rows, per=per)
        if entry.endswith("fork"):
            a.update(reserve=1, t_out=2 * X, l_out=2 * X, r_out=2 * X, rep=2 * X, ws=X, stream=None)
        else:
            a.update(t_out=2 * X, r_out=2 * X, remap=3 * X, rep=2 * X, ws=X, stream=None)
        assert getattr(hlib, entry)(*a.values()) == INVALID


# ---------------------------------------------------------------------------
# tree attention
# ---------------------------------------------------------------------------
def pack_mask(sees):
    """u32 words [B, T, ceil(T / 32)] of bool [B, T, T]."""
    B, T, _ = sees.shape
    words = (T + 31) // 32
    bits = np.zeros((B, T, words * 32), np.uint64)
    bits[:, :, :T] = sees
    return (bits.reshape(B, T, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def random_trees(rng, B, T):
    sees = np.zeros((B, T, T), bool)
    for b in range(B):
        for t in range(T):
            p = int(rng.integers(-1, t)) if t else -1
            if p >= 0:
                sees[b, t] = sees[b, p]
            sees[b, t, t] = True
    return sees


class Tree:
    """One call's host data and its 64-bit answer."""

    def __init__(self, seed, B, T, H, G, d, L, base, count=None, page=0, sees=None, spare=2):
        rng = np.random.default_rng(seed)
        self.dims = (B, T, H, G, d, L, page)
        n = lambda *s: bf(rng.standard_normal(s))  # noqa: E731
        self.q, self.k, self.v = n(B * T, H * d), n(B * T, G * d), n(B * T, G * d)
        self.base = np.asarray(base, np.int32)
        self.count = None if count is None else np.asarray(count, np.int32)
        self.sees = random_trees(rng, B, T) if sees is None else sees
        if page:
            per = L // page
            self.pages = B * per + spare
            self.table = rng.permutation(self.pages)[:B * per].reshape(B, per).astype(np.int32)
            self.kc, self.vc = n(self.pages, G, page, d), n(self.pages, G, page, d)
        else:
            self.pages, self.table = 0, None
            self.kc, self.vc = n(B, G, L, d), n(B, G, L, d)

    def at(self, b, p):
        page = self.dims[6]
        return (self.table[b, p // page], p % page) if page else (b, p)

    def live(self, b):
        return self.dims[1] if self.count is None else int(self.count[b])

    def stale(self, value):
        """Fills every position from base on, and unused pages, with `value`."""
        B, T, H, G, d, L, page = self.dims
        fill = bf([value])[0]
        keep = np.zeros(self.kc.shape[:1] + (self.kc.shape[2],), bool)
        for b in range(B):
            for p in range(int(self.base[b])):
                keep[self.at(b, p)] = True
        for c in (self.kc, self.vc):
            c[...] = np.where(keep[:, None, :, None], c, fill)

    def answer(self):
        """(out, bound of its error, k cache, v cache) after the call.

        The kernels round each probability to bf16 (half a step, 2^-8 relative)
        and the result once more; sums are f32.  So an output may be off by
        2^-8 sum(w |v|) + 2^-8 |o|, and 2^-12 sum(w |v|) for all 32-bit roundings."""
        B, T, H, G, d, L, page = self.dims
        kc, vc = self.kc.copy(), self.vc.copy()
        out, tol = np.zeros((B, T, H, d)), np.zeros((B, T, H, d))
        q = ora.from_bf16(self.q).astype(np.float64).reshape(B, T, H, d)
        for b in range(B):
            n, p0 = self.live(b), int(self.base[b])
            for i in range(n):
                f, r = self.at(b, p0 + i)
                kc[f, :, r] = self.k.reshape(B, T, G, d)[b, i]
                vc[f, :, r] = self.v.reshape(B, T, G, d)[b, i]
            spots = [self.at(b, p) for p in range(p0 + n)]
            if not spots:
                continue
            f, r = np.array(spots).T
            K = ora.from_bf16(kc[f, :, r]).astype(np.float64)  # [positions, G, d]
            V = ora.from_bf16(vc[f, :, r]).astype(np.float64)
            for t in range(n):
                see = np.concatenate([np.ones(p0, bool), self.sees[b, t, :n]])
                if not see.any():
                    continue
                for h in range(H):
                    g = h // (H // G)
                    with np.errstate(invalid="ignore", over="ignore"):
                        s = K[see, g] @ q[b, t, h] / np.sqrt(d)
                        w = np.exp(s - s.max())
                        w /= w.sum()
                        o = w @ V[see, g]
                        a = w @ np.abs(V[see, g])
                    out[b, t, h] = o
                    tol[b, t, h] = a * (2.0 ** -8 + 2.0 ** -12) + np.abs(o) * 2.0 ** -8
        return out.reshape(B * T, H * d), tol.reshape(B * T, H * d), kc, vc

    def call(self, torch, lib, stream=None, state=None):
        B, T, H, G, d, L, page = self.dims
        D = Dev(torch)
        s = state or {}
        if not s:
            s.update(q=D(self.q), k=D(self.k), v=D(self.v), kc=D(self.kc), vc=D(self.vc),
                     table=None if self.table is None else D(self.table), base=D(self.base),
                     count=None if self.count is None else D(self.count), mask=D(pack_mask(self.sees)),
                     ws=D.empty(lib.strata_b200_tree_attention_workspace_bytes(T, H, G, d), torch.uint8),
                     out=D(np.full((B * T, H * d), 0x7FC0, np.uint16)), status=D(np.zeros(1, np.int32)))
            s["ws"].fill_(0xFF)
        st = torch.cuda.current_stream().cuda_stream if stream is None else stream
        rc = lib.strata_b200_tree_attention_bf16(
            ptr(s["q"]), ptr(s["k"]), ptr(s["v"]), ptr(s["kc"]), ptr(s["vc"]), ptr(s["table"]), ptr(s["base"]),
            ptr(s["count"]), ptr(s["mask"]), B, T, H, G, d, L, page, self.pages, ptr(s["ws"]), ptr(s["out"]),
            ptr(s["status"]), st)
        assert rc == 0
        return s

    def check(self, torch, s, status=0):
        torch.cuda.synchronize()
        out, tol, kc, vc = self.answer()
        u16 = lambda t: t.cpu().numpy().view(np.uint16)  # noqa: E731
        assert int(s["status"].item()) == status
        assert np.array_equal(u16(s["kc"]), kc), "k cache"
        assert np.array_equal(u16(s["vc"]), vc), "v cache"
        got = ora.from_bf16(u16(s["out"])).astype(np.float64)
        fine = np.isfinite(out)
        assert np.array_equal(np.isfinite(got), fine)
        off = np.abs(got - out)[fine] - tol[fine]
        assert off.size == 0 or off.max() <= 0, f"off by {np.abs(got - out)[fine].max():.3e}, {off.max():.3e} past the bound"

    def go(self, torch, lib, status=0):
        self.check(torch, self.call(torch, lib), status)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,G,d,page,base", [
    (1, 1, 8, 8, 128, 0, [0]),                 # a single token with nothing before it
    (2, 1, 32, 8, 128, 0, [300, 1]),           # single tokens
    (3, 16, 8, 8, 128, 0, [128, 127, 129]),    # around a tile's end
    (1, 33, 6, 2, 64, 0, [250]),               # two mask words
    (2, 23, 28, 4, 64, 16, [77, 500]),         # 7 heads a kv head
    (2, 16, 64, 4, 128, 32, [640, 0]),         # 16 heads a kv head
    (2, 40, 16, 2, 128, 64, [100, 1000]),      # more than 256 rows a kv head
    (1, 130, 4, 4, 64, 128, [200]),            # a tree longer than a tile
    (1, 300, 2, 1, 128, 0, [64]),
    (1, 9, 128, 1, 64, 256, [511]),            # 128 heads a kv head
    (4, 5, 8, 4, 128, 4096, [4000, 4090, 17, 4096]),
    (1, 64, 3, 1, 128, 16, [2000]),            # split over many blocks
    (1, 3, 40, 8, 128, 16, [5000]),
    (37, 2, 2, 1, 64, 16, None),               # many short sequences
])
def test_tree_attention(cuda, lib, B, T, H, G, d, page, base):
    if base is None:
        base = np.random.default_rng(1).integers(0, 90, B)
    L = -(-(max(base) + T + 7) // (page or 1)) * (page or 1)
    Tree(B * 1000 + T, B, T, H, G, d, L, base, page=page).go(cuda, lib)


@pytest.mark.gpu
@pytest.mark.parametrize("d,page", [(128, 0), (64, 16)])
def test_tree_attention_ragged_counts_and_stale_rows(cuda, lib, d, page):
    """Rows past count are zero, nothing of them is appended, and whatever the
    cache held at or past base (NaN, infinities) reaches no output."""
    for seed, stale in ((1, np.nan), (2, np.inf), (3, 1.0)):
        t = Tree(seed, 5, 20, 8, 2, d, 320, [0, 255, 256, 31, 290], count=[20, 0, 7, 1, 19], page=page)
        t.stale(stale)
        t.go(cuda, lib)


@pytest.mark.gpu
@pytest.mark.parametrize("value", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("H,d,page", [(2, 128, 0), (16, 128, 16), (8, 64, 0)])
def test_tree_attention_keeps_masked_nodes_out(cuda, lib, value, H, d, page):
    """A node with non-finite k and v reaches exactly the nodes that see it."""
    T = 40
    t = Tree(11, 2, T, H, 2, d, 256, [130, 100], page=page)
    G = 2
    t.sees[:, :, 5] = False
    t.sees[:, 5, 5] = True
    t.sees[0, 17, 5] = True
    k, v = t.k.reshape(2, T, G, d), t.v.reshape(2, T, G, d)
    v[:, 5, :, 3] = bf([value])[0]
    if np.isnan(value):
        k[:, 5] = bf([value])[0]
    t.go(cuda, lib)


@pytest.mark.gpu
def test_tree_attention_empty_and_full_masks(cuda, lib):
    T = 37
    none, every = np.zeros((3, T, T), bool), np.ones((3, T, T), bool)
    Tree(5, 3, T, 4, 2, 64, 200, [0, 0, 90], count=[T, 3, T], sees=none).go(cuda, lib)
    Tree(6, 3, T, 4, 2, 64, 200, [0, 0, 90], count=[T, 3, T], sees=every).go(cuda, lib)
    rng = np.random.default_rng(3)
    Tree(7, 3, T, 4, 2, 128, 200, [0, 9, 90], sees=rng.random((3, T, T)) < 0.2).go(cuda, lib)


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,H,G,d,page,top,extra", [
    (230, 4, 8, 4, 128, 0, 300, 3),    # several sequences a block, a cache of an odd length
    (230, 9, 4, 2, 64, 16, 500, 0),
    (60, 40, 16, 2, 128, 0, 700, 0),   # two query tiles of one kv head at once, the second often empty
    (70, 33, 32, 4, 64, 16, 600, 0),
    (3, 20, 16, 2, 128, 0, 9000, 5),   # one sequence over many blocks, many tiles each
])
def test_tree_attention_many_sequences_with_stale_rows(cuda, lib, B, T, H, G, d, page, top, extra):
    """Blocks that go through several sequences, or through one for long, with
    ragged counts and NaN in every row that no live position holds."""
    rng = np.random.default_rng(B + T)
    base, count = rng.integers(0, top, B), rng.integers(0, T + 1, B)
    base[:3], count[:3] = [top, 0, top - 1], [T, 1, 1]
    L = -(-(top + T + extra) // (page or 1)) * (page or 1)
    if not page:
        L += (extra - L) % 8  # a multiple of 8, or off by `extra`
    t = Tree(B, B, T, H, G, d, L, base, count=count, page=page)
    t.stale(np.nan)
    t.go(cuda, lib)


@pytest.mark.gpu
def test_tree_attention_large_scores(cuda, lib):
    """Scores far apart: the running maximum moves by hundreds between tiles."""
    t = Tree(8, 2, 12, 4, 2, 128, 700, [600, 650])
    t.kc = bf(ora.from_bf16(t.kc) * np.linspace(0.1, 12.0, 700)[None, None, :, None])
    t.go(cuda, lib)
    t = Tree(8, 2, 12, 4, 2, 128, 700, [600, 650])
    t.kc = bf(ora.from_bf16(t.kc) * np.linspace(12.0, 0.1, 700)[None, None, :, None])
    t.go(cuda, lib)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 16])
def test_tree_attention_reports_unusable_sequences(cuda, lib, page):
    torch = cuda
    t = Tree(9, 5, 8, 4, 2, 128, 64, [10, -1, 60, 20, 30], count=[8, 8, 8, 9, -3], page=page)
    s = t.call(torch, lib)
    # the other sequences compute; these give zeros and append nothing
    t.count = np.array([8, 0, 0, 0, 0], np.int32)
    t.check(torch, s, status=2)


@pytest.mark.gpu
def test_tree_attention_reports_a_missing_page(cuda, lib):
    torch = cuda
    t = Tree(10, 2, 8, 4, 2, 128, 64, [10, 40], page=16)
    good = t.table.copy()
    for bad in (-1, t.pages, 1 << 30):
        t.table = good.copy()
        t.table[1, 2] = bad
        before_k, before_v = t.kc.copy(), t.vc.copy()
        s = t.call(torch, lib)
        torch.cuda.synchronize()
        assert int(s["status"].item()) == 6
        # nothing is written outside the sequences' own pages; sequence 0 is complete
        spare = np.setdiff1d(np.arange(t.pages), np.r_[good[0], good[1]])
        assert np.array_equal(s["kc"].cpu().numpy().view(np.uint16)[spare], before_k[spare])
        assert np.array_equal(s["vc"].cpu().numpy().view(np.uint16)[spare], before_v[spare])
        one = Tree(10, 2, 8, 4, 2, 128, 64, [10, 40], page=16)
        one.count = np.array([8, 0], np.int32)
        out, tol, _, _ = one.answer()
        got = ora.from_bf16(s["out"].cpu().numpy().view(np.uint16)).astype(np.float64)
        assert np.all(np.abs(got - out)[:8] <= tol[:8])
    # entries no live position needs may be anything
    t.table = good.copy()
    t.table[0, 2:] = -1
    t.go(torch, lib)


class HoledTree(Tree):
    """A paged call some of whose table entries name no page: cached positions there read as zero
    rows (score 0 and value 0, counted in the softmax), and nodes there are attended but not stored."""

    def punch(self, holes):
        """holes: (sequence, page of the sequence, the entry put there)."""
        self.stale(np.nan)
        self.sound = self.table.copy()
        for b, i, entry in holes:
            self.table[b, i] = entry

    def answer(self):
        named, caches = self.table, (self.kc, self.vc)
        bad = (named < 0) | (named >= self.pages)
        # every hole a zero page of its own, behind the pool
        self.table = named.copy()
        self.table[bad] = self.pages + np.arange(bad.sum())
        self.kc, self.vc = (np.concatenate([c, np.zeros((bad.sum(), *c.shape[1:]), c.dtype)]) for c in caches)
        out, tol, kc, vc = super().answer()
        self.table, (self.kc, self.vc) = named, caches
        return out, tol, kc[:self.pages], vc[:self.pages]


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,G,d,page,base,holes", [
    (8, 4, 2, 128, 16, [200, 40], [(0, 1, -1)]),                          # inside the first tile
    (8, 4, 2, 64, 16, [200, 140], [(0, 9, 1 << 30), (1, 0, -7)]),         # in a later tile; the first page
    (3, 8, 1, 128, 64, [640, 250], [(0, 2, -1), (0, 3, -1), (1, 1, 10 ** 6)]),  # a whole tile
    (5, 4, 4, 64, 128, [500, 129], [(0, 1, -1), (1, 0, -1)]),
    (40, 8, 1, 128, 16, [390, 64], [(0, 3, -1), (0, 20, -1), (1, 3, -1)]),  # two query tiles a kv head
    (40, 8, 1, 64, 256, [390, 600], [(0, 0, -1), (1, 2, -1)]),
    (20, 4, 2, 128, 16, [100, 37], [(0, 7, -1), (1, 2, -1), (1, 3, 1 << 30)]),  # pages of nodes, and of both
])
def test_tree_attention_reads_missing_pages_as_zero_rows(cuda, lib, T, H, G, d, page, base, holes):
    L = -(-(max(base) + T) // page) * page
    t = HoledTree(T + d + page, 2, T, H, G, d, L, base, page=page)
    t.punch(holes)
    t.go(cuda, lib, status=6)
    t.table = t.sound  # the same call with all its pages
    t.go(cuda, lib)


@pytest.mark.gpu
def test_tree_attention_in_graphs_and_on_two_streams(cuda, lib):
    """A captured call replayed on new inputs, and two calls in flight at once
    on streams of their own with workspaces of their own."""
    torch = cuda
    a, b = Tree(21, 2, 16, 8, 2, 128, 2100, [2000, 1500]), Tree(22, 3, 30, 8, 8, 64, 1000, [900, 0, 500])
    sa, sb = a.call(torch, lib), b.call(torch, lib)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a.call(torch, lib, state=sa)
    fresh = Tree(23, 2, 16, 8, 2, 128, 2100, [1999, 3])
    for k in ("q", "k", "v", "kc", "vc"):
        sa[k].copy_(torch.from_numpy(getattr(fresh, k).view(np.int16)))
    sa["base"].copy_(torch.from_numpy(fresh.base))
    sa["mask"].copy_(torch.from_numpy(pack_mask(fresh.sees).view(np.int32)))
    g.replay()
    fresh.check(torch, sa)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        fresh.call(torch, lib, stream=s1.cuda_stream, state=sa)
        b.call(torch, lib, stream=s2.cuda_stream, state=sb)
    fresh.check(torch, sa)
    b.check(torch, sb)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [0, 64])
def test_tree_attention_past_32_bit_offsets(cuda, lib, page):
    """Caches of more than 2^31 elements: the last kv head's rows lie past every
    32-bit offset.  Checked on the device in 64 bits, bound as in Tree.answer."""
    torch = cuda
    G, d, L, T = 16, 128, 1_100_032, 3
    g = torch.Generator(device="cuda").manual_seed(5)
    new = lambda *s: torch.randn(s, device="cuda", generator=g, dtype=torch.bfloat16)  # noqa: E731
    kc, vc = (new(L // page, G, page, d) if page else new(1, G, L, d) for _ in range(2))
    q, k, v = new(T, G * d), new(T, G * d), new(T, G * d)
    at = L - 7
    base = torch.tensor([at], dtype=torch.int32, device="cuda")
    table = torch.arange(L // page - 1, -1, -1, dtype=torch.int32, device="cuda")[None].contiguous() if page else None
    mask = torch.tensor([1, 3, 5], dtype=torch.int32, device="cuda")
    ws = torch.empty(lib.strata_b200_tree_attention_workspace_bytes(T, G, G, d), dtype=torch.uint8, device="cuda")
    out, status = torch.empty_like(q), torch.zeros(1, dtype=torch.int32, device="cuda")
    assert kc.numel() > 2 ** 31
    assert lib.strata_b200_tree_attention_bf16(
        ptr(q), ptr(k), ptr(v), ptr(kc), ptr(vc), ptr(table), ptr(base), None, ptr(mask), 1, T, G, G, d, L, page,
        L // page if page else 0, ptr(ws), ptr(out), ptr(status), torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    assert int(status.item()) == 0
    for h in (0, G - 1):
        rows = [(c.flip(0)[:, h] if page else c[0, h]).reshape(L, d)[:at + T] for c in (kc, vc)]
        for r, x in zip(rows, (k, v)):
            assert torch.equal(r[at:].view(torch.int16), x.view(T, G, d)[:, h].view(torch.int16))
        s = rows[0].double() @ q.view(T, G, d)[:, h].double().T / d ** 0.5
        s[at:][~torch.tensor([[1, 1, 1], [0, 1, 0], [0, 0, 1]], dtype=torch.bool, device="cuda")] = -np.inf
        w = torch.softmax(s, 0).T
        o, a = w @ rows[1].double(), w @ rows[1].double().abs()
        off = (out.view(T, G, d)[:, h].double() - o).abs() - a * (2.0 ** -8 + 2.0 ** -12) - o.abs() * 2.0 ** -8
        assert off.max().item() <= 0
    if page:  # the same pool: a row forked, and an accepted path moved, near the pool's end
        P = L // page
        lens, parents = torch.tensor([70, 0], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
        ti = torch.full((2, 3), -1, dtype=torch.int32, device="cuda")
        ti[0, :2] = torch.tensor([P - 1, P - 2])
        refs = torch.ones(P, dtype=torch.int32, device="cuda")
        refs[P - 3] = 0  # the only free page
        to, lo, ro = torch.empty_like(ti), torch.empty_like(lens), torch.empty_like(refs)
        rep = torch.zeros(4, dtype=torch.int32, device="cuda")
        fws = torch.empty(lib.strata_b200_kv_fork_workspace_bytes(2, 3, P), dtype=torch.uint8, device="cuda")
        st = torch.cuda.current_stream().cuda_stream
        assert lib.strata_b200_kv_fork(pools_array([kc]), 1, 2 * d, G, page, P, ptr(ti), ptr(lens), ptr(refs), ptr(parents),
                                       2, 3, 1, ptr(to), ptr(lo), ptr(ro), ptr(rep), ptr(fws), st) == 0
        torch.cuda.synchronize()
        assert rep.tolist() == [0, 1, 0, 0] and to.tolist() == [[P - 1, P - 2, -1], [P - 1, P - 3, -1]]
        assert torch.equal(kc[P - 3, :, :6].view(torch.int16), kc[P - 2, :, :6].view(torch.int16))
        want = kc[P - 3, :, 9].clone()
        nb, path, n = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 70], [[0], [3]], [0, 1]))
        assert lib.strata_b200_kv_accept(pools_array([kc]), 1, 2 * d, ptr(to), ptr(nb), ptr(path), ptr(n), 2, G, 3 * page,
                                         1, page, P, ptr(status), st) == 0
        torch.cuda.synchronize()
        assert int(status.item()) == 0
        assert torch.equal(kc[P - 3, :, 6].view(torch.int16), want.view(torch.int16))


@pytest.mark.gpu
def test_tree_attention_repeats_exactly(cuda, lib):
    torch = cuda
    t = Tree(31, 4, 31, 16, 2, 128, 3000, [2900, 1, 700, 2048])
    s = t.call(torch, lib)
    torch.cuda.synchronize()
    first = s["out"].clone()
    for _ in range(3):
        t.call(torch, lib, state=s)
        torch.cuda.synchronize()
        assert torch.equal(first, s["out"])


# ---------------------------------------------------------------------------
# beam selection
# ---------------------------------------------------------------------------
def beam_answer(logits, scores, done, batch, beams, keep, eos):
    R, V = logits.shape
    x = logits.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    got = ([], [], [], [])
    gap = np.inf
    for b in range(batch):
        cand = []
        for w in range(beams):
            r = b * beams + w
            s = float(scores[r])
            if not s > -np.inf:
                continue
            if done is not None and done[r]:
                cand.append((-s, w * V + max(eos, 0), r, eos, 1))
                continue
            m = x[r].max()
            if m == -np.inf:
                continue
            with np.errstate(invalid="ignore"):
                y = np.where(x[r] == m, 0.0, x[r] - m)
            y = y - np.log(np.exp(y).sum())
            ids = np.lexsort((np.arange(V), -y))[:keep + 1]
            cand += [(-(s + y[v]), w * V + v, r, int(v), int(v == eos)) for v in ids if y[v] > -np.inf]
        cand = sorted(cand)
        d = np.diff([c[0] for c in cand[:keep + 1]])
        d = d[d > 0]
        gap = min(gap, d.min() if d.size else np.inf)
        cand = cand[:keep] + [(np.inf, 0, -1, -1, 0)] * max(0, keep - len(cand))
        got[0].append([-c[0] for c in cand])
        for i in (1, 2, 3):
            got[i].append([c[i + 1] for c in cand])
    return [np.array(g) for g in got], gap


def beam_check(torch, lib, logits, scores, done, batch, beams, keep, eos, offset=0):
    """logits: f32 array, or uint16 bf16 bits.  offset: elements the tensor starts after an aligned address."""
    D = Dev(torch)
    half = logits.dtype == np.uint16
    ref = ora.from_bf16(logits) if half else logits
    V = logits.shape[1]
    flat = np.concatenate([np.zeros(offset, logits.dtype), logits.reshape(-1)])
    dl = D(flat)
    ds, dd = D(np.asarray(scores, np.float32)), None if done is None else D(np.asarray(done, np.int32))
    ws = D.empty(lib.strata_b200_beam_select_workspace_bytes(batch, beams, V, keep), torch.uint8)
    ws.fill_(0xFF)
    n = batch * keep
    outs = [D(np.full(n, 9, np.float32))] + [D(np.full(n, 9, np.int32)) for _ in range(3)]
    f = lib.strata_b200_beam_select_bf16 if half else lib.strata_b200_beam_select_f32
    assert f(ptr(dl) + offset * logits.itemsize, ptr(ds), ptr(dd), batch, beams, V, keep, eos, *map(ptr, outs), ptr(ws),
             torch.cuda.current_stream().cuda_stream) == 0
    torch.cuda.synchronize()
    want, gap = beam_answer(ref, np.asarray(scores, np.float32), done, batch, beams, keep, eos)
    # A term of the softmax is off by a few 2^-23, so lse and a score by less than 2^-20, and the
    # score is rounded to f32 once.  Candidates closer than that have no order to check.
    assert gap > 2.0 ** -19, "the inputs do not decide the order"
    got = [o.cpu().numpy().reshape(batch, keep) for o in outs]
    for g, w, name in zip(got[1:], want[1:], ("parent", "token", "done")):
        assert np.array_equal(g, w), name
    fine = np.isfinite(want[0])
    assert np.array_equal(got[0][~fine], want[0][~fine].astype(np.float32))
    assert np.all(np.abs(got[0] - want[0])[fine] <= 2.0 ** -20 + np.abs(want[0])[fine] * 2.0 ** -24)
    return got


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("batch,beams,vocab,keep", [
    (1, 1, 1, 1), (1, 1, 5, 8), (2, 4, 1000, 4), (3, 3, 8192, 6), (1, 4, 32000, 8), (2, 5, 32003, 10),
    (1, 16, 50021, 64), (33, 8, 4099, 8), (1, 64, 8193, 64), (1, 1, 200001, 64), (1, 1024, 130, 64)])
def test_beam_select(cuda, lib, batch, beams, vocab, keep, half):
    rng = np.random.default_rng(vocab + beams)
    x = (rng.standard_normal((batch * beams, vocab)) * 3).astype(np.float32)
    scores = (-20 - 3 * rng.random(batch * beams)).astype(np.float32)
    beam_check(cuda, lib, bf(x) if half else x, scores, None, batch, beams, keep, -1)
    done = rng.random(batch * beams) < 0.3
    beam_check(cuda, lib, bf(x) if half else x, scores, done, batch, beams, keep, min(2, vocab - 1))


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("offset", [1, 2, 3, 5])
def test_beam_select_at_any_alignment(cuda, lib, half, offset):
    """Rows of an odd length from an odd address; equal rows with equal scores
    give equal candidates, so the lowest beam comes first wherever its row starts."""
    rng = np.random.default_rng(offset)
    row = (rng.standard_normal(9001) * 3).astype(np.float32)
    x = np.tile(row, (6, 1))
    beam_check(cuda, lib, bf(x) if half else x, np.full(6, -4.25), None, 2, 3, 9, 7, offset=offset)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 8200, 70001])
def test_beam_select_ties_and_orders(cuda, lib, vocab):
    """Every logit equal, ascending and descending rows (each tile replaces
    the whole list, or nothing), and two values only."""
    up = np.arange(vocab, dtype=np.float32)[None] * np.float32(0.001)
    for x in (np.zeros((1, vocab), np.float32), up, up[:, ::-1].copy(),
              (np.arange(vocab) % 97 == 5).astype(np.float32)[None]):
        for keep in (1, 17, 64):
            beam_check(cuda, lib, x, [-1.0], None, 1, 1, min(keep, vocab), 3)
    beam_check(cuda, lib, bf(np.zeros((8, vocab), np.float32)), np.full(8, -3.0), None, 2, 4, 64, -1)
    # a block of high logits that one thread holds, and one that a warp's threads hold
    x = np.zeros((2, vocab), np.float32)
    x[0, 8:16] = 5 + np.arange(8)
    x[1, vocab // 2:] = 1 + np.arange(vocab - vocab // 2) * np.float32(0.01)
    beam_check(cuda, lib, x, [-1.0, -1.5], None, 1, 2, 40, -1)


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [100, 20011])
def test_beam_select_non_finite(cuda, lib, vocab):
    """-inf and NaN logits are never chosen, empty beams offer nothing, infinite
    logits share their row's probability, slots without a candidate say so."""
    rng = np.random.default_rng(vocab)
    x = (rng.standard_normal((8, vocab)) * 3).astype(np.float32)
    x[0] = -np.inf
    x[1, :] = np.nan
    x[2, 7:] = -np.inf
    x[3, ::3] = np.nan
    x[4, [3, 50]] = np.inf
    x[5, 20:] = -np.inf
    scores = np.array([-1, -1, -2, -3, -2.5, -np.inf, np.nan, -30], np.float32)
    beam_check(cuda, lib, x, scores, None, 1, 8, 20, 4)
    beam_check(cuda, lib, x, scores, [1, 0, 0, 1, 0, 1, 0, 0], 2, 4, 30, 4)
    got = beam_check(cuda, lib, x[:3], scores[:3], None, 1, 3, 12, -1)
    assert (got[1][0, 7:] == -1).all() and np.isneginf(got[0][0, 7:]).all()
    beam_check(cuda, lib, x[:2], scores[:2], None, 1, 2, 3, 0)
    beam_check(cuda, lib, x[:2], scores[:2], [1, 1], 2, 1, 3, -1)


@pytest.mark.gpu
def test_beam_select_in_a_graph(cuda, lib):
    torch = cuda
    D = Dev(torch)
    rng = np.random.default_rng(2)
    x1, x2 = ((rng.standard_normal((8, 5000)) * 3).astype(np.float32) for _ in range(2))
    dl, ds = D(x1), D(np.full(8, -2.0, np.float32))
    ws = D.empty(lib.strata_b200_beam_select_workspace_bytes(2, 4, 5000, 4), torch.uint8)
    outs = [D(np.zeros(8, np.float32))] + [D(np.zeros(8, np.int32)) for _ in range(3)]

    def call():
        assert lib.strata_b200_beam_select_f32(ptr(dl), ptr(ds), None, 2, 4, 5000, 4, -1, *map(ptr, outs), ptr(ws),
                                               torch.cuda.current_stream().cuda_stream) == 0
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        call()
    dl.copy_(torch.from_numpy(x2))
    g.replay()
    torch.cuda.synchronize()
    want, _ = beam_answer(x2, np.full(8, -2.0), None, 2, 4, 4, -1)
    assert np.array_equal(outs[1].cpu().numpy().reshape(2, 4), want[1])
    assert np.array_equal(outs[2].cpu().numpy().reshape(2, 4), want[2])


def _hard_pairs(rng, lo, hi, n, half):
    """n pairs (a, x), x - a in [lo, hi], for which (x - a) log2(e) in f32 is farthest from the
    exact product, so 2^it from exp(x - a)."""
    a = rng.uniform(-3, 3, 200 * n).astype(np.float32)
    x = (a + rng.uniform(lo, hi, a.size)).astype(np.float32)
    if half:
        a, x = ora.round_bf16(a), ora.round_bf16(x)
    d = x.astype(np.float64) - a
    e = (x - a).astype(np.float32) * np.float32(1.4426950408889634)
    off = np.where((d >= lo) & (d <= hi), np.abs(e.astype(np.float64) - d * 1.4426950408889634074), -1.0)
    order = np.argsort(-off)[:n]
    rng.shuffle(order)
    return a[order], x[order]


@pytest.mark.gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("lo,hi", [(0.5, 2.0), (2.0, 4.0), (4.0, 8.0), (11.1, 15.99), (15.99, 40.0)])
def test_beam_select_a_logit_far_above_the_ones_before(cuda, lib, lo, hi, half):
    """Two logits a row, which one thread meets in turn, the larger one last: the sum of
    exponentials keeps its bound however far the second lies above the first."""
    rng = np.random.default_rng(int(lo * 100) + half)
    batch, beams, vocab = 8, 32, 32768
    a, x = _hard_pairs(rng, lo, hi, batch * beams, half)
    rows = np.full((batch * beams, vocab), -np.inf, np.float32)
    for r in range(batch * beams):
        at = int(rng.integers(0, 8)) * 1024 + int(rng.integers(0, 32)) * (8 if half else 4)
        rows[r, at], rows[r, at + 8192] = a[r], x[r]
    scores = np.log1p(np.exp(a.astype(np.float64) - x)) - np.tile(np.arange(beams) * 2.0 ** -10, batch)  # a step apart
    beam_check(cuda, lib, bf(rows) if half else rows, scores, None, batch, beams, beams, -1)


# ---------------------------------------------------------------------------
# kv_accept
# ---------------------------------------------------------------------------
def pools_array(ts):
    return (P * len(ts))(*[t.data_ptr() for t in ts])


@pytest.mark.gpu
@pytest.mark.parametrize("n_caches,G,row,page,dtype", [
    (1, 1, 16, 0, np.uint8), (3, 2, 256, 0, np.uint8), (7, 3, 128, 16, np.uint8), (2, 8, 48, 64, np.uint8),
    (256, 1, 16, 32, np.uint8)])
def test_kv_accept(cuda, lib, n_caches, G, row, page, dtype):
    torch = cuda
    D = Dev(torch)
    rng = np.random.default_rng(n_caches)
    B, L, width = 6, 192, 40
    base = np.array([0, 100, 37, 152, 10, 64], np.int32)
    paths = [[], [0, 1, 2], [3], list(range(1, 40, 2)), list(range(40)), [0, 1, 4, 5, 6, 20, 21, 22, 23, 24, 39]]
    path = np.full((B, width), -7, np.int32)
    for b, p in enumerate(paths):
        path[b, :len(p)] = p
    n = np.array([len(p) for p in paths], np.int32)
    if page:
        per = L // page
        pages = B * per + 2
        table = rng.permutation(pages)[:B * per].reshape(B, per).astype(np.int32)
        shape = (pages, G, page, row)
    else:
        pages, table, shape = 0, None, (B, G, L, row)
    host = [rng.integers(0, 256, shape).astype(np.uint8) for _ in range(n_caches)]
    dev = [D(h) for h in host]
    status = D(np.zeros(1, np.int32))
    t = None if table is None else D(table)
    db, dp, dn = D(base), D(path), D(n)

    def call():
        assert lib.strata_b200_kv_accept(pools_array(dev), n_caches, row, ptr(t), ptr(db), ptr(dp), ptr(dn), B, G, L,
                                         width, page, pages, ptr(status),
                                         torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()

    def spot(b, p):
        return (table[b, p // page], p % page) if page else (b, p)

    def expect(skip=()):
        for h in host:
            for b in range(B):
                if b in skip:
                    continue
                rows = [h[spot(b, base[b] + x)[0], :, spot(b, base[b] + x)[1]].copy() for x in path[b, :n[b]]]
                for i, r in enumerate(rows):
                    f, s = spot(b, base[b] + i)
                    h[f, :, s] = r
        for h, d in zip(host, dev):
            assert np.array_equal(d.cpu().numpy(), h)

    call()
    expect()
    assert int(status.item()) == 0
    # paths that are refused leave their sequence alone and the others go ahead
    path[1, :3] = [2, 2, 3]
    path[3, :2] = [39, 40]
    n[3] = 2  # 152 + 40 is past the end
    n[4] = 41
    path[5, 0] = -1
    dp.copy_(torch.from_numpy(path))
    dn.copy_(torch.from_numpy(n))
    call()
    expect(skip=(1, 3, 4, 5))
    assert int(status.item()) == 2
    if page:
        status.zero_()
        path[5, 0] = 0
        n[4], n[1], n[3] = 0, 0, 0
        table[5, (64 + 39) // page] = pages
        t.copy_(torch.from_numpy(table))
        dp.copy_(torch.from_numpy(path))
        dn.copy_(torch.from_numpy(n))
        call()
        expect(skip=(1, 3, 4, 5))
        assert int(status.item()) == 6


# ---------------------------------------------------------------------------
# kv_fork and kv_compact
# ---------------------------------------------------------------------------
def fork_answer(table, lens, refs, parents, ps, reserve, pools):
    """(table, lens, refs, report, pools) after the call, row by row."""
    R, per = table.shape
    same = lambda e, n=0: (table.copy(), lens.copy(), refs.copy(), [e, 0, 0, n], [p.copy() for p in pools])  # noqa: E731
    pages = len(refs)
    for r, p in enumerate(parents):
        if p < -1 or p >= R or (p >= 0 and (lens[p] < 0 or lens[p] + reserve > per * ps)):
            bad = 2
            break
    else:
        bad = 0
    named = [int(g) for g in table.reshape(-1) if g >= 0]
    if any(g >= pages for g in named):
        bad = 6
    elif not bad:
        for p in parents:
            if p >= 0 and any(table[p, i] < 0 for i in range(-(-lens[p] // ps))):
                bad = 6
    if bad:
        return same(bad)
    left = refs.astype(int).copy()
    for g in named:
        left[g] -= 1
    if (left < 0).any():
        return same(3)
    out = np.full_like(table, -1)
    ln = np.array([lens[p] if p >= 0 else 0 for p in parents], np.int32)
    for r, p in enumerate(parents):
        for i in range(ln[r] // ps):
            out[r, i] = table[p, i]
            left[out[r, i]] += 1
    kept, copies = {}, {}
    for r, p in enumerate(parents):
        if ln[r] % ps:
            g = int(table[p, ln[r] // ps])
            if left[g] == 0 and g not in kept:
                kept[g] = r
                out[r, ln[r] // ps] = g
            else:
                copies[r] = g
    for g in kept:
        left[g] = 1
    free = [g for g in range(pages) if left[g] == 0]
    want = sum(-(-(ln[r] + reserve) // ps) - (out[r] >= 0).sum() for r, p in enumerate(parents) if p >= 0)
    if want > len(free):
        return same(5, want - len(free))
    res = [p.copy() for p in pools]
    k = 0
    for r, p in enumerate(parents):
        for i in range(-(-(ln[r] + reserve) // ps) if p >= 0 else 0):
            if out[r, i] < 0:
                out[r, i] = free[k]
                left[free[k]] = 1
                if r in copies and i == ln[r] // ps:
                    for a, b in zip(res, pools):
                        a[free[k], :, :ln[r] % ps] = b[copies[r], :, :ln[r] % ps]
                k += 1
    return out, ln, left.astype(np.int32), [0, len(copies), want - len(copies), len(free) - want], res


class Fork:
    def __init__(self, torch, lib, pages, ps, rows, per, pools=2, G=2, row=32, seed=0):
        self.torch, self.lib, self.D = torch, lib, Dev(torch)
        rng = np.random.default_rng(seed)
        self.pages, self.ps, self.rows, self.per, self.G, self.row = pages, ps, rows, per, G, row
        self.pools = [rng.integers(0, 256, (pages, G, ps, row)).astype(np.uint8) for _ in range(pools)]
        self.dev = [self.D(p) for p in self.pools]
        self.table = np.full((rows, per), -1, np.int32)
        self.lens = np.zeros(rows, np.int32)
        self.refs = np.zeros(pages, np.int32)

    def step(self, parents, reserve=1):
        torch, D = self.torch, self.D
        want = fork_answer(self.table, self.lens, self.refs, list(parents), self.ps, reserve, self.pools)
        ti, li, ri, pa = D(self.table), D(self.lens), D(self.refs), D(np.asarray(parents, np.int32))
        to, lo, ro = D(np.full_like(self.table, 77)), D(np.full_like(self.lens, 77)), D(np.full_like(self.refs, 77))
        rep = D(np.full(4, 77, np.int32))
        ws = D.empty(self.lib.strata_b200_kv_fork_workspace_bytes(self.rows, self.per, self.pages), torch.uint8)
        ws.fill_(0xFF)
        assert self.lib.strata_b200_kv_fork(
            pools_array(self.dev), len(self.dev), self.row, self.G, self.ps, self.pages, ptr(ti), ptr(li), ptr(ri),
            ptr(pa), self.rows, self.per, reserve, ptr(to), ptr(lo), ptr(ro), ptr(rep), ptr(ws),
            torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        got = [x.cpu().numpy() for x in (to, lo, ro, rep)]
        for g, w, name in zip(got, want, ("table", "lens", "refs", "report")):
            assert np.array_equal(g, np.asarray(w)), (name, g, w)
        self.table, self.lens, self.refs, report, self.pools = want
        for d, h in zip(self.dev, self.pools):
            assert np.array_equal(d.cpu().numpy(), h)
        return report


@pytest.mark.gpu
@pytest.mark.parametrize("pages,ps,rows,per", [(40, 16, 5, 6), (9000, 16, 300, 9), (60, 64, 4, 5), (1800, 16, 1100, 2),
                                               (6000, 32, 1500, 3)])
def test_kv_fork_from_a_prompt_through_beam_steps(cuda, lib, pages, ps, rows, per):
    """Grow one row, fan it out, then steps of random survivors and growth,
    ended rows and rows taken up again; every state equal to the definition's."""
    f = Fork(cuda, lib, pages, ps, rows, per, seed=pages)
    rng = np.random.default_rng(3)
    none = [-1] * rows
    assert f.step([0] + none[1:], reserve=ps + 5)[:3] == [0, 0, 2]
    f.lens[0] = ps + 5
    rep = f.step([0] * rows)
    assert rep[0] == 0 and rep[1] == rows - 1
    for step in range(6):
        f.lens = np.where(f.lens > 0, np.minimum(f.lens + (1 if step < 4 else ps // 2), per * ps - 1), 0).astype(np.int32)
        # growth past the reserved pages is not allowed: lens stays inside what the table holds
        held = (f.table >= 0).sum(1) * ps
        f.lens = np.minimum(f.lens, held).astype(np.int32)
        f.step(rng.integers(0, rows, rows), reserve=1)
    parents = rng.integers(0, rows, rows)
    parents[::2] = -1
    f.step(parents, reserve=0)
    f.step(rng.integers(0, rows, rows), reserve=1)
    f.step(none)
    assert (f.refs == 0).all()


@pytest.mark.gpu
def test_kv_fork_pages_held_elsewhere(cuda, lib):
    """A partly filled page that a prefix cache also holds, or that is another
    row's full page, is copied by everyone; held pages are never handed out."""
    f = Fork(cuda, lib, 12, 16, 3, 4)
    f.table[0, :2] = [4, 7]
    f.table[1, :2] = [4, 7]
    f.lens[:] = [20, 32, 0]
    f.refs[[4, 7, 0]] = [3, 2, 1]  # page 4 is also held elsewhere, page 0 only elsewhere
    f.step([0, 1, -1], reserve=1)   # row 0's tail page is row 1's full page: copied
    f = Fork(cuda, lib, 12, 16, 3, 4)
    f.table[0, :2] = [4, 7]
    f.lens[0] = 20
    f.refs[[4, 7]] = [1, 2]
    f.step([0, 0, 0], reserve=0)
    f.lens[:] = [20, 20, 20]
    f.step([1, 1, 2], reserve=13)


@pytest.mark.gpu
def test_kv_fork_errors_change_nothing(cuda, lib):
    f = Fork(cuda, lib, 4, 16, 2, 4)
    f.table[0, :2] = [1, 3]
    f.lens[0] = 20
    f.refs[[1, 3]] = 1
    assert f.step([0, 0], reserve=30)[0] == 5
    assert f.step([0, 2])[0] == 2
    assert f.step([0, -2])[0] == 2
    assert f.step([0, 0], reserve=45)[0] == 2
    f.lens[0] = -1
    assert f.step([0, 0])[0] == 2
    f.lens[0] = 20
    f.refs[3] = 0
    assert f.step([0, 0])[0] == 3
    f.refs[3] = 1
    f.table[0, 1] = -1
    assert f.step([0, 0])[0] == 6
    f.table[0, 1] = 4
    assert f.step([0, 0])[0] == 6
    f.table[0, 1] = 3
    assert f.step([0, 0])[0] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("pages,live,rows", [(1, 1, 1), (10, 0, 2), (10, 10, 2), (50, 20, 3), (5000, 3500, 40),
                                             (30011, 9000, 64)])
def test_kv_compact(cuda, lib, pages, live, rows):
    torch = cuda
    D = Dev(torch)
    rng = np.random.default_rng(pages)
    ps, G, row = 16, 2, 16
    used = rng.permutation(pages)[:live].astype(np.int32)
    per = max(1, -(-live // rows)) + 1
    table = np.full((rows, per), -1, np.int32)
    for i, g in enumerate(used):
        table[i % rows, i // rows] = g
    refs = np.zeros(pages, np.int32)
    refs[used] = rng.integers(1, 5, live)
    pools = [rng.integers(0, 256, (pages, G, ps, row)).astype(np.uint8) for _ in range(3)]
    dev = [D(p) for p in pools]
    ti, ri = D(table), D(refs)
    ws = D.empty(lib.strata_b200_kv_compact_workspace_bytes(pages), torch.uint8)

    def call():
        ws.fill_(0xFF)
        outs = [D(np.full_like(table, 77)), D(np.full_like(refs, 77)), D(np.full_like(refs, 77)), D(np.zeros(4, np.int32))]
        assert lib.strata_b200_kv_compact(pools_array(dev), 3, row, G, ps, pages, ptr(ti), ptr(ri), rows, per,
                                          *map(ptr, outs), ptr(ws), torch.cuda.current_stream().cuda_stream) == 0
        torch.cuda.synchronize()
        return [o.cpu().numpy() for o in outs]

    if live:  # refused: a table entry without references, one past the pool, a negative count
        for entry, ref, code in ((None, 0, 3), (pages, None, 6), (None, -1, 3)):
            t2, r2 = table.copy(), refs.copy()
            if entry is not None:
                t2[0, 0] = entry
            if ref is not None:
                r2[used[0]] = ref
            ti.copy_(torch.from_numpy(t2))
            ri.copy_(torch.from_numpy(r2))
            to, ro, mo, rep = call()
            assert rep[0] == code and np.array_equal(to, t2) and np.array_equal(ro, r2)
            assert np.array_equal(mo, np.arange(pages))
        ti.copy_(torch.from_numpy(table))
        ri.copy_(torch.from_numpy(refs))
    to, ro, mo, rep = call()
    holes = [g for g in range(live) if refs[g] == 0]
    movers = [g for g in range(live, pages) if refs[g] > 0]
    remap = np.where(refs > 0, np.arange(pages), -1)
    want = [p.copy() for p in pools]
    for a, b in zip(movers, holes):
        remap[a] = b
        for w, p in zip(want, pools):
            w[b] = p[a]
    new = np.zeros_like(refs)
    new[remap[refs > 0]] = refs[refs > 0]
    assert list(rep) == [0, live, len(movers), pages - live]
    assert np.array_equal(mo, remap) and np.array_equal(ro, new)
    assert np.array_equal(to, np.where(table >= 0, remap[np.maximum(table, 0)], -1))
    for d, w in zip(dev, want):
        assert np.array_equal(d.cpu().numpy(), w)


# ---------------------------------------------------------------------------
# What one call writes is there for the next one on its stream
# ---------------------------------------------------------------------------
class DecodeAttention:
    """Calls of the framework's decode attention, which reads cache rows below the position
    before its wait for the kernel ahead of it."""

    def __init__(self, torch, lib, B, H, G, d, L):
        self.torch, self.lib, self.dims = torch, lib, (B, H, G, d, L)
        lib.strata_b200_attention_decode_bf16.argtypes = [P] * 6 + [I64] * 5 + [P] * 3
        lib.strata_b200_attention_decode_scratch_bytes.argtypes = [I64] * 4
        lib.strata_b200_attention_decode_scratch_bytes.restype = C.c_uint64
        new = lambda *s: torch.randn(s, device="cuda", generator=torch.Generator("cuda").manual_seed(s[-1]),  # noqa: E731
                                     dtype=torch.bfloat16)
        self.q, self.k, self.v = new(B, H * d), new(B, G * d), new(B, G * d)
        self.scratch = torch.empty(lib.strata_b200_attention_decode_scratch_bytes(B, H, d, L), dtype=torch.uint8,
                                   device="cuda")

    def __call__(self, kc, vc, pos, out):
        B, H, G, d, L = self.dims
        assert self.lib.strata_b200_attention_decode_bf16(
            ptr(self.q), ptr(self.k), ptr(self.v), ptr(kc), ptr(vc), ptr(pos), B, H, G, d, L, ptr(self.scratch), ptr(out),
            self.torch.cuda.current_stream().cuda_stream) == 0


def _back_to_back(torch, first, then, restore):
    """Bits of `then()`'s outputs where the GPU is waited for between the two, and without, eagerly and
    in a graph; two sets of inputs in turn, so that what one left in a cache is wrong for the other."""
    def go(between, which):
        restore(which)
        torch.cuda.synchronize()
        first()
        if between:
            torch.cuda.synchronize()
        outs = then()
        torch.cuda.synchronize()
        return [o.view(torch.int16).clone() for o in outs]

    want = [go(True, 0), go(True, 1)]
    assert not any(torch.equal(a, b) for a, b in zip(*want))
    for i in range(12):
        assert all(torch.equal(a, b) for a, b in zip(want[i % 2], go(False, i % 2)))
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        restore(0)
        s.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            first()
            outs = then()
        for i in range(6):
            restore(i % 2)
            g.replay()
            s.synchronize()
            assert all(torch.equal(a, b.view(torch.int16)) for a, b in zip(want[i % 2], outs))


@pytest.mark.gpu
@pytest.mark.parametrize("G,d", [(8, 128), (2, 64)])
def test_decode_attention_right_behind_an_accept(cuda, lib, G, d):
    """An accept moves rows of 64 caches, and the next step's attention over each of them is
    launched at once: it reads the moved rows."""
    torch = cuda
    B, L, H, layers, width = 8, 320, 4 * G, 32, 40
    rng = np.random.default_rng(G)
    D = Dev(torch)
    gen = torch.Generator("cuda").manual_seed(1)
    init = torch.randn((2 * layers, B, G, L, d), device="cuda", generator=gen, dtype=torch.bfloat16)
    caches = init.clone()
    bases = [D(rng.integers(0, L - 2 * width, B).astype(np.int32)) for _ in range(2)]
    paths = [D(np.stack([np.sort(rng.choice(2 * width, width, replace=False)) for _ in range(B)]).astype(np.int32))
             for _ in range(2)]
    base, path = torch.empty_like(bases[0]), torch.empty_like(paths[0])
    n = D(np.full(B, width, np.int32))
    pos = torch.empty_like(base)
    attend = DecodeAttention(torch, lib, B, H, G, d, L)
    outs = [torch.empty(B, H * d, dtype=torch.bfloat16, device="cuda") for _ in range(layers)]

    def accept():
        assert lib.strata_b200_kv_accept(pools_array(list(caches)), 2 * layers, 2 * d, None, ptr(base), ptr(path), ptr(n),
                                         B, G, L, width, 0, 0, None, torch.cuda.current_stream().cuda_stream) == 0

    def step():
        for i in reversed(range(layers)):
            attend(caches[2 * i], caches[2 * i + 1], pos, outs[i])
        return outs

    def restore(which):
        caches.copy_(init)
        base.copy_(bases[which])
        path.copy_(paths[which])
        pos.copy_(bases[which] + width)  # the next token's position

    _back_to_back(torch, accept, step, restore)


@pytest.mark.gpu
@pytest.mark.parametrize("T,H,G,d", [(24, 32, 8, 128), (40, 8, 1, 64), (3, 4, 4, 128)])
def test_decode_attention_right_behind_tree_attention(cuda, lib, T, H, G, d):
    """The tree's rows are appended before a step behind it reads them."""
    torch = cuda
    B, L = 6, 640
    t = Tree(T, B, T, H, G, d, L, [500, 3, 0, 129, 600 - T, 255])
    s = t.call(torch, lib)
    torch.cuda.synchronize()
    init = [torch.from_numpy(x.view(np.int16)).cuda() for x in (t.kc, t.vc)]
    pos = s["base"] + T
    attend = DecodeAttention(torch, lib, B, H, G, d, L)
    out = torch.empty(B, H * d, dtype=torch.bfloat16, device="cuda")

    new = [(s["k"].clone(), s["v"].clone()), (s["k"].flip(0).clone(), s["v"].flip(0).clone())]

    def restore(which):
        for c, x in zip((s["kc"], s["vc"]), init):
            c.copy_(x)
        for c, x in zip((s["k"], s["v"]), new[which]):
            c.copy_(x)

    def step():
        attend(s["kc"], s["vc"], pos, out)
        return [out]

    _back_to_back(torch, lambda: t.call(torch, lib, state=s), step, restore)


def _under_counted(case):
    """(pages, rows, per, table, lens, refs, parents) whose counts are below the table's own references."""
    if case == "one row keeps the page, another lets it go":
        return 4, 2, 2, [[0, -1], [0, -1]], [16, 16], [1, 0, 0, 0], [0, -1]
    if case == "a page without a reference is shared out":
        return 3, 2, 2, [[0, 1], [-1, -1]], [32, 0], [0, 1, 0], [0, 0]
    if case == "every row keeps it":
        return 3, 3, 1, [[2], [2], [2]], [16] * 3, [0, 0, 2], [0, 1, 2]
    if case == "a row takes it from another that keeps it":
        return 3, 3, 2, [[2, -1], [1, 2], [-1, -1]], [16, 32, 0], [0, 1, 1], [0, 0, 1]
    # planned by a cluster: one reference is missing among many
    return 5000, 1100, 2, [[7, -1]] * 1100, [16] * 1100, [1099 if g == 7 else 0 for g in range(5000)], \
        [r if r % 3 else (r * 7) % 1100 for r in range(1100)]


@pytest.mark.gpu
@pytest.mark.parametrize("case", ["one row keeps the page, another lets it go", "a page without a reference is shared out",
                                  "every row keeps it", "a row takes it from another that keeps it", "many rows"])
def test_kv_fork_counts_the_old_references_before_the_new_ones(cuda, lib, case):
    """Error 3 compares the counts with the old table, whatever the new one shares: an
    under-counted page must not come out free beside a row that holds it."""
    pages, rows, per, table, lens, refs, parents = _under_counted(case)
    f = Fork(cuda, lib, pages, 16, rows, per, pools=1)
    f.table[:], f.lens[:], f.refs[:] = table, lens, refs
    assert f.step(parents, reserve=0)[0] == 3
    named = f.table[f.table >= 0]
    f.refs = np.bincount(named, minlength=pages).astype(np.int32)  # with all references counted it goes through
    assert f.step(parents, reserve=0)[0] == 0
