"""The operators for several continuations of a sequence: attention of a tree of
drafted tokens over a KV cache, keeping the accepted branch's rows, forking and
compacting a paged cache, and a beam step's selection.

Each case is one call.  ``run`` computes it in plain torch, or, with ``own``
true, through the C entry points of include/strata_b200.h.  Plain forms work
in 32 bits (the beam scores, which are compared with one another, in 64).
"""
import ctypes
import math

import torch

own = False

DEV = "cuda"
LIB_PATH = "ferrite-strata_b200/libstrata_b200.so"


# ---------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------
def listed():
    return [
        # One user of the 7B decoder shape (32 heads of 128), a draft of 16 tokens after a short
        # prompt: what a single verification step's latency is made of.
        {"name": "tree 1x16 over 500, 32/32", "op": "tree", "batch": 1, "tokens": 16, "heads": 32, "kv_heads": 32,
         "dim": 128, "max_len": 640, "base_lo": 500, "base_hi": 500, "page": 0, "full": True},
        # The 7B shape at batch 8, contiguous caches, ragged lengths and odd ragged drafts.
        {"name": "tree 8x25 over 2048, 32/32", "op": "tree", "batch": 8, "tokens": 25, "heads": 32, "kv_heads": 32,
         "dim": 128, "max_len": 2176, "base_lo": 1100, "base_hi": 2048, "page": 0, "full": False},
        # The 70B shape (64 query heads on 8), batch 32, caches in 16-position pages.
        {"name": "tree 32x16 over 4096, 64/8 paged", "op": "tree", "batch": 32, "tokens": 16, "heads": 64,
         "kv_heads": 8, "dim": 128, "max_len": 4224, "base_lo": 3000, "base_hi": 4096, "page": 16, "full": True},
        # Wide trees over long prompts: 512 query rows a kv head, the largest call.
        {"name": "tree 8x64 over 16384, 64/8 paged", "op": "tree", "batch": 8, "tokens": 64, "heads": 64,
         "kv_heads": 8, "dim": 128, "max_len": 16512, "base_lo": 12000, "base_hi": 16384, "page": 64, "full": False},
        # One sentence, 4 beams, the 7B vocabulary, f32 logits.
        {"name": "beam 1x4 of 32000 f32", "op": "beam", "batch": 1, "beams": 4, "vocab": 32000, "keep": 4,
         "bf16": False, "masked": False},
        # A serving batch of 32 x 16 beams over a large, odd vocabulary, some beams finished,
        # twice as many continuations kept as beams.
        {"name": "beam 32x16 of 128001 bf16", "op": "beam", "batch": 32, "beams": 16, "vocab": 128001, "keep": 32,
         "bf16": True, "masked": True},
        # The accepted branch of one sequence in the 32 layers' k and v caches of the 7B shape.
        {"name": "accept 1 of 64 caches", "op": "accept", "batch": 1, "caches": 64, "kv_heads": 32, "dim": 128,
         "max_len": 128, "tokens": 16, "page": 0},
        # A batch of 32 over paged pools of 80 layers with 8 kv heads.
        {"name": "accept 32 of 160 pools paged", "op": "accept", "batch": 32, "caches": 160, "kv_heads": 8, "dim": 128,
         "max_len": 256, "tokens": 33, "page": 16},
        # Beams of one sentence after a step.
        {"name": "fork 4 rows of 64 pools", "op": "fork", "batch": 1, "beams": 4, "pools": 64, "kv_heads": 8,
         "dim": 128, "page": 16, "prompt": 300, "own_len": 60, "spare": 32, "reserve": 1},
        # 16 sentences of 8 beams, multi-head caches.
        {"name": "fork 128 rows of 32 pools", "op": "fork", "batch": 16, "beams": 8, "pools": 32, "kv_heads": 32,
         "dim": 128, "page": 16, "prompt": 200, "own_len": 90, "spare": 256, "reserve": 1},
        # A small pool with holes after a few sequences ended.
        {"name": "compact 100 pages of 16 pools", "op": "compact", "pages": 100, "live": 0.7, "rows": 8, "pools": 16,
         "kv_heads": 8, "dim": 128, "page": 16},
        # A large pool, a third of it free.
        {"name": "compact 3000 pages of 32 pools", "op": "compact", "pages": 3000, "live": 0.65, "rows": 61,
         "pools": 32, "kv_heads": 8, "dim": 128, "page": 16},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["tree", "tree", "tree", "beam", "beam", "accept", "fork", "compact"])
    if op == "tree":
        group = rng.choice([1, 1, 2, 3, 4, 7, 8, 8, 12, 16])
        kv_heads = rng.choice([1, 2, 4, 8, 8, 16, 32])
        dim = rng.choice([64, 128, 128])
        tokens = _log_int(rng, 1, 140)
        page = rng.choice([0, 0, 16, 32, 64, 128, 256])
        base_hi = _log_int(rng, 1, 16000)
        # at most the largest listed case's cached bytes and products
        top = min(500e6 / (4.0 * dim * kv_heads * (base_hi + (2 + group) * tokens)),
                  250e9 / (4.0 * dim * kv_heads * group * tokens * (base_hi + tokens)))
        batch = _log_int(rng, 1, max(1, min(64, int(top))))
        unit = page or 1
        max_len = -(-(base_hi + tokens + rng.randint(0, 200)) // unit) * unit
        return {"op": "tree", "batch": batch, "tokens": tokens, "heads": group * kv_heads, "kv_heads": kv_heads,
                "dim": dim, "max_len": max_len, "base_lo": rng.choice([0, base_hi // 2, base_hi]),
                "base_hi": base_hi, "page": page, "full": rng.random() < 0.4}
    if op == "beam":
        vocab = _log_int(rng, 500, 200000)
        beams = _log_int(rng, 1, 32)
        keep = min(64, max(1, beams * rng.choice([1, 1, 2])), beams * vocab)
        batch = _log_int(rng, 1, max(1, min(64, int(60e6 / (vocab * beams)))))
        return {"op": "beam", "batch": batch, "beams": beams, "vocab": vocab, "keep": keep,
                "bf16": rng.random() < 0.5, "masked": rng.random() < 0.5}
    kv_heads = rng.choice([1, 2, 8, 8, 32])
    dim = rng.choice([64, 128])
    page = rng.choice([16, 16, 32, 64])
    if op == "accept":
        tokens = _log_int(rng, 2, 100)
        unit = page if rng.random() < 0.5 else 0
        max_len = -(-(tokens + rng.randint(1, 200)) // (unit or 1)) * (unit or 1)
        caches = _log_int(rng, 1, 160)
        batch = _log_int(rng, 1, max(1, min(64, int(2e9 / (2.0 * caches * kv_heads * dim * max_len)))))
        return {"op": "accept", "batch": batch, "caches": caches, "kv_heads": kv_heads, "dim": dim,
                "max_len": max_len, "tokens": tokens, "page": unit}
    if op == "fork":
        beams = _log_int(rng, 1, 16)
        prompt, own_len = _log_int(rng, 1, 500), rng.randint(1, 100)
        pools = _log_int(rng, 1, 64)
        seq = 2.0 * pools * kv_heads * dim * (prompt + beams * (own_len + 2 * page))
        batch = _log_int(rng, 1, max(1, min(32, int(3e9 / seq))))
        return {"op": "fork", "batch": batch, "beams": beams, "pools": pools, "kv_heads": kv_heads, "dim": dim,
                "page": page, "prompt": prompt, "own_len": own_len, "spare": batch * beams * (2 + 40 // page) + 1,
                "reserve": rng.choice([0, 1, 1, 2, 33])}
    pools = _log_int(rng, 1, 64)
    pages = _log_int(rng, 10, max(10, min(20000, int(3e9 / (2.0 * pools * kv_heads * dim * page)))))
    return {"op": "compact", "pages": pages, "live": rng.choice([0.1, 0.5, 0.9]), "rows": _log_int(rng, 1, 100),
            "pools": pools, "kv_heads": kv_heads, "dim": dim, "page": page}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed))


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32).to(torch.bfloat16)


def _randint(g, lo, hi, shape):
    """Uniform in [lo, hi], I32."""
    return torch.randint(lo, hi + 1, shape, generator=g, device=DEV, dtype=torch.int32)


def _page_table(g, rows, per, pages):
    return torch.randperm(pages, generator=g, device=DEV)[:rows * per].reshape(rows, per).to(torch.int32)


def _tree_masks(g, batch, tokens):
    """Ancestor masks [batch, tokens, words] of random trees: node t's parent is one of the
    nodes before it (mostly a near one), or the prompt; a node sees itself and its ancestors."""
    words = (tokens + 31) // 32
    sees = torch.zeros(batch, tokens, tokens, dtype=torch.bool, device=DEV)
    back = torch.empty(batch, tokens, device=DEV).exponential_(0.4, generator=g).long() + 1
    rows = torch.arange(batch, device=DEV)
    for t in range(tokens):
        parent = t - back[:, t]
        sees[:, t] = torch.where((parent >= 0)[:, None], sees[rows, parent.clamp(min=0)], False)
        sees[:, t, t] = True
    bits = torch.zeros(batch, tokens, words * 32, dtype=torch.int64, device=DEV)
    bits[:, :, :tokens] = sees.long()
    packed = (bits.reshape(batch, tokens, words, 32) << torch.arange(32, device=DEV)).sum(-1)
    return torch.where(packed >= 1 << 31, packed - (1 << 32), packed).to(torch.int32)


def _prepare_tree(c, g):
    B, T, H, G, d, L, ps = (c[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "max_len", "page"))
    s = {"q": _normal(g, B * T, H * d), "k": _normal(g, B * T, G * d), "v": _normal(g, B * T, G * d),
         "base": _randint(g, min(c["base_lo"], c["base_hi"]), c["base_hi"], (B,)),
         "count": torch.full((B,), T, dtype=torch.int32, device=DEV) if c["full"] else _randint(g, max(1, T // 2), T, (B,)),
         "mask": _tree_masks(g, B, T), "table": None, "pages": 0,
         "out": torch.empty(B * T, H * d, dtype=torch.bfloat16, device=DEV)}
    if ps:
        per = L // ps
        s["pages"] = B * per + 3
        s["table"] = _page_table(g, B, per, s["pages"])
        s["kc"], s["vc"] = _normal(g, s["pages"], G, ps, d), _normal(g, s["pages"], G, ps, d)
    else:
        s["kc"], s["vc"] = _normal(g, B, G, L, d), _normal(g, B, G, L, d)
    return s


def _prepare_beam(c, g):
    R, V = c["batch"] * c["beams"], c["vocab"]
    logits = torch.randn(R, V, generator=g, device=DEV) * 2.5
    done = torch.zeros(R, dtype=torch.int32, device=DEV)
    if c["masked"]:  # tokens that may not follow, and beams that have ended
        logits[:, ::7] = float("-inf")
        done = (torch.rand(R, generator=g, device=DEV) < 0.15).int()
    # accumulated log probabilities of beams that compete: some tens below zero
    scores = -30.0 - 4.0 * torch.rand(R, generator=g, device=DEV)
    n = (c["batch"], c["keep"])
    i32 = {"dtype": torch.int32, "device": DEV}
    return {"logits": logits.to(torch.bfloat16) if c["bf16"] else logits, "scores": scores, "done": done, "eos": 2,
            "out": (torch.empty(n, device=DEV), torch.empty(n, **i32), torch.empty(n, **i32), torch.empty(n, **i32))}


def _prepare_accept(c, g):
    B, C, G, d, L, T, ps = (c[k] for k in ("batch", "caches", "kv_heads", "dim", "max_len", "tokens", "page"))
    depth = max(1, min(T, 8))
    # a root-to-leaf path: strictly increasing node indices
    path = torch.rand(B, T, generator=g, device=DEV).argsort(-1)[:, :depth].sort(-1).values.int()
    s = {"base": _randint(g, 0, L - T, (B,)), "path": path, "n": _randint(g, 0, depth, (B,)), "table": None,
         "pages": 0}
    if ps:
        s["pages"] = B * (L // ps) + 1
        s["table"] = _page_table(g, B, L // ps, s["pages"])
        s["caches"] = _normal(g, C, s["pages"], G, ps, d)
    else:
        s["caches"] = _normal(g, C, B, G, L, d)
    return s


def _prepare_fork(c, g):
    B, W, N, G, d, ps = (c[k] for k in ("batch", "beams", "pools", "kv_heads", "dim", "page"))
    R = B * W
    # beams of one sentence share the prompt's full pages and hold the rest alone
    length = c["prompt"] + _randint(g, 0, c["own_len"], (B,)).repeat_interleave(W)
    shared = c["prompt"] // ps
    per = -(-(c["prompt"] + c["own_len"] + max(c["reserve"], 1)) // ps) + 1
    pages = B * shared + R * (per - shared) + c["spare"]
    perm = torch.randperm(pages, generator=g, device=DEV).int()
    col = torch.arange(per, device=DEV)
    row = torch.arange(R, device=DEV)[:, None]
    ident = torch.where(col < shared, (row // W) * shared + col, B * shared + row * (per - shared) + col - shared)
    used = -(-(length + 1) // ps)  # each row also holds the page of its next position
    table = torch.where(col < used[:, None], perm[ident], -1).int()
    refs = torch.bincount(table[table >= 0].long(), minlength=pages).int()
    # survivors keep their slot, the others' slots go to a survivor of the same sentence
    alive = torch.rand(B, W, generator=g, device=DEV) < 0.5
    alive[:, 0] = True
    rank = torch.rand(B, W, W, generator=g, device=DEV) * alive[:, None, :]
    pick = torch.where(alive, torch.arange(W, device=DEV), rank.argmax(-1))
    parents = (pick + torch.arange(B, device=DEV)[:, None] * W).reshape(-1).int()
    return {"pools": _normal(g, N, pages, G, ps, d), "table": table, "lens": length.int(), "refs": refs,
            "parents": parents, "reserve": c["reserve"],
            "out": (torch.empty_like(table), torch.empty_like(length.int()), torch.empty_like(refs),
                    torch.empty(4, dtype=torch.int32, device=DEV))}


def _prepare_compact(c, g):
    P, R, N, G, d, ps = (c[k] for k in ("pages", "rows", "pools", "kv_heads", "dim", "page"))
    order = torch.randperm(P, generator=g, device=DEV).int()
    n = max(1, int(P * c["live"]))
    per = -(-n // R) + 1
    table = torch.full((R, per), -1, dtype=torch.int32, device=DEV)
    at = torch.arange(n, device=DEV)
    table[at % R, at // R] = order[:n]
    refs = torch.zeros(P, dtype=torch.int32, device=DEV)
    refs[order[:n].long()] = _randint(g, 1, 3, (n,))
    return {"pools": _normal(g, N, P, G, ps, d), "table": table, "refs": refs,
            "out": (torch.empty_like(table), torch.empty_like(refs), torch.empty_like(refs),
                    torch.empty(4, dtype=torch.int32, device=DEV))}


_PREPARE = {"tree": _prepare_tree, "beam": _prepare_beam, "accept": _prepare_accept, "fork": _prepare_fork,
            "compact": _prepare_compact}


def prepare(case, seed):
    state = _PREPARE[case["op"]](case, _gen(seed))
    state["case"] = case
    return state


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
def _bit_rows(mask, tokens):
    """bool [B, T, T] of packed mask words."""
    bits = (mask.long()[..., None] >> torch.arange(32, device=mask.device)) & 1
    return bits.flatten(-2)[..., :tokens].bool()


def _cache_index(s, ps, seq, pos):
    """First and row index of positions `pos` of sequences `seq` in a cache or a page pool."""
    if not ps:
        return seq, pos
    return s["table"].long()[seq, pos // ps], pos % ps


def _plain_tree(s):
    c = s["case"]
    B, T, H, G, d, ps = (c[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "page"))
    base, count = s["base"].long(), s["count"].long()
    node = torch.arange(T, device=DEV)
    seq, t = (node < count[:, None]).nonzero(as_tuple=True)
    first, row = _cache_index(s, ps, seq, base[seq] + t)
    s["kc"][first, :, row] = s["k"].view(B, T, G, d)[seq, t]
    s["vc"][first, :, row] = s["v"].view(B, T, G, d)[seq, t]
    top = int(c["base_hi"]) + T
    if ps:
        need = -(-top // ps)
        k, v = (x[s["table"][:, :need].long()].transpose(1, 2).reshape(B, G, need * ps, d)
                for x in (s["kc"], s["vc"]))
    else:
        k, v = s["kc"][:, :, :top], s["vc"][:, :, :top]
    q = s["q"].view(B, T, G, H // G, d).permute(0, 2, 3, 1, 4).reshape(B, G, H // G * T, d).float()
    score = (q @ k.float().transpose(-1, -2)).view(B, G, H // G, T, -1) / math.sqrt(d)
    at = torch.arange(k.shape[2], device=DEV) - base[:, None]  # [B, L], relative to the first node
    tree = _bit_rows(s["mask"], T).gather(2, at.clamp(0, T - 1)[:, None, :].expand(B, T, -1))
    sees = (at < 0)[:, None] | (tree & ((at >= 0) & (at < count[:, None]))[:, None])
    sees = (sees & (node < count[:, None])[..., None])[:, None, None]
    score = score.masked_fill_(~sees, float("-inf"))
    most = score.amax(-1, keepdim=True)
    e = (score - torch.where(torch.isinf(most), 0.0, most)).exp_()
    o = (e.view(B, G, H // G * T, -1) @ v.float()).view(B, G, H // G, T, d)
    total = e.sum(-1, keepdim=True)
    o = torch.where(total > 0, o / total, 0.0)
    return o.permute(0, 3, 1, 2, 4).reshape(B * T, H * d).to(torch.bfloat16), s["kc"], s["vc"]


def _plain_beam(s):
    c = s["case"]
    B, W, V, keep = c["batch"], c["beams"], c["vocab"], c["keep"]
    x = s["logits"].double()
    x = torch.where(x.isnan(), float("-inf"), x)
    most = x.amax(-1, keepdim=True)
    logp = x - most
    logp = logp - logp.exp().sum(-1, keepdim=True).log()
    done = s["done"].bool()[:, None]
    eos = torch.arange(V, device=DEV) == s["eos"]
    logp = torch.where(done, torch.where(eos, 0.0, float("-inf")), logp)
    score = (s["scores"].double()[:, None] + logp).view(B, W * V)
    best, at = score.sort(dim=-1, descending=True, stable=True)
    best, at = best[:, :keep], at[:, :keep]
    none = best == float("-inf")
    parent = at // V + torch.arange(B, device=DEV)[:, None] * W
    token = at % V
    ended = done.view(-1)[parent] | (token == s["eos"])
    return (best.float(), torch.where(none, -1, parent).int(), torch.where(none, -1, token).int(),
            (ended & ~none).int())


def _plain_accept(s):
    c = s["case"]
    base, path, n = s["base"].long(), s["path"].long(), s["n"].long()
    seq, i = (torch.arange(path.shape[1], device=DEV) < n[:, None]).nonzero(as_tuple=True)
    first, row = _cache_index(s, c["page"], seq, base[seq] + path[seq, i])
    rows = s["caches"][:, first, :, row]
    first, row = _cache_index(s, c["page"], seq, base[seq] + i)
    s["caches"][:, first, :, row] = rows
    return s["caches"]


def _plain_fork(s):
    c = s["case"]
    ps, pages = c["page"], s["refs"].shape[0]
    table, refs, parents = s["table"].long(), s["refs"].long(), s["parents"].long()
    R, per = table.shape
    r = torch.arange(R, device=DEV)
    col = torch.arange(per, device=DEV)
    live = parents >= 0
    length = torch.where(live, s["lens"].long()[parents.clamp(min=0)], 0)
    full, part = length // ps, length % ps > 0
    mine = table[parents.clamp(min=0)]
    shared = live[:, None] & (col < full[:, None])
    left = refs - torch.bincount(table[table >= 0], minlength=pages) + torch.bincount(mine[shared], minlength=pages)
    tail = mine.gather(1, full.clamp(max=per - 1)[:, None])[:, 0]
    spot = torch.where(part, tail, 0)
    first = torch.full((pages,), R, device=DEV).scatter_reduce(0, spot, torch.where(part, r, R), "amin")
    kept = part & (left[spot] == 0) & (first[spot] == r)
    left = left.index_add(0, spot[kept], torch.ones_like(spot[kept]))
    copied = part & ~kept
    need = torch.where(live, (length + s["reserve"] + ps - 1) // ps, 0)
    fresh = need - full - kept.long()
    offset = fresh.cumsum(0) - fresh
    free = (left == 0).nonzero()[:, 0]
    new = (col >= (full + kept.long())[:, None]) & (col < need[:, None])
    nth = (offset - full - kept.long())[:, None] + col
    out = torch.where(shared | (kept[:, None] & (col == full[:, None])), mine, -1)
    out = torch.where(new, free[nth.clamp(0, free.shape[0] - 1)], out)
    left = left.index_add(0, out[new], torch.ones_like(out[new]))
    src, dst = tail[copied], out[r[copied], full[copied]]
    used = (length % ps)[copied]
    take = (torch.arange(ps, device=DEV) < used[:, None])[None, :, None, :, None]
    s["pools"][:, dst] = torch.where(take, s["pools"][:, src], s["pools"][:, dst])
    total = fresh.sum()
    report = torch.stack([total * 0, copied.sum(), total - copied.sum(), free.shape[0] - total])
    return out.int(), length.int(), left.int(), report.int(), s["pools"]


def _plain_compact(s):
    table, refs = s["table"].long(), s["refs"].long()
    live = refs > 0
    ident = torch.arange(refs.shape[0], device=DEV)
    n = live.sum()
    hole = (~live & (ident < n)).nonzero()[:, 0]
    mover = (live & (ident >= n)).nonzero()[:, 0]
    remap = torch.where(live, ident, -1)
    remap[mover] = hole
    new = torch.zeros_like(refs)
    new[remap[live]] = refs[live]
    out = torch.where(table >= 0, remap[table.clamp(min=0)], -1)
    s["pools"][:, hole] = s["pools"][:, mover]
    report = torch.stack([n * 0, n, n * 0 + mover.shape[0], refs.shape[0] - n])
    return out.int(), new.int(), remap.int(), report.int(), s["pools"]


_PLAIN = {"tree": _plain_tree, "beam": _plain_beam, "accept": _plain_accept, "fork": _plain_fork,
          "compact": _plain_compact}


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------
_P, _I = ctypes.c_void_p, ctypes.c_int64
_SIGNATURES = {
    "strata_b200_tree_attention_workspace_bytes": [_I] * 4,
    "strata_b200_tree_attention_bf16": [_P] * 9 + [_I] * 8 + [_P] * 4,
    "strata_b200_beam_select_workspace_bytes": [_I] * 4,
    "strata_b200_beam_select_bf16": [_P] * 3 + [_I] * 5 + [_P] * 6,
    "strata_b200_beam_select_f32": [_P] * 3 + [_I] * 5 + [_P] * 6,
    "strata_b200_kv_accept": [_P] + [_I] * 2 + [_P] * 4 + [_I] * 6 + [_P] * 2,
    "strata_b200_kv_fork_workspace_bytes": [_I] * 3,
    "strata_b200_kv_fork": [_P] + [_I] * 5 + [_P] * 4 + [_I] * 3 + [_P] * 6,
    "strata_b200_kv_compact_workspace_bytes": [_I],
    "strata_b200_kv_compact": [_P] + [_I] * 5 + [_P] * 2 + [_I] * 2 + [_P] * 6,
}
_loaded = {}


def _lib():
    if not _loaded:
        lib = ctypes.CDLL(LIB_PATH)
        for name, args in _SIGNATURES.items():
            f = getattr(lib, name)
            f.argtypes = args
            f.restype = ctypes.c_uint64 if name.endswith("bytes") else ctypes.c_int32
        _loaded["lib"] = lib
    return _loaded["lib"]


def _workspace(s, size_of, *sizes):
    """The state's workspace, allocated at its first call as a user's program would."""
    if "ws" not in s:
        s["ws"] = torch.empty(max(size_of(*sizes), 1), dtype=torch.uint8, device=DEV)
    return s["ws"].data_ptr()


def _at(t):
    return None if t is None else t.data_ptr()


def _pointers(s, stacked):
    """A host array of the device addresses of stacked[0], stacked[1], ... (one per layer's k or v)."""
    if "ptrs" not in s:
        n, step = stacked.shape[0], stacked.stride(0) * stacked.element_size()
        s["ptrs"] = (ctypes.c_void_p * n)(*range(stacked.data_ptr(), stacked.data_ptr() + n * step, step))
    return s["ptrs"]


def _ok(rc):
    if rc:
        raise RuntimeError("entry point returned %d" % rc)


def _own_tree(s, lib, stream):
    c = s["case"]
    B, T, H, G, d, L, ps = (c[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "max_len", "page"))
    ws = _workspace(s, lib.strata_b200_tree_attention_workspace_bytes, T, H, G, d)
    _ok(lib.strata_b200_tree_attention_bf16(
        _at(s["q"]), _at(s["k"]), _at(s["v"]), _at(s["kc"]), _at(s["vc"]), _at(s["table"]), _at(s["base"]),
        _at(s["count"]), _at(s["mask"]), B, T, H, G, d, L, ps, s["pages"], ws, _at(s["out"]), None, stream))
    return s["out"], s["kc"], s["vc"]


def _own_beam(s, lib, stream):
    c = s["case"]
    B, W, V, keep = c["batch"], c["beams"], c["vocab"], c["keep"]
    ws = _workspace(s, lib.strata_b200_beam_select_workspace_bytes, B, W, V, keep)
    f = lib.strata_b200_beam_select_bf16 if c["bf16"] else lib.strata_b200_beam_select_f32
    _ok(f(_at(s["logits"]), _at(s["scores"]), _at(s["done"]), B, W, V, keep, s["eos"],
          *(t.data_ptr() for t in s["out"]), ws, stream))
    return s["out"]


def _own_accept(s, lib, stream):
    c = s["case"]
    B, C, G, d, L, ps = (c[k] for k in ("batch", "caches", "kv_heads", "dim", "max_len", "page"))
    _ok(lib.strata_b200_kv_accept(_pointers(s, s["caches"]), C, 2 * d, _at(s["table"]), _at(s["base"]),
                                  _at(s["path"]), _at(s["n"]), B, G, L, s["path"].shape[1], ps, s["pages"], None,
                                  stream))
    return s["caches"]


def _own_fork(s, lib, stream):
    c = s["case"]
    (R, per), pages = s["table"].shape, s["refs"].shape[0]
    ws = _workspace(s, lib.strata_b200_kv_fork_workspace_bytes, R, per, pages)
    _ok(lib.strata_b200_kv_fork(_pointers(s, s["pools"]), c["pools"], 2 * c["dim"], c["kv_heads"], c["page"], pages,
                                _at(s["table"]), _at(s["lens"]), _at(s["refs"]), _at(s["parents"]), R, per,
                                s["reserve"], *(t.data_ptr() for t in s["out"]), ws, stream))
    return *s["out"], s["pools"]


def _own_compact(s, lib, stream):
    c = s["case"]
    (R, per), pages = s["table"].shape, s["refs"].shape[0]
    ws = _workspace(s, lib.strata_b200_kv_compact_workspace_bytes, pages)
    _ok(lib.strata_b200_kv_compact(_pointers(s, s["pools"]), c["pools"], 2 * c["dim"], c["kv_heads"], c["page"],
                                   pages, _at(s["table"]), _at(s["refs"]), R, per,
                                   *(t.data_ptr() for t in s["out"]), ws, stream))
    return *s["out"], s["pools"]


_OWN = {"tree": _own_tree, "beam": _own_beam, "accept": _own_accept, "fork": _own_fork, "compact": _own_compact}


def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state, _lib(), torch.cuda.current_stream().cuda_stream)
    return _PLAIN[op](state)


# ---------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------
def work(case):
    c = case
    if c["op"] == "tree":
        B, T, H, G, d = (c[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
        base = (min(c["base_lo"], c["base_hi"]) + c["base_hi"]) / 2
        n = T if c["full"] else (max(1, T // 2) + T) / 2
        cached = 4.0 * B * G * d * base
        rows = 2.0 * B * (2 * T * H * d + 4 * n * G * d)  # q and out; k, v read and written
        return {"bytes": cached + rows, "flops": 4.0 * d * H * B * n * (base + n)}
    if c["op"] == "beam":
        n = c["batch"] * c["beams"] * c["vocab"]
        return {"bytes": n * (2.0 if c["bf16"] else 4.0) + 16.0 * c["batch"] * c["keep"], "flops": 4.0 * n}
    row = 2.0 * c["dim"] * c["kv_heads"]
    if c["op"] == "accept":
        depth = max(1, min(c["tokens"], 8))
        moved = depth / 2 * (1 - depth / (2.0 * c["tokens"]))  # about: rows that are not in place already
        return {"bytes": 2 * row * c["caches"] * c["batch"] * moved + 4.0 * c["batch"] * (depth + 2), "flops": 0}
    if c["op"] == "fork":
        rows = c["batch"] * c["beams"]
        per = -(-(c["prompt"] + c["own_len"] + max(c["reserve"], 1)) // c["page"]) + 1
        pages = rows * per + c["spare"]
        copies = c["batch"] * (c["beams"] - 1) / 2 * (c["page"] - 1) / 2.0
        return {"bytes": 2 * row * c["pools"] * copies + 8.0 * (rows * per + pages) + 12.0 * rows, "flops": 0}
    n = max(1, int(c["pages"] * c["live"]))
    moved = n * (1 - n / c["pages"])
    return {"bytes": 2 * row * c["page"] * c["pools"] * moved + 8.0 * n + 12.0 * c["pages"], "flops": 0}


# ---------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------
def _exact_tree(c, s):
    B, T, H, G, d, ps = (c[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim", "page"))
    base, count = s["base"].tolist(), s["count"].tolist()
    words = s["mask"].tolist()
    out = torch.zeros(B, T, G, H // G, d, dtype=torch.float64, device=DEV)
    for b in range(B):
        n, p = count[b], base[b]
        if ps:
            ids = s["table"][b].long()
            keys, vals = (x[ids].double().permute(1, 0, 2, 3).flatten(1, 2)[:, :p] for x in (s["kc"], s["vc"]))
        else:
            keys, vals = s["kc"][b, :, :p].double(), s["vc"][b, :, :p].double()
        kn = s["k"].view(B, T, G, d)[b, :n].double().transpose(0, 1)
        vn = s["v"].view(B, T, G, d)[b, :n].double().transpose(0, 1)
        hide = torch.tensor([[0.0 if (words[b][t][j // 32] >> (j % 32)) & 1 else -math.inf for j in range(n)]
                             for t in range(n)], dtype=torch.float64, device=DEV)
        for h in range(H // G):
            q = s["q"].view(B, T, G, H // G, d)[b, :n, :, h].double().transpose(0, 1) * d ** -0.5
            z = torch.cat([torch.einsum("gtd,gpd->gtp", q, keys), torch.einsum("gtd,gjd->gtj", q, kn) + hide], 2)
            z = z - torch.logsumexp(z, 2, keepdim=True).nan_to_num(neginf=0.0)
            w = z.exp()
            o = torch.einsum("gtp,gpd->tgd", w[:, :, :p], vals) + torch.einsum("gtj,gjd->tgd", w[:, :, p:], vn)
            out[b, :n, :, h] = o
        for i in range(n):
            at = (int(s["table"][b, (p + i) // ps]), slice(None), (p + i) % ps) if ps else (b, slice(None), p + i)
            s["kc"][at] = s["k"].view(B, T, G, d)[b, i]
            s["vc"][at] = s["v"].view(B, T, G, d)[b, i]
    return out.view(B * T, H * d), s["kc"], s["vc"]


def _exact_beam(c, s):
    B, W, V, keep = c["batch"], c["beams"], c["vocab"], c["keep"]
    got = [[], [], [], []]
    done = s["done"].tolist()
    for b in range(B):
        cand = []
        for w in range(W):
            r = b * W + w
            if done[r]:
                cand.append((-float(s["scores"][r]), w * V + s["eos"], r, s["eos"], 1))
                continue
            x = s["logits"][r].double()
            total = torch.logsumexp(x, 0)
            cut = x.topk(min(keep, V)).values[-1]
            ids = (x >= cut).nonzero()[:, 0]
            for v, z in zip(ids.tolist(), (x[ids] - total + s["scores"][r].double()).tolist()):
                if z > -math.inf:
                    cand.append((-z, w * V + v, r, v, int(v == s["eos"])))
        cand = sorted(cand)[:keep]
        cand += [(math.inf, 0, -1, -1, 0)] * (keep - len(cand))
        for k, f in enumerate((lambda e: -e[0], lambda e: e[2], lambda e: e[3], lambda e: e[4])):
            got[k].append([f(e) for e in cand])
    return [torch.tensor(got[0], dtype=torch.float64, device=DEV)] + [
        torch.tensor(x, dtype=torch.int32, device=DEV) for x in got[1:]]


def _exact_accept(c, s):
    ps, table = c["page"], s["table"].tolist() if c["page"] else None
    spot = lambda b, p: (table[b][p // ps], p % ps) if ps else (b, p)  # noqa: E731
    for b, (p, path, n) in enumerate(zip(s["base"].tolist(), s["path"].tolist(), s["n"].tolist())):
        for i in range(n):  # path[i] >= i, so a row is read before it is written
            (x, y), (u, v) = spot(b, p + path[i]), spot(b, p + i)
            s["caches"][:, u, :, v] = s["caches"][:, x, :, y].clone()
    return s["caches"]


def _exact_fork(c, s):
    ps = c["page"]
    table, lens, refs, parents = (s[k].tolist() for k in ("table", "lens", "refs", "parents"))
    left = list(refs)
    for row in table:
        for g in row:
            if g >= 0:
                left[g] -= 1
    out = [[-1] * len(table[0]) for _ in table]
    length = [lens[p] if p >= 0 else 0 for p in parents]
    for r, p in enumerate(parents):
        for i in range(length[r] // ps):
            out[r][i] = table[p][i]
            left[table[p][i]] += 1
    copies, taken = [], set()
    for r, p in enumerate(parents):
        i = length[r] // ps
        if length[r] % ps:
            g = table[p][i]
            if left[g] == 0 and g not in taken:
                taken.add(g)
                out[r][i] = g
            else:
                copies.append((r, i, g, length[r] % ps))
    for g in taken:
        left[g] = 1
    free = [g for g, n in enumerate(left) if n == 0]
    todo = {r: (i, g, n) for r, i, g, n in copies}
    used = fresh = 0
    for r, p in enumerate(parents):
        for i in range(-(-(length[r] + s["reserve"]) // ps) if p >= 0 else 0):
            if out[r][i] < 0:
                out[r][i] = free[used]
                left[free[used]] = 1
                used += 1
                if r in todo and todo[r][0] == i:
                    _, g, n = todo[r]
                    s["pools"][:, out[r][i], :, :n] = s["pools"][:, g, :, :n]
                else:
                    fresh += 1
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return t(out), t(length), t(left), t([0, len(copies), fresh, len(free) - used]), s["pools"]


def _exact_compact(c, s):
    table, refs = s["table"].tolist(), s["refs"].tolist()
    n = sum(x > 0 for x in refs)
    holes = [g for g in range(n) if refs[g] == 0]
    remap = [g if refs[g] > 0 else -1 for g in range(len(refs))]
    moves = list(zip([g for g in range(n, len(refs)) if refs[g] > 0], holes))
    new = [refs[g] if g < n else 0 for g in range(len(refs))]
    for a, b in moves:
        remap[a], new[b] = b, refs[a]
        s["pools"][:, b] = s["pools"][:, a]
    t = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    return (t([[remap[g] if g >= 0 else -1 for g in row] for row in table]), t(new), t(remap),
            t([0, n, len(moves), len(refs) - n]), s["pools"])


_EXACT = {"tree": _exact_tree, "beam": _exact_beam, "accept": _exact_accept, "fork": _exact_fork,
          "compact": _exact_compact}


def exact(case, seed):
    return _EXACT[case["op"]](case, prepare(case, seed))
