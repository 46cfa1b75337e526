"""Operators of a paged key/value cache, as a serving loop calls them.

* ``paged``: attention of new tokens, or of a tree of drafted tokens, over a
  cache whose keys lie in pages (or one row of tokens a sequence);
* ``write``: the rows of new tokens put into the cache;
* ``draft``: one step of drafting without its attention: the drafted rows of
  every layer written, then those of the accepted path moved together;
* ``fork``: sequences that continue others, in several copies or not at all
  (beams, samples of one prompt), with room for new tokens;
* ``compact``: the pages in use moved to the front of the pool.

``run`` computes the plain form of each (elementary torch operations, sums in 32
bits) or, with ``own``, calls the library.
"""
import math
import os
import random
import sys

import torch

own = False

_DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _fa():
    root = os.path.join(os.getcwd(), "flash-attn-v100_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import flash_attention_v100
    return flash_attention_v100


# ---------------------------------------------------------------------------
# cases

def _paged(name, B, N, cap_tokens, page, H, Hkv, D, dtype, lens, tree=0, cap=0.0, slopes=False):
    """``cap_tokens``: tokens a sequence may hold; ``page``: 0 for one row of
    tokens a sequence; ``lens``, ``tree``: numbers that the filled lengths and the
    trees are drawn from (tree 0: the new tokens follow one another)."""
    return {"name": name, "op": "paged", "B": B, "N": N, "S": cap_tokens, "page": page, "H": H, "Hkv": Hkv, "D": D,
            "dtype": dtype, "lens": lens, "tree": tree, "cap": cap, "slopes": slopes, "L": 1}


def _cache(name, op, B, N, cap_tokens, page, Hkv, D, dtype, lens, L):
    return {"name": name, "op": op, "B": B, "N": N, "S": cap_tokens, "page": page, "Hkv": Hkv, "D": D, "dtype": dtype,
            "lens": lens, "L": L}


def listed():
    return [
        # the smallest call: one new token of one sequence over 512 cached ones
        _paged("paged_one", 1, 1, 512, 16, 8, 8, 64, "fp16", lens=2),
        # serving: one new token of each of 32 sequences, lengths from a quarter of the room to all of it
        _paged("paged_tokens", 32, 1, 4096, 16, 32, 8, 128, "bf16", lens=3),
        # verifying trees of up to 64 drafted tokens of 16 sequences over long caches
        _paged("tree_batch", 16, 64, 8192, 64, 32, 8, 128, "bf16", lens=5, tree=7),
        # full precision: a small batch's trees with capped scores and a distance bias, caches of one row a sequence
        _paged("tree_rows", 2, 26, 1001, 0, 12, 4, 80, "fp32", lens=11, tree=13, cap=30.0, slopes=True),
        # prompts' keys and values into the cache: three, and a free slot of the batch
        _cache("write_prompt", "write", 4, 2048, 2112, 16, 8, 128, "bf16", lens=19, L=1),
        # one new token of 64 sequences into the cache
        _cache("write_tokens", "write", 64, 1, 1024, 16, 8, 128, "bf16", lens=23, L=1),
        # a small batch's drafts
        _cache("draft_small", "draft", 4, 26, 400, 16, 8, 64, "fp16", lens=29, L=2),
        # drafts of 64 tokens, 64 sequences, 8 layers
        _cache("draft_batch", "draft", 64, 64, 256, 16, 8, 128, "bf16", lens=31, L=8),
        # the best of 32 beams continued, over 4 layers
        _cache("fork_beams", "fork", 32, 1, 1024, 16, 8, 128, "bf16", lens=37, L=4),
        # samples of one prompt, full precision
        _cache("fork_small", "fork", 5, 3, 200, 32, 4, 80, "fp32", lens=41, L=1),
        # the pages of 64 sequences, half of the pool's, in 2 layers
        _cache("compact_pool", "compact", 64, 0, 512, 16, 8, 128, "bf16", lens=43, L=2),
        # a small pool
        _cache("compact_small", "compact", 6, 0, 300, 32, 4, 64, "fp16", lens=47, L=1),
    ]


# what a drawn case may cost by its plain arithmetic (the largest listed case has 1.1e11) and hold in bytes
_MOST_FLOPS = {"fp16": 1.0e11, "bf16": 1.0e11, "fp32": 2.0e10}
_MOST_BYTES = 4.0e8


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_one(rng):
    dt = rng.choice(["bf16", "fp16", "bf16", "fp16", "fp32"])
    Hkv = rng.choice([1, 2, 4, 8, 12, 16])
    D = rng.choice([32, 64, 64, 80, 96, 128, 128])
    page = rng.choice([16, 16, 32, 48, 64, 128, 256])
    seed = rng.randint(1, 10 ** 6)
    what = rng.choice(["paged", "paged", "paged", "write", "draft", "fork", "compact"])
    if what == "paged":
        tree = rng.random() < 0.5
        N = _log(rng, 2, 128) if tree else rng.choice([1, 1, 1, rng.randint(2, 9), _log(rng, 10, 300)])
        return _paged("", _log(rng, 1, 48), N, N + _log(rng, 8, 16000), rng.choice([0, page, page, page]),
                      Hkv * rng.choice([1, 1, 2, 4, 8]), Hkv, D, dt, lens=seed, tree=seed + 1 if tree else 0,
                      cap=rng.choice([0.0, 0.0, 30.0, 50.0]), slopes=rng.random() < 0.3)
    if what == "write":
        N = rng.choice([1, 1, rng.randint(2, 64), _log(rng, 65, 4000)])
        return _cache("", "write", _log(rng, 1, 96), N, N + _log(rng, 8, 500), page, Hkv, D, dt, lens=seed, L=1)
    if what == "draft":
        N = _log(rng, 2, 128)
        return _cache("", "draft", _log(rng, 1, 64), N, N + _log(rng, 8, 300), page, Hkv, D, dt, lens=seed,
                      L=rng.randint(1, 8))
    return _cache("", what, _log(rng, 2, 96), rng.choice([0, 1, 1, 17]) if what == "fork" else 0, _log(rng, 40, 2000),
                  page, Hkv, D, dt, lens=seed, L=rng.randint(1, 4))


def draw(rng):
    while True:
        c = _draw_one(rng)
        w = work(c)
        if w["flops"] <= _MOST_FLOPS[c["dtype"]] and w["bytes"] <= _MOST_BYTES and _pool_bytes(c) <= 1.2e9:
            del c["name"]
            return c


# ---------------------------------------------------------------------------
# lengths, trees, paths and sources, from the case alone

def _lengths(case):
    """Filled tokens of each sequence, the new ones among them; a free slot now and then."""
    rng = random.Random(case["lens"])
    S, N = case["S"], case["N"]
    top = S - (N if case["op"] == "fork" else 0)
    lo = max(1, N, top // 4) if case["op"] != "write" or N < 65 else max(N, top * 15 // 16)
    lens = [rng.randint(min(lo, top), top) for _ in range(case["B"])]
    if case["B"] > 3:
        lens[rng.randrange(case["B"])] = 0
    return lens


def _tree(case):
    """(B, N) parents: -1 follows the context, -2 is padding; at most 4 children, depth below 9."""
    rng = random.Random(case["tree"])
    rows = []
    for _ in range(case["B"]):
        N = case["N"]
        n = rng.randint(max(1, N - N // 4), N)
        row, depth, kids = [], [], []
        for i in range(n):
            may = [j for j in range(i) if depth[j] < 8 and kids[j] < 4]
            p = rng.choice(may[-12:]) if may and (i > 3 or rng.random() < 0.5) else -1
            row.append(p)
            depth.append(0 if p < 0 else depth[p] + 1)
            kids.append(0)
            if p >= 0:
                kids[p] += 1
        rows.append(row + [-2] * (N - n))
    return rows


def _paths(case):
    """(B, A) accepted nodes of each draft, -1 behind the last."""
    rng = random.Random(case["lens"] + 1)
    N = case["N"]
    A = min(N, 9)
    rows = []
    for _ in range(case["B"]):
        path = sorted(rng.sample(range(N), rng.randint(0, A)))
        rows.append(path + [-1] * (A - len(path)))
    return rows


def _sources(case):
    """Which sequence each one continues: few of them several times, now and then none."""
    rng = random.Random(case["lens"] + 2)
    B = case["B"]
    best = rng.sample(range(B), max(1, B // 2))
    src = [rng.choice(best) for _ in range(B)]
    if B > 3:
        src[rng.randrange(B)] = -1
    return src


def _columns(case):
    return -(-case["S"] // case["page"])


def _used_pages(case, lens):
    return sum(-(-n // case["page"]) for n in lens)


def _pool_pages(case):
    """What the sequences hold, and as much again where pages are to be found."""
    lens = _lengths(case)
    n = _used_pages(case, lens)
    if case["op"] == "fork":
        return n + _used_pages(case, [case["S"]] * case["B"])
    return 2 * n if case["op"] == "compact" else n + n // 8 + 1


def _pool_bytes(case):
    es = 4 if case["dtype"] == "fp32" else 2
    tokens = _pool_pages(case) * case["page"] if case["page"] else case["B"] * case["S"]
    return 2 * case["L"] * tokens * case["Hkv"] * case["D"] * es


def _ancestors(row):
    """For each node the nodes it sees, itself the last."""
    out = []
    for i, p in enumerate(row):
        out.append((out[p] if p >= 0 else []) + [i] if p >= -1 else [])
    return out


def work(case):
    es = 4 if case["dtype"] == "fp32" else 2
    B, N, Hkv, D, L = case["B"], case["N"], case["Hkv"], case["D"], case["L"]
    lens = _lengths(case)
    row = 2 * L * Hkv * D * es  # one token's K and V of all layers
    tables = 0 if not case["page"] else 4 * _used_pages(case, lens)
    if case["op"] == "paged":
        H = case["H"]
        if case["tree"]:
            pairs = sum(max(0, n - N) + len(a) if a and n >= N else 0 for n, r in zip(lens, _tree(case)) for a in _ancestors(r))
        else:
            pairs = sum(max(0, n - N + i + 1) for n in lens for i in range(N))
        return {"bytes": 2 * B * N * H * D * es + row * sum(lens) + tables, "flops": 4 * D * H * pairs}
    if case["op"] == "write":
        return {"bytes": 2 * row * sum(min(N, n) for n in lens), "flops": 0}
    if case["op"] == "draft":
        moved = sum(j != a for p, n in zip(_paths(case), lens) for j, a in enumerate(p) if a >= 0 and n >= N)
        return {"bytes": 2 * row * (sum(min(N, n) for n in lens) + moved), "flops": 0}
    if case["op"] == "fork":
        src, ps = _sources(case), case["page"]
        seen, rows = set(), 0
        for s in src:
            if s >= 0 and s in seen:
                rows += lens[s] % ps
            seen.add(s)
        out = _used_pages(case, [lens[s] + N if s >= 0 else 0 for s in src])
        return {"bytes": 2 * row * rows + tables + 4 * out, "flops": 0}
    live = [n for n in lens]
    used = _used_pages(case, live)
    # half of the pages in use lie behind their number, as the pool has twice as many
    return {"bytes": 2 * row * case["page"] * (used // 2) + 2 * tables, "flops": 0}


# ---------------------------------------------------------------------------
# inputs

def _page_table(case, lens, g):
    """(B, columns) pages in no order; what no token needs holds -1."""
    M, ps, P = _columns(case), case["page"], _pool_pages(case)
    order = torch.randperm(P, generator=g, device="cuda").to(torch.int32)
    n = torch.tensor([-(-x // ps) for x in lens], device="cuda")
    at = (torch.cumsum(n, 0) - n)[:, None] + torch.arange(M, device="cuda")
    table = order[at.clamp(max=P - 1)]
    return torch.where(torch.arange(M, device="cuda") < n[:, None], table, torch.full_like(table, -1))


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    dt = _DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(shape, generator=g, device="cuda", dtype=dt)

    B, N, Hkv, D, L = case["B"], case["N"], case["Hkv"], case["D"], case["L"]
    lens = _lengths(case)
    st = {"case": case, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"), "table": None}
    if case["page"]:
        st["table"] = _page_table(case, lens, g)
        pool = (_pool_pages(case), case["page"], Hkv, D)
    else:
        pool = (B, case["S"], Hkv, D)
    if case["op"] in ("draft", "fork", "compact"):  # every layer's pages in one pool
        pool = (L,) + pool
    st["kc"], st["vc"] = randn(*pool), randn(*pool)
    if case["op"] == "paged":
        H = case["H"]
        st["q"] = randn(B, N, H, D)
        st["slopes"] = st["parents"] = None
        if case["slopes"]:
            e = torch.arange(1, H + 1, device="cuda", dtype=torch.float32) * (-8.0 / H)
            st["slopes"] = torch.exp2(e) * (1.0 + 0.05 * torch.randn(H, generator=g, device="cuda"))
        if case["tree"]:
            st["parents"] = torch.tensor(_tree(case), dtype=torch.int32, device="cuda")
    if case["op"] == "write":
        st["k"], st["v"] = randn(B, N, Hkv, D), randn(B, N, Hkv, D)
    if case["op"] == "draft":
        st["k"], st["v"] = randn(L, B, N, Hkv, D), randn(L, B, N, Hkv, D)
        st["path"] = torch.tensor(_paths(case), dtype=torch.int32, device="cuda")
    if case["op"] == "fork":
        st["sources"] = torch.tensor(_sources(case), dtype=torch.int32, device="cuda")
    return st


# ---------------------------------------------------------------------------
# the library's calls

def _run_own(st):
    fa, case = _fa(), st["case"]
    with torch.no_grad():
        if case["op"] == "paged":
            return fa.flash_attention_v100_paged(st["q"], st["kc"], st["vc"], st["lens"], st["table"],
                                                 parents=st["parents"], softcap=case["cap"],
                                                 distance_slopes=st["slopes"])
        if case["op"] == "write":
            return fa.paged_cache_write_v100(st["k"], st["v"], st["kc"], st["vc"], st["lens"], st["table"])
        if case["op"] == "draft":
            fa.paged_cache_write_v100(st["k"], st["v"], st["kc"], st["vc"], st["lens"], st["table"])
            lens = fa.paged_cache_accept_v100(st["kc"], st["vc"], st["lens"], st["path"], case["N"], st["table"])
            return st["kc"], st["vc"], lens
        if case["op"] == "fork":
            table, lens = fa.paged_cache_fork_v100(st["kc"], st["vc"], st["table"], st["lens"], st["sources"],
                                                   new_tokens=case["N"])
            return st["kc"], st["vc"], table, lens
        table, used = fa.paged_cache_compact_v100(st["kc"], st["vc"], st["table"], st["lens"])
        return st["kc"], st["vc"], table, used


# ---------------------------------------------------------------------------
# the plain form

def _seen_by_nodes(parents, B, N, device):
    """(B, N, N): which nodes each sees, and (B, N): which are in the tree."""
    if parents is None:
        return (torch.ones(N, N, dtype=torch.bool, device=device).tril().expand(B, N, N),
                torch.ones(B, N, dtype=torch.bool, device=device))
    i = torch.arange(N, device=device)
    reach = ((parents[..., None] == i) | (i[:, None] == i)).float()
    for _ in range(N.bit_length()):  # paths of twice the length each time
        reach = (torch.matmul(reach, reach) > 0).float()
    return reach > 0, parents >= -1


def _plain_paged(st):
    case, q, lens = st["case"], st["q"], st["lens"].long()
    B, N, H, D = q.shape
    Hkv, dev = case["Hkv"], q.device
    G = H // Hkv
    if st["table"] is None:
        k, v = st["kc"], st["vc"]
    else:
        t = st["table"].clamp(min=0).long()
        k, v = (x[t].flatten(1, 2) for x in (st["kc"], st["vc"]))
    kh, vh = (x.float().transpose(1, 2).contiguous() for x in (k, v))  # (B, Hkv, S, D)
    S = kh.shape[2]
    qh = q.float().view(B, N, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, N * G, D)
    x = torch.matmul(qh, kh.transpose(-1, -2).contiguous()) * D ** -0.5
    if case["cap"]:
        x = case["cap"] * torch.tanh(x / case["cap"])
    reach, inside = _seen_by_nodes(st["parents"], B, N, dev)
    c = lens - N
    j = torch.arange(S, device=dev)
    node = (j - c[:, None]).clamp(0, N - 1)  # (B, S)
    new = (j >= c[:, None]) & (j < lens[:, None])
    seen = (j < c[:, None])[:, None] | (new[:, None] & reach.gather(2, node[:, None].expand(B, N, S)))
    seen = seen & (inside & (c[:, None] + torch.arange(N, device=dev) >= 0))[..., None]
    if st["slopes"] is not None:
        pos = c[:, None] + reach.sum(-1) - 1
        key = torch.where(new, pos.gather(1, node), j)
        dist = (pos[..., None] - key[:, None]).abs().float().repeat_interleave(G, dim=1)[:, None]
        x = x - st["slopes"].view(1, Hkv, 1, G, 1).expand(1, Hkv, N, G, 1).reshape(1, Hkv, N * G, 1) * dist
    x = x.masked_fill(~seen.repeat_interleave(G, dim=1)[:, None], float("-inf"))
    m = x.amax(dim=-1, keepdim=True)
    e = torch.exp(x - torch.where(m == float("-inf"), torch.zeros_like(m), m))
    n = e.sum(dim=-1, keepdim=True)
    o = torch.matmul(e / torch.where(n == 0, torch.ones_like(n), n), vh)
    return o.view(B, Hkv, N, G, D).permute(0, 2, 1, 3, 4).reshape(B, N, H, D).to(q.dtype)


def _places(st, pos):
    """Page and row of positions (B, n)."""
    ps = st["case"]["page"]
    return st["table"].long().gather(1, (pos // ps).clamp(0, st["table"].shape[1] - 1)), pos % ps


def _plain_write(st):
    N, lens = st["case"]["N"], st["lens"].long()
    pos = lens[:, None] - N + torch.arange(N, device=lens.device)
    keep = pos >= 0
    page, row = _places(st, pos.clamp(min=0))
    page, row = page[keep], row[keep]
    if st["kc"].dim() == 5:
        st["kc"][:, page, row] = st["k"][:, keep]
        st["vc"][:, page, row] = st["v"][:, keep]
    else:
        st["kc"][page, row] = st["k"][keep]
        st["vc"][page, row] = st["v"][keep]
    return st["kc"], st["vc"]


def _plain_draft(st):
    _plain_write(st)
    N, lens, path = st["case"]["N"], st["lens"].long(), st["path"].long()
    c = lens - N
    moved = (path >= 0) & (c >= 0)[:, None]
    sp, sr = _places(st, (c[:, None] + path).clamp(min=0))
    dp, dr = _places(st, (c[:, None] + torch.arange(path.shape[1], device=lens.device)).clamp(min=0))
    sp, sr, dp, dr = (t[moved] for t in (sp, sr, dp, dr))
    st["kc"][:, dp, dr] = st["kc"][:, sp, sr]
    st["vc"][:, dp, dr] = st["vc"][:, sp, sr]
    return st["kc"], st["vc"], torch.where(c >= 0, c + moved.sum(1), lens).int()


def _plain_fork(st):
    case, table, src = st["case"], st["table"].long(), st["sources"].long()
    ps, N, dev = case["page"], case["N"], table.device
    B, M = table.shape
    P = st["kc"].shape[1]
    valid = src >= 0
    s = src.clamp(min=0)
    n = torch.where(valid, st["lens"].long()[s], torch.zeros_like(s))
    full, part = n // ps, n % ps
    b = torch.arange(B, device=dev)
    again = ((src[:, None] == src) & (b < b[:, None])).any(1)  # an earlier one continues the same
    copy = valid & again & (part > 0)
    kept = full + ((part > 0) & ~copy)
    pages = torch.where(valid, (n + N + ps - 1) // ps, torch.zeros_like(n))
    m = torch.arange(M, device=dev)
    old = table[s]
    holds = m < kept[:, None]
    free = torch.ones(P, dtype=torch.bool, device=dev)
    free[old[holds]] = False
    order = torch.argsort((~free).int(), stable=True)
    need = pages - kept
    first = torch.cumsum(need, 0) - need
    fresh = order[(first[:, None] + m - kept[:, None]).clamp(0, P - 1)]
    out = torch.where(holds, old, torch.where(m < pages[:, None], fresh, torch.full_like(fresh, -1)))
    which = copy.nonzero().squeeze(1)
    frm, to = old[which, full[which]], out[which, full[which]]
    rows = (torch.arange(ps, device=dev) < part[which][:, None])[None, ..., None, None]
    for x in (st["kc"], st["vc"]):
        x[:, to] = torch.where(rows, x[:, frm], x[:, to])
    return st["kc"], st["vc"], out.int(), torch.where(valid, n + N, n).int()


def _plain_compact(st):
    ps, table = st["case"]["page"], st["table"].long()
    P = st["kc"].shape[1]
    holds = torch.arange(table.shape[1], device=table.device) < ((st["lens"].long() + ps - 1) // ps)[:, None]
    live = torch.zeros(P, dtype=torch.bool, device=table.device)
    live[table[holds]] = True
    used = live.sum()
    p = torch.arange(P, device=table.device)
    holes, movers = (~live & (p < used)).nonzero().squeeze(1), (live & (p >= used)).nonzero().squeeze(1)
    to = p.clone()
    to[movers] = holes
    st["kc"][:, holes] = st["kc"][:, movers]
    st["vc"][:, holes] = st["vc"][:, movers]
    out = torch.where(holds, to[table.clamp(min=0)], torch.full_like(table, -1))
    return st["kc"], st["vc"], out.int(), used.int()


def run(state):
    if own:
        return _run_own(state)
    return {"paged": _plain_paged, "write": _plain_write, "draft": _plain_draft, "fork": _plain_fork,
            "compact": _plain_compact}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------
# the definition in 64 bits

def _exact_paged(case, st):
    q, slopes = st["q"], st["slopes"]
    B, N, H, D = q.shape
    G, ps = H // case["Hkv"], case["page"]
    trees = _tree(case) if case["tree"] else [list(range(-1, N - 1))] * B
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, n in enumerate(_lengths(case)):
        if n == 0:
            continue
        if ps:
            t = st["table"][b].tolist()[:-(-n // ps)]
            kb, vb = (torch.cat([x[p] for p in t])[:n].double() for x in (st["kc"], st["vc"]))
        else:
            kb, vb = st["kc"][b, :n].double(), st["vc"][b, :n].double()
        c = n - N
        hidden = torch.ones(N, n, dtype=torch.bool)
        place = [float(x) for x in range(n)]
        for i, line in enumerate(_ancestors(trees[b])):
            if not line or c + i < 0:
                continue
            hidden[i, :max(c, 0)] = False
            for a in line:
                if c + a >= 0:
                    hidden[i, c + a] = False
            place[c + i] = float(c + len(line) - 1)
        hidden = hidden.to(q.device)
        empty = hidden.all(dim=1)
        kp = torch.tensor(place, dtype=torch.float64, device=q.device)
        qp = torch.cat([torch.zeros(max(0, -c), dtype=torch.float64, device=q.device), kp[max(c, 0):]])
        for h in range(H):
            s = q[b, :, h].double() @ kb[:, h // G].T / math.sqrt(D)
            if case["cap"]:
                e = torch.exp(-2.0 * (s / case["cap"]).abs())
                s = case["cap"] * torch.sign(s) * (1.0 - e) / (1.0 + e)
            if slopes is not None:
                s = s - slopes[h].double() * (qp[:, None] - kp[None, :]).abs()
            w = torch.softmax(s.masked_fill(hidden, -1e300), dim=1)
            out[b, :, h] = torch.where(empty[:, None], torch.zeros_like(vb[:1, 0]), w @ vb[:, h // G])
    return out


def exact(case, seed):
    st = prepare(case, seed)
    op, ps, N = case["op"], case["page"], case["N"]
    if op == "paged":
        return _exact_paged(case, st)
    kc, vc = st["kc"].double(), st["vc"].double()
    table, lens = st["table"].tolist(), _lengths(case)
    if op in ("write", "draft"):
        lead = (slice(None),) if op == "draft" else ()
        for b, n in enumerate(lens):
            p = [(table[b][x // ps] * ps + x % ps) for x in range(max(0, n - N), n)]
            if not p:
                continue
            at = torch.tensor(p, device=kc.device)
            for x, y in ((kc, st["k"]), (vc, st["v"])):
                flat = x.view(*x.shape[:-4], -1, *x.shape[-2:])
                flat[lead + (at,)] = y[lead + (b, slice(N - len(p), N))].double()
        if op == "write":
            return kc, vc
        new = []
        for b, (n, path) in enumerate(zip(lens, _paths(case))):
            path = [a for a in path if a >= 0]
            new.append(n - N + len(path) if n >= N else n)
            for x in (kc, vc):
                flat = x.view(x.shape[0], -1, *x.shape[-2:])
                place = [table[b][(n - N + a) // ps] * ps + (n - N + a) % ps for a in range(N)] if n >= N else []
                for j, a in enumerate(path if place else []):
                    flat[:, place[j]] = flat[:, place[a]]
        return kc, vc, torch.tensor(new, dtype=torch.int32, device=kc.device)
    M, P = len(table[0]), kc.shape[1]
    if op == "fork":
        rows, new, taken, copies, first = [], [], set(), [], set()
        for s in _sources(case):
            n = lens[s] if s >= 0 else 0
            have = table[s][:n // ps]
            if n % ps and s not in first:
                have = table[s][:n // ps + 1]
            elif n % ps:
                copies.append((len(rows), table[s][n // ps], n // ps, n % ps))
            first.add(s)
            taken.update(have)
            rows.append(list(have))
            new.append(n + N if s >= 0 else 0)
        free = iter(p for p in range(P) if p not in taken)
        for r, n in zip(rows, new):
            while len(r) * ps < n:
                r.append(next(free))
        for b, frm, col, part in copies:
            for x in (kc, vc):
                x[:, rows[b][col], :part] = x[:, frm, :part]
        rows = [r + [-1] * (M - len(r)) for r in rows]
        return (kc, vc, torch.tensor(rows, dtype=torch.int32, device=kc.device),
                torch.tensor(new, dtype=torch.int32, device=kc.device))
    rows = [r[:-(-n // ps)] for r, n in zip(table, lens)]
    live = sorted({p for r in rows for p in r})
    holes = [p for p in range(len(live)) if p not in set(live)]
    to = {p: p for p in live}
    to.update(zip([p for p in live if p >= len(live)], holes))
    for p, h in to.items():
        if p != h:
            kc[:, h], vc[:, h] = kc[:, p], vc[:, p]
    rows = [[to[p] for p in r] + [-1] * (M - len(r)) for r in rows]
    return (kc, vc, torch.tensor(rows, dtype=torch.int32, device=kc.device),
            torch.tensor(len(live), dtype=torch.int32, device=kc.device))
