"""Oracle of the paged key/value cache: attention over it in 64 bits, sequence by
sequence (bounds of :mod:`ops_oracle`), and what its operators leave in pools, tables
and lengths, by lists."""
import random

import torch

import ops_oracle as oo


def ancestors(parents):
    """Per token the tokens it sees, itself the last; none for what is no token."""
    out = []
    for i, p in enumerate(parents):
        if p == -1:
            out.append([i])
        elif 0 <= p < i and out[p]:
            out.append(out[p] + [i])
        else:
            out.append([])
    return out


def draw_tree(rng, n, depth=9):
    row, deep = [], []
    for i in range(n):
        may = [j for j in range(i) if deep[j] < depth - 1]
        p = rng.choice(may) if may and rng.random() < 0.85 else -1
        row.append(p)
        deep.append(0 if p < 0 else deep[p] + 1)
    return row


def place(table, b, x, size):
    """(page, row) of token x of sequence b, None where there is no page."""
    if table is None:
        return b, x
    return table[b][x // size], x % size


def attention(q, kc, vc, lens, table=None, parents=None, softcap=0.0, slopes=None, scale=None):
    """{"o", "lse"}: (value, bound).  Integers as lists; pools may hold anything in places
    that nothing sees."""
    B, N, H, D = q.shape
    P, size = kc.shape[:2]
    room = size if table is None else len(table[0]) * size
    dev = q.device
    outs = []
    for b in range(B):
        n = room if lens is None else max(0, min(room, lens[b]))
        c = n - N
        rows = parents if parents is None or not isinstance(parents[0], list) else parents[b]
        sees = [list(range(i + 1)) for i in range(N)] if rows is None else ancestors(rows)
        pos = [c + len(s) - 1 for s in sees]
        seen = torch.zeros(1, N, max(n, 1), dtype=torch.bool)
        for i, s in enumerate(sees):
            if s and c + i >= 0:
                seen[0, i, :max(c, 0)] = True
                for a in s:
                    if c + a >= 0:
                        seen[0, i, c + a] = True
        k = torch.zeros(1, max(n, 1), *kc.shape[2:], dtype=kc.dtype, device=dev)
        v = torch.zeros_like(k)
        at = [place(table, b, x, size) for x in range(n)]
        ok = [x for x in range(n) if 0 <= at[x][0] < P]
        for x in set(range(n)) - set(ok):
            seen[0, :, x] = False
        if ok:
            pages = torch.tensor([at[x][0] for x in ok], device=dev)
            rs = torch.tensor([at[x][1] for x in ok], device=dev)
            k[0, ok], v[0, ok] = kc[pages, rs], vc[pages, rs]
        hidden = ~seen[0].any(0)  # keys that no token sees: whatever they hold
        k[0, hidden.to(dev)] = 0
        v[0, hidden.to(dev)] = 0
        kpos = torch.arange(max(n, 1), device=dev)
        for i in range(N):
            if 0 <= c + i:
                kpos[c + i] = pos[i] if sees[i] else c + i
        sl = slopes if slopes is None or slopes.dim() == 1 else slopes[b:b + 1]
        outs.append(oo.scored(q[b:b + 1], k, v, None, scale, softcap, sl, 0, seen, kpos=kpos,
                              qpos=torch.tensor([pos], device=dev)))
    return {x: tuple(torch.cat([o[x][y] for o in outs]) for y in (0, 1)) for x in ("o", "lse")}


def write(kc, vc, k, v, lens, table):
    """The pools after a write; leading layers on all of them."""
    kc, vc = kc.clone(), vc.clone()
    P, size = kc.shape[1:3]
    N = k.shape[2]
    for b, n in enumerate(lens):
        for i in range(N):
            x = n - N + i
            if x < 0:
                continue
            p, r = place(table, b, x, size)
            if 0 <= p < P:
                kc[:, p, r], vc[:, p, r] = k[:, b, i], v[:, b, i]
    return kc, vc


def accept(kc, vc, lens, path, N, table):
    kc, vc, new = kc.clone(), vc.clone(), []
    P, size = kc.shape[1:3]
    for b, n in enumerate(lens):
        if n < N:
            new.append(n)
            continue
        keep, last = [], -1
        for a in path[b]:
            if a <= last or a >= N:
                break
            keep.append(a)
            last = a
        for j, a in enumerate(keep):
            (p0, r0), (p1, r1) = place(table, b, n - N + a, size), place(table, b, n - N + j, size)
            if 0 <= p0 < P and 0 <= p1 < P:
                for x in (kc, vc):
                    x[:, p1, r1] = x[:, p0, r0].clone()
        new.append(n - N + len(keep))
    return kc, vc, new


def fork(kc, vc, table, lens, sources, more):
    """(pools, table, lengths) as paged_cache_fork_v100 documents them."""
    kc, vc = kc.clone(), vc.clone()
    P, size = kc.shape[1:3]
    M, B = len(table[0]) if table else 0, len(table)
    kept, plans, heirs = set(), [], set()
    for b, s in enumerate(sources):
        if not 0 <= s < B:
            plans.append(None)
            continue
        n, add = max(0, min(lens[s], M * size)), max(0, more[b])
        if n + add > M * size:
            plans.append(None)
            continue
        have, copy = list(table[s][:n // size]), None
        if n % size:
            page = table[s][n // size]
            if s in heirs and 0 <= page < P:
                copy = (page, n % size)
            else:
                have.append(page)
            heirs.add(s)
        kept.update(p for p in have if 0 <= p < P)
        plans.append((have, copy, n + add))
    free = [p for p in range(P) if p not in kept]
    rows, new, wanted = [], [], 0
    for plan in plans:
        if plan is not None:
            have, copy, n = plan
            need = -(-n // size) - len(have)
            first, wanted = wanted, wanted + need
            if need == 0 or wanted <= len(free):
                row = have + free[first:first + need]
                if copy:
                    for x in (kc, vc):
                        x[:, row[len(have)], :copy[1]] = x[:, copy[0], :copy[1]].clone()
                rows.append([p if 0 <= p < P else -1 for p in row] + [-1] * (M - len(row)))
                new.append(n)
                continue
        rows.append([-1] * M)
        new.append(0)
    return kc, vc, rows, new


def compact(kc, vc, table, lens):
    kc, vc = kc.clone(), vc.clone()
    P, size = kc.shape[1:3]
    M = len(table[0]) if table else 0
    rows = [r[:-(-max(0, min(n, M * size)) // size)] for r, n in zip(table, lens)]
    live = sorted({p for r in rows for p in r if 0 <= p < P})
    U = len(live)
    to = {p: p for p in live}
    to.update(zip([p for p in live if p >= U], [p for p in range(U) if p not in set(live)]))
    for p, h in to.items():
        if p != h:
            for x in (kc, vc):
                x[:, h] = x[:, p].clone()
    return kc, vc, [[to.get(p, -1) for p in r] + [-1] * (M - len(r)) for r in rows], U


def draw_table(rng, lens, size, M, P):
    """A page table of pages in no order, -1 behind each sequence's."""
    pages = list(range(P))
    rng.shuffle(pages)
    rows = []
    for n in lens:
        k = -(-n // size)
        rows.append([pages.pop() for _ in range(k)] + [-1] * (M - k))
    return rows


def rng(*seed):
    return random.Random(str(seed))
