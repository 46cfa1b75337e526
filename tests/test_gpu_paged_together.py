"""The paged cache as a serving loop runs it: a layer that decodes over it, drafts that
are verified and accepted, beams, compaction; captured and replayed, on other streams,
two calls at once."""
import math

import pytest
import torch

import flash_attention_v100 as fa
import ops_oracle as oo
import paged_oracle as po

pytestmark = pytest.mark.gpu
DEV = "cuda"


def ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEV)


def layer(dt, seed=0, **kw):
    torch.manual_seed(seed)
    return fa.EnhancedMultiHeadAttention(256, 4, **kw).to(DEV, dt).eval()


def cache(pages, size, Hkv, D, dt, layers=None):
    s = (pages, size, Hkv, D) if layers is None else (layers, pages, size, Hkv, D)
    return torch.full(s, math.nan, dtype=dt, device=DEV), torch.full(s, math.nan, dtype=dt, device=DEV)


OPTIONS = [{}, {"rotary_dim": 32}, {"rotary_dim": 64, "rotary_interleaved": True, "softcap": 5.0}, {"distance_bias": True}]


@pytest.mark.parametrize("dt,tol", [(torch.float32, 2e-5), (torch.bfloat16, 3e-2)])
@pytest.mark.parametrize("kw", OPTIONS)
@pytest.mark.parametrize("batch_first", [True, False])
def test_layer_decodes_what_it_computes_at_once(dt, tol, kw, batch_first):
    # the causal layer over whole sequences, and token by token over the cache: the same
    # sums in another order.  float32: outputs near 1 of 256 products, 2^-24 each way a few
    # times; bf16: projections rounded to 2^-8 of values near 1, in both.
    m = layer(dt, batch_first=batch_first, **kw)
    B, S = 3, 70
    x = torch.randn(B, S, 256, generator=torch.Generator("cpu").manual_seed(1)).to(DEV, dt)
    with torch.no_grad():
        want = (m(x, is_causal=True)[0] if batch_first else m(x.transpose(0, 1), is_causal=True)[0].transpose(0, 1))
    kc, vc = cache(20, 16, 4, 64, dt)
    table, lens = ints([[3, 9, 4, 17, 0], [5, 1, 19, 2, 11], [7, 8, 10, 12, 13]]), torch.zeros(B, dtype=torch.int32, device=DEV)
    got = []
    for a, b in ((0, 40), (40, 41), (41, 42), (42, 60), (60, 70)):
        lens = lens + (b - a)
        y = x[:, a:b] if batch_first else x[:, a:b].transpose(0, 1)
        o = m.decode(y, kc, vc, lens, table)
        got.append(o if batch_first else o.transpose(0, 1))
    assert (torch.cat(got, 1).float() - want.float()).abs().max() <= tol


def test_layer_refuses():
    m = layer(torch.float32, rotary_dim=32)
    kc, vc = cache(4, 16, 4, 64, torch.float32)
    x = torch.randn(1, 3, 256, device=DEV)
    with pytest.raises(ValueError, match="positions"):
        m.decode(x, kc, vc, ints([3]), ints([[0]]), parents=ints([-1, 0, 0]))
    with pytest.raises(ValueError, match="rotary_dim"):
        layer(torch.float32).decode(x, kc, vc, ints([3]), ints([[0]]), positions=ints([0, 1, 2]))
    d = layer(torch.float32, dropout=0.1)
    d.train()
    with pytest.raises(ValueError, match="dropout"):
        d.decode(x, kc, vc, ints([3]), ints([[0]]))
    assert not m.decode(x, kc, vc, ints([3]), ints([[0]])).requires_grad


def test_draft_accept_fork_compact():
    # prompt, a tree verified and accepted, beams forked, compaction: at every step attention
    # over the cache is that over the tokens that each sequence is supposed to hold
    g = torch.Generator("cpu").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.float16).to(DEV)  # noqa: E731
    B, Hkv, H, D, size, P, M, L = 3, 2, 8, 64, 16, 64, 12, 2
    kc, vc = cache(P, size, Hkv, D, torch.float16, L)
    table, lens = ints([[-1] * M] * B), ints([0] * B)
    text = [[[] for _ in range(B)] for _ in range(L)]  # (k, v) rows of each layer and sequence

    def look(label):
        q = r(len(text[0]), 1, H, D)
        for x in range(L):
            o = fa.flash_attention_v100_paged(q, kc[x], vc[x], lens, table)
            n = max(len(t) for t in text[x])
            ks, vs = (torch.zeros(len(text[x]), n, Hkv, D, dtype=torch.float16, device=DEV) for _ in range(2))
            for b, t in enumerate(text[x]):
                for i, (a, c) in enumerate(t):
                    ks[b, i], vs[b, i] = a, c
            full = torch.tensor([len(t) for t in text[x]])
            assert lens.tolist() == full.tolist()
            ref = po.attention(q, ks, vs, full.tolist())
            oo.check({"o": o}, ref, ["o"], f"{label}, layer {x}")

    def write(N, keep):
        k, v = r(L, len(text[0]), N, Hkv, D), r(L, len(text[0]), N, Hkv, D)
        fa.paged_cache_write_v100(k, v, kc, vc, lens, table)
        for x in range(L):
            for b in range(len(text[0])):
                text[x][b] += [(k[x, b, i], v[x, b, i]) for i in keep(b)]

    # prompts of 37 tokens (room by a fork of each sequence to itself)
    table, lens = fa.paged_cache_fork_v100(kc, vc, table, lens, ints([0, 1, 2]), 37)
    write(37, lambda b: range(37))
    look("prompt")
    # trees of 10 drafted tokens, of which paths are kept
    paths = [[0, 2, 5], [1, 9], []]
    table, lens = fa.paged_cache_fork_v100(kc, vc, table, lens, ints([0, 1, 2]), 10)
    write(10, lambda b: paths[b])
    lens = fa.paged_cache_accept_v100(kc, vc, lens, ints([p + [-1] * (4 - len(p)) for p in paths]), 10, table)
    look("accepted")
    # beams: the first in three copies, the last dropped; new tokens of their own
    table, lens = fa.paged_cache_fork_v100(kc, vc, table, lens, ints([0, 1, 0, -1, 0]), ints([3, 3, 3, 0, 3]))
    text = [[list(t[0]), list(t[1]), list(t[0]), [], list(t[0])] for t in text]
    k, v = r(L, 5, 3, Hkv, D), r(L, 5, 3, Hkv, D)
    fa.paged_cache_write_v100(k, v, kc, vc, lens, table)
    for x in range(L):
        for b in (0, 1, 2, 4):
            text[x][b] += [(k[x, b, i], v[x, b, i]) for i in range(3)]
    look("beams")
    table, used = fa.paged_cache_compact_v100(kc, vc, table, lens)
    live = {p for row, n in zip(table.tolist(), lens.tolist()) for p in row[:-(-n // size)]}
    assert live == set(range(int(used)))
    look("compact")


def tree_step(state):
    """One step of drafting as it is captured: rows written, trees attended, paths kept."""
    fa.paged_cache_write_v100(state["k"], state["v"], state["kc"], state["vc"], state["lens"], state["table"])
    o = fa.flash_attention_v100_paged(state["q"], state["kc"], state["vc"], state["lens"], state["table"], parents=state["par"])
    lens = fa.paged_cache_accept_v100(state["kc"], state["vc"], state["lens"], state["path"], state["q"].shape[1], state["table"])
    table, more = fa.paged_cache_fork_v100(state["kc"], state["vc"], state["table"], lens, state["src"], 2)
    table2, used = fa.paged_cache_compact_v100(state["kc"], state["vc"], table, more)
    return o, lens, table, more, table2, used


def tree_state(seed, big=False):
    rng, g = po.rng("step", seed), torch.Generator("cpu").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).to(torch.bfloat16).to(DEV)  # noqa: E731
    B, N, H, Hkv, D, size, M = (6, 40, 16, 4, 128, 16, 130) if big else (4, 9, 8, 2, 64, 16, 40)
    lens = [rng.randint(N, M * size - 2) for _ in range(B)]
    P = B * M
    return {"q": r(B, N, H, D), "k": r(B, N, Hkv, D), "v": r(B, N, Hkv, D), "kc": r(P, size, Hkv, D), "vc": r(P, size, Hkv, D),
            "lens": ints(lens), "table": ints(po.draw_table(rng, lens, size, M, P)),
            "par": ints([po.draw_tree(rng, N) for _ in range(B)]),
            "path": ints([sorted(rng.sample(range(N), 4)) + [-1] for _ in range(B)]), "src": ints([0, 0] + list(range(B - 2)))}


def clone(st):
    return {k: v.clone() for k, v in st.items()}


@pytest.mark.parametrize("big", [False, True])
def test_captured_and_replayed(big):
    # replays on new inputs, with eager work and synchronizations between them, equal the eager step
    first = tree_state(1, big)
    st = clone(first)
    tree_step(clone(first))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = tree_step(st)
    for seed in (1, 2, 3, 2):
        fresh = tree_state(seed, big)
        for name in st:
            st[name].copy_(fresh[name])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (*out, st["kc"], st["vc"])]
        eager = clone(fresh)
        want = (*tree_step(eager), eager["kc"], eager["vc"])
        assert all(torch.equal(a, b) for a, b in zip(got, want)), seed


def test_other_streams_and_two_calls_at_once():
    # each stream's tensors are its own: what runs beside them changes nothing
    states = [tree_state(s, s % 2 == 0) for s in range(4)]
    want = []
    for s in states:
        c = clone(s)
        want.append((*tree_step(c), c["kc"], c["vc"]))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    for _ in range(3):
        runs = [clone(s) for s in states]
        torch.cuda.synchronize()
        outs = []
        for st, stream in zip(runs, streams):
            with torch.cuda.stream(stream):
                outs.append(tree_step(st))
        torch.cuda.synchronize()
        for o, c, w in zip(outs, runs, want):
            assert all(torch.equal(a, b) for a, b in zip((*o, c["kc"], c["vc"]), w))


def test_versions_of_written_caches():
    # autograd learns that a cache it saved has been written
    st = tree_state(5)
    before = st["kc"]._version, st["vc"]._version
    fa.paged_cache_write_v100(st["k"], st["v"], st["kc"], st["vc"], st["lens"], st["table"])
    assert st["kc"]._version > before[0] and st["vc"]._version > before[1]
    with torch.inference_mode():
        st = tree_state(5)
        tree_step(st)


def test_refusals_on_the_gpu():
    st = tree_state(6)
    q, kc, vc, lens, table = (st[x] for x in ("q", "kc", "vc", "lens", "table"))
    call = fa.flash_attention_v100_paged
    with pytest.raises(ValueError, match="page_table"):
        call(q, kc, vc, lens, table[:2])
    with pytest.raises(ValueError, match="page_table"):
        call(q, kc, vc, lens, table.float())
    with pytest.raises(ValueError, match="key_lengths"):
        call(q, kc, vc, lens[:2], table)
    with pytest.raises(ValueError, match="without a page_table"):
        call(q, kc, vc, lens)
    with pytest.raises(ValueError, match="multiple of 16"):
        call(q, kc[:, :8].contiguous(), vc[:, :8].contiguous(), lens, table)
    with pytest.raises(ValueError, match="does not match"):
        call(q.half(), kc, vc, lens, table)
    with pytest.raises(ValueError, match="multiple of num_heads_kv"):
        call(q[:, :, :3], kc, vc, lens, table)
    with pytest.raises(ValueError, match="unit stride"):
        call(q, kc.transpose(2, 3).contiguous().transpose(2, 3), vc, lens, table)
    with pytest.raises(ValueError, match="parents"):
        call(q, kc, vc, lens, table, parents=st["par"][:, :3])
    with pytest.raises(NotImplementedError, match="256"):
        call(q[:, :1].expand(-1, 257, -1, -1), kc, vc, lens, table, parents=torch.zeros(257, dtype=torch.int32, device=DEV))
    with pytest.raises(NotImplementedError, match="head_dim"):
        call(q[..., :60], kc[..., :60].contiguous(), vc[..., :60].contiguous(), lens, table)
    with pytest.raises(ValueError, match="same memory"):
        fa.paged_cache_write_v100(st["k"], st["v"], kc, kc, lens, table)
    with pytest.raises(ValueError, match="overlapping"):
        fa.paged_cache_write_v100(st["k"], st["v"], kc[:1].expand(kc.shape), vc, lens, table)
    with pytest.raises(ValueError, match="do not match the cache"):
        fa.paged_cache_write_v100(st["k"][:, :, :1], st["v"][:, :, :1], kc, vc, lens, table)
    with pytest.raises(ValueError, match="dtype"):
        fa.paged_cache_write_v100(st["k"].half(), st["v"], kc, vc, lens, table)
    with pytest.raises(NotImplementedError, match="no_grad"):
        fa.paged_cache_write_v100(st["k"].requires_grad_(True), st["v"], kc, vc, lens, table)
    with pytest.raises(NotImplementedError, match="grad"):
        call(q, kc.clone().requires_grad_(True), vc, lens, table)
    with pytest.raises(ValueError, match="drafted"):
        fa.paged_cache_accept_v100(kc, vc, lens, st["path"], -1, table)
    with pytest.raises(ValueError, match="path"):
        fa.paged_cache_accept_v100(kc, vc, lens, st["path"].float(), 3, table)
    with pytest.raises(ValueError, match="new_tokens"):
        fa.paged_cache_fork_v100(kc, vc, table, lens, st["src"], -1)
    with pytest.raises(ValueError, match="new_tokens"):
        fa.paged_cache_fork_v100(kc, vc, table, lens, st["src"], lens[:2])
    with pytest.raises(ValueError, match="sources"):
        fa.paged_cache_fork_v100(kc, vc, table, lens, st["src"][None])
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        dual = fwd.make_dual(q.clone(), torch.ones_like(q))
        with pytest.raises(NotImplementedError, match="forward"):
            call(dual, kc, vc, lens, table)
