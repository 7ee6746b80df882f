"""The references of a beam search's ops on CPU tensors against definitions written apart, their refusals, and a whole search on them."""
import itertools
import math

import pytest
import torch

from distributed_sse_for_llm_response_amd import ops
from distributed_sse_for_llm_response_amd.engine import kv_cache
from distributed_sse_for_llm_response_amd.ops import beams_reference as bref

INF = math.inf
i32 = torch.int32


def _outs(G, K):
    return torch.zeros(G, K), torch.zeros(G, K, dtype=i32), torch.zeros(G, K, dtype=i32)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("G,W,V,K,eos", [(1, 1, 4, 6, -1), (2, 3, 50, 7, 3), (3, 4, 33, 64, -1), (1, 8, 200, 16, 199)])
def test_select_against_all_scores(dtype, G, W, V, K, eos):
    gen = torch.Generator().manual_seed(V)
    x = torch.randn(G * W, V, generator=gen).to(dtype)
    x[torch.rand(G * W, V, generator=gen) < 0.2] = -INF
    s = -torch.rand(G, W, generator=gen)
    s[0, 0] = -INF
    o, end = _outs(G, K), torch.zeros(G, W)
    ops.beam_select(x, s, *o, eos, end if eos >= 0 else None)
    lp = s.double().view(-1, 1) + torch.log_softmax(x.double(), 1)
    for g in range(G):
        all_ = sorted((-float(lp[r, t]), r, t) for r in range(g * W, g * W + W) for t in range(V) if t != eos and lp[r, t] > -INF)[:K]
        n = len(all_)
        assert o[1][g].tolist() == [r for _, r, _ in all_] + [-1] * (K - n)
        assert o[2][g].tolist() == [t for _, _, t in all_] + [-1] * (K - n)
        assert torch.allclose(o[0][g, :n], torch.tensor([-v for v, _, _ in all_]), rtol=2.0 ** -23, atol=0)
        assert bool((o[0][g, n:] == -INF).all())
    if eos >= 0:
        assert torch.allclose(end, lp[:, eos].float().view(G, W), rtol=2.0 ** -22, atol=0)


def test_select_orders_equal_scores():
    o = _outs(1, 5)
    ops.beam_select(torch.zeros(3, 4), torch.tensor([[-1.0, 0.0, 0.0]]), *o)
    assert o[1].tolist() == [[1, 1, 1, 1, 2]] and o[2].tolist() == [[0, 1, 2, 3, 0]]


def test_select_scores_in_place():
    """The new scores may take the old ones' place."""
    gen = torch.Generator().manual_seed(31)
    x, s = torch.randn(12, 900, generator=gen), -torch.rand(3, 4, generator=gen)
    apart = torch.zeros(3, 4), torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, 4, dtype=torch.int32)
    end, end2 = torch.zeros(3, 4), torch.zeros(3, 4)
    ops.beam_select(x, s, *apart, 5, end)
    rows, tokens = torch.zeros_like(apart[1]), torch.zeros_like(apart[2])
    ops.beam_select(x, s, s, rows, tokens, 5, end2)
    assert torch.equal(s, apart[0]) and torch.equal(rows, apart[1]) and torch.equal(tokens, apart[2]) and torch.equal(end, end2)


def test_select_refusals():
    x, s, o = torch.zeros(4, 9), torch.zeros(2, 2), _outs(2, 3)
    bad = [dict(logits=x.half()), dict(logits=x.t().contiguous().t()), dict(logits=x[:3]), dict(scores=s.double()), dict(scores=s.view(1, 4)),
           dict(out_rows=o[1].long()), dict(out_tokens=o[2][:, :2].contiguous()), dict(out_scores=torch.zeros(2, 65)), dict(eos_id=9),
           dict(eos_id=-2), dict(end_scores=torch.zeros(2, 2)), dict(end_scores=torch.zeros(2, 3), eos_id=1), dict(logits=x[:, :0])]
    for change in bad:
        a = dict(logits=x, scores=s, out_scores=o[0], out_rows=o[1], out_tokens=o[2], eos_id=-1, end_scores=None)
        a.update(change)
        with pytest.raises(RuntimeError):
            ops.beam_select(**a)
    with pytest.raises(RuntimeError):
        ops.beam_select(torch.zeros(33, 9), torch.zeros(1, 33), *_outs(1, 3))


def test_shared_pages():
    bt = torch.tensor([[5, 6, 7, 8], [5, 6, 9, 8], [1, 2, 3, 4], [1, 2, 3, 4]], dtype=i32)
    sh = torch.zeros(2, dtype=i32)
    for ctx, want in (([128, 128, 128, 128], [2, 4]), ([40, 128, 127, 128], [1, 3]), ([0, 90, 0, 0], [2, 0]), ([31, 128, 500, 500], [0, 4])):
        ops.beam_shared(bt, torch.tensor(ctx, dtype=i32), 2, sh)
        assert sh.tolist() == want
    with pytest.raises(RuntimeError):
        ops.beam_shared(bt, torch.zeros(4, dtype=i32), 3, sh)
    with pytest.raises(RuntimeError):
        ops.beam_shared(bt, torch.zeros(3, dtype=i32), 2, sh)


def test_attention_refusals():
    b = torch.bfloat16
    a = dict(q=torch.zeros(4, 8, 128, dtype=b), k_cache=torch.zeros(3, 2, 32, 128, dtype=b), v_cache=torch.zeros(3, 2, 128, 32, dtype=b),
             block_tables=torch.zeros(4, 2, dtype=i32), ctx_len=torch.ones(4, dtype=i32), shared=torch.zeros(2, dtype=i32),
             out=torch.zeros(4, 8, 128, dtype=b), width=2)
    ops.beam_attention(**a)
    for change in (dict(q=a["q"].float()), dict(q=a["q"][:, :, :64].contiguous()), dict(q=a["q"][:, :7].contiguous(), out=a["out"][:, :7].contiguous()),
                   dict(out=a["out"][:3]), dict(k_cache=a["k_cache"][:, :, :16].contiguous()), dict(v_cache=a["k_cache"]), dict(width=3),
                   dict(width=0), dict(shared=torch.zeros(4, dtype=i32)), dict(ctx_len=torch.ones(3, dtype=i32)),
                   dict(block_tables=torch.zeros(4, 2, dtype=torch.int64)), dict(block_tables=torch.zeros(3, 2, dtype=i32)),
                   dict(q=torch.zeros(4, 34, 128, dtype=b), out=torch.zeros(4, 34, 128, dtype=b))):
        with pytest.raises(RuntimeError):
            ops.beam_attention(**{**a, **change})


def _fork_args(S=4, M=3, P=9):
    return dict(block_tables=torch.zeros(S, M, dtype=i32), held=torch.zeros(S, dtype=i32), lens=torch.zeros(S, dtype=i32),
                parents=torch.arange(S, dtype=i32), refs=torch.zeros(P, dtype=i32), copies=torch.zeros(S, 2, dtype=i32),
                starved=torch.zeros(1, dtype=i32), pools=[torch.zeros(2, P, 4)])


def test_fork_refusals():
    a = _fork_args()
    ops.page_fork(**a)
    for change in (dict(held=a["held"].long()), dict(lens=a["lens"][:3]), dict(parents=a["parents"][:3]), dict(copies=torch.zeros(4, dtype=i32)),
                   dict(starved=torch.zeros(2, dtype=i32)), dict(refs=a["refs"][:0]), dict(pools=[torch.zeros(2, 8, 4)]),
                   dict(pools=[torch.zeros(2, 9, 3)]), dict(pools=[torch.zeros(9, 4)]), dict(pools=[torch.zeros(2, 9, 4, 2)[..., 0]]),
                   dict(block_tables=a["block_tables"][:, :0])):
        with pytest.raises(RuntimeError):
            ops.page_fork(**{**a, **change})
    with pytest.raises(RuntimeError):
        ops.page_fork(**_fork_args(S=2049))


def test_fork_as_sequences():
    """Whatever the forks, every slot's pages hold its own sequence: tokens written page by page against lists of tokens."""
    gen = torch.Generator().manual_seed(1)
    S, M, P = 6, 4, 6 * 4 + 6
    a = _fork_args(S, M, P)
    a["pools"] = [torch.full((1, P, 32, 4), -1.0)]
    texts = [[] for _ in range(S)]
    for step in range(100):
        parents = [int(x) for x in torch.randint(-1, S, (S,), generator=gen)] if step % 3 == 0 else list(range(S))
        if all(q < 0 for q in parents):
            continue
        a["parents"].copy_(torch.tensor(parents, dtype=i32))
        ops.page_fork(**a)
        texts = [list(texts[q]) if q >= 0 else [] for q in parents]
        assert int(a["starved"]) == 0
        held = torch.zeros(P, dtype=i32)
        for s in range(S):
            assert int(a["lens"][s]) == len(texts[s])
            for p in a["block_tables"][s, : int(a["held"][s])].tolist():
                held[p] += 1
            if parents[s] < 0 or len(texts[s]) == 32 * M:
                assert parents[s] >= 0 or int(a["held"][s]) == 0
                continue
            n = len(texts[s])
            page = int(a["block_tables"][s, n // 32])
            assert int(a["refs"][page]) == 1
            a["pools"][0][0, page, n % 32] = step * S + s
            texts[s].append(step * S + s)
            a["lens"][s] += 1
            for i, t in enumerate(texts[s]):
                assert float(a["pools"][0][0, int(a["block_tables"][s, i // 32]), i % 32, 0]) == t
        assert torch.equal(held, a["refs"])


def test_fork_starves_and_recovers():
    a = _fork_args(S=3, M=2, P=3)
    a["parents"].copy_(torch.tensor([0, -1, -1]))
    ops.page_fork(**a)
    a["lens"][0] = 5
    a["refs"][2] = 1  # somebody else's
    a["parents"].zero_()
    ops.page_fork(**a)
    assert int(a["starved"]) == 1 and a["held"].tolist() == [1, 1, 1]
    assert a["refs"].tolist() == [2, 1, 1] and sorted(a["copies"][:, 1].tolist()) == [-1, -1, 1]
    a["refs"][2] = 0
    a["parents"].copy_(torch.arange(3))
    ops.page_fork(**a)
    assert int(a["starved"]) == 0 or int(a["refs"][0]) <= 1


def test_reorder_and_refusals():
    t, h = torch.arange(12.0).view(6, 2), torch.arange(6).to(torch.bfloat16)
    ops.state_reorder([t, h], torch.tensor([1, 0, 2, 4, 4, -1], dtype=i32), 3)
    assert t[:, 0].tolist() == [2, 0, 4, 8, 8, 10] and h.tolist() == [1, 0, 2, 4, 4, 5]
    p = torch.arange(6, dtype=i32)
    for states, width in (([t], 4), ([t[:5]], 3), ([torch.zeros(6, 3, dtype=torch.uint8)], 3), ([torch.zeros(6, 4, 2).transpose(1, 2)], 3),
                          ([torch.zeros(1, 4).expand(6, 4)], 3), ([t], 0), ([t], 33), ([t, h, t], 3)):
        with pytest.raises(RuntimeError):
            ops.state_reorder(states, p, width)
    with pytest.raises(RuntimeError):
        ops.state_reorder([t], p.long(), 3)


def test_pools_of_the_caches():
    """Every cache's pools are its own tensors as [layers, pages, ..]."""
    for c in (kv_cache.KVCache(2, 5, 3, "cpu"), kv_cache.LatentKVCache({0: 24}, 5, "cpu", transposed={0: 16}),
              kv_cache.PagedKVCache({0: (2, 16, 8)}, 5, "cpu", transposed=(0,)),
              kv_cache.MixedKVCache({0: 24}, {1: (2, 16, 8)}, 5, "cpu", latent_transposed={0: 16}, kv_transposed=(1,))):
        pools = c.pools()
        assert pools and all(p.dim() >= 3 and p.shape[1] == 5 for p in pools)
        a = _fork_args(S=2, M=2, P=5)
        a["lens"][0], a["held"][0], a["refs"][0] = 3, 1, 1
        a["parents"].zero_()
        for p in pools:
            p[:, 0] = 2.0
        a["pools"] = pools
        ops.page_fork(**a)
        new = int(a["copies"][0, 1])
        assert new > 0 and all(bool((p[:, new] == 2).all()) for p in c.pools())


def search(dev, steps=70, width=3, groups=2, V=61, fork_pages=None):
    """A search of a model with one attention layer and one recurrent state, run through the ops, and the same search over lists of
    tokens with everything recomputed in 64 bits.  Returns both sides' beams."""
    gen = torch.Generator().manual_seed(5)
    S, H, M, P = width * groups, 2, 4, 64
    E = torch.randn(V, 128, generator=gen, dtype=torch.float64)
    head = torch.randn(V, 128, generator=gen, dtype=torch.float64) * 0.4
    bf = lambda t: t.to(torch.bfloat16)  # noqa: E731

    def tok_kv(t, pos):  # key, value and query of a token at a position, exact in bf16
        c = math.cos(0.7 * pos + 0.3)
        e = bf(E[t] * c)
        return e, bf(E[t].roll(17) * 0.5), bf(E[t].flip(0) * c)

    def logits_of(o, state):
        return ((o.double() + state.double() * 0.05) @ head.T).float()

    # ---- the ops
    kv = kv_cache.KVCache(1, P, H, dev)
    rec = kv_cache.RecurrentStateCache({0: (128, 2)}, S, dev)
    z = lambda *s: torch.zeros(*s, dtype=i32, device=dev)  # noqa: E731
    bt, held, lens, refs, copies, starved, shared = z(S, M), z(S), z(S), z(P), z(S, 2), z(1), z(groups)
    scores = torch.full((groups, width), -INF, device=dev)
    scores[:, 0] = 0
    out = (torch.empty(groups, width, device=dev), z(groups, width), z(groups, width))
    ids, parents = torch.tensor([7 + s // width for s in range(S)]), torch.arange(S)
    texts = [[int(t)] for t in ids]
    perm = [((t & 15) >> 2) * 8 + (t >> 4) * 4 + (t & 3) for t in range(32)]
    for step in range(steps):
        ops.page_fork(bt, held, lens, parents.to(dev, i32), refs, copies, starved, kv.pools())
        rec.reorder(parents.to(dev, i32), width)
        assert int(starved) == 0
        qs = []
        for s in range(S):
            n = int(lens[s])
            k, v, q = tok_kv(int(ids[s]), n)
            page = int(bt[s, n // 32])
            kv.k[0, page, :, n % 32] = k.to(dev)
            kv.v[0, page, :, :, perm[n % 32]] = v.to(dev)
            rec.state[0][s] = 0.9 * rec.state[0][s] + k.to(dev).float()
            qs.append(q.expand(4, 128))
        lens += 1
        q = torch.stack(qs).to(dev).contiguous()
        o = torch.zeros_like(q)
        ops.beam_shared(bt, lens, width, shared)
        ops.beam_attention(q, kv.k[0], kv.v[0], bt, lens, shared, o, width)
        x = logits_of(o.float().mean(1).cpu(), rec.state[0].cpu())
        ops.beam_select(x.to(dev), scores, *out)
        scores = out[0].clone()
        parents, ids = out[1].flatten().cpu().long(), out[2].flatten().cpu()
        texts = [texts[int(p)] + [int(t)] for p, t in zip(parents, ids)]
    # ---- every beam's score from its text alone
    exact = []
    for text in texts:
        total, state = 0.0, torch.zeros(128)
        ks, vs = [], []
        for i, t in enumerate(text[:-1]):
            k, v, q = tok_kv(t, i)
            ks.append(k.double()), vs.append(v.double())
            state = 0.9 * state + k.float()
            p = torch.softmax(torch.stack(ks) @ q.double() / math.sqrt(128), 0)
            x = logits_of(bf(p @ torch.stack(vs))[None].float(), state[None])
            total += float(torch.log_softmax(x[0].double(), 0)[text[i + 1]])
        exact.append(total)
    return texts, scores.flatten().cpu(), torch.tensor(exact, dtype=torch.float64), (bt.cpu(), held.cpu(), refs.cpu(), rec.state[0].cpu(), shared.cpu())


def check_search(result):
    texts, scores, exact, (bt, held, refs, _, shared) = result
    # the attention's result is off by at most 2^-7 of about one in each of 128 dims (weights and result round to bf16), a logit, its
    # product with 128 factors of 0.4, by 0.4 sqrt(128) 2^-7 = 0.035 as independent errors add, a log-probability by sqrt(2) of
    # that and a sum of 70 by sqrt(70) of it: 0.42, five times of which no beam passes
    assert float((scores.double() - exact).abs().max()) < 5 * 0.42
    for a, b in itertools.combinations(texts, 2):
        assert a != b
    count = torch.zeros_like(refs)
    for s in range(bt.shape[0]):
        for p in bt[s, : int(held[s])].tolist():
            count[p] += 1
    assert torch.equal(count, refs)


def test_a_search():
    check_search(search("cpu"))


def test_fork_entries_that_are_no_pages():
    """Ids outside the pool, negative ones too, are carried along and count nowhere."""
    a = _fork_args(2, 4, 9)
    a["block_tables"].copy_(torch.tensor([[3, 4, 5, 0], [-4, 10 ** 6, 6, 0]]))
    a["held"].fill_(3)
    a["lens"].fill_(70)
    a["refs"].copy_(torch.tensor([0, 0, 0, 1, 1, 1, 1, 0, 0]))
    a["parents"].fill_(1)
    ops.page_fork(**a)
    assert a["block_tables"].tolist() == [[-4, 10 ** 6, 0, 0], [-4, 10 ** 6, 6, 0]]
    assert a["refs"].tolist() == [1, 0, 0, 0, 0, 0, 1, 0, 0] and a["copies"].tolist() == [[6, 0], [-1, -1]] and int(a["starved"]) == 0


def too_large(device):
    """Calls that a limit of sizes refuses, of tensors that nothing reads."""
    e, z = lambda *s: torch.empty(*s, dtype=torch.uint8, device=device), lambda *s: torch.zeros(*s, dtype=i32, device=device)
    q = torch.empty((1 << 19) + 2, 8, 128, dtype=torch.bfloat16, device=device)
    k, v = (torch.zeros(1, 8, *s, dtype=torch.bfloat16, device=device) for s in ((32, 128), (128, 32)))
    many = e((1 << 31) - (1 << 17) + 100)
    return [lambda: ops.page_fork(z(2, 1), z(2), z(2), z(2), z(1), z(2, 2), z(1), [e(1, 1, (1 << 30) + 16)]),
            lambda: ops.state_reorder([many[None, 2 * i: many.numel() - 100 + 2 * i] for i in range(17)], z(1), 1),
            lambda: ops.beam_attention(q, k, v, z(q.shape[0], 1), z(q.shape[0]), z(q.shape[0] // 2), q, 2)]


@pytest.mark.parametrize("which", [0, 1, 2])
def test_sizes_past_the_limits(which):
    with pytest.raises(RuntimeError, match="at most"):
        too_large("cpu")[which]()


def refused_fork(device):
    """A fork with more pieces to copy than a launch counts, its state, and a copy of that."""
    a = {k: v if k == "pools" else v.to(device) for k, v in _fork_args(S=2048, M=1, P=1).items()}
    a["held"][0], a["lens"][0], a["refs"][0] = 1, 3, 1
    a["parents"].zero_()
    a["pools"] = [torch.zeros(1 << 20, 1, 16, dtype=torch.uint8, device=device)]
    return a, {k: v.clone() for k, v in a.items() if k != "pools"}


def test_fork_refuses_before_it_moves():
    a, before = refused_fork("cpu")
    with pytest.raises(RuntimeError, match="pieces"):
        ops.page_fork(**a)
    assert all(torch.equal(a[k], v) for k, v in before.items())


def starved_forks(sharers, free):
    """One sequence of 5 tokens that `sharers` slots go on from without a free page, then `free` pages given back and the call that
    serves them: its arguments, and what it has to leave."""
    S, P = sharers + 1, sharers + 7
    a = _fork_args(S, 3, P)
    a["held"][0], a["lens"][0] = 1, 5
    a["block_tables"][0, 0] = 1
    a["refs"].fill_(1)
    a["parents"].copy_(torch.tensor([0] * sharers + [-1]))
    bref.page_fork(**a)
    assert int(a["starved"]) == sharers - 1 and a["refs"].tolist() == [1, sharers] + [1] * (P - 2)
    a["refs"][3: 3 + free] = 0
    a["parents"].copy_(torch.tensor(list(range(sharers)) + [-1]))
    a["pools"] = [torch.arange(2 * P * 4.0).view(2, P, 4)]
    served = min(free, sharers - 1)
    pages = [3 + s for s in range(served)] + [1] * (sharers - served)
    refs = [1, sharers - served] + [1] * (P - 2)
    refs[3 + served: 3 + free] = [0] * (free - served)
    return a, dict(block_tables=[[p, 0, 0] for p in pages] + [[0, 0, 0]], refs=refs, starved=[sharers - 1 - served],
                   copies=[[1, 3 + s] for s in range(served)] + [[-1, -1]] * (S - served), held=[1] * sharers + [0],
                   lens=[5] * sharers + [0])


@pytest.mark.parametrize("sharers", [2, 3, 5])
@pytest.mark.parametrize("free", [0, 1, 2, 4])
def test_fork_serves_the_starved_with_as_many_pages(sharers, free):
    a, want = starved_forks(sharers, free)
    ops.page_fork(**a)
    assert {k: a[k].tolist() for k in want} == want
    for old, new in want["copies"]:
        assert old < 0 or torch.equal(a["pools"][0][:, new], a["pools"][0][:, old])


def test_shared_of_too_many_slots():
    e = torch.empty(1 << 26, 1, dtype=i32)  # nothing reads it
    with pytest.raises(RuntimeError, match="at most"):
        ops.beam_shared(e, e.view(-1), 1, e.view(-1))
