"""A beam search's kernels (selection over beams and vocabulary, attention over shared pages, forks of block tables, states that change
slots) against their references in 64 bits, which the CPU tests hold against definitions of their own."""
import math

import pytest
import torch

from distributed_sse_for_llm_response_amd import ops
from distributed_sse_for_llm_response_amd.engine import kv_cache
from distributed_sse_for_llm_response_amd.ops import beams_reference as bref
from distributed_sse_for_llm_response_amd.ops.reference import gather_kv

pytestmark = pytest.mark.gpu
INF = math.inf


# ------------------------------------------------------------------------------------------------------------ selection
# A row's log-sum: each exponential has an argument y in (-42, 0] rounded twice (|y| 2^-23) and one step of its own (2^-23), what is
# below 2^-42 of the largest counts for nothing; a value goes through at most 80 additions (2^-24 each).  The score rounds once.
LOG_SUM = 43 * 2.0 ** -23 + 80 * 2.0 ** -24


def _logits(gen, rows, V, dtype):
    """Multiples of 1/8, exact in both types: many equal logits in a row, while scores of different rows are told apart by their
    log-sums and base scores."""
    return (torch.randn(rows, V, generator=gen) * 16).round().clamp(-120, 120).div(8).to(dtype)


def _apart(logits, scores):
    """Whether no two rows' scores are as near as two log-sums may be off (modulo the logits' steps of 1/8)."""
    z = torch.logsumexp(logits.double(), 1)
    off = (scores.double().flatten() - z).view(scores.shape)
    for row in off:
        f = sorted(float(v) % 0.125 for v in row if math.isfinite(v))
        if any(b - a < 2.1 * LOG_SUM for a, b in zip(f, f[1:])) or (len(f) > 1 and f[0] + 0.125 - f[-1] < 2.1 * LOG_SUM):
            return False
    return True


def _scores(gen, logits, groups, width, most):
    """Base scores that keep the rows apart."""
    while True:
        scores = -torch.rand(groups, width, generator=gen) * most
        if _apart(logits, scores):
            return scores


def _select(dev, logits, scores, K, eos=-1):
    G, W = scores.shape
    outs = []
    for f, d in ((bref.beam_select, "cpu"), (ops.beam_select, dev)):
        o = (torch.full((G, K), 7.0, device=d), torch.full((G, K), 7, device=d, dtype=torch.int32),
             torch.full((G, K), 7, device=d, dtype=torch.int32))
        end = torch.full((G, W), 7.0, device=d) if eos >= 0 else None
        f(logits.cpu() if d == "cpu" else logits, scores.to(d), *o, eos, end)
        outs.append([t.cpu() for t in o] + ([end.cpu()] if eos >= 0 else []))
    return outs


def _same_choice(want, got):
    assert torch.equal(want[1], got[1]) and torch.equal(want[2], got[2])
    for a, b in zip([want[0]] + want[3:], [got[0]] + got[3:]):
        live = a > -INF
        assert torch.equal(live, b > -INF)
        a, b = a[live].double(), b[live].double()
        assert bool(((a - b).abs() <= LOG_SUM + 2 * 2.0 ** -24 * a.abs()).all()), float((a - b).abs().max())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,width,V,K", [(1, 1, 1, 1), (1, 1, 5, 8), (2, 3, 63, 64), (1, 4, 1000, 4), (3, 5, 2048, 10),
                                              (1, 8, 32768, 16), (2, 32, 4099, 64), (1, 2, 50001, 3), (5, 4, 777, 8), (1, 3, 9000, 33)])
def test_select(gpu, dtype, groups, width, V, K):
    gen = torch.Generator().manual_seed(1000 * groups + V + K)
    logits = _logits(gen, groups * width, V, dtype)
    scores = _scores(gen, logits, groups, width, 9)
    for eos in {-1, V // 2, V - 1}:
        _same_choice(*_select(gpu, logits.to(gpu), scores, K, eos))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("start", [1, 2, 3, 5])
def test_select_strided_rows(gpu, dtype, start):
    """Rows of a wider buffer at addresses of every alignment."""
    gen = torch.Generator().manual_seed(start)
    wide = _logits(gen, 8, 5003, dtype).to(gpu)
    logits = wide[:, start: start + 4700]
    scores = _scores(gen, logits.cpu(), 2, 4, 5)
    _same_choice(*_select(gpu, logits, scores, 8, 17))


def test_select_equal_logits(gpu):
    """Every token equal: the first tokens of the best row, in order; of two equal rows the first one's."""
    for dtype in (torch.float32, torch.bfloat16):
        logits = torch.full((4, 9001), 0.5, device=gpu, dtype=dtype)
        want, got = _select(gpu, logits, torch.tensor([[-2.0, -1.0, -1.0, -3.0]]), 64)
        assert got[1].tolist() == [[1] * 64] and got[2].tolist() == [list(range(64))]
        _same_choice(want, got)
        want, got = _select(gpu, logits[:, :40], torch.tensor([[-2.0, -1.0, -1.0, -3.0]]), 64)
        assert got[1].tolist() == [[1] * 40 + [2] * 24]
        _same_choice(want, got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,width,V,K", [(1, 4, 50001, 64), (64, 8, 2100, 3)])
def test_select_more_than_gathered(gpu, dtype, groups, width, V, K):
    """Rows of equal logits, more of them than LDS holds candidates: in a workgroup of the rows, or over a row's workgroups."""
    logits = torch.full((groups * width, V), -0.25, device=gpu, dtype=dtype)
    scores = -torch.arange(groups * width, dtype=torch.float32).view(groups, width)
    want, got = _select(gpu, logits, scores, K, 1)
    assert got[1].tolist() == [[g * width] * K for g in range(groups)] and got[2][0].tolist() == [0] + list(range(2, K + 1))
    _same_choice(want, got)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [7, 1001, 50001])
def test_select_rows_of_equal_logits_tie(gpu, V, dtype):
    """Beams of the same logits and scores tie whatever addresses their rows have: the lowest row first, the scores the same bits."""
    gen = torch.Generator().manual_seed(V)
    row = torch.randn(V, generator=gen).clamp(-3, 3)
    row[V // 2], row[V // 3] = 5.0, 4.0
    G, W = 3, 8
    logits = row.to(dtype).to(gpu).expand(G * W, V).contiguous()
    o = torch.zeros(G, 16, device=gpu), torch.zeros(G, 16, dtype=torch.int32, device=gpu), torch.zeros(G, 16, dtype=torch.int32, device=gpu)
    ops.beam_select(logits, torch.full((G, W), -0.7, device=gpu), *o)
    for g in range(G):
        assert o[1][g].tolist() == 2 * list(range(g * W, g * W + W)) and o[2][g].tolist() == W * [V // 2] + W * [V // 3]
    assert bool((o[0].view(-1, W) == o[0][0].view(2, W)[:, :1].repeat(G, 1)).all())


def test_select_scores_in_place(gpu):
    """The new scores may take the old ones' place."""
    gen = torch.Generator().manual_seed(31)
    x, s = torch.randn(12, 900, generator=gen).to(gpu), -torch.rand(3, 4, generator=gen).to(gpu)
    apart = torch.zeros(3, 4, device=gpu), torch.zeros(3, 4, dtype=torch.int32, device=gpu), torch.zeros(3, 4, dtype=torch.int32, device=gpu)
    end, end2 = torch.zeros(3, 4, device=gpu), torch.zeros(3, 4, device=gpu)
    ops.beam_select(x, s, *apart, 5, end)
    rows, tokens = torch.zeros_like(apart[1]), torch.zeros_like(apart[2])
    ops.beam_select(x, s, s, rows, tokens, 5, end2)
    assert torch.equal(s, apart[0]) and torch.equal(rows, apart[1]) and torch.equal(tokens, apart[2]) and torch.equal(end, end2)


def test_select_more_lists_than_noted(gpu):
    """A vocabulary so long that the merge cannot note every list that goes on: all rows equal, or one ahead."""
    V, K = 1 << 23, 5
    logits = torch.zeros(32, V, device=gpu, dtype=torch.bfloat16)
    o = (torch.zeros(1, K, device=gpu), torch.zeros(1, K, device=gpu, dtype=torch.int32), torch.zeros(1, K, device=gpu, dtype=torch.int32))
    for ahead in (0, 7):
        scores = torch.zeros(1, 32, device=gpu)
        scores[0, ahead] = 1.0 if ahead else 0.0
        ops.beam_select(logits, scores, *o, 1)
        assert o[1].tolist() == [[ahead] * K] and o[2].tolist() == [[0, 2, 3, 4, 5]]
        assert float((o[0] - (scores[0, ahead] - math.log(V))).abs().max()) < LOG_SUM + 2.0 ** -23 * 16


def test_select_what_is_not_finite(gpu):
    gen = torch.Generator().manual_seed(3)
    logits = _logits(gen, 12, 3000, torch.float32)
    scores = _scores(gen, logits, 2, 6, 1)
    logits[1, 7] = math.nan          # a row with NaN, with +inf, of -inf alone, of two values only
    logits[2, 2999] = INF
    logits[3] = -INF
    logits[4, 5:] = -INF
    logits[4, :3] = -INF
    logits[6:, ::2] = -INF
    logits[8] = torch.finfo(torch.float32).min   # masked by the type's lowest value throughout, and in part
    logits[9, 10:] = torch.finfo(torch.float32).min
    scores[0, 5], scores[1, 1], scores[1, 5] = -INF, math.nan, INF
    for eos in (-1, 3, 7):
        _same_choice(*_select(gpu, logits.to(gpu), scores, 16, eos))
    scores.fill_(-INF)
    _, got = _select(gpu, logits.to(gpu), scores, 16, 3)
    assert bool((got[0] == -INF).all()) and bool((got[1] == -1).all()) and bool((got[2] == -1).all()) and bool((got[3] == -INF).all())


@pytest.mark.parametrize("V", [4096, 40000])
def test_select_best_in_one_lane(gpu, V):
    """The best tokens 256 or 1024 apart, where a workgroup's lanes meet the same few: the bound of the chunk's best is low then, and
    a long list is gathered."""
    for step in (4, 256, 1024, 2048):
        logits = torch.zeros(1, V)
        logits[0, ::step] = 20 + torch.arange(0, V, step).flip(0) / 8192
        _same_choice(*_select(gpu, logits.to(gpu), torch.tensor([[-1.0]]), 64))


def test_select_more_candidates_than_gathered(gpu):
    """One row of 32 far ahead: the merge meets all of the group's best in few lists."""
    V = 40960
    logits = torch.zeros(32, V)
    logits[5] = torch.linspace(0, 4, V)
    logits[6] = torch.linspace(4, 0, V)
    scores = torch.full((1, 32), -500.0) - torch.arange(32) * 3
    scores[0, 5], scores[0, 6] = -1.0, -1.01
    _same_choice(*_select(gpu, logits.to(gpu), scores, 64))


def test_select_first_step_and_graph(gpu):
    """One beam in use, then a captured selection replayed over new logits."""
    gen = torch.Generator().manual_seed(9)
    logits = _logits(gen, 8, 2500, torch.float32).to(gpu)
    scores = torch.tensor([[-0.5, -INF, -INF, -INF], [-INF, -INF, -1.5, -INF]])
    _same_choice(*_select(gpu, logits, scores, 4, 2))
    o = (torch.empty(2, 4, device=gpu), torch.empty(2, 4, device=gpu, dtype=torch.int32), torch.empty(2, 4, device=gpu, dtype=torch.int32))
    s = scores.to(gpu)
    ops.beam_select(logits, s, *o, 2)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.beam_select(logits, s, *o, 2)
    for seed in range(4):
        gen = torch.Generator().manual_seed(20 + seed)
        new = _logits(gen, 8, 2500, torch.float32)
        sc = _scores(gen, new, 2, 4, 4)
        logits.copy_(new)
        s.copy_(sc)
        g.replay()
        torch.cuda.synchronize()
        want, got = _select(gpu, logits, sc, 4, 2)
        _same_choice(want[:3], [t.cpu() for t in o])
        _same_choice(want, got)


# ------------------------------------------------------------------------------------------------------------ attention
def _cache(gen, pages, hkv, dev):
    k = torch.randn(pages, hkv, 32, 128, generator=gen).to(torch.bfloat16)
    v = torch.randn(pages, hkv, 128, 32, generator=gen).to(torch.bfloat16)
    return k.to(dev), v.to(dev)


def _tables(gen, lens, common, width, extra=1):
    """Block tables of groups whose beams have common[g] leading pages the same and the others their own, in random order."""
    S = len(lens)
    need = [max(common[s // width], -(-n // 32)) for s, n in enumerate(lens)]
    total = sum(common) + sum(n - common[s // width] for s, n in enumerate(need)) + 3
    perm, at = torch.randperm(total, generator=gen).tolist(), 0
    bt = torch.zeros(S, max(need) + extra, dtype=torch.int32)
    for g in range(S // width):
        for j in range(common[g]):
            bt[g * width: (g + 1) * width, j] = perm[at]
            at += 1
    for s in range(S):
        for j in range(common[s // width], need[s]):
            bt[s, j] = perm[at]
            at += 1
    return bt, total


def _attend(dev, gen, lens, common, width, hq, hkv, poison=False):
    bt, pages = _tables(gen, lens, common, width)
    k, v = _cache(gen, pages, hkv, "cpu")
    if poison:  # what stands in a page past the sequence's end is not finite
        for s, n in enumerate(lens):
            if n % 32:
                t = torch.arange(n % 32, 32)
                k[int(bt[s, n // 32])][:, t] = math.nan
                v[int(bt[s, n // 32])][:, :, ((t & 15) >> 2) * 8 + (t >> 4) * 4 + (t & 3)] = INF
    q = torch.randn(len(lens), hq, 128, generator=gen).to(torch.bfloat16)
    ctx = torch.tensor(lens, dtype=torch.int32)
    shared = torch.zeros(len(lens) // width, dtype=torch.int32)
    bref.beam_shared(bt, ctx, width, shared)
    dsh = torch.full_like(shared, -5).to(dev)
    ops.beam_shared(bt.to(dev), ctx.to(dev), width, dsh)
    assert torch.equal(dsh.cpu(), shared)
    out = torch.full(q.shape, 3.0, dtype=torch.bfloat16, device=dev)
    args = (q.to(dev), k.to(dev), v.to(dev), bt.to(dev), ctx.to(dev))
    ops.beam_attention(*args, dsh, out, width)
    # weights and result round to bf16 (half a step, 2^-8, each); a score is 128 products of some 0.1 summed in 32 bits
    for s, n in enumerate(lens):
        got = out[s].cpu().double()
        if n == 0:
            assert bool((got == 3.0).all())
            continue
        K, V = (x.double().repeat_interleave(hq // hkv, 1) for x in gather_kv(k, v, bt[s], n))
        p = torch.softmax((q[s].double()[None] * K).sum(-1) / math.sqrt(128), 0)[..., None]
        want, size = (p * V).sum(0), (p * V.abs()).sum(0)
        assert bool(((got - want).abs() <= (2.0 ** -8 + 1e-4) * size + 2.0 ** -8 * want.abs()).all()), (s, float((got - want).abs().max()))
    return args, dsh, out


@pytest.mark.parametrize("hq,hkv", [(8, 8), (8, 4), (32, 8), (8, 1), (16, 1), (12, 4), (5, 1)])
@pytest.mark.parametrize("width", [1, 3, 4, 8])
def test_attention_heads(gpu, hq, hkv, width):
    gen = torch.Generator().manual_seed(hq * 100 + width)
    lens = [97 + 13 * s for s in range(2 * width)]
    _attend(gpu, gen, lens, [2, 3], width, hq, hkv)


@pytest.mark.parametrize("width,lens,common", [
    (2, [1, 1], [0]), (2, [1, 0], [0]), (2, [0, 0, 5, 31], [0, 0]), (4, [32, 32, 32, 32], [1]), (4, [33, 32, 64, 65], [1]),
    (3, [64, 65, 66, 0, 0, 0, 40, 0, 90], [2, 0, 1]), (2, [4000, 4001], [120]), (2, [4000, 4001], [0]), (16, [700] * 16, [20]),
    (32, [100 + i for i in range(32)], [3]), (1, [2500, 31, 1], [0, 0, 0])])
def test_attention_lengths(gpu, width, lens, common):
    gen = torch.Generator().manual_seed(sum(lens) + width)
    _attend(gpu, gen, lens, common, width, 8, 2)


def test_attention_past_the_end_not_finite(gpu):
    gen = torch.Generator().manual_seed(4)
    _attend(gpu, gen, [70, 65, 64, 83, 0, 95, 31, 161], [2, 0], 4, 8, 2, poison=True)  # no end lies in a page that others read


def test_attention_shared_is_a_choice(gpu):
    """Any number of pages up to the common ones gives the same numbers, more than are whole counts as those."""
    gen = torch.Generator().manual_seed(5)
    args, dsh, out = _attend(gpu, gen, [300, 290, 320, 310], [8], 4, 8, 2)
    for n in (0, 1, 5, 9, 10 ** 6, -3):
        o = torch.zeros_like(out)
        ops.beam_attention(*args, torch.tensor([min(n, 8) if n < 10 ** 6 else 8], dtype=torch.int32, device=gpu), o, 4)
        assert float((o.float() - out.float()).abs().max()) < 0.03
    same = torch.zeros(1, 40, dtype=torch.int32).expand(4, 40).contiguous().to(gpu)
    a, b = torch.zeros_like(out), torch.zeros_like(out)  # equal tables: pages that are not whole in every slot are not shared
    ops.beam_attention(args[0], args[1], args[2], same, args[4], torch.tensor([40], dtype=torch.int32, device=gpu), a, 4)
    ops.beam_attention(args[0], args[1], args[2], same, args[4], torch.tensor([9], dtype=torch.int32, device=gpu), b, 4)
    assert torch.equal(a, b)


def test_attention_as_paged_attention(gpu):
    """Groups of one: the decode attention that the engine runs."""
    gen = torch.Generator().manual_seed(6)
    lens = [513, 40, 700, 1]
    args, _, out = _attend(gpu, gen, lens, [0] * 4, 1, 8, 2)
    i32 = dict(dtype=torch.int32, device=gpu)
    o = torch.empty_like(out)
    e = torch.empty(1, device=gpu)
    ops.paged_attention(0, *args[:4], torch.arange(4, **i32), torch.ones(4, **i32), args[4], torch.arange(4, **i32), torch.zeros(4, **i32),
                        o, e, e, 1024, 1)
    assert float((o.float() - out.float()).abs().max()) < 0.03


def test_attention_graph_and_stream(gpu):
    gen = torch.Generator().manual_seed(7)
    args, dsh, out = _attend(gpu, gen, [200, 210, 190, 220], [4], 2 * 2, 8, 2)
    side = torch.cuda.Stream()
    o = torch.zeros_like(out)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.beam_attention(*args, dsh, o, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, out)
    graphs = []
    for _ in range(2):  # two graphs of the same call have work areas of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ops.beam_attention(*args, dsh, o, 4)
        graphs.append(g)
    for n in (150, 220, 35):
        args[4].copy_(torch.tensor([n, n + 1, n, n - 3], dtype=torch.int32))
        ops.beam_shared(args[3], args[4], 4, dsh)
        want = torch.zeros_like(out)
        ops.beam_attention(*args, dsh, want, 4)
        for g in graphs:
            o.zero_()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o, want)


@pytest.mark.parametrize("width,hq,hkv", [(16, 16, 1), (32, 10, 1), (7, 16, 1)])
def test_attention_many_columns(gpu, width, hq, hkv):
    """More (beam, head) columns than one workgroup holds, and a last tile that is not full."""
    gen = torch.Generator().manual_seed(width)
    _attend(gpu, gen, [64 + 5 * s for s in range(width)], [2], width, hq, hkv)


@pytest.mark.parametrize("width,hq", [(2, 16), (4, 32)])
def test_attention_far_pages(gpu, width, hq):
    """Pages beyond 2^31 elements and 2^32 bytes of a pool."""
    gen = torch.Generator().manual_seed(width)
    lens, common = [100 + s for s in range(width)], [2]
    bt, small = _tables(gen, lens, common, width)
    k, v = _cache(gen, small, 8, "cpu")
    pages = 2 ** 31 // (8 * 32 * 128) + 64
    bk = torch.zeros(pages, 8, 32, 128, dtype=torch.bfloat16, device=gpu)
    bv = torch.zeros(pages, 8, 128, 32, dtype=torch.bfloat16, device=gpu)
    far = pages - 1 - torch.arange(small)
    bk[far], bv[far] = k.to(gpu), v.to(gpu)
    q = torch.randn(width, hq, 128, generator=gen).to(torch.bfloat16).to(gpu)
    ctx = torch.tensor(lens, dtype=torch.int32, device=gpu)
    sh = torch.tensor(common, dtype=torch.int32, device=gpu)
    a, b = torch.zeros_like(q), torch.zeros_like(q)
    ops.beam_attention(q, k.to(gpu), v.to(gpu), bt.to(gpu), ctx, sh, a, width)
    ops.beam_attention(q, bk, bv, far[bt.long()].to(torch.int32).to(gpu), ctx, sh, b, width)
    assert torch.equal(a, b) and bool(a.any())


def test_attention_entries_that_are_no_pages(gpu):
    """Ids outside the cache read page 0."""
    gen = torch.Generator().manual_seed(8)
    for width in (4, 8):  # pages to registers, pages through LDS
        k, v = _cache(gen, 4, 2, gpu)
        q = torch.randn(width, 8, 128, generator=gen).to(torch.bfloat16).to(gpu)
        bad = torch.tensor([[1, 10 ** 6, 2, -3]] * width, dtype=torch.int32, device=gpu)
        good = torch.tensor([[1, 0, 2, 0]] * width, dtype=torch.int32, device=gpu)
        ctx = torch.full((width,), 128, dtype=torch.int32, device=gpu)
        for shared in (0, 3):
            sh = torch.tensor([shared], dtype=torch.int32, device=gpu)
            a, b = torch.zeros_like(q), torch.zeros_like(q)
            ops.beam_attention(q, k, v, bad, ctx, sh, a, width)
            ops.beam_attention(q, k, v, good, ctx, sh, b, width)
            assert torch.equal(a, b)


def test_two_streams(gpu):
    """Calls of every op on two streams at once, each with its own tensors: work areas are the calls' own."""
    gen = torch.Generator().manual_seed(10)
    sides = []
    for n in (200, 333):
        args, dsh, out = _attend(gpu, gen, [n, n + 9, n - 5, n + 1], [4], 4, 8, 2)
        logits = _logits(gen, 4, 30000, torch.float32)
        scores = _scores(gen, logits, 1, 4, 3)
        sides.append((args, dsh, out, logits.to(gpu), scores, _select(gpu, logits.to(gpu), scores, 8)[0]))
    streams = [torch.cuda.Stream() for _ in sides]
    got = []
    torch.cuda.synchronize()
    for _ in range(10):
        for st, (args, dsh, out, logits, scores, _) in zip(streams, sides):
            with torch.cuda.stream(st):
                o = torch.zeros_like(out)
                ops.beam_attention(*args, dsh, o, 4)
                t = (torch.zeros(1, 8, device=gpu), torch.zeros(1, 8, device=gpu, dtype=torch.int32), torch.zeros(1, 8, device=gpu, dtype=torch.int32))
                ops.beam_select(logits, scores.to(gpu), *t)
                got.append((o, t))
    torch.cuda.synchronize()
    for i, (o, t) in enumerate(got):
        assert torch.equal(o, sides[i % 2][2])
        _same_choice(sides[i % 2][5], [x.cpu() for x in t])


# ---------------------------------------------------------------------------------------------------------------- forks
def _fork_state(gen, lens, common, width, spare, M=None):
    bt, used = _tables(gen, lens, common, width, extra=2)
    if M is not None:
        bt = bt[:, :M].contiguous()
    held = torch.tensor([-(-n // 32) for n in lens], dtype=torch.int32)
    refs = torch.zeros(used - 3 + spare, dtype=torch.int32)
    # the tables' pages are a part of [0, used): number them anew, so that `spare` pages are free
    pages = sorted({int(bt[s, j]) for s in range(len(lens)) for j in range(int(held[s]))})
    places = torch.randperm(refs.numel(), generator=gen)[: len(pages)].tolist()
    new = dict(zip(pages, places))
    for s in range(len(lens)):
        for j in range(bt.shape[1]):
            bt[s, j] = new[int(bt[s, j])] if j < int(held[s]) else 0
            if j < int(held[s]):
                refs[int(bt[s, j])] += 1
    return [bt, held, torch.tensor(lens, dtype=torch.int32)], refs


def _fork(dev, state, refs, parents, pools):
    S = state[0].shape[0]
    sides = []
    for f, d in ((bref.page_fork, "cpu"), (ops.page_fork, dev)):
        t = [x.clone().to(d) for x in state] + [torch.tensor(parents, dtype=torch.int32, device=d), refs.clone().to(d),
                                                torch.full((S, 2), 9, dtype=torch.int32, device=d),
                                                torch.full((1,), 9, dtype=torch.int32, device=d)]
        p = [x.clone().to(d) for x in pools]
        f(*t, p)
        sides.append([x.cpu() for x in t + p])
    for a, b in zip(*sides):
        assert torch.equal(a, b)
    return sides[0]


def _pools(gen, pages):
    return [torch.randn(2, pages, 3, 32, 8, generator=gen).to(torch.bfloat16), torch.randn(1, pages, 32, 4, generator=gen),
            torch.randint(0, 255, (3, pages, 16), generator=gen, dtype=torch.uint8)]


@pytest.mark.parametrize("lens,common,width,parents", [
    ([40, 40], [1], 2, [0, 0]), ([40, 40], [1], 2, [1, 0]), ([40, 40], [1], 2, [-1, 1]), ([40, 40], [1], 2, [-1, -1]),
    ([64, 64, 64], [2], 3, [2, 2, 2]), ([64, 64, 64], [2], 3, [0, 1, 2]), ([96, 96, 96, 96], [1], 4, [3, 0, 0, -1]),
    ([1, 0, 0, 0], [0], 4, [0, 0, 0, 0]), ([70, 0, 0, 0], [0], 4, [0, 0, 0, 0]), ([33, 65, 97, 129] * 4, [0, 0, 1, 1], 4, list(range(15, -1, -1))),
    ([500 + s // 8 for s in range(80)], [15] * 10, 8, [8 * (s // 8) + (s * 5 + 3) % 8 // 2 for s in range(80)]),
    ([31] * 6, [0], 6, [99, -7, 2, 2, 6, 5])])
def test_fork(gpu, lens, common, width, parents):
    gen = torch.Generator().manual_seed(len(lens) + sum(lens))
    state, refs = _fork_state(gen, lens, common, width, 2 * len(lens) + 5)
    pools = _pools(gen, refs.numel())
    got = _fork(gpu, state, refs, parents, pools)
    live = [s for s, q in enumerate(parents) if 0 <= q < len(lens)]
    at = [int(got[0][s, int(got[2][s]) // 32]) for s in live]
    assert len(set(at)) == len(at) and all(int(got[4][p]) == 1 for p in at) and int(got[6]) == 0
    held = torch.zeros_like(got[4])
    for s in range(len(lens)):
        for j in range(int(got[1][s])):
            held[int(got[0][s, j])] += 1
    assert torch.equal(held, got[4])


@pytest.mark.parametrize("spare", [0, 1, 2, 3])
def test_fork_without_room(gpu, spare):
    """Pages run out: who finds none keeps sharing, and a second call once pages are free serves them."""
    gen = torch.Generator().manual_seed(spare)
    state, refs = _fork_state(gen, [40, 41, 64, 64], [1], 4, spare)
    pools = _pools(gen, refs.numel())
    got = _fork(gpu, state, refs, [0, 0, 2, 0], pools)
    freed = 2  # slots 1 and 3 give a page of their own up
    assert int(got[6]) == max(0, 3 - spare - freed)
    again = _fork(gpu, got[:3], got[4], [0, 1, 2, -1], got[7:])
    assert int(again[6]) <= int(got[6])


def test_fork_full_tables_and_other_holders(gpu):
    gen = torch.Generator().manual_seed(11)
    state, refs = _fork_state(gen, [128, 128, 100, 97], [2, 2], 2, 6, M=4)
    _fork(gpu, state, refs, [1, 1, 2, 2], _pools(gen, refs.numel()))   # slots 0 and 1 have no further page
    refs[int(state[0][2, 3])] += 1                                     # somebody else holds slot 2's last page too
    got = _fork(gpu, state, refs, [0, 1, 2, 2], _pools(gen, refs.numel()))
    assert int(got[5][2, 0]) == int(got[5][3, 0]) == int(state[0][2, 3])


def test_fork_entries_that_are_no_pages(gpu):
    """Ids outside the pool are carried along, count nowhere and are copied nowhere."""
    gen = torch.Generator().manual_seed(12)
    state, refs = _fork_state(gen, [70, 70], [2], 2, 6)
    t = [x.clone().to(gpu) for x in state]
    t[0][0, 2], t[0][1, 0] = 10 ** 6, -4
    r = refs.to(gpu)
    pools = [p.to(gpu) for p in _pools(gen, refs.numel())]
    before = [p.clone() for p in pools]
    copies, starved = torch.zeros(2, 2, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)
    ops.page_fork(*t, torch.tensor([0, 0], dtype=torch.int32, device=gpu), r, copies, starved, pools)
    assert copies.tolist() == [[-1, -1], [-1, -1]] and all(torch.equal(a, b) for a, b in zip(pools, before))


@pytest.mark.parametrize("columns", [4, 2000])
def test_fork_takes_on_entries_that_are_no_pages(gpu, columns):
    """Where the parent has such an id, its follower has it too, not the page that it gave up: one launch, and one for the tables."""
    state, refs = _fork_state(torch.Generator().manual_seed(14), [70, 70], [0], 2, 5)
    state[0] = torch.cat([state[0], torch.zeros(2, columns, dtype=torch.int32)], 1)[:, :columns].contiguous()
    refs[int(state[0][1, 0])] = refs[int(state[0][1, 1])] = 0
    state[0][1, 0], state[0][1, 1] = -4, 10 ** 6
    for parents in ([1, 1], [1, 0], [0, 0]):
        got = _fork(gpu, state, refs, parents, _pools(torch.Generator().manual_seed(15), refs.numel()))
        assert got[0][0, :2].tolist() == state[0][parents[0], :2].tolist()


def test_fork_many_slots_and_pages(gpu):
    gen = torch.Generator().manual_seed(13)
    S, W = 2048, 8
    lens = [35 + 3 * (s // W) % 60 for s in range(S)]
    state, refs = _fork_state(gen, lens, [1] * (S // W), W, 20000)
    parents = [W * (s // W) + int(x) for s, x in enumerate(torch.randint(0, W, (S,), generator=gen))]
    parents[5 * W: 6 * W] = [-1] * W
    _fork(gpu, state, refs, parents, [torch.randn(1, refs.numel(), 8, generator=gen)])


def test_fork_far_pages(gpu):
    """A pool beyond 2^32 bytes, its layers strided."""
    pages = 70000
    pool = torch.zeros(2, pages + 7, 16384, dtype=torch.float32, device=gpu)[:, :pages]
    t = lambda *x: torch.tensor(x, dtype=torch.int32, device=gpu)  # noqa: E731
    refs = torch.ones(pages, dtype=torch.int32, device=gpu)
    refs[pages - 2] = 0
    refs[pages - 1] = 2
    pool[:, pages - 1] = torch.randn(2, 16384, device=gpu)
    bt, copies, starved = t([pages - 1], [0]), torch.zeros(2, 2, dtype=torch.int32, device=gpu), t(5)
    held, lens = t(1, 0), t(31, 0)
    refs[pages - 1] = 1
    ops.page_fork(bt, held, lens, t(0, 0), refs, copies, starved, [pool])
    assert copies.tolist() == [[pages - 1, pages - 2], [-1, -1]] and bt.tolist() == [[pages - 2], [pages - 1]] and int(starved) == 0
    assert torch.equal(pool[:, pages - 2], pool[:, pages - 1]) and bool(pool[:, pages - 2].any()) and not bool(pool[:, : pages - 2].any())


def test_fork_many_pools_and_a_graph(gpu):
    gen = torch.Generator().manual_seed(14)
    state, refs = _fork_state(gen, [40, 45, 50, 55], [1], 4, 40)
    pools = [torch.randn(1, refs.numel(), 4, generator=gen) for _ in range(130)]
    _fork(gpu, state, refs, [2, 2, 0, 3], pools)
    t = [x.clone().to(gpu) for x in state] + [torch.arange(4, dtype=torch.int32, device=gpu), refs.clone().to(gpu),
                                              torch.zeros(4, 2, dtype=torch.int32, device=gpu), torch.zeros(1, dtype=torch.int32, device=gpu)]
    dp = [p.to(gpu) for p in pools[:3]]
    ops.page_fork(*t, dp)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.page_fork(*t, dp)
    now, r, p = [x.cpu() for x in t[:3]], t[4].cpu(), [x.cpu() for x in dp]
    for parents in ([1, 1, 1, 3], [0, 0, 2, 2], [-1, 1, 1, 1], [1, 1, 2, 3]):
        t[3].copy_(torch.tensor(parents, dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        cpu = now + [torch.tensor(parents, dtype=torch.int32), r, torch.zeros(4, 2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)]
        bref.page_fork(*cpu, p)
        for a, b in zip(cpu + p, t + dp):
            assert torch.equal(a, b.cpu())


# --------------------------------------------------------------------------------------------------------------- states
@pytest.mark.parametrize("width,groups", [(1, 3), (2, 5), (4, 1), (5, 3), (8, 2), (9, 2), (16, 1), (17, 2), (32, 1)])
@pytest.mark.parametrize("kind", ["matrices", "odd", "halves"])
def test_reorder(gpu, width, groups, kind):
    gen = torch.Generator().manual_seed(width + groups)
    S = width * groups
    shapes = {"matrices": [(torch.float32, (4, 32, 16)), (torch.float32, (3, 96)), (torch.bfloat16, (64,))],
              "odd": [(torch.float32, (3, 801)), (torch.float32, (5,)), (torch.float32, ())],
              "halves": [(torch.bfloat16, (7,)), (torch.bfloat16, (3, 11)), (torch.float32, (9,))]}[kind]
    for trial in range(4):
        states = [torch.randn(S, *s, generator=gen).to(t) for t, s in shapes]
        parents = width * (torch.arange(S) // width) + torch.randint(0, width, (S,), generator=gen)
        if trial == 1:
            parents = width * (torch.arange(S) // width) + (torch.arange(S) + 1) % width  # a cycle
        if trial == 2:
            parents[::3] = -1
        if trial == 3:
            parents = parents.flip(0)  # other groups' slots: left alone
        parents = parents.to(torch.int32)
        dev = [s.to(gpu) for s in states]
        ops.state_reorder(dev, parents.to(gpu), width)
        bref.state_reorder(states, parents, width)
        for a, b in zip(states, dev):
            assert torch.equal(a, b.cpu())


def test_reorder_views_and_many(gpu):
    """Slots of a wider buffer, more tensors than a launch takes, empty ones among them."""
    gen = torch.Generator().manual_seed(2)
    wide = torch.randn(6, 40, generator=gen)
    states = [torch.randn(6, 1 + i % 7, generator=gen) for i in range(150)] + [torch.empty(6, 0), wide[:, 3:20]]
    parents = torch.tensor([2, 0, 0, 3, 5, 4], dtype=torch.int32)
    dw = wide.to(gpu)
    dev = [s.to(gpu) for s in states[:-1]] + [dw[:, 3:20]]
    ops.state_reorder(dev, parents.to(gpu), 3)
    bref.state_reorder(states, parents, 3)
    for a, b in zip(states, dev):
        assert torch.equal(a, b.cpu())
    assert torch.equal(dw.cpu(), wide)
    ops.state_reorder([], parents.to(gpu), 3)


def test_reorder_far_slots(gpu):
    """Slots beyond 2^32 bytes of a state."""
    big = torch.zeros(5, 2 ** 28 + 4, device=gpu)
    big[4, -3:] = 2.0
    big[1, :2] = 3.0
    ops.state_reorder([big], torch.tensor([4, 1, 2, 4, 1], dtype=torch.int32, device=gpu), 5)
    want = [(0, 2), (3, 0), (0, 0), (0, 2), (3, 0)]
    assert [(float(big[s, 0]), float(big[s, -1])) for s in range(5)] == want and float(big.sum()) == 2 * 3 * 2 + 2 * 2 * 3


def test_refusals(gpu):
    """What the CPU tests refuse, the bindings refuse too; and what only they can tell."""
    import test_beams as cpu

    i32 = dict(dtype=torch.int32, device=gpu)
    b = dict(dtype=torch.bfloat16, device=gpu)
    x, s = torch.zeros(4, 9, device=gpu), torch.zeros(2, 2, device=gpu)
    o = [t.to(gpu) for t in cpu._outs(2, 3)]
    for change in (dict(logits=x.half()), dict(logits=x.t().contiguous().t()), dict(logits=x[:3]), dict(scores=s.double()), dict(scores=s.cpu()),
                   dict(scores=s.view(1, 4)), dict(out_rows=o[1].long()), dict(out_tokens=o[2][:, :2].contiguous()),
                   dict(out_scores=torch.zeros(2, 65, device=gpu)), dict(eos_id=9), dict(eos_id=-2), dict(end_scores=torch.zeros(2, 2, device=gpu)),
                   dict(end_scores=torch.zeros(2, 3, device=gpu), eos_id=1), dict(logits=x[:, :0]), dict(logits=x[:1].expand(4, 9))):
        with pytest.raises(RuntimeError):
            ops.beam_select(**{**dict(logits=x, scores=s, out_scores=o[0], out_rows=o[1], out_tokens=o[2], eos_id=-1, end_scores=None), **change})
    a = dict(q=torch.zeros(4, 8, 128, **b), k_cache=torch.zeros(3, 2, 32, 128, **b), v_cache=torch.zeros(3, 2, 128, 32, **b),
             block_tables=torch.zeros(4, 2, **i32), ctx_len=torch.ones(4, **i32), shared=torch.zeros(2, **i32), out=torch.zeros(4, 8, 128, **b),
             width=2)
    ops.beam_attention(**a)
    odd = torch.zeros(4 * 8 * 128 + 1, **b)[1:].view(4, 8, 128)
    for change in (dict(q=a["q"].float()), dict(q=a["q"][:, :, :64].contiguous()), dict(out=a["out"][:3]), dict(v_cache=a["k_cache"]), dict(width=3),
                   dict(width=0), dict(width=33), dict(shared=torch.zeros(4, **i32)), dict(ctx_len=torch.ones(3, **i32)), dict(ctx_len=a["ctx_len"].cpu()),
                   dict(block_tables=torch.zeros(4, 2, device=gpu, dtype=torch.int64)), dict(block_tables=torch.zeros(4, 4, **i32)[:, ::2]),
                   dict(q=torch.zeros(4, 34, 128, **b), out=torch.zeros(4, 34, 128, **b)), dict(q=odd), dict(k_cache=a["k_cache"][:0], v_cache=a["v_cache"][:0])):
        with pytest.raises(RuntimeError):
            ops.beam_attention(**{**a, **change})
    f = {k: [t.to(gpu) for t in v] if k == "pools" else v.to(gpu) for k, v in cpu._fork_args().items()}
    ops.page_fork(**f)
    far = torch.zeros(2 * 9 * 4 + 1, device=gpu)[1:].view(2, 9, 4)
    for change in (dict(held=f["held"].long()), dict(lens=f["lens"][:3]), dict(parents=f["parents"][:3]), dict(copies=torch.zeros(4, **i32)),
                   dict(starved=torch.zeros(2, **i32)), dict(refs=f["refs"][:0]), dict(pools=[torch.zeros(2, 8, 4, device=gpu)]),
                   dict(pools=[torch.zeros(2, 9, 3, device=gpu)]), dict(pools=[torch.zeros(9, 4, device=gpu)]), dict(pools=[far]),
                   dict(pools=[torch.zeros(2, 9, 4, 2, device=gpu)[..., 0]]), dict(pools=[torch.zeros(2, 9, 4)]),
                   dict(pools=[torch.zeros(2, 9, 8, device=gpu)[:, :, :4]]), dict(block_tables=f["block_tables"].t())):
        with pytest.raises(RuntimeError):
            ops.page_fork(**{**f, **change})
    t, p = torch.zeros(6, 2, device=gpu), torch.arange(6, **i32)
    for states, width in (([t], 4), ([t[:5]], 3), ([torch.zeros(6, 3, dtype=torch.uint8, device=gpu)], 3), ([t.cpu()], 3), ([t, t], 3),
                          ([torch.zeros(6, 4, 2, device=gpu).transpose(1, 2)], 3), ([torch.zeros(1, 4, device=gpu).expand(6, 4)], 3), ([t], 0), ([t], 33)):
        with pytest.raises(RuntimeError):
            ops.state_reorder(states, p, width)
    with pytest.raises(RuntimeError):
        ops.state_reorder([t], p.long(), 3)
    torch.cuda.synchronize()


@pytest.mark.parametrize("which", [0, 1, 2])
def test_sizes_past_the_limits(gpu, which):
    import test_beams as cpu

    with pytest.raises(RuntimeError, match="at most"):
        cpu.too_large(gpu)[which]()


def test_most_rows(gpu):
    """Attention over 2^22 rows of one key each is that key's value; choice over 65535 rows is the same in every group."""
    S, H = 1 << 18, 16
    k, v = _cache(torch.Generator().manual_seed(3), 1, H, gpu)
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)  # noqa: E731
    q = torch.ones(S, H, 128, dtype=torch.bfloat16, device=gpu)
    out = torch.zeros_like(q)
    ops.beam_attention(q, k, v, z(S, 1), z(S) + 1, z(S), out, 1)
    _, mine = gather_kv(k.cpu(), v.cpu(), torch.zeros(1, dtype=torch.int32), 1)
    assert bool((out == mine[0].to(gpu)).all())
    G, W = 13107, 5
    logits = (torch.arange(W * 7, device=gpu).float() * 3 % 11).view(1, W, 7).expand(G, W, 7).reshape(G * W, 7).contiguous()
    o = torch.zeros(G, 9, device=gpu), z(G, 9), z(G, 9)
    ops.beam_select(logits, torch.zeros(G, W, device=gpu), *o)
    one = torch.zeros(1, 9), torch.zeros(1, 9, dtype=torch.int32), torch.zeros(1, 9, dtype=torch.int32)
    bref.beam_select(logits[:W].cpu(), torch.zeros(1, W), *one)
    assert torch.equal(o[2].cpu(), one[2].expand(G, 9)) and bool((o[0] == o[0][0]).all())
    assert torch.equal(o[1].cpu(), one[1] + W * torch.arange(G, dtype=torch.int32)[:, None])


def test_nothing_to_do(gpu):
    z = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)  # noqa: E731
    ops.beam_select(torch.zeros(0, 9, device=gpu), torch.zeros(0, 2, device=gpu), torch.zeros(0, 3, device=gpu), z(0, 3), z(0, 3))
    e = torch.zeros(0, 8, 128, dtype=torch.bfloat16, device=gpu)
    ops.beam_attention(e, torch.zeros(1, 2, 32, 128, dtype=torch.bfloat16, device=gpu), torch.zeros(1, 2, 128, 32, dtype=torch.bfloat16, device=gpu),
                       z(0, 2), z(0), z(0), e.clone(), 4)
    ops.beam_shared(z(0, 2), z(0), 4, z(0))
    ops.page_fork(z(0, 2), z(0), z(0), z(0), z(3), z(0, 2), z(1))
    ops.state_reorder([torch.zeros(0, 4, device=gpu)], z(0), 4)
    torch.cuda.synchronize()


def test_reorder_caches(gpu):
    gen = torch.Generator().manual_seed(8)
    parents = torch.tensor([1, 1, 0, 3, 7, 4, 4, 6], dtype=torch.int32)
    for make in (lambda d: kv_cache.RecurrentStateCache({0: (160, 4), 3: (96, 2)}, 8, d),
                 lambda d: kv_cache.MatrixStateCache({0: ((4, 32, 16), 0, 0), 1: ((2, 8, 8), 24, 4)}, 8, d),
                 lambda d: kv_cache.MemoryStateCache({0: (2, 32, 64)}, {0: (64, 4)}, 8, d)):
        a, b = make("cpu"), make(gpu)
        for name in ("state", "tail", "norm"):
            for key, t in getattr(a, name, {}).items():
                t.copy_(torch.randn(t.shape, generator=gen))
                getattr(b, name)[key].copy_(t)
        a.reorder(parents, 4)
        b.reorder(parents.to(gpu), 4)
        for name in ("state", "tail", "norm"):
            for key, t in getattr(a, name, {}).items():
                assert torch.equal(t, getattr(b, name)[key].cpu())


# ----------------------------------------------------------------------------------------------------------- all together
def test_a_step_in_a_graph(gpu):
    """Choice, fork, states, shared pages and attention of a step as one graph, replayed over its own results, against the same calls made
    one by one on copies."""
    gen = torch.Generator().manual_seed(21)
    W, G, V, H = 4, 3, 3000, 2
    S = W * G
    state, refs = _fork_state(gen, [70 + 9 * (s // W) for s in range(S)], [2] * G, W, 60)
    state[0] = torch.cat([state[0], torch.zeros(S, 6, dtype=torch.int32)], 1)
    k, v = _cache(gen, refs.numel(), H, "cpu")

    def make():
        d = dict(bt=state[0], held=state[1], lens=state[2], refs=refs, k=k[None], v=v[None], state=torch.randn(S, 64, 3, generator=torch.Generator().manual_seed(1)),
                 scores=-torch.arange(S, dtype=torch.float32).view(G, W) / 7, logits=torch.zeros(S, V), q=torch.zeros(S, 8, 128, dtype=torch.bfloat16),
                 rows=torch.zeros(G, W, dtype=torch.int32), tokens=torch.zeros(G, W, dtype=torch.int32), copies=torch.zeros(S, 2, dtype=torch.int32),
                 starved=torch.zeros(1, dtype=torch.int32), shared=torch.zeros(G, dtype=torch.int32), out=torch.zeros(S, 8, 128, dtype=torch.bfloat16),
                 new=torch.zeros(G, W))
        return {n: t.clone().to(gpu) for n, t in d.items()}

    def step(d):
        ops.beam_select(d["logits"], d["scores"], d["new"], d["rows"], d["tokens"], 2)
        d["scores"].copy_(d["new"])
        ops.page_fork(d["bt"], d["held"], d["lens"], d["rows"].view(-1), d["refs"], d["copies"], d["starved"], [d["k"], d["v"]])
        ops.state_reorder([d["state"]], d["rows"].view(-1), W)
        d["lens"].add_(1)
        ops.beam_shared(d["bt"], d["lens"], W, d["shared"])
        ops.beam_attention(d["q"], d["k"][0], d["v"][0], d["bt"], d["lens"], d["shared"], d["out"], W)

    a, b = make(), make()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(make())
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step(a)
    for i in range(40):
        gen = torch.Generator().manual_seed(100 + i)
        logits, q = _logits(gen, S, V, torch.float32), torch.randn(S, 8, 128, generator=gen).to(torch.bfloat16)
        for d in (a, b):
            d["logits"].copy_(logits)
            d["q"].copy_(q)
        g.replay()
        torch.cuda.synchronize()
        step(b)
        for n in a:
            assert torch.equal(a[n], b[n]), (i, n)
    assert int(a["starved"]) == 0 and len({tuple(t) for t in a["copies"].tolist()}) > 1


def test_a_search(gpu):
    from test_beams import check_search, search

    check_search(search(gpu))


# ------------------------------------------------------------------------------------------------------ calls at the borders
def test_fork_refuses_before_it_moves(gpu):
    import test_beams as cpu

    a, before = cpu.refused_fork(gpu)
    with pytest.raises(RuntimeError, match="pieces"):
        ops.page_fork(**a)
    assert all(torch.equal(a[k], v) for k, v in before.items())


@pytest.mark.parametrize("sharers", [2, 3, 5])
@pytest.mark.parametrize("free", [0, 1, 2, 4])
def test_fork_serves_the_starved_with_as_many_pages(gpu, sharers, free):
    import test_beams as cpu

    a, want = cpu.starved_forks(sharers, free)
    b = {k: [t.to(gpu) for t in v] if k == "pools" else v.to(gpu) for k, v in a.items()}
    ops.page_fork(**b)
    bref.page_fork(**a)
    assert {k: b[k].tolist() for k in want} == want
    assert torch.equal(a["pools"][0], b["pools"][0].cpu())


def test_fork_of_many_that_share(gpu):
    """Pages that slots of several parents go on in, some with a holder beside them, over tables of one launch and of two."""
    for S, M, seed in ((60, 4, 1), (700, 9, 2), (2048, 3, 3)):
        gen = torch.Generator().manual_seed(seed)
        P = S + 50
        shared = torch.randint(0, S // 3, (S,), generator=gen).to(torch.int32)  # the page that a slot goes on in
        bt = torch.zeros(S, M, dtype=torch.int32)
        bt[:, 0] = shared
        refs = torch.bincount(shared.long(), minlength=P).to(torch.int32)
        refs[: S // 3: 5] += 1
        refs[S // 3: S // 3 + S // 4] = 1
        parents = torch.where(torch.rand(S, generator=gen) < 0.8, torch.arange(S), torch.randint(-1, S, (S,), generator=gen))
        state = [bt, torch.ones(S, dtype=torch.int32), torch.full((S,), 7, dtype=torch.int32)]
        got = _fork(gpu, state, refs, parents.tolist(), [torch.randn(1, P, 8, generator=gen)])
        assert int((got[5][:, 0] >= 0).sum()) > S // 4 and (S < 100 or int(got[6]) > 0)


def _masked(gen, rows, V, dtype, low, allowed):
    """Rows of which `allowed` tokens are left (the first one among them), the others at a finite value."""
    x = _logits(gen, rows, V, dtype)
    keep = torch.zeros(rows, V, dtype=torch.bool)
    for r in range(rows):
        keep[r, torch.randperm(V, generator=gen)[: allowed]] = True
    keep[:, 0] = allowed > 0
    return torch.where(keep, x, torch.tensor(low, dtype=dtype))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", ["lowest", -1e9, -16.0])
@pytest.mark.parametrize("groups,width,V,K,allowed", [(2, 4, 33001, 16, 3), (1, 8, 5000, 64, 1), (3, 2, 40000, 5, 0), (1, 32, 7257, 58, 2),
                                                     (4, 4, 2051, 33, 40)])
def test_select_masked_by_a_finite_value(gpu, dtype, low, groups, width, V, K, allowed):
    """Few tokens left in a row, the others equal: the rest of the places goes to the lowest of those."""
    gen = torch.Generator().manual_seed(V + K)
    logits = _masked(gen, groups * width, V, dtype, torch.finfo(dtype).min if low == "lowest" else low, allowed)
    scores = _scores(gen, logits if allowed else torch.zeros_like(logits), groups, width, 9)
    for eos in (-1, 2):
        _same_choice(*_select(gpu, logits.to(gpu), scores, K, eos))


def _microseconds(f):
    times = []
    for _ in range(7):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        for _ in range(5):
            f()
        b.record()
        torch.cuda.synchronize()
        times.append(a.elapsed_time(b) * 200)
    return sorted(times)[3]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("groups,width,V,K", [(64, 8, 131072, 16), (8, 32, 7257, 58), (16, 5, 50001, 10)])
def test_select_of_masked_rows_takes_no_longer(gpu, dtype, groups, width, V, K):
    """Equal logits do not cost a walk of the row per candidate."""
    gen = torch.Generator(device=gpu).manual_seed(V)
    x = (torch.randn(groups * width, V, device=gpu, generator=gen) * 2.5).to(dtype)
    keep = torch.rand(groups * width, V, device=gpu, generator=gen) < 5 / V
    scores = -torch.rand(groups, width, device=gpu, generator=gen)
    o = (torch.zeros(groups, K, device=gpu), torch.zeros(groups, K, dtype=torch.int32, device=gpu),
         torch.zeros(groups, K, dtype=torch.int32, device=gpu))
    usual = _microseconds(lambda: ops.beam_select(x, scores, *o, 2))
    for low in (torch.finfo(dtype).min, -1e9):
        masked = torch.where(keep, x, torch.tensor(low, dtype=dtype, device=gpu))
        assert _microseconds(lambda: ops.beam_select(masked, scores, *o, 2)) < 2 * usual + 5
    equal = torch.full_like(x, 0.5)
    assert _microseconds(lambda: ops.beam_select(equal, scores, *o, 2)) < 2 * usual + 5


@pytest.mark.parametrize("dtype,piece", [(torch.float32, 4), (torch.bfloat16, 8)])
@pytest.mark.parametrize("K,lanes", [(16, 9), (32, 20), (64, 40)])
def test_select_best_in_few_lanes(gpu, dtype, piece, K, lanes):
    """The best tokens all in the pieces that a few lanes read: more of them are above the bound than LDS holds."""
    gen = torch.Generator().manual_seed(K)
    V = 70000
    logits = _logits(gen, 2, V, dtype) / 8
    hot = torch.arange(V) // piece % (64 if K <= 32 else 128) < lanes
    logits[:, hot] += 8
    scores = _scores(gen, logits, 1, 2, 3)
    _same_choice(*_select(gpu, logits.to(gpu), scores, K, 3))


def _end_errors(gpu, x):
    """By how much the scores of ending with token 1 are off, from base scores that bring them near zero, where they round by nothing."""
    want = x[:, 1].double() - torch.logsumexp(x.double(), 1)
    base = (-want).float().view(-1, 1)
    end, o = torch.zeros_like(base), (torch.zeros(len(x), 1, device=gpu), torch.zeros(len(x), 1, dtype=torch.int32, device=gpu),
                                      torch.zeros(len(x), 1, dtype=torch.int32, device=gpu))
    ops.beam_select(x, base, *o, 1, end)
    return end.view(-1).double() - (want + base.view(-1).double())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("where", ["end", "candidate"])
def test_select_log_sums(gpu, dtype, where):
    """Half of a row's sum in one token, the other half in 131071.  A wave's sum is scaled by an exponential whose argument, up to 16,
    rounds by 2^-21 at most, 2^-21 / sqrt(3) rms: 1.9e-7 of the value.  There are 32 waves at least, their errors independent, over
    half of the sum: 1.9e-7 / sqrt(32) / 2 = 1.7e-8.  A candidate's exponential is added to in its thread, 15 times at most, by half a
    step of a number from 1 to 2, 2^-24 / sqrt(3) rms: sqrt(15) 3.4e-8 / 2 = 6.7e-8 of the sum."""
    rows, V = 64, 131072
    x = (torch.randn(rows, V, device=gpu, generator=torch.Generator(device=gpu).manual_seed(1)) * 0.5).to(dtype)
    x[:, 1] = -20.0
    top = torch.logsumexp(x.double(), 1)
    at = torch.randint(2, V, (rows,), device=gpu, generator=torch.Generator(device=gpu).manual_seed(2))
    if where == "end":
        at = torch.ones_like(at)
    x[torch.arange(rows, device=gpu), at] = top.to(dtype)
    rms = float(_end_errors(gpu, x).pow(2).mean().sqrt())
    assert rms < (2.5e-8 if where == "end" else (1.7e-8 ** 2 + 6.7e-8 ** 2) ** 0.5), rms


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 5000, 50001])
def test_select_scores_a_step_apart(gpu, dtype, V):
    """Rows of the same logits and base scores one 32-bit step apart, the best in the last row: in 32 bits the scores are the same."""
    gen = torch.Generator().manual_seed(V)
    row = torch.randn(V, generator=gen).clamp(-3, 3)
    row[V // 2], row[V // 3] = 4.0, 3.5
    W, K = 8, 16
    logits = row.to(dtype).expand(W, V).contiguous()
    base = torch.tensor([-0.7])
    bases = [float(base)]
    while len(bases) < W:
        base = torch.nextafter(base, torch.zeros(1))
        bases.append(float(base))
    scores = torch.tensor([bases])
    want, got = _select(gpu, logits.to(gpu), scores, K)
    assert got[1].tolist() == [2 * list(range(W - 1, -1, -1))] and got[2].tolist() == [W * [V // 2] + W * [V // 3]]
    assert torch.equal(want[1], got[1]) and torch.equal(want[2], got[2])


@pytest.mark.parametrize("width,hq,hkv", [(3, 4, 2), (6, 8, 2), (4, 16, 1), (10, 16, 1)])
def test_attention_scores_far_below_zero(gpu, width, hq, hkv):
    """Keys that all score -3.7e33: equal weights, over shared pages and a slot's own."""
    gen = torch.Generator().manual_seed(width)
    lens, common = [100 + 7 * s for s in range(width)], [2]
    bt, pages = _tables(gen, lens, common, width)
    _, v = _cache(gen, pages, hkv, "cpu")
    k = torch.full((pages, hkv, 32, 128), -2.0 ** 54, dtype=torch.bfloat16)
    q = torch.full((width, hq, 128), 2.0 ** 54, dtype=torch.bfloat16)
    ctx, shared = torch.tensor(lens, dtype=torch.int32), torch.tensor(common, dtype=torch.int32)
    out = torch.zeros_like(q).to(gpu)
    ops.beam_attention(q.to(gpu), k.to(gpu), v.to(gpu), bt.to(gpu), ctx.to(gpu), shared.to(gpu), out, width)
    for s, n in enumerate(lens):  # weights of one are exact: the result rounds, and its sum in 32 bits
        V = gather_kv(k, v, bt[s], n)[1].double().repeat_interleave(hq // hkv, 1)
        want = V.mean(0)
        assert bool(((out[s].cpu().double() - want).abs() <= 2.0 ** -8 * want.abs() + n * 2.0 ** -24 * V.abs().mean(0)).all())


@pytest.mark.parametrize("width,hq", [(4, 4), (8, 12), (16, 16), (20, 24), (32, 16)])
def test_attention_in_a_large_pool(gpu, width, hq):
    """A cache allocated ahead, its live pages anywhere in it, and tables as wide as the longest sequence: the same numbers."""
    gen = torch.Generator().manual_seed(width + hq)
    lens, common = [0 if s % 7 == 3 else 400 + 3 * s for s in range(2 * width)], [11, 0]
    bt, small = _tables(gen, lens, common, width)
    k, v = (x.to(gpu) for x in _cache(gen, small, 4, "cpu"))
    pages = 2500  # 164 MB
    bk, bv = torch.full((pages, 4, 32, 128), math.nan, dtype=torch.bfloat16, device=gpu), torch.full((pages, 4, 128, 32), math.nan, dtype=torch.bfloat16, device=gpu)
    at = torch.randperm(pages, generator=gen)[:small]
    bk[at], bv[at] = k, v
    wide = torch.full((2 * width, 1025), -1, dtype=torch.int32)
    wide[:, : bt.shape[1]] = at[bt.long()].to(torch.int32)
    q = torch.randn(2 * width, hq, 128, generator=gen).to(torch.bfloat16).to(gpu)
    ctx, shared = torch.tensor(lens, dtype=torch.int32, device=gpu), torch.tensor(common, dtype=torch.int32, device=gpu)
    out = torch.full_like(q, 3.0)
    ops.beam_attention(q, bk, bv, wide.to(gpu), ctx, shared, out, width)
    for s, n in enumerate(lens):
        got = out[s].cpu().double()
        if n == 0:
            assert bool((got == 3.0).all())
            continue
        K, V = (x.double().repeat_interleave(hq // 4, 1) for x in gather_kv(k.cpu(), v.cpu(), bt[s], n))
        p = torch.softmax((q[s].cpu().double()[None] * K).sum(-1) / math.sqrt(128), 0)[..., None]
        want, size = (p * V).sum(0), (p * V.abs()).sum(0)
        assert bool(((got - want).abs() <= (2.0 ** -8 + 1e-4) * size + 2.0 ** -8 * want.abs()).all()), s


def test_shared_of_too_many_slots(gpu):
    e = torch.empty(1 << 26, 1, dtype=torch.int32, device=gpu)  # nothing reads it
    with pytest.raises(RuntimeError, match="at most"):
        ops.beam_shared(e, e.view(-1), 1, e.view(-1))


@pytest.mark.parametrize("width,hq", [(4, 4), (6, 12), (9, 16), (20, 16)])
def test_attention_more_shared_pages_than_whole_ones(gpu, width, hq):
    """Counts past the whole pages of every slot are those, negative ones none, with 1 to 8 column tiles."""
    gen = torch.Generator().manual_seed(width)
    k, v = _cache(gen, 12, 2, gpu)
    bt = torch.randperm(12, generator=gen).to(torch.int32).expand(width, 12).contiguous().to(gpu)
    q = torch.randn(width, hq, 128, generator=gen).to(torch.bfloat16).to(gpu)
    ctx = torch.tensor([290 + s for s in range(width)], dtype=torch.int32, device=gpu)
    outs = []
    for n in (9, 10, 10 ** 6, 2 ** 31 - 1, 0, -3, -2 ** 31):
        outs.append(torch.zeros_like(q))
        ops.beam_attention(q, k, v, bt, ctx, torch.tensor([n], dtype=torch.int32, device=gpu), outs[-1], width)
    assert all(torch.equal(outs[0], o) for o in outs[1:4]) and all(torch.equal(outs[4], o) for o in outs[5:])
    for s in range(width):
        K, V = (x.double().repeat_interleave(hq // 2, 1) for x in gather_kv(k.cpu(), v.cpu(), bt[s].cpu(), 290 + s))
        p = torch.softmax((q[s].cpu().double()[None] * K).sum(-1) / math.sqrt(128), 0)[..., None]
        want, size = (p * V).sum(0), (p * V.abs()).sum(0)
        for o in (outs[0], outs[4]):
            assert bool(((o[s].cpu().double() - want).abs() <= (2.0 ** -8 + 1e-4) * size + 2.0 ** -8 * want.abs()).all()), s
