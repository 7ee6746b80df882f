"""PyTorch references of the ops of a beam search (``ops/beams.py`` has their definitions): what CPU tensors run on and what the
kernels are tested against.  Plain loops over groups and slots, sums and scores in 64 bits."""
from __future__ import annotations

import math

import torch

from .reference import PAGE, gather_kv

BEAM_WIDTH, BEAM_KEEP, FORK_SLOTS, BEAM_ROWS = 32, 64, 2048, 1 << 22
COPY_PIECE, COPY_PIECES, SHARED_SLOTS = 1 << 14, (1 << 31) - 1, (1 << 26) - 1


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise RuntimeError(text)


def _typed(t, dtype, name: str) -> None:
    _need(t.dtype == dtype, f"{name} must be {dtype}")
    _need(t.is_contiguous(), f"{name} must be contiguous")


def _beams(slots: int, width: int) -> int:
    _need(1 <= width <= BEAM_WIDTH, f"a group has 1 to {BEAM_WIDTH} beams")
    _need(slots % width == 0, "slots must be whole groups of `width` beams")
    return slots // width


def beam_select(logits, scores, out_scores, out_rows, out_tokens, eos_id=-1, end_scores=None):
    _need(logits.dtype in (torch.float32, torch.bfloat16), "logits must be fp32 or bf16")
    _need(logits.dim() == 2 and (logits.shape[1] == 1 or logits.stride(1) == 1), "logits must be [rows, V] with a unit innermost stride")
    _typed(scores, torch.float32, "scores")
    _typed(out_scores, torch.float32, "out_scores")
    _typed(out_rows, torch.int32, "out_rows")
    _typed(out_tokens, torch.int32, "out_tokens")
    _need(scores.dim() == 2 and scores.numel() == logits.shape[0], "scores must be [groups, width], a number per row of logits")
    W, V = scores.shape[1], logits.shape[1]
    G = _beams(logits.shape[0], W)
    _need(out_scores.dim() == 2 and out_scores.shape[0] == G and 1 <= out_scores.shape[1] <= BEAM_KEEP,
          f"out_scores must be [groups, 1 to {BEAM_KEEP}]")
    _need(out_rows.shape == out_scores.shape and out_tokens.shape == out_scores.shape, "outputs differ in shape")
    _need(1 <= V <= 1 << 24 and logits.shape[0] <= 65535, "1 to 2^24 tokens, at most 65535 rows")
    _need(-1 <= eos_id < V, "eos_id must be a token or -1")
    if end_scores is not None:
        _typed(end_scores, torch.float32, "end_scores")
        _need(end_scores.shape == scores.shape, "end_scores must match scores")
        _need(eos_id >= 0, "end_scores needs an eos_id")
        end_scores.fill_(-math.inf)
    K = out_scores.shape[1]
    for g in range(G):
        best = []
        for w in range(W):
            row, x = g * W + w, logits[g * W + w].double()
            base, top = float(scores[g, w]), float(x.max())
            if not (math.isfinite(base) and math.isfinite(top)) or bool(x.isnan().any()):
                continue
            y = (x - top) + (base - math.log(float((x - top).exp().sum())))
            if eos_id >= 0:
                if end_scores is not None:
                    end_scores[g, w] = y[eos_id]
                y[eos_id] = -math.inf
            order = torch.sort(x, descending=True, stable=True).indices
            order = order[y[order] > -math.inf][:K].tolist()
            best += [(-float(y[t]), row, t) for t in order]
        best = sorted(best)[:K]
        for i in range(K):
            s, row, t = best[i] if i < len(best) else (math.inf, -1, -1)
            out_scores[g, i], out_rows[g, i], out_tokens[g, i] = -s, row, t


def beam_shared(block_tables, ctx_len, width, shared):
    for t, n in ((block_tables, "block_tables"), (ctx_len, "ctx_len"), (shared, "shared")):
        _typed(t, torch.int32, n)
    _need(block_tables.dim() == 2 and block_tables.shape[1] >= 1, "block_tables must be [slots, max_blocks]")
    _need(block_tables.shape[0] <= SHARED_SLOTS, f"at most {SHARED_SLOTS} slots")
    G = _beams(block_tables.shape[0], width)
    _need(ctx_len.numel() == block_tables.shape[0] and shared.numel() == G, "ctx_len must be [slots], shared [groups]")
    for g in range(G):
        live = [s for s in range(g * width, (g + 1) * width) if int(ctx_len[s]) > 0]
        n = min([int(ctx_len[s]) // PAGE for s in live] + [block_tables.shape[1]]) if live else 0
        same = [len({int(block_tables[s, j]) for s in live}) == 1 for j in range(n)]
        shared[g] = same.index(False) if False in same else n


def beam_attention(q, k_cache, v_cache, block_tables, ctx_len, shared, out, width):
    for t, n in ((q, "q"), (k_cache, "k_cache"), (v_cache, "v_cache"), (out, "out")):
        _typed(t, torch.bfloat16, n)
    for t, n in ((block_tables, "block_tables"), (ctx_len, "ctx_len"), (shared, "shared")):
        _typed(t, torch.int32, n)
    _need(q.dim() == 3 and q.shape[2] == 128, "q must be [slots, Hq, 128]")
    _need(out.shape == q.shape, "out must match q")
    _need(k_cache.dim() == 4 and k_cache.shape[2:] == (PAGE, 128), "k_cache must be [blocks, Hkv, 32, 128]")
    _need(v_cache.shape == (*k_cache.shape[:2], 128, PAGE), "v_cache must be [blocks, Hkv, 128, 32]")
    S, hq, hkv = q.shape[0], q.shape[1], k_cache.shape[1]
    _need(hkv >= 1 and hq >= 1 and hq % hkv == 0 and hq // hkv <= 16, "up to 16 q heads per key/value head, the same for each")
    _need(S * hq <= BEAM_ROWS, f"at most {BEAM_ROWS} slots times q heads")
    G = _beams(S, width)
    _need(block_tables.dim() == 2 and block_tables.shape[0] == S and block_tables.shape[1] >= 1, "block_tables must be [slots, max_blocks]")
    _need(ctx_len.numel() == S and shared.numel() == G, "ctx_len must be [slots], shared [groups]")
    for s in range(S):
        n = int(ctx_len[s])
        if n <= 0:
            continue
        k, v = (x.double().repeat_interleave(hq // hkv, dim=1) for x in gather_kv(k_cache, v_cache, block_tables[s], n))
        score = (q[s].double()[None] * k).sum(-1) / math.sqrt(128)      # [n, hq]
        p = torch.softmax(score, 0)
        out[s] = (p[..., None] * v).sum(0).to(out.dtype)


def page_fork(block_tables, held, lens, parents, refs, copies, starved, pools=()):
    for t, n in ((block_tables, "block_tables"), (held, "held"), (lens, "lens"), (parents, "parents"), (refs, "refs"),
                 (copies, "copies"), (starved, "starved")):
        _typed(t, torch.int32, n)
    _need(block_tables.dim() == 2 and block_tables.shape[1] >= 1, "block_tables must be [slots, max_blocks]")
    S, M = block_tables.shape
    _need(S <= FORK_SLOTS, f"at most {FORK_SLOTS} slots")
    _need(held.numel() == S and lens.numel() == S and parents.numel() == S, "held, lens and parents must be [slots]")
    _need(copies.shape == (S, 2) and starved.numel() == 1, "copies must be [slots, 2], starved [1]")
    _need(refs.numel() >= 1, "refs must have a count per page")
    pieces = 0
    for t in pools:
        _need(t.dim() >= 3 and t.shape[1] == refs.numel(), "a pool must be [layers, pages, ..]")
        if t.numel():
            _need(t[0, 0].is_contiguous() and t[0].is_contiguous(), "a pool's pages must be contiguous")
            _need(t[0, 0].numel() * t.element_size() % 16 == 0, "a pool's pages must start and end at 16 bytes")
            _need(t[0, 0].numel() * t.element_size() <= 1 << 30, "a page of a pool's layer is at most 1 GiB")
            pieces += t.shape[0] * -(-t[0, 0].numel() * t.element_size() // COPY_PIECE)
            _need(S * pieces <= COPY_PIECES, "pages of all slots, pools and layers are at most 2^31 - 1 pieces of 16 KiB")
    P = refs.numel()  # an entry outside of the pool goes along with the others, but has no count
    before, had, size = block_tables.clone(), held.clamp(0, M).tolist(), lens.tolist()
    goes = [q if 0 <= q < S else -1 for q in parents.tolist()]
    for s, q in enumerate(goes):  # every slot gives its pages up and takes its parent's
        n = had[q] if q >= 0 else 0
        for page in before[s, :had[s]].tolist():
            if 0 <= page < P:
                refs[page] -= 1
        block_tables[s, :n] = before[q, :n]
        for page in before[q, :n].tolist():
            if 0 <= page < P:
                refs[page] += 1
        held[s], lens[s] = n, size[q] if q >= 0 else 0
    counts = refs.clone()
    free = (counts == 0).nonzero()[:, 0].tolist()
    copies.fill_(-1)
    starved.zero_()
    at = [int(lens[s]) // PAGE for s in range(S)]
    goes_to = [int(block_tables[s, j]) if q >= 0 and 0 <= j < min(M, int(held[s])) else -1 for s, (q, j) in enumerate(zip(goes, at))]
    for s, q in enumerate(goes):
        j, page = at[s], goes_to[s]
        if q < 0 or not 0 <= j < M:
            continue
        if j < int(held[s]) and not 0 <= page < P:
            continue
        alike = [t for t in range(S) if goes_to[t] == page]
        if page >= 0 and s == alike[-1] and int(counts[page]) == len(alike):
            continue
        if not free:
            starved += 1
            continue
        new = free.pop(0)
        refs[new] = 1
        block_tables[s, j] = new
        held[s] = max(int(held[s]), j + 1)
        if page >= 0:
            refs[page] -= 1
            if int(lens[s]) % PAGE:
                copies[s] = torch.tensor([page, new], dtype=torch.int32)
    for a, b in copies.tolist():
        for t in pools:
            if a >= 0 and t.numel():
                t[:, b] = t[:, a]


def state_reorder(states, parents, width):
    _typed(parents, torch.int32, "parents")
    S = parents.numel()
    _beams(S, width)
    for t in states:
        _need(t.dim() >= 1 and t.shape[0] == S, "a state must be [slots, ..]")
        if t.numel():
            _need(t[0].is_contiguous() and (S == 1 or t.stride(0) >= t[0].numel()), "a slot's state must be contiguous")
            _need(t[0].numel() * t.element_size() % 2 == 0 and t[0].numel() * t.element_size() < (1 << 31) - 1 - (1 << 16),
                  "a slot's state must have an even number of bytes, under 2 GiB")
            _need(sum(u.data_ptr() == t.data_ptr() and u.numel() > 0 for u in states) == 1, "a state is listed twice")
    _need(sum(t[0].numel() * t.element_size() for t in states if t.numel()) <= 1 << 35, "at most 32 GiB of a slot in all")
    src = [q if q // width == s // width and q >= 0 else s for s, q in enumerate(parents.tolist())]
    for t in states:
        t.copy_(t.clone()[torch.tensor(src, dtype=torch.long)])
