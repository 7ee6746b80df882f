"""Ops of a beam search over the paged cache: HIP kernels on GPU tensors, ``beams_reference`` on CPU tensors.

A request is a group of ``width`` neighbouring decode slots, slot ``g * width + w`` its beam w.  One step of a search: the logits of
all slots go through ``beam_select``; its rows are the parents that ``page_fork`` and ``state_reorder`` move pages and states by, its
tokens the next inputs; ``beam_shared`` says how many pages a group's tables have in common, and ``beam_attention`` reads those once
in every layer.  Dispatch and errors follow ``ops/__init__.py``: a GPU tensor takes the kernel, which raises RuntimeError on
arguments that it does not take.  All ops can be captured into a graph, run on the current stream of their tensors' device and keep
no work area of their own between calls.
"""
from __future__ import annotations

import torch

from . import beams_reference as bref
from .layers import _hip

BEAM_WIDTH = 32   # beams of a group
BEAM_KEEP = 64    # candidates of a group
FORK_SLOTS = 2048


def beam_select(logits, scores, out_scores, out_rows, out_tokens, eos_id: int = -1, end_scores=None):
    """The K best continuations of each group over its beams and the vocabulary.

    logits [groups * width, V] (fp32 or bf16, whole vocabularies, rows may be strided), scores [groups, width] fp32
    (log-probabilities of the beams so far, -inf for a beam that is not in use).  A continuation's score is scores[w] + log
    softmax(logits[row])[token]; out_scores, out_rows, out_tokens [groups, K] receive the K <= 64 best by (score descending,
    row, token ascending): the score, the row of `logits` it came from -- the slot whose pages and state go on -- and the token.
    Equal logits of a row are ordered by token; scores are compared in 64 bits, over log-sums of 32-bit terms (rows of the same
    logits have the same), and returned in 32.  A token of logit -inf is no candidate, and neither is anything of a row whose
    score or log-sum is not finite (NaN or +inf among its logits, all of them -inf); places that nothing is left for hold -inf,
    -1, -1.  eos_id >= 0: that token counts in the softmax but is not offered; end_scores [groups, width] (optional) receives
    each beam's score with it.  Outputs overlap neither the inputs nor each other, but with K = width out_scores may be `scores`."""
    if _hip(logits):
        torch.ops.dsse.beam_select(logits, scores, out_scores, out_rows, out_tokens, eos_id, end_scores)
    else:
        bref.beam_select(logits, scores, out_scores, out_rows, out_tokens, eos_id, end_scores)


def beam_shared(block_tables, ctx_len, width: int, shared):
    """shared [groups] = how many leading whole pages (of all ctx_len tokens) the tables of a group's live slots have in common;
    0 without a live slot (ctx_len 0 = idle).  Once per step, for all layers.  At most 2^26 - 1 slots."""
    if _hip(block_tables):
        torch.ops.dsse.beam_shared(block_tables, ctx_len, width, shared)
    else:
        bref.beam_shared(block_tables, ctx_len, width, shared)


def beam_attention(q, k_cache, v_cache, block_tables, ctx_len, shared, out, width: int):
    """Decode attention (paged_attention mode 0) of groups of `width` slots, one query each, over the dense cache's pages.

    q, out [slots, Hq, 128] bf16, k_cache [blocks, Hkv, 32, 128], v_cache [blocks, Hkv, 128, 32] (KVCache's pages), up to 16 q heads
    per key/value head; slot s attends to its ctx_len[s] keys (its own among them), and a slot of ctx_len 0 is idle: its row of out
    stays as it was.  The first shared[g] pages must be the same in the tables of group g's live slots (beam_shared); they are read
    once for the group, the others once per slot.  0 is always right.  At most 2^22 rows (slots times Hq)."""
    if _hip(q):
        torch.ops.dsse.beam_attention(q, k_cache, v_cache, block_tables, ctx_len, shared, out, width)
    else:
        bref.beam_attention(q, k_cache, v_cache, block_tables, ctx_len, shared, out, width)


def page_fork(block_tables, held, lens, parents, refs, copies, starved, pools=()):
    """Slot s goes on with the sequence of slot parents[s], for all slots at once and in place.

    block_tables [slots, max_blocks], held [slots] (pages of a slot), lens [slots] (tokens of a slot), refs [pages] (holders of a
    page, 0 = free), all int32.  Every slot takes its parent's pages and length; a parent outside [0, slots) ends the slot: it holds
    nothing any more.  Pages that nobody holds are free from then on.  The page that a slot's next token goes to (number
    lens // 32) then becomes its own: of the slots that go on in one page (those of a parent; of several where an earlier call found
    no free page) the last keeps it if they alone hold it, the others -- and every slot that has no such page yet -- get the lowest
    free pages in slot order.  copies [slots, 2] receives (old, new) where the old page holds tokens already, (-1, -1) elsewhere, and
    the page is copied in every pool: `pools` are tensors [layers, pages, ..] (KVCache.pools() and its like), whole pages of whole
    16-byte units, at most 1 GiB in a layer and, a page of each slot in every pool and layer together, 2^31 - 1 pieces of 16 KiB.  A
    slot that finds no free page keeps what it has, shared: starved [1] counts those, and once pages are free a call with parents[s]
    = s serves them: as many as were starved are enough.  A slot whose max_blocks pages are full needs none.  Entries of a table past
    the slot's pages stay as they were; a number that is no page goes along with the others, but counts nowhere and is copied
    nowhere.  At most 2048 slots."""
    if _hip(block_tables):
        torch.ops.dsse.page_fork(block_tables, held, lens, parents, refs, copies, starved, pools)
    else:
        bref.page_fork(block_tables, held, lens, parents, refs, copies, starved, pools)


def state_reorder(states, parents, width: int):
    """In every tensor of `states` ([slots, ..], any type, a slot's part contiguous and under 2 GiB, at most 32 GiB in all, no two
    of them overlapping), slot s takes what slot parents[s] held, in place and for all slots at once.  parents [slots] int32 stay
    within their group of `width` slots; a slot whose parent is itself, or lies outside its group (an ended slot's -1), stays as it
    is."""
    if _hip(parents):
        torch.ops.dsse.state_reorder(states, parents, width)
    else:
        bref.state_reorder(states, parents, width)
