"""Generation with drafted tokens: a draft model proposes a few tokens a step, the target verifies them in one.

One round for a batch: the draft model steps ``drafts`` + 1 times from a recorded single-token step
(``DecodeSession``), each sample feeding the next; the target then runs the tokens so far unseen (the last one kept and
the drafts) as ONE step with the logits of every position wanted, which costs it little more than a single token does;
``ops.verify_drafts`` says which drafts stand and what follows them, so that the tokens are distributed as the
target's own (greedy: are the target's own).  Both caches are then cut back to what stood.

Any two models over one vocabulary will do; the natural draft is the same weights in 4 bits.  Caches that cannot be cut
back (windows, fixed-size state) are refused.  Random numbers: a request's draws, and which of them meets which of its
tokens, depend on its seed and index alone, whatever else its batch holds: every round takes ``drafts`` + 1 numbers of the
request's stream and of the draft's, also where the context's end leaves fewer drafts.  The draft's samples and the
verification use streams of their own.
"""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np
import torch

from ..sampling import Sampler, SamplingParams
from ..sampling.sampler import uniform_draws
from .batch import StepEntry
from .decode_session import drop_sessions, session_for
from .generate import check_kernels, settle, take_token

_DRAFT_STREAM = 0x5851F42D4C957F2D         # what the draft's seed differs by


def check_draftable(model, draft, cache, draft_cache) -> None:
    """Raises ValueError where the two cannot work together."""
    if model.vocab_size != draft.vocab_size:
        raise ValueError(f"the draft has a vocabulary of {draft.vocab_size}, the model one of {model.vocab_size}")
    for what, m, c in (("model", model, cache), ("draft", draft, draft_cache)):
        if c.has_running_state or any(g.spec.window > 0 for g in c.kv_groups):
            raise ValueError(f"drafted tokens need caches that can be cut back: the {what} has windows or fixed-size state")
        if not m.graph_safe:
            raise ValueError(f"drafted tokens need a {what} whose single-token step can be recorded")


def room_for_drafts(model, draft, lengths: Sequence[int], drafts: int, context: int) -> int:
    """How many tokens may be drafted in a round for sequences of these lengths (positions in the cache): the step runs
    one token more, and no position past the context or either model's last is touched."""
    most = min(context, model.max_positions, draft.max_positions)
    return max(0, min([drafts] + [most - n - 1 for n in lengths]))


def acquire_pair(cache, draft_cache):
    """A slot of each cache, or of neither."""
    slot = cache.acquire()
    try:
        return slot, draft_cache.acquire()
    except Exception:
        cache.release(slot)
        raise


def run_drafted(model, draft, cache, draft_cache, params: SamplingParams, states, stop_ids, max_tokens: int, context: int,
                drafts: int, kept_slots: Optional[Sequence] = None, first_sample: Optional[list] = None,
                counts: Optional[dict] = None) -> None:
    """One batch from start to end, as ``run_batch_graphed`` but with ``drafts`` tokens drafted a round.
    ``kept_slots``: a (slot, draft slot) pair for each request, taken by the caller; they are not given back, and at the end
    hold exactly what was fed and emitted.  ``counts``: receives ``rounds``, ``drafted`` and ``kept``."""
    check_draftable(model, draft, cache, draft_cache)
    context = min(context, model.max_positions, draft.max_positions)
    ops, device = model.runtime.ops, model.runtime.device
    draft_params = SamplingParams(params.temperature, params.top_k, params.seed ^ _DRAFT_STREAM)
    tally = counts if counts is not None else {}
    tally.update(rounds=0, drafted=0, kept=0)
    slots = {}
    try:
        live = []
        for k, st in enumerate(states):
            if max_tokens <= 0 or st.held + len(st.prompt) >= context:
                st.finished, st.reason = True, "max_tokens" if max_tokens <= 0 else "context"
                continue
            slots[k] = kept_slots[k] if kept_slots is not None else acquire_pair(cache, draft_cache)
            live.append(k)
        if not live:
            return

        def leave(k):
            pair = slots.pop(k)
            if kept_slots is None:
                cache.release(pair[0])
                draft_cache.release(pair[1])

        prompts = [list(states[k].prompt) for k in live]
        sampler = Sampler(params, [states[k].index for k in live], device, ops)
        logits = model.step(cache, [StepEntry(slots[k][0], p, [len(p) - 1]) for k, p in zip(live, prompts)])
        first = sampler.sample(logits)
        draft.step(draft_cache, [StepEntry(slots[k][1], p) for k, p in zip(live, prompts)])
        last = dict(zip(live, first.cpu().tolist()))           # the token each request has produced and not been fed
        if first_sample is not None:
            import time
            first_sample.append(time.perf_counter())
        check_kernels(model)
        for k in list(live):
            if not take_token(states[k], last[k], stop_ids, max_tokens, context):
                live.remove(k)
                leave(k)
        members = list(live)        # whom the draft's recorded step runs: those that have ended stay until half of them have
        drawn = 0                   # numbers that the rounds so far have taken of each request's streams
        while live:
            if len(live) * 2 <= len(members):
                for k in members:
                    if k not in live:
                        leave(k)
                members = list(live)
            starts = {k: cache.length(slots[k][0]) for k in live}
            room = {k: room_for_drafts(model, draft, [starts[k]], drafts, context) for k in live}
            g, n = max(room.values()), len(live)
            ids, qs = _draft(draft, draft_cache, draft_params, [slots[k][1] for k in members], [states[k].index for k in members],
                             [last[k] for k in members], [room.get(k) for k in members], g, drawn, context)
            if n < len(members):
                at = torch.tensor([members.index(k) for k in live], device=device)
                ids, qs = ids[at], None if qs is None else qs[at]
            rows = [row[:room[k]] for k, row in zip(live, ids.cpu().tolist())] if g else [[] for _ in live]
            logits = model.step(cache, [StepEntry(slots[k][0], [last[k]] + r, range(len(r) + 1)) for k, r in zip(live, rows)])
            if min(room.values()) < g:                             # near the context's end: every sequence in g + 1 rows, the drafts end at a -1
                places = torch.arange(g, device=device)
                ids = ids.masked_fill(places >= torch.tensor([room[k] for k in live], device=device)[:, None], -1)
                wide = logits.new_zeros((n * (g + 1), logits.shape[1]))
                wide[torch.tensor([i * (g + 1) + j for i, r in enumerate(rows) for j in range(len(r) + 1)], device=device)] = logits
                logits = wide
            # the token behind the drafts taken comes from the round's last number, however many drafts there were
            draws = np.stack([uniform_draws(params.seed, states[k].index, 1 + drawn, drafts + 1) for k in live])
            draws = np.concatenate([draws[:, :g], draws[:, drafts:]], axis=1)
            tokens, kept = ops.verify_drafts(logits.view(n, g + 1, -1), qs, ids, torch.from_numpy(draws).to(device),
                                             params.temperature if not params.greedy else 0.0, params.kept)
            answer = torch.cat([tokens, kept[:, None]], dim=1).cpu().tolist()
            check_kernels(model)
            drawn += drafts + 1
            tally["rounds"] += 1
            tally["drafted"] += sum(room.values())
            for k, row in zip(list(live), answer):
                start, stood = starts[k], row[-1]
                tally["kept"] += stood
                # what both models have been fed and what stands of it: the last token and the drafts kept
                cache.truncate(slots[k][0], start + 1 + stood)
                draft_cache.truncate(slots[k][1], start + 1 + stood)
                goes_on = True
                for i, token in enumerate(row[:stood + 1]):
                    goes_on = take_token(states[k], token, stop_ids, max_tokens, context)
                    if not goes_on:
                        # what was kept behind this token has been fed, but is no part of the answer
                        cut = start + 1 + min(i, stood)
                        cache.truncate(slots[k][0], cut)
                        draft_cache.truncate(slots[k][1], cut)
                        break
                last[k] = states[k].produced[-1] if states[k].produced else last[k]
                if not goes_on:
                    live.remove(k)
        if kept_slots is not None:
            settle(model, cache, states, [pair[0] for pair in kept_slots], context)
            settle(draft, draft_cache, states, [pair[1] for pair in kept_slots], context)
    finally:
        if kept_slots is None:
            for a, b in slots.values():
                cache.release(a)
                draft_cache.release(b)


def _draft(draft, cache, params: SamplingParams, slots: Sequence[int], requests: Sequence[int], tokens: Sequence[int],
           rooms: Sequence[Optional[int]], g: int, drawn: int, context: int):
    """``g`` tokens drafted behind ``tokens``: (ids int32 [n, g], the logits they were sampled from [n, g, vocab], or None
    where greedy).  The draft is stepped once more, so that its cache holds the last one too.

    ``rooms``: how many of the g each sequence has room for, None for one that has ended.  The recorded step moves every
    sequence on g + 1 times, but none past the context's last position, where one without room for more stays: what it writes
    there is no part of it, since a sequence that fills the context ends without that position.  One that has ended writes
    behind its end, on pages of its own."""
    n, device = len(slots), draft.runtime.device
    session = session_for(draft, cache, params, n, pipelined=False, kv_bound=context)
    state = (list(slots), list(requests), drawn)
    if getattr(session, "drafts_for", None) != state:          # (else it is where the round before left it)
        session.rebind(slots, requests, [drawn] * n)
    session.drafts_for = (list(slots), list(requests), drawn + g + 1)
    starts = [min(cache.length(s), context - 1) for s in slots]
    for s, start, room in zip(slots, starts, rooms):
        cache.reserve(s, room + 1 if room is not None else min(start + g + 1, context) - cache.length(s))
    session.sync_block_tables()
    session.feed(tokens, starts)
    ids = torch.empty((n, g), dtype=torch.int32, device=device)
    qs = None if params.greedy else torch.empty((n, g, draft.vocab_size), dtype=torch.float32, device=device)
    for i in range(g + 1):
        session.launch()
        if i < g:
            ids[:, i] = session.next_tokens
            if qs is not None:
                qs[:, i] = session.logits
    for s, room in zip(slots, rooms):
        if room is not None:
            cache.commit(s, room + 1)
    return ids, qs


def cache_room(prompts: Sequence[Sequence[int]], max_tokens: int, drafts: int, context: int, max_batch: int) -> int:
    """Positions that each of the two caches needs for these requests: a round may run ``drafts`` positions past a request's
    last."""
    from ..cache import PAGE_TOKENS
    from .generate import round_up
    need = sorted((round_up(min(context, len(p) + max_tokens + drafts), PAGE_TOKENS) for p in prompts), reverse=True)
    return max(sum(need[:max_batch]), PAGE_TOKENS)


def generate_drafted(model, draft, prompts: Sequence[Sequence[int]], max_tokens: int, params: SamplingParams, drafts: int,
                     stop_ids=None, context: Optional[int] = None, max_batch: int = 64, cache=None, draft_cache=None,
                     counts: Optional[dict] = None) -> List[List[int]]:
    """``generate`` with ``drafts`` tokens drafted a round by ``draft``.  ``cache`` and ``draft_cache``: the caller's, who calls
    again and wants neither them nor the recorded steps made anew; without them they are made here and dropped at the end."""
    from .generate import RequestState, plan_batches
    if drafts < 1:
        raise ValueError(f"at least one token is drafted a round, got {drafts}")
    context = min(context or model.max_positions, model.max_positions, draft.max_positions)
    stop = frozenset(model.stop_ids if stop_ids is None else stop_ids)
    for i, p in enumerate(prompts):
        if len(p) == 0:
            raise ValueError(f"prompt {i} is empty")
        if len(p) > context:
            raise ValueError(f"prompt {i} has {len(p)} tokens, the context holds {context}")
    total = cache_room(prompts, max_tokens, drafts, context, max_batch)
    if cache is None:
        cache = model.new_cache(max_tokens=total, n_slots=max_batch)
    made = draft_cache is None
    if made:
        draft_cache = draft.new_cache(max_tokens=total, n_slots=max_batch)
    page = cache.page_tokens
    batches = plan_batches([len(p) for p in prompts], max_tokens + drafts + 1, context, min(max_batch, cache.n_slots, draft_cache.n_slots),
                           min(cache.n_pages, draft_cache.n_pages) * page, page)
    states = [RequestState(i, p) for i, p in enumerate(prompts)]
    sums = {"rounds": 0, "drafted": 0, "kept": 0}
    try:
        for batch in batches:
            here: dict = {}
            run_drafted(model, draft, cache, draft_cache, params, [states[i] for i in batch], stop, max_tokens, context, drafts, counts=here)
            for key in sums:
                sums[key] += here[key]
    finally:
        if made:
            drop_sessions(draft, draft_cache)
    if counts is not None:
        counts.update(sums)
    return [s.produced for s in states]
