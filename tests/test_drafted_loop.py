"""The loop of generation with drafted tokens against a fake device: which draws meet which tokens, what stands in both caches,
where a round near the context's end writes."""
import numpy as np
import pytest
import torch

import plain_q4 as plain
from math_utils_b200.cache import SequenceCache
from math_utils_b200.engine import drafted
from math_utils_b200.engine.generate import RequestState, plan_batches
from math_utils_b200.parts.base import KVCacheSpec
from math_utils_b200.sampling import SamplingParams

VOCAB = 50


def next_of(tokens):
    """The target's own next token: a function of the whole sequence."""
    h = 7
    for t in tokens:
        h = (h * 31 + int(t) + 1) % 1000003
    return h % VOCAB


def draft_of(tokens):
    """The draft's: the target's but for every third sequence."""
    t = next_of(tokens)
    return t if (sum(map(int, tokens)) + len(tokens)) % 3 else (t + 1) % VOCAB


class Memory:
    """What a cache's pages hold: a token for every position written, page by page, so that a write on another sequence's page
    shows."""

    def __init__(self, cache):
        self.cache, self.pages = cache, {}

    def _page(self, slot, position):
        page = int(self.cache.kv_groups[0].table[slot, position // 64])
        assert page >= 0, f"slot {slot} has no page for position {position}"
        return page, position % 64

    def write(self, slot, position, token):
        self.pages[self._page(slot, position)] = int(token)

    def read(self, slot, length):
        return [self.pages[self._page(slot, p)] for p in range(length)]


class FakeOps:
    def __init__(self, params):
        self.params, self.seen = params, []

    def check_status(self, device):
        pass

    def verify_drafts(self, logits, draft_logits, drafts, draws, temperature, top_k):
        tokens, kept = [], []
        self.seen.append((drafts.clone(), draws.clone()))
        for i in range(drafts.shape[0]):
            t, n, _ = plain.verify(logits[i].numpy(), None, drafts[i].tolist(), draws[i].numpy(), 0.0, 0)
            tokens.append(t)
            kept.append(n)
        return torch.tensor(tokens, dtype=torch.int32), torch.tensor(kept, dtype=torch.int32)


class FakeModel:
    vocab_size, max_positions, graph_safe = VOCAB, 200, True

    def __init__(self, cache, ops, of, most):
        self.cache, self.memory, self.of, self.max_positions = cache, Memory(cache), of, most
        self.runtime = type("Runtime", (), dict(ops=ops, device=torch.device("cpu")))

    def step(self, cache, entries):
        rows = []
        for e in entries:
            start = cache.reserve(e.slot, len(e.tokens))
            held = self.memory.read(e.slot, start)
            for i, t in enumerate(e.tokens):
                self.memory.write(e.slot, start + i, t)
            for w in e.want:
                row = torch.zeros(VOCAB)
                row[self.of(held + list(e.tokens)[:w + 1])] = 1.0
                rows.append(row)
            cache.commit(e.slot, len(e.tokens))
        return torch.stack(rows) if rows else None


class FakeSession:
    """The recorded step of the draft: a token each, the samples fed on, positions up to kv_bound - 1."""

    def __init__(self, model, cache, n, kv_bound):
        self.model, self.cache, self.n, self.kv_bound = model, cache, n, kv_bound
        self.slots, self.draws, self.next_tokens, self.logits = None, None, torch.zeros(n, dtype=torch.int32), torch.zeros(n, VOCAB)

    def rebind(self, slots, requests, draws):
        assert len(slots) == self.n
        self.slots, self.draws = list(slots), list(draws)

    def sync_block_tables(self):
        pass

    def feed(self, tokens, positions):
        self.tokens, self.positions = list(tokens), list(positions)

    def launch(self):
        for i, slot in enumerate(self.slots):
            p = self.positions[i]
            held = self.model.memory.read(slot, p)
            self.model.memory.write(slot, p, self.tokens[i])
            self.next_tokens[i] = self.tokens[i] = self.model.of(held + [self.tokens[i]])
            self.positions[i] = min(p + 1, self.kv_bound - 1)
            self.draws[i] += 1


class World:
    """Two caches of exactly the pages that ``plan_batches`` counts, and what is recorded of a run."""

    def __init__(self, monkeypatch, lens, max_tokens, context, drafts, most=200, n_slots=None):
        params = SamplingParams(0.0, 0, 3)
        need = sum(-(-min(context, n + max_tokens + drafts) // 64) * 64 for n in lens)
        caches = [SequenceCache([KVCacheSpec(1, 16, 0)], max(need, 64), most, torch.float32, "cpu", n_slots=n_slots or len(lens)) for _ in range(2)]
        self.ops = FakeOps(params)
        self.model = FakeModel(caches[0], self.ops, next_of, most)
        self.draft = FakeModel(caches[1], self.ops, draft_of, most)
        self.caches, self.params, self.sessions, self.asked = caches, params, {}, []
        world = self

        class FakeSampler:
            def __init__(self, *a):
                pass

            def sample(self, logits):
                return logits.argmax(dim=1).int()

        def session_for(model, cache, params, n, pipelined=True, kv_bound=None):
            bound = model.max_positions if kv_bound is None else kv_bound
            return world.sessions.setdefault((n, bound), FakeSession(model, cache, n, bound))

        def draws_of(seed, request, first, count):
            world.asked.append((request, first, count))
            return np.array([request + (first + i) / 1024.0 for i in range(count)])

        monkeypatch.setattr(drafted, "Sampler", FakeSampler)
        monkeypatch.setattr(drafted, "session_for", session_for)
        monkeypatch.setattr(drafted, "uniform_draws", draws_of)

    def run(self, prompts, stop, max_tokens, context, drafts, kept_slots=None, states=None):
        states = states or [RequestState(i, p) for i, p in enumerate(prompts)]
        counts = {}
        drafted.run_drafted(self.model, self.draft, *self.caches, self.params, states, frozenset(stop), max_tokens, context, drafts,
                            kept_slots=kept_slots, counts=counts)
        return states, counts


def expected(prompt, max_tokens, stop, context):
    out, seq = [], list(prompt)
    while len(out) < max_tokens and len(seq) < context:
        t = next_of(seq)
        if t in stop:
            break
        out.append(t)
        seq.append(t)
    return out


def test_drawn_cases(monkeypatch):
    rng = np.random.default_rng(11)
    reasons = set()
    for case in range(80):
        n, context, drafts = int(rng.integers(1, 7)), int(rng.integers(2, 200)), int(rng.integers(1, 6))
        lens = [int(rng.integers(1, context + 1)) for _ in range(n)]
        max_tokens = int(rng.choice([1, 2, 3, 17, 64, 300]))
        stop = set(rng.integers(0, VOCAB, size=int(rng.integers(0, 4))).tolist())
        world = World(monkeypatch, lens, max_tokens, context, drafts)
        assert len(plan_batches(lens, max_tokens + drafts + 1, context, n, world.caches[0].n_pages * 64, 64)) == 1
        for _ in range(2):                                # the same slots again
            prompts = [rng.integers(0, VOCAB, size=k).tolist() for k in lens]
            states, counts = world.run(prompts, stop, max_tokens, context, drafts)
            for st, p in zip(states, prompts):
                assert st.finished and st.produced == expected(p, max_tokens, stop, context), (case, lens, max_tokens, context, drafts)
                reasons.add(st.reason)
            for c in world.caches:
                assert c.slots.n_free == n and c.free_pages(0) == c.n_pages
            assert counts["kept"] <= counts["drafted"]
    assert reasons == {"stop", "max_tokens", "context"}


@pytest.mark.parametrize("beside", [[], [95], [99, 60, 97], [1, 2, 3, 98]])
def test_what_a_request_draws_is_its_own_matter(monkeypatch, beside):
    """Beside requests that run into the context's end a request drafts as many tokens, and takes the same numbers for them and for
    the token behind them, as alone."""
    prompt = np.random.default_rng(1).integers(0, VOCAB, size=20).tolist()
    others = [np.random.default_rng(n).integers(0, VOCAB, size=n).tolist() for n in beside]
    drafts = 4

    def met(prompts):
        """Round by round: the drafts of request 0 and the numbers that decide about them."""
        world = World(monkeypatch, [len(p) for p in prompts], 50, 100, drafts)
        states, _ = world.run(prompts, (), 50, 100, drafts)
        assert states[0].produced == expected(prompt, 50, (), 100)
        firsts = [first for request, first, count in world.asked if request == 0]
        assert all(count == drafts + 1 for _, _, count in world.asked)
        return firsts, [(d[0].tolist(), u[0].tolist()) for d, u in world.ops.seen][:len(firsts)]

    alone = met([prompt])
    assert alone[0] == [1 + i * (drafts + 1) for i in range(len(alone[0]))]
    assert all(len(d) == drafts and min(d) >= 0 for d, _ in alone[1][:8])
    assert met([prompt] + others) == alone


def test_a_conversation_up_to_the_end_of_the_context(monkeypatch):
    """Kept slots hold, turn after turn, exactly what was fed and emitted, in both caches."""
    for context, drafts, max_tokens in ((90, 4, 11), (64, 3, 200), (100, 5, 1), (70, 1, 30)):
        world = World(monkeypatch, [context], max_tokens, context, drafts)
        pair = tuple(c.acquire() for c in world.caches)
        said = []
        for turn in range(30):
            ids = np.random.default_rng(turn).integers(0, VOCAB, size=7).tolist()
            if len(said) + len(ids) >= context:
                break
            st = RequestState(turn, ids, held=len(said))
            want = expected(said + ids, max_tokens, (), context)
            world.run(None, (), max_tokens, context, drafts, kept_slots=[pair], states=[st])
            assert st.produced == want
            said += ids + want
            for model, cache, slot in zip((world.model, world.draft), world.caches, pair):
                assert cache.length(slot) == len(said) and model.memory.read(slot, len(said)) == said


def test_slots_are_had_in_pairs(monkeypatch):
    """Where the draft's cache has no slot left, or cannot be made, none of the model's stays taken."""
    from math_utils_b200 import LLM, Options
    from math_utils_b200.cache import CacheFull
    world = World(monkeypatch, [5, 5], 3, 100, 2)
    taken = world.caches[1].acquire()
    with pytest.raises(CacheFull):
        world.run([[1, 2, 3], [4, 5]], (), 3, 100, 2)
    assert world.caches[0].slots.n_free == 2 and world.caches[1].slots.n_free == 1
    world.caches[1].release(taken)
    assert [len(s.produced) for s in world.run([[1, 2, 3], [4, 5]], (), 3, 100, 2)[0]] == [3, 3]

    class Model:
        max_positions = 100

        def __init__(self, cache):
            self.cache = cache

        def new_cache(self, **how):
            if self.cache is None:
                raise MemoryError("no room")
            return self.cache

    llm = LLM(options=Options(drafts=2))
    llm.model, llm.draft = Model(world.caches[0]), Model(None)
    for _ in range(2):
        with pytest.raises(MemoryError):
            llm.prompt([1, 2, 3])
        assert llm._slot is None and world.caches[0].slots.n_free == 2
