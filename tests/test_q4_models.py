"""Whole models with 4-bit matrices and 8-bit rows, and generation with drafted tokens, through the library's entry points."""
import json

import numpy as np
import pytest
import torch

import plain_gpt2
import plain_q4 as plain
import test_forisun_gpu as forisun
import test_lusalorn_gpu as lusalorn
import test_pelenex_gpu as pelenex
import test_seledra_gpu as seledra
import test_tibopel_gpu as tibopel
import test_tokolorn_gpu as tokolorn
from helpers import BF16_NEAR_TIE, check_logits, run_batch, run_tail_one_by_one, run_whole
from math_utils_b200 import LLM, DecoderModel, Options, write_random_model
from math_utils_b200.csrc import ops
from math_utils_b200.engine.drafted import generate_drafted, room_for_drafts, run_drafted
from math_utils_b200.engine.runtime import Runtime
from math_utils_b200.sampling import SamplingParams
from math_utils_b200.sampling.sampler import uniform_draws

gpu = pytest.mark.gpu


def tokens_for(vocab, n, seed):
    return np.random.default_rng(seed).integers(0, vocab, size=n).tolist()


# ------------------------------------------------------------------------------------------------ 4-bit matrices
def in_four_bits(weights):
    """A GPT-2's weights with the layers' matrices ([in, out] in the file) as their 4-bit values."""
    out = dict(weights)
    for name, w in weights.items():
        if w.ndim == 2 and name.split(".")[-2] in ("c_attn", "c_proj", "c_fc"):
            q = ops.quantize_q4(torch.from_numpy(w).to(torch.bfloat16).t().contiguous().cuda())
            u8 = lambda t: t.contiguous().view(torch.uint8).cpu().numpy()
            out[name] = plain.q4_values(u8(q.codes), u8(q.scales))[:, :w.shape[0]].T
    return out


@gpu
@pytest.mark.parametrize("name", ["tiny_a", "tiny_b", "tiny_c"])
def test_gpt2_with_4_bit_matrices_against_plain(name, model_dirs, plain_models):
    """Whole prompts, single tokens and an unequal batch: bfloat16 rows are taken as they are, so the bounds are those
    of the bfloat16 path with the matrices' 4-bit values in the plain model."""
    cfg, w = plain_models[name]
    w = in_four_bits(w)
    model = DecoderModel.from_dir(model_dirs[name], weight_bits=4)
    cache = model.new_cache(max_tokens=3 * 192, n_slots=3)
    toks = tokens_for(cfg["vocab_size"], 70, 5)
    want = plain_gpt2.forward(toks, cfg, w)
    check_logits(run_whole(model, cache, toks), want, "bfloat16", f"{name} whole")
    check_logits(run_tail_one_by_one(model, cache, toks, 20), want, "bfloat16", f"{name} tail")
    requests = [tokens_for(cfg["vocab_size"], n, 6 + n) for n in (33, 70, 9)]
    for got, r in zip(run_batch(model, cache, requests, [30, 41, 1]), requests):
        check_logits(got, plain_gpt2.forward(r, cfg, w), "bfloat16", f"{name} batch")
    full = DecoderModel.from_dir(model_dirs[name])
    matrices = sum(v.size for k, v in w.items() if v.ndim == 2 and k.split(".")[-2] in ("c_attn", "c_proj", "c_fc"))
    assert model.weight_bytes < full.weight_bytes
    if name == "tiny_a":
        assert full.weight_bytes - model.weight_bytes >= matrices * 2 * 0.4        # (padding to 128 takes some of it)


class PlainOps:
    """The kernels' 8-bit norm and 4-bit product in plain torch, put in their place: a model's other launches stay."""

    def __init__(self, monkeypatch):
        self.norms = self.products = 0
        monkeypatch.setattr(ops, "residual_add_norm_q8", self.norm)
        monkeypatch.setattr(ops, "linear_q4", self.linear)

    @staticmethod
    def rows(h):
        return ops.quantize_q8(h.float().contiguous())

    def norm(self, x, y, mult, weight, eps, y2=None, mult2=0.0, scale=None):
        self.norms += 1
        if y is not None:
            add = mult * y + (mult2 * y2 if y2 is not None else 0.0)
            x += add * scale if scale is not None else add
        h = x.double() / torch.sqrt((x.double() ** 2).mean(dim=1, keepdim=True) + eps) * weight.double()
        return self.rows(h)

    def linear(self, x, weight, bias=None, act=None, residual=None, out=None, out_dtype=None, way=0):
        self.products += 1
        codes, scales = weight
        table = torch.tensor([0, .5, 1, 1.5, 2, 3, 4, 6], device=codes.device)
        c = torch.stack((codes & 15, codes >> 4), dim=2).flatten(1).long()
        w = table[c % 8] * torch.where(c >= 8, -1.0, 1.0)
        e = scales.view(torch.uint8).permute(0, 3, 2, 1, 4).reshape(-1, w.shape[1] // 32)[:w.shape[0]]
        w = (w.unflatten(1, (-1, 32)) * torch.exp2(e.float() - 127)[..., None]).flatten(1).double()
        rows = ops.q8_values(x).double() if isinstance(x, ops.Q8Rows) else x.double()
        z = rows @ w[:, :rows.shape[1]].t()
        if bias is not None:
            z = z + bias
        if act == "gelu_new":
            z = 0.5 * z * (1 + torch.tanh(np.sqrt(2 / np.pi) * (z + 0.044715 * z ** 3)))
        elif act == "gelu":
            z = 0.5 * z * (1 + torch.erf(z / np.sqrt(2)))
        elif act == "relu2":
            z = z.clamp(min=0) ** 2
        else:
            assert act in (None, "none")
        if residual is not None:
            z = z + residual
        if out is None:
            return z.to(out_dtype or torch.bfloat16)
        return out.copy_(z)


@pytest.fixture(scope="module")
def seledra_dirs(tmp_path_factory):
    out = {}
    for name, cfg in seledra.CONFIGS.items():
        d = tmp_path_factory.mktemp("seledra_" + name)
        (d / "config.json").write_text(json.dumps(cfg))
        seledra.write_safetensors(str(d / "model.safetensors"), {k: torch.from_numpy(np.array(v)).to(torch.bfloat16)
                                                                 for k, v in seledra.weights_of(name).items()})
        out[name] = str(d)
    return out


@gpu
@pytest.mark.parametrize("name", ["a", "b", "c"])
@pytest.mark.parametrize("row_bits", [16, 8])
def test_a_model_of_norms_in_8_bits(name, row_bits, seledra_dirs, monkeypatch):
    """Attention, recurrences and feed-forwards whose rows come from the norm that adds to the stream: the model against
    itself with the norm and the products in plain torch, everything else as it is; prompts, single tokens, a batch."""
    model = DecoderModel.from_dir(seledra_dirs[name], weight_bits=4, row_bits=row_bits)
    vocab = seledra.CONFIGS[name]["vocab"]
    cache = model.new_cache(max_tokens=4 * 192, n_slots=4)
    toks = tokens_for(vocab, 150, 3)
    requests = [tokens_for(vocab, n, 40 + n) for n in (20, 90, 3)]

    def all_ways():
        whole = run_whole(model, cache, toks)
        tail = run_tail_one_by_one(model, cache, toks[:60], 20)
        batch = np.concatenate(run_batch(model, cache, requests, [17, 70, 1]))
        return whole, tail, batch

    got = all_ways()
    ops.check_status()
    with monkeypatch.context() as patch:
        stand_in = PlainOps(patch)
        want = all_ways()
    assert stand_in.products > 0 and (stand_in.norms > 0) == (row_bits == 8)
    # an entry that lies at an edge between two 8-bit codes goes to the other one where the stream before it differs in a
    # last bit: half a step of e4m3 is 2^-4 of one entry in hundreds, as noise no more than the bfloat16 path's own
    for g, w, what in zip(got, want, ("whole", "tail", "batch")):
        check_logits(g, w, "bfloat16", f"seledra {name} {what}", bf16_rms=seledra.BF16_RMS[name] * (1.5 if row_bits == 8 else 1.0))


class CheckedOps(PlainOps):
    """The kernels themselves, each product and each norm compared with plain torch on the same inputs."""

    def __init__(self, monkeypatch):
        self.kernels = ops.residual_add_norm_q8, ops.linear_q4
        super().__init__(monkeypatch)

    def norm(self, x, y, mult, weight, eps, y2=None, mult2=0.0, scale=None):
        before = x.clone()
        rows = self.kernels[0](x, y, mult, weight, eps, y2=y2, mult2=mult2, scale=scale)
        want = super().norm(before, y, mult, weight, eps, y2=y2, mult2=mult2, scale=scale)
        assert torch.allclose(x, before, rtol=1e-5, atol=1e-6)
        got, want = ops.q8_values(rows), ops.q8_values(want)
        # a whole step of e4m3 where an entry lies at an edge between two codes, and for a group's small ones at that of its largest
        top = want.unflatten(1, (-1, 32)).abs().amax(dim=2, keepdim=True).expand(-1, -1, 32).flatten(1)
        assert ((got - want).abs() <= 2.0 ** -3 * want.abs() + 2.0 ** -15 * top).all()
        return rows

    def linear(self, x, weight, bias=None, act=None, residual=None, out=None, out_dtype=None, way=0):
        given = x.materialize_copy() if isinstance(x, ops.NormedInput) else x
        res = None if residual is None else residual.clone()
        got = self.kernels[1](x, weight, bias, act=act, residual=residual, out=out, out_dtype=out_dtype)
        want = super().linear(given, weight, bias, act, res, None, torch.float64)
        # half a step of bfloat16 of the answer and of the row's largest sum's own errors
        assert torch.isfinite(got).all()
        assert ((got.double() - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -10 * want.abs().amax(dim=1, keepdim=True)).all()
        return got


FAMILIES = {"forisun": forisun, "lusalorn": lusalorn, "pelenex": pelenex, "seledra": seledra, "tibopel": tibopel, "tokolorn": tokolorn}


@gpu
@pytest.mark.parametrize("name", ["a", "b", "c"])
@pytest.mark.parametrize("family", FAMILIES)
def test_every_design_with_4_bit_matrices(family, name, tmp_path, monkeypatch):
    """What each mixer and feed-forward hands to the products and takes from the norm, in a prompt, a batch and single tokens."""
    d = write_random_model(str(tmp_path), FAMILIES[family].CONFIGS[name], seed=5)
    for row_bits in (16, 8):
        model = DecoderModel.from_dir(d, weight_bits=4, row_bits=row_bits)
        cache = model.new_cache(max_tokens=4 * 192, n_slots=4)
        with monkeypatch.context() as patch:
            checked = CheckedOps(patch)
            whole = run_whole(model, cache, tokens_for(model.vocab_size, 70, 3))
            run_tail_one_by_one(model, cache, tokens_for(model.vocab_size, 24, 4), 6)
            run_batch(model, cache, [tokens_for(model.vocab_size, n, n) for n in (20, 40, 3)], [17, 36, 1])
        assert checked.products > 0 and np.isfinite(whole).all()
        ops.check_status()


@gpu
def test_4_bit_single_token_steps_from_graphs(model_dirs):
    """Generation replays recorded steps: the same tokens as steps run one by one."""
    from math_utils_b200.engine.generate import generate
    model = DecoderModel.from_dir(model_dirs["tiny_a"], weight_bits=4, row_bits=8)
    prompts = [tokens_for(512, n, n) for n in (3, 17, 40)]
    for params in (SamplingParams(0.0, 0, 0), SamplingParams(0.9, 20, 7)):
        a = generate(model, prompts, 30, params, stop_ids=[])
        b = generate(model, prompts, 30, params, stop_ids=[], use_graph=False)
        assert a == b and all(len(x) == 30 for x in a)


def test_refused_combinations():
    for args, words in (((torch.float32, "cpu", 4), "bfloat16"), (("bfloat16", "cpu", 8), "16 or 4"), (("bfloat16", "cpu", 4, 4), "16 or 8"),
                        (("bfloat16", "cpu", 16, 8), "4-bit weights")):
        with pytest.raises(ValueError, match=words):
            Runtime.create(*args)
    with pytest.raises(ValueError, match="drafted tokens"):
        LLM(options=Options(drafts=2, dtype="float32")).use("/nowhere")
    with pytest.raises(ValueError, match="drafted tokens"):
        LLM(options=Options(drafts=-1)).use("/nowhere")


@pytest.mark.parametrize("error", [RuntimeError, MemoryError, ValueError])
def test_a_draft_that_cannot_be_loaded_leaves_no_model(monkeypatch, error):
    """Whatever ends the load of the draft, the model does not stay behind to answer without drafts."""
    from math_utils_b200 import llm as module
    loads = []

    class Models:
        @staticmethod
        def from_dir(folder, **how):
            loads.append(how["weight_bits"])
            if len(loads) == 2:
                raise error("no room")
            return object()

    monkeypatch.setattr(module, "DecoderModel", Models)
    llm = LLM(options=Options(drafts=2))
    with pytest.raises(error, match="no room"):
        llm.use("/nowhere")
    assert loads == [16, 4] and not llm.loaded and llm.draft is None
    with pytest.raises(RuntimeError, match="no model loaded"):
        llm.generate([[1, 2]])


def test_a_model_in_4_bits_is_its_own_draft(monkeypatch):
    """Its draft would hold the same numbers: it is loaded once."""
    from math_utils_b200 import llm as module
    from math_utils_b200.engine import drafted
    loads = []

    class Models:
        @staticmethod
        def from_dir(folder, **how):
            loads.append((how["weight_bits"], how["row_bits"]))
            return Models()

        def new_cache(self, *a):
            return None

    monkeypatch.setattr(module, "DecoderModel", Models)
    monkeypatch.setattr(drafted, "check_draftable", lambda *a: None)
    llm = LLM(options=Options(drafts=2, weight_bits=4, row_bits=8)).use("/nowhere")
    assert loads == [(4, 8)] and llm.draft is llm.model
    llm.use("/nowhere", Options(drafts=2))
    assert loads[1:] == [(16, 16), (4, 16)] and llm.draft is not llm.model


# ------------------------------------------------------------------------------------------------ drafted tokens
def test_rooms_and_draws():
    class Model:
        max_positions = 100
    assert room_for_drafts(Model, Model, [10, 95], 4, 80) == 0          # past the context: one token at a time
    assert room_for_drafts(Model, Model, [10, 75], 4, 80) == 4
    assert room_for_drafts(Model, Model, [10, 77], 4, 80) == 2
    assert room_for_drafts(Model, Model, [10, 79], 4, 80) == 0
    for request in (0, 3, 1 << 40):
        want = [plain_gpt2.uniform_draw(11, request, n) for n in range(4, 9)]
        assert uniform_draws(11, request, 4, 5).tolist() == want


def greedy_or_near_tie(model, prompt, produced):
    """Every produced token is the largest logit of the model itself over the whole sequence, or as near as the bfloat16
    path's noise can bridge (steps of one and of several tokens go through other kernels)."""
    cache = model.new_cache(max_tokens=256, n_slots=1)
    logits = run_whole(model, cache, list(prompt) + produced)[len(prompt) - 1:-1]
    for row, token in zip(logits, produced):
        assert row.max() - row[token] <= BF16_NEAR_TIE * row.std()


@gpu
@pytest.mark.parametrize("name,drafts", [("tiny_a", 1), ("tiny_a", 4), ("tiny_b", 3)])
def test_greedy_drafts_give_the_models_own_tokens(name, drafts, model_dirs, plain_models):
    cfg, _ = plain_models[name]
    llm = LLM(model_dirs[name], Options(temperature=0.0, drafts=drafts, max_batch=3))
    prompts = [tokens_for(cfg["vocab_size"], n, n) for n in (1, 9, 40, 63, 5)]
    out = llm.generate(prompts, max_tokens=40, stop_ids=[])
    for p, o in zip(prompts, out):
        assert len(o) == min(40, llm.context - len(p))
        greedy_or_near_tie(llm.model, p, o)
    counts = llm.draft_counts
    assert 0 < counts["kept"] <= counts["drafted"]
    # a draft that is the model itself is right but for near ties
    model = llm.model
    counts = {}
    generate_drafted(model, model, prompts[:3], 24, SamplingParams(0.0, 0, 0), drafts, stop_ids=[], counts=counts)
    assert counts["kept"] >= 0.9 * counts["drafted"]


@gpu
def test_drafted_samples_depend_on_seed_alone(model_dirs):
    llm = LLM(model_dirs["tiny_a"], Options(temperature=0.9, top_k=30, seed=5, drafts=3))
    prompts = [tokens_for(512, n, n) for n in (4, 30, 11)]
    first = llm.generate(prompts, max_tokens=30, stop_ids=[])
    assert llm.generate(prompts, max_tokens=30, stop_ids=[]) == first
    assert llm.generate(prompts, max_tokens=30, stop_ids=[], seed=6) != first
    assert all(len(x) == 30 for x in first) and all(0 <= t < 512 for x in first for t in x)
    everything = llm.generate(prompts, max_tokens=12, stop_ids=[], top_k=-1)
    assert all(len(x) == 12 for x in everything)


@gpu
def test_drafted_generation_keeps_its_caches_and_graphs(model_dirs, monkeypatch):
    """Call after call on one pair of caches and the same recordings; a batch that thins out one by one moves to a smaller graph only where
    it has halved; larger calls take the place of what was held, and nothing else keeps it."""
    import gc
    import weakref
    from math_utils_b200.engine.decode_session import DecodeSession
    recorded = []
    record = DecodeSession._record_graph
    monkeypatch.setattr(DecodeSession, "_record_graph", lambda self, *a: recorded.append(self.n) or record(self, *a))
    llm = LLM(model_dirs["tiny_b"], Options(temperature=0.0, drafts=3, max_batch=16))            # 80 positions
    thinning = [tokens_for(1031, 48 + 2 * i, i) for i in range(16)]
    first = llm.generate(thinning, max_tokens=60, stop_ids=[])
    assert [len(o) for o in first] == [32 - 2 * i for i in range(16)]
    assert len(recorded) <= 5 and recorded[0] == 16 and all(b * 2 <= a for a, b in zip(recorded, recorded[1:]))
    pair = llm._batch_cache, llm._draft_batch_cache
    held, n = None, len(recorded)
    for _ in range(4):
        assert llm.generate(thinning, max_tokens=60, stop_ids=[]) == first
        assert (llm._batch_cache, llm._draft_batch_cache) == pair and len(recorded) == n
        gc.collect()
        torch.cuda.synchronize()
        now = torch.cuda.memory_allocated()
        assert held is None or now - held <= 2 ** 20
        held = now
    for c in pair:
        assert c.slots.n_free == 16 and c.free_pages(0) == c.n_pages
    old = [weakref.ref(c) for c in pair]
    del pair, c
    llm.options = Options(temperature=0.0, drafts=3, max_batch=24)
    assert len(llm.generate([thinning[0]] * 24, max_tokens=4, stop_ids=[])) == 24
    gc.collect()
    assert all(r() is None for r in old)
    sessions = dict(llm.draft.__dict__["_decode_sessions"])
    assert [len(o) for o in generate_drafted(llm.model, llm.draft, thinning[:2], 4, SamplingParams(0.0, 0, 0), 3, stop_ids=[])] == [4, 4]
    assert dict(llm.draft.__dict__["_decode_sessions"]) == sessions


@gpu
def test_the_first_drafted_tokens_are_distributed_as_the_models(model_dirs):
    """The second token of 2,048 requests with one prompt, given the commonest first token: frequencies of the four likeliest
    against the model's own softmax, within 5 standard deviations of a binomial count."""
    llm = LLM(model_dirs["tiny_a"], Options(temperature=1.0, top_k=8, seed=3, drafts=2, max_batch=64))
    prompt = tokens_for(512, 12, 2)
    out = llm.generate([prompt] * 2048, max_tokens=3, stop_ids=[])
    firsts = np.array([o[0] for o in out])
    common = np.bincount(firsts).argmax()
    seconds = np.array([o[1] for o in out if o[0] == common])
    cache = llm.model.new_cache(max_tokens=64, n_slots=1)
    row = run_whole(llm.model, cache, prompt + [int(common)])[-1]
    p = plain.softmax_kept(row, 1.0, 8)
    n = len(seconds)
    assert n >= 200
    for t in np.argsort(-p)[:4]:
        # (the bfloat16 path's logits differ by a hundredth of their spread between steps of one and of several tokens)
        slack = 5 * np.sqrt(n * p[t] * (1 - p[t])) + n * p[t] * BF16_NEAR_TIE * row.std()
        assert abs((seconds == t).sum() - n * p[t]) <= slack


@gpu
def test_drafted_requests_end_as_others_do(model_dirs):
    """Stop tokens among drafts, the context's end, one token, none; a batch that thins out."""
    folder = model_dirs["tiny_b"]                               # 80 positions
    llm = LLM(folder, Options(temperature=0.0, drafts=4))
    prompts = [tokens_for(1031, n, n) for n in (2, 30, 75, 79, 80)]
    free = llm.generate(prompts, max_tokens=60, stop_ids=[])
    assert [len(x) for x in free] == [60, 50, 5, 1, 0]
    stop = sorted({free[0][7], free[1][2]})
    got = llm.generate(prompts, max_tokens=60, stop_ids=stop)
    for f, g in zip(free, got):
        at = min([f.index(s) for s in stop if s in f] + [len(f)])
        assert g == f[:at]
    assert llm.generate(prompts[:2], max_tokens=1, stop_ids=[]) == [free[0][:1], free[1][:1]]
    assert llm.generate(prompts[:2], max_tokens=0, stop_ids=[]) == [[], []]


@gpu
def test_a_drafted_conversation_keeps_both_caches(model_dirs):
    llm = LLM(model_dirs["tiny_a"], Options(temperature=0.0, drafts=3, context=128))
    plain_llm = LLM(model_dirs["tiny_a"], Options(temperature=0.0, context=128))
    said, held = [], 0
    for turn, n in enumerate((5, 9, 1)):
        ids = tokens_for(512, n, turn)
        answer = llm.prompt(ids, max_tokens=11)
        assert len(answer) <= 11
        greedy_or_near_tie(plain_llm.model, said + ids, answer)
        said += ids + answer
        held = len(said)
        assert llm._cache.length(llm._slot) == llm._draft_cache.length(llm._draft_slot) == held == llm.last["context_used"]
    llm.reset()
    assert llm.prompt([3, 4, 5], max_tokens=4) == LLM(model_dirs["tiny_a"], Options(temperature=0.0, drafts=3, context=128)).prompt([3, 4, 5], max_tokens=4)


@gpu
def test_drafts_of_a_latent_attention_model(tmp_path):
    """Caches of one row a position are cut back too."""
    d = write_random_model(str(tmp_path), forisun.CONFIGS["a"], seed=2)
    llm = LLM(d, Options(temperature=0.0, drafts=3))
    prompt = tokens_for(llm.model.vocab_size, 20, 1)
    out = llm.generate([prompt], max_tokens=20, stop_ids=[])[0]
    assert len(out) == 20
    greedy_or_near_tie(llm.model, prompt, out)


@gpu
def test_models_that_cannot_draft_are_refused(seledra_dirs, model_dirs):
    with pytest.raises(ValueError, match="cut back"):
        LLM(seledra_dirs["a"], Options(drafts=2))
    a, b = (DecoderModel.from_dir(model_dirs[n]) for n in ("tiny_a", "tiny_b"))
    with pytest.raises(ValueError, match="vocabulary"):
        generate_drafted(a, b, [[1, 2]], 4, SamplingParams(), 2)
    with pytest.raises(ValueError, match="at least one"):
        generate_drafted(a, a, [[1, 2]], 4, SamplingParams(), 0)


@gpu
def test_the_command_line_drafts(model_dirs, capsys):
    from math_utils_b200.cli import main
    assert main([model_dirs["tiny_a"], "--prompt", "1 2 3", "--tokens", "6", "--temp", "0", "--drafts", "2"]) == 0
    drafted = capsys.readouterr().out.split()
    assert len(drafted) <= 6 and all(t.isdigit() for t in drafted)
    assert main([model_dirs["tiny_a"], "--prompt", "1 2 3", "--tokens", "6", "--temp", "0", "--q4", "--rows8"]) == 0
    assert capsys.readouterr().out.strip()


def test_the_command_line_refuses(capsys):
    from math_utils_b200.cli import main
    for flags in (["--rows8"], ["--q4", "--fp32"], ["--drafts", "2", "--fp32"], ["--drafts", "2", "--profile"]):
        assert main(["nowhere", *flags]) == 1
        assert "--rows8 goes with --q4" in capsys.readouterr().err
