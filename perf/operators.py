"""Cases for timing the operators of answering with 4-bit weights, with their plain forms and their results in 64 bits.

Four operators that a quantised model's step is made of, and the one that lets such a model draft for another:

``product16``  act(x W^T + bias) (+ residual): bfloat16 rows, weights in 4 bits with a scale for every 32 along k
``product8``   the same with rows in 8 bits with a scale for every 32
``norm8``      x += mult * y on the float32 stream, then the normed row in 8 bits with a scale for every 32
``verify``     which drafted tokens the target's distribution takes, and the token that follows them

Formats.  Weights: codes [n, kp / 2] uint8, kp = k rounded up to 128, the code of an even column in the low half of its
byte; a code is a sign bit and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6.  Rows: codes [m, kp] float8_e4m3fn.  Scales of both are
powers of two (float8_e8m0fnu) laid out as [tiles of 128 rows, kp / 128, 32, 4, 4]: row r of a tile at [r % 32, r // 32],
its four groups of 32 columns last.  Columns from k on are zeros.

Sizes are those of GPT-2 medium and XL (width 1,024 and 1,600, inner width 4,096 and 6,400), of the benchmark's families
at size m (width 2,048, inner width 5,632), and generic ones for the largest calls.
"""
import math

import torch
import torch.nn.functional as F

own = False

DEVICE = "cuda:0"
EPS = 1e-5
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


# ---------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one token of a conversation through the first feed-forward product (GPT-2 XL): the smallest call
        {"name": "up_single", "op": "product16", "m": 1, "n": 6400, "k": 1600, "bias": True, "act": "gelu_new", "residual": False},
        # one token for each of eight conversations through the second one, added to the float32 stream: long k, few columns
        {"name": "down_single_b8", "op": "product16", "m": 8, "n": 1600, "k": 6400, "bias": True, "act": "none", "residual": True},
        # a full batch of single tokens through a gate and up projection (size m)
        {"name": "gate_up_single_b48", "op": "product16", "m": 48, "n": 11264, "k": 2048, "bias": False, "act": "none", "residual": False},
        # two whole prompts through the first feed-forward product (GPT-2 medium)
        {"name": "up_prompt_2x1024", "op": "product16", "m": 2048, "n": 4096, "k": 1024, "bias": True, "act": "gelu_new", "residual": False},
        # eight single tokens, normed rows in 8 bits, through the mixer's projections (size m)
        {"name": "proj_single_b8_rows8", "op": "product8", "m": 8, "n": 4096, "k": 2048, "bias": False, "act": "none", "residual": False},
        # an odd number of prompt tokens through the fused q | k | v projection (GPT-2 XL)
        {"name": "qkv_prompt_777_rows8", "op": "product8", "m": 777, "n": 4800, "k": 1600, "bias": True, "act": "none", "residual": False},
        # a long prompt through a wide model's feed-forward: the largest product
        {"name": "up_prompt_4096_rows8", "op": "product8", "m": 4096, "n": 16384, "k": 4096, "bias": False, "act": "none", "residual": False},
        # the norm between two sublayers of a single-token step (size m)
        {"name": "norm_single_b8", "op": "norm8", "m": 8, "k": 2048, "mult": 0.5},
        # the same over an odd number of prompt tokens, a width that is no multiple of 128 (GPT-2 XL)
        {"name": "norm_prompt_777", "op": "norm8", "m": 777, "k": 1600, "mult": 1.0},
        # a long prompt step of a wide model
        {"name": "norm_prompt_4096", "op": "norm8", "m": 4096, "k": 8192, "mult": 0.25},
        # four drafted tokens in each of eight conversations, at the library's default temperature and top-k
        {"name": "verify_b8_top40", "op": "verify", "batch": 8, "drafts": 4, "vocab": 50257, "temperature": 0.7, "top_k": 40},
        # a full batch, the whole vocabulary kept
        {"name": "verify_b64_all", "op": "verify", "batch": 64, "drafts": 5, "vocab": 50257, "temperature": 1.0, "top_k": 0},
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _size(rng, low, high, unit):
    """A size from the range, a multiple of ``unit`` three times out of four and any number otherwise."""
    n = _spread(rng, low, high)
    return n if rng.random() < 0.25 else max(unit, n // unit * unit)


def draw(rng):
    op = rng.choice(["product16", "product8", "norm8", "verify"])
    if op in ("product16", "product8"):
        residual = rng.random() < 0.4
        return {"op": op, "m": _spread(rng, 1, 4096), "n": _size(rng, 200, 12000, 64), "k": _size(rng, 100, 6400, 64),
                "bias": rng.random() < 0.5, "act": "none" if residual else rng.choice(["none", "gelu_new", "gelu", "relu2"]),
                "residual": residual}
    if op == "norm8":
        return {"op": op, "m": _spread(rng, 1, 4096), "k": _size(rng, 100, 8192, 64), "mult": round(rng.uniform(0.1, 1.5), 3)}
    return {"op": op, "batch": _spread(rng, 1, 64), "drafts": rng.randint(1, 5), "vocab": _spread(rng, 500, 50257),
            "temperature": rng.choice([0.0, 0.3, 0.7, 1.0, 1.3]), "top_k": rng.choice([-1, 0, 5, 40, 200])}


# ---------------------------------------------------------------------------------------------------- layouts
def _tiles(s):
    """Scale bytes [rows, groups] (groups a multiple of four) -> the layout of the formats above."""
    rows, groups = s.shape
    s = F.pad(s, (0, 0, 0, -rows % 128))
    return s.view(-1, 4, 32, groups // 4, 4).permute(0, 3, 2, 1, 4).contiguous().view(torch.float8_e8m0fnu)


def _untiled(s, rows):
    """The layout's scales as float32 [rows, groups]."""
    t, kb = s.shape[:2]
    e = s.view(torch.uint8).permute(0, 3, 2, 1, 4).reshape(t * 128, kb * 4)[:rows]
    return torch.exp2(e.float() - 127.0)


def _exponent(top, most):
    """The smallest e with top <= most * 2^e (0 where top is 0), as a byte with a bias of 127."""
    mantissa, exp = torch.frexp(top)
    m, e = math.frexp(most)
    e = exp - e + (mantissa > m).to(exp.dtype)
    return torch.where(top > 0, (e + 127).clamp(0, 254), torch.zeros_like(e)).to(torch.uint8)


def _scaled_groups(x, most):
    """Rows [m, k] padded to whole 128s as groups [m, groups, 32], and each group's scale byte."""
    g = F.pad(x, (0, -x.shape[1] % 128)).unflatten(1, (-1, 32))
    return g, _exponent(g.abs().amax(dim=2), most)


def _weights(n, k, gen):
    """A weight matrix of normal numbers in 4 bits: (codes, scales)."""
    w = torch.randn((n, k), generator=gen, device=DEVICE) * 0.02
    g, e = _scaled_groups(w, 6.0)
    v = g * torch.exp2(127.0 - e.float())[..., None]
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=DEVICE)
    code = torch.bucketize(v.abs(), edges) + 8 * (v < 0)
    code = code.flatten(1).to(torch.uint8)
    return (code[:, 0::2] | code[:, 1::2] << 4).contiguous(), _tiles(e)


def _rows8(x):
    g, e = _scaled_groups(x, 448.0)
    return (g * torch.exp2(127.0 - e.float())[..., None]).flatten(1).to(torch.float8_e4m3fn), _tiles(e)


# ---------------------------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=DEVICE)      # noqa: E731
    s = {"case": case}
    op = case["op"]
    if op in ("product16", "product8"):
        m, n, k = case["m"], case["n"], case["k"]
        x = normal(m, k)
        x[:, :: 61] *= 12.0                                 # the few wide channels of a model's activations
        s["x"] = x.bfloat16() if op == "product16" else _rows8(x)
        s["w"] = _weights(n, k, gen)
        s["bias"] = normal(n) * 0.1 if case["bias"] else None
        s["residual"] = normal(m, n) if case["residual"] else None
    elif op == "norm8":
        m, k = case["m"], case["k"]
        s["x"], s["y"] = normal(m, k) * 2.0, normal(m, k)
        s["y"][:, :: 61] *= 12.0
        s["weight"] = 1.0 + 0.1 * normal(k)
    else:
        b, g, v = case["batch"], case["drafts"], case["vocab"]
        s["logits"] = normal(b, g + 1, v) * 2.5
        # a draft model near the target, as one of the same weights in fewer bits is
        s["draft_logits"] = s["logits"][:, :g] + 0.6 * normal(b, g, v)
        s["draws"] = torch.rand((b, g + 1), generator=gen, device=DEVICE, dtype=torch.float64)
        if _greedy(case):
            s["drafts"] = s["draft_logits"].argmax(dim=2).int()
        else:
            q = _distribution(s["draft_logits"], case["temperature"], case["top_k"])
            pick = torch.rand((b, g, 1), generator=gen, device=DEVICE, dtype=torch.float64)
            s["drafts"] = _walk(q, pick).int()
    return s


# ---------------------------------------------------------------------------------------------------- one pass
def _ops():
    from math_utils_b200.csrc import ops
    return ops


def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        ops = _ops()
        if op == "product16":
            out_dtype = torch.float32 if case["residual"] else torch.bfloat16
            return ops.linear_q4(state["x"], ops.Q4Weight(*state["w"]), bias=state["bias"], act=case["act"],
                                 residual=state["residual"], out_dtype=out_dtype)
        if op == "product8":
            out_dtype = torch.float32 if case["residual"] else torch.bfloat16
            return ops.linear_q4(ops.Q8Rows(*state["x"]), ops.Q4Weight(*state["w"]), bias=state["bias"], act=case["act"],
                                 residual=state["residual"], out_dtype=out_dtype)
        if op == "norm8":
            rows = ops.residual_add_norm_q8(state["x"], state["y"], case["mult"], state["weight"], EPS)
            return [state["x"], rows.codes, rows.scales]
        return list(ops.verify_drafts(state["logits"], state["draft_logits"], state["drafts"], state["draws"],
                                      case["temperature"], case["top_k"]))
    if op in ("product16", "product8"):
        return _plain_product(state, case)
    if op == "norm8":
        return _plain_norm(state, case)
    return _plain_verify(state, case)


def _activation(z, act):
    if act == "gelu_new":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z / math.sqrt(2.0)))
    return torch.relu(z) ** 2 if act == "relu2" else z


def _plain_product(state, case):
    codes, scales = state["w"]
    table = torch.tensor(MAGNITUDES + tuple(-v for v in MAGNITUDES), device=DEVICE)
    w = table[torch.stack((codes & 15, codes >> 4), dim=2).int()].flatten(1)
    w = (w.unflatten(1, (-1, 32)) * _untiled(scales, w.shape[0])[..., None]).flatten(1)
    if case["op"] == "product8":
        x = (state["x"][0].float().unflatten(1, (-1, 32)) * _untiled(state["x"][1], case["m"])[..., None]).flatten(1)
    else:
        x, w = state["x"].float(), w[:, :case["k"]]
    z = x @ w.t()
    if state["bias"] is not None:
        z = z + state["bias"]
    z = _activation(z, case["act"])
    return z + state["residual"] if case["residual"] else z.bfloat16()


def _plain_norm(state, case):
    x = state["x"]
    x += case["mult"] * state["y"]
    h = x * torch.rsqrt((x * x).mean(dim=1, keepdim=True) + EPS) * state["weight"]
    return [x, *_rows8(h)]


def _greedy(case):
    return case["temperature"] <= 0.0 or 0 < case["top_k"] <= 1


def _distribution(logits, temperature, top_k):
    """Softmax at the temperature over the ``top_k`` largest logits (ties: the lowest index first), in 64 bits."""
    z = logits.double()
    p = torch.exp((z - z.amax(dim=-1, keepdim=True)) / temperature)
    if 0 < top_k < logits.shape[-1]:
        at = torch.sort(logits, dim=-1, descending=True, stable=True).indices[..., :top_k]
        p = torch.zeros_like(p).scatter(-1, at, p.gather(-1, at))
    return p / p.sum(dim=-1, keepdim=True)


def _walk(p, pick):
    """The first token at which the running sum of the masses ``p``, in the order of the vocabulary, passes pick of it all."""
    run_ = p.cumsum(dim=-1)
    passed = (run_ > pick * run_[..., -1:]) & (p > 0)
    return passed.byte().argmax(dim=-1)


def _plain_verify(state, case):
    logits, drafts = state["logits"], state["drafts"].long()
    b, g = drafts.shape
    if _greedy(case):
        best = logits.argmax(dim=2)
        taken = best[:, :g] == drafts
        then = None
    else:
        p = _distribution(logits, case["temperature"], case["top_k"])
        q = _distribution(state["draft_logits"], case["temperature"], case["top_k"])
        px, qx = (t[:, :g].gather(2, drafts[..., None])[..., 0] for t in (p, q))
        taken = state["draws"][:, :g] * qx < px
    kept = taken.long().cumprod(dim=1).sum(dim=1)
    if _greedy(case):
        then = best.gather(1, kept[:, None])[:, 0]
    else:
        row = kept[:, None, None].expand(-1, 1, p.shape[2])
        at, other = p.gather(1, row)[:, 0], F.pad(q, (0, 0, 0, 1)).gather(1, row)[:, 0]
        rest = torch.relu(at - other)
        rest = torch.where(rest.sum(dim=1, keepdim=True) > 0, rest, at)
        then = _walk(rest, state["draws"][:, g:])
    place = torch.arange(g + 1, device=DEVICE)
    tokens = torch.where(place < kept[:, None], F.pad(drafts, (0, 1)), torch.where(place == kept[:, None], then[:, None], -1))
    return [tokens.int(), kept.int()]


# ---------------------------------------------------------------------------------------------------- work and values
def work(case):
    op = case["op"]
    if op in ("product16", "product8"):
        m, n, k = case["m"], case["n"], case["k"]
        row = 2.0 * k if op == "product16" else k + k / 32.0
        out = 8.0 if case["residual"] else 2.0
        return {"bytes": n * k * (0.5 + 1.0 / 32.0) + m * row + m * n * out + 4.0 * n * case["bias"], "flops": 2.0 * m * n * k}
    if op == "norm8":
        m, k = case["m"], case["k"]
        return {"bytes": m * k * (13.0 + 1.0 / 32.0) + 4.0 * k, "flops": 8.0 * m * k}
    b, g, v = case["batch"], case["drafts"], case["vocab"]
    rows = g + 1 if _greedy(case) else 2 * g + 1
    return {"bytes": b * (4.0 * rows * v + 16.0 * g), "flops": 4.0 * b * rows * v}


def _values(codes_of, scales, rows):
    """What codes with scales stand for, in 64 bits; ``codes_of``: the codes' values [rows, kp]."""
    t, kb = scales.shape[:2]
    byte = scales.view(torch.uint8).double()
    out = torch.empty((rows, kb * 128), dtype=torch.float64, device=DEVICE)
    for block in range(4):
        for group in range(4):
            s = torch.pow(2.0, byte[:, :, :, block, group] - 127.0).permute(0, 2, 1)           # [tile, 32, kb]
            for tile in range(t):
                first = tile * 128 + block * 32
                n = min(32, rows - first)
                if n > 0:
                    at = codes_of[first:first + n].view(n, kb, 4, 32)[:, :, group].double()
                    out[first:first + n].view(n, kb, 4, 32)[:, :, group] = at * s[tile, :n, :, None]
    return out


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "verify":
        return None                                        # whole numbers alone
    if case["op"] == "norm8":
        return _exact_norm(state, case)
    codes, scales = state["w"]
    n, m, k = case["n"], case["m"], case["k"]
    both = torch.empty((n, codes.shape[1] * 2), dtype=torch.float64, device=DEVICE)
    for half in (0, 1):
        c = ((codes >> (4 * half)) & 15).double()
        low, exp = c % 2, torch.div(c, 2, rounding_mode="floor") % 4
        size = torch.where(exp == 0, low * 0.5, (1.0 + low * 0.5) * torch.pow(2.0, exp - 1.0))
        both[:, half::2] = torch.where(c >= 8, -size, size)
    w = _values(both, scales, n)[:, :k]
    x = _values(state["x"][0].double(), state["x"][1], m)[:, :k] if case["op"] == "product8" else state["x"].double()
    z = torch.matmul(x, w.transpose(0, 1))
    if state["bias"] is not None:
        z += state["bias"].double()
    if case["act"] == "gelu_new":
        z = z / (1.0 + torch.exp(-2.0 * 0.79788456080286535588 * (z + 0.044715 * z * z * z)))
    elif case["act"] == "gelu":
        z = z * 0.5 * torch.special.erfc(-z * 0.70710678118654752440)
    elif case["act"] == "relu2":
        z = torch.clamp(z, min=0.0).square()
    return z + state["residual"].double() if case["residual"] else z


def _exact_norm(state, case):
    x = state["x"].double() + case["mult"] * state["y"].double()
    h = x / torch.sqrt(x.square().sum(dim=1, keepdim=True) / case["k"] + EPS) * state["weight"].double()
    m, k = h.shape
    kp = -(-k // 128) * 128
    wide = torch.zeros((m, kp), dtype=torch.float64, device=DEVICE)
    wide[:, :k] = h
    groups = wide.view(m, kp // 32, 32)
    top = groups.abs().max(dim=2).values
    e = torch.ceil(torch.log2(top / 448.0))
    e = torch.where(top > 448.0 * torch.pow(2.0, e), e + 1.0, e)
    e = torch.where(top <= 448.0 * torch.pow(2.0, e - 1.0), e - 1.0, e)
    e = torch.where(top > 0, e.clamp(min=-127.0), torch.full_like(e, -127.0))
    v = groups / torch.pow(2.0, e)[..., None]
    step = torch.pow(2.0, torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6))) - 3.0)
    codes = torch.round(v / step) * step
    tiles = -(-m // 128)
    scales = torch.full((tiles * 128, kp // 32), 2.0 ** -127, dtype=torch.float64, device=DEVICE)
    scales[:m] = torch.pow(2.0, e)
    laid = torch.stack([scales.view(tiles, 4, 32, kp // 128, 4)[:, b] for b in range(4)], dim=2)       # [tile, 32, 4, kb, 4]
    return [x, codes.view(m, kp), laid.movedim(3, 1)]
