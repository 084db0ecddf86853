"""4-bit weights, 8-bit rows, their products, the norm that writes 8-bit rows and the verification of drafted tokens,
against plain statements in 64 bits (``plain_q4``)."""
import numpy as np
import pytest
import torch

import plain_q4 as plain
from math_utils_b200.csrc import ops
from math_utils_b200.csrc.ops import KernelError, Q4Weight, Q8Rows

gpu = pytest.mark.gpu
BF16_HALF = 2.0 ** -8               # half a step of bfloat16, relative
ACTS = {
    None: lambda z: z,
    "gelu_new": lambda z: 0.5 * z * (1.0 + np.tanh(np.sqrt(2.0 / np.pi) * (z + 0.044715 * z ** 3))),
    "gelu": lambda z: 0.5 * z * (1.0 + torch.erf(torch.from_numpy(z / np.sqrt(2.0))).numpy()),
    "relu2": lambda z: np.maximum(z, 0.0) ** 2,
}


def u8(t):
    return t.contiguous().view(torch.uint8).cpu().numpy()


def f64(t):
    return t.double().cpu().numpy()


def normal(shape, seed, scale=1.0, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def rough(shape, seed, dtype=torch.bfloat16):
    """Rows whose entries spread over many magnitudes, with zeros and a group of nothing else."""
    x = normal(shape, seed) * torch.exp2(torch.randint(-12, 6, shape, generator=torch.Generator().manual_seed(seed + 1)).float())
    x[:, ::7] = 0.0
    if shape[1] >= 64:
        x[:, 32:64] = 0.0
    return x.to(dtype)


# ------------------------------------------------------------------------------------------------ formats
@gpu
@pytest.mark.parametrize("m,k", [(1, 1), (1, 32), (3, 100), (130, 128), (5, 257), (257, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_in_eight_bits(m, k, dtype):
    x = rough((m, k), 3 * m + k, dtype)
    got = ops.quantize_q8(x.cuda())
    values, e = plain.q8_of(f64(x))
    assert np.array_equal(plain.scale_bytes(u8(got.scales), m) - 127.0, e)
    assert np.array_equal(plain.e4m3(u8(got.codes)), values)


@gpu
def test_rows_in_eight_bits_of_strided_and_unaligned_rows():
    x = rough((9, 300), 5)
    for view in (x.cuda()[:, 1:258], x.cuda()[::2, :200], x.cuda()[3:4, 5:8]):
        values, e = plain.q8_of(f64(view))
        got = ops.quantize_q8(view)
        assert np.array_equal(plain.e4m3(u8(got.codes)), values)
        assert np.array_equal(plain.scale_bytes(u8(got.scales), view.shape[0]) - 127.0, e)


@gpu
def test_rows_in_eight_bits_at_the_ends_of_the_range():
    x = torch.zeros(6, 64)
    x[0, :3] = torch.tensor([448.0, 449.0, -17.0])                # one step above what an exponent of 0 holds
    x[1, 0], x[1, 40] = 448.0, 3.0e38
    x[2, 0], x[2, 1] = 1.0e-38, 1.0e-45                           # subnormal numbers: the lowest exponent
    x[3, 3], x[3, 33] = float("inf"), 1.0
    x[4, 5], x[4, 6], x[4, 33] = float("nan"), 2.0, -2.0
    got = ops.quantize_q8(x.cuda())
    values = plain.q8_values(u8(got.codes), u8(got.scales))[:, :64]
    for row in (0, 1, 2, 5):
        want, e = plain.q8_of(f64(x[row:row + 1]))
        assert np.array_equal(values[row], (want.reshape(-1, 32) * 2.0 ** e.reshape(-1, 1)).reshape(-1)[:64])
    for row in (3, 4):                                            # a group with an infinity or NaN is NaN, its neighbours are not
        assert np.isnan(values[row, :32]).all() and np.isfinite(values[row, 32:]).all() and values[row, 33] != 0


@gpu
@pytest.mark.parametrize("n,k", [(1, 1), (3, 100), (128, 128), (130, 257), (300, 640)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_weights_in_four_bits(n, k, dtype):
    w = rough((n, k), n + k, dtype)
    got = ops.quantize_q4(w.cuda())
    groups = plain.groups_of(f64(w))
    values = plain.q4_values(u8(got.codes), u8(got.scales)).reshape(groups.shape)
    e = plain.scale_bytes(u8(got.scales), n) - 127.0
    top = plain.smallest_exponent(np.abs(groups).max(axis=2), 6.0)
    assert ((e == top) | (e == top - 1)).all()
    # the codes are the nearest at the scale taken
    assert np.array_equal(values, plain.round_e2m1(groups / 2.0 ** e[..., None]) * 2.0 ** e[..., None])
    # and of the two scales it is the one with the smaller squared error (sums of 32 squares in 32 bits: 64 roundings)
    err = lambda x: ((plain.round_e2m1(np.clip(groups / 2.0 ** x[..., None], -6, 6)) * 2.0 ** x[..., None] - groups) ** 2).sum(axis=2)
    best, other = err(top), err(np.maximum(top - 1, -127.0))
    slack = 64 * 2.0 ** -24 * np.maximum(best, other)
    assert (np.where(e == top, best <= other + slack, other <= best + slack)).all()


@gpu
def test_a_weight_that_is_no_number():
    w = torch.ones(4, 128)
    w[1, 40] = float("inf")
    w[2, 3] = float("nan")
    got = ops.quantize_q4(w.cuda())
    y = f64(ops.linear_q4(torch.ones(2, 128, dtype=torch.bfloat16, device="cuda"), got, out_dtype=torch.float32))
    assert np.isnan(y[:, 1:3]).all() and (y[:, [0, 3]] == 128.0).all()


# ------------------------------------------------------------------------------------------------ products
def product_bound(x, w, out_dtype, pieces):
    """What the sum of k products may be off by: its operands are exact (bfloat16 rows up to 2^-22 of their group's largest
    entry); a product of 32 along k adds to the float32 sum with a handful of roundings, 2^-23 of the largest partial sum
    each where the tensor cores cut instead of rounding, and up to 16 parts of k are added at the end."""
    size = np.abs(x) @ np.abs(w).T
    steps = pieces * w.shape[1] / 32
    off = (2 * steps + 40) * 2.0 ** -23 * size
    if pieces == 2:
        g = np.abs(plain.groups_of(x)).max(axis=2)
        off = off + 2.0 ** -22 * np.repeat(g, 32, axis=1)[:, :w.shape[1]] @ np.abs(w).T
    return off


def check_product(x_values, w_values, got, bias, act, residual, out_dtype, pieces):
    z = x_values @ w_values.T + (0.0 if bias is None else f64(bias))
    want = ACTS[act](z)
    off = product_bound(x_values, w_values, out_dtype, pieces) + 2.0 ** -23 * np.abs(z)
    if act == "relu2":
        off = 2.2 * np.abs(z) * off + off ** 2
    elif act is not None:
        off = 1.2 * off + 2.0 ** -19 * np.abs(z)                  # gelu's slope is at most 1.13; its own error a few 2^-22
    if residual is not None:
        want = want + f64(residual)
    off = off + 2.0 ** -23 * np.abs(want)
    if out_dtype == torch.bfloat16:
        off = off + BF16_HALF * (np.abs(want) + off)
    d = np.abs(f64(got) - want)
    assert got.dtype == out_dtype and np.isfinite(f64(got)).all()
    worst = np.unravel_index(np.argmax(d - off), d.shape)
    assert (d <= off + 1e-30).all(), f"at {worst}: {f64(got)[worst]} for {want[worst]}, {d[worst]:.3g} off, {off[worst]:.3g} allowed"


SHAPES = [(1, 1, 1), (1, 128, 128), (2, 100, 31), (16, 300, 200), (17, 129, 640), (33, 256, 1600), (64, 1000, 96),
          (65, 130, 384), (128, 128, 4224), (129, 520, 256), (257, 640, 128), (300, 1030, 900)]


@gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("rows", ["bfloat16", "eight"])
def test_products(m, n, k, rows):
    x, w = rough((m, k), m + n), normal((n, k), k, 0.05)
    weight = ops.quantize_q4(w.cuda())
    w_values = plain.q4_values(u8(weight.codes), u8(weight.scales))
    if rows == "eight":
        given = ops.quantize_q8(x.cuda())
        x_values, pieces = plain.q8_values(u8(given.codes), u8(given.scales)), 1
    else:
        given, x_values, pieces = x.cuda(), f64(x), 2
        w_values = w_values[:, :k]
    bias, residual = normal((n,), 7), normal((m, n), 8)
    for act, res, dtype in ((None, None, torch.bfloat16), (None, residual, torch.float32), ("gelu_new", None, torch.bfloat16),
                            ("gelu", residual, torch.float32), ("relu2", None, torch.float32)):
        b = bias if act != "relu2" else None
        got = ops.linear_q4(given, weight, bias=None if b is None else b.cuda(), act=act,
                            residual=None if res is None else res.cuda(), out_dtype=dtype)
        check_product(x_values, w_values, got, b, act, res, dtype, pieces)
    ops.check_status()


@gpu
@pytest.mark.parametrize("rows", ["bfloat16", "eight"])
@pytest.mark.parametrize("m", [1, 8, 12, 40, 64, 150, 300])
def test_products_by_every_way(m, rows):
    """Each kernel, however many blocks share a tile and however wide the tiles are, over several tiles and stages."""
    n, k = 700, 1300
    x, w = rough((m, k), m), normal((n, k), 2, 0.05)
    weight = ops.quantize_q4(w.cuda())
    w_values = plain.q4_values(u8(weight.codes), u8(weight.scales))
    if rows == "eight":
        given = ops.quantize_q8(x.cuda())
        x_values, pieces = plain.q8_values(u8(given.codes), u8(given.scales)), 1
    else:
        given, x_values, pieces, w_values = x.cuda(), f64(x), 2, w_values[:, :k]
    bias = normal((n,), 7)
    ways = [-64, -128, -192, -256] + ([1 + b for b in range(9)] if m <= 64 else [])
    for way in ways:
        got = ops.linear_q4(given, weight, bias=bias.cuda(), out_dtype=torch.float32, way=way)
        check_product(x_values, w_values, got, bias, None, None, torch.float32, pieces)
    ops.check_status()
    with pytest.raises(KernelError, match="bad argument"):
        ops.linear_q4(given, weight, way=-100)
    with pytest.raises(KernelError, match="bad argument" if m <= 64 else "unsupported"):
        ops.linear_q4(given, weight, way=10)


@gpu
@pytest.mark.parametrize("m", [1, 20, 200])
def test_products_into_views_and_into_their_residual(m):
    """Rows that lie apart, outputs that are columns of a wider buffer, the residual that is the output; what lies
    between the columns stays."""
    n, k = 200, 250
    wide = rough((m, 2 * k), 1).cuda()
    x, w = wide[:, 3:3 + k], normal((n, k), 2, 0.05)
    weight = ops.quantize_q4(w.cuda())
    w_values = plain.q4_values(u8(weight.codes), u8(weight.scales))[:, :k]
    buf = normal((m, n + 13), 3).cuda()
    before = buf.clone()
    out = buf[:, 5:5 + n]
    ops.linear_q4(x, weight, residual=out, out=out)
    check_product(f64(x), w_values, out, None, None, before[:, 5:5 + n], torch.float32, 2)
    assert torch.equal(buf[:, :5], before[:, :5]) and torch.equal(buf[:, 5 + n:], before[:, 5 + n:])


@gpu
@pytest.mark.parametrize("m,n,k", [(1, 130, 8), (3, 300, 104), (8, 200, 1600), (2, 1000, 2048), (5, 129, 4104), (8, 140, 8192), (9, 140, 256), (40, 140, 256)])
@pytest.mark.parametrize("beta", [True, False])
def test_products_of_normed_rows(m, n, k, beta):
    """LayerNorm made inside the product (up to 8 rows) or before it: against the norm in 64 bits, each of whose entries may go
    either way where it is rounded to bfloat16 (half a step, 2^-8 of it, and the norm's own 32-bit sums)."""
    x = normal((m + 3, k), 1, 2.0) + 0.7
    gamma, b = 1.0 + 0.2 * normal((k,), 2), 0.3 * normal((k,), 3) if beta else None
    weight = ops.quantize_q4(normal((n, k), 4, 0.05).cuda())
    w = plain.q4_values(u8(weight.codes), u8(weight.scales))[:, :k]
    pick = torch.randperm(m + 3, generator=torch.Generator().manual_seed(5))[:m].int()
    for rows in (None, pick):
        chosen = f64(x if rows is None else x[rows.long()])
        h = (chosen - chosen.mean(axis=1, keepdims=True)) / np.sqrt(chosen.var(axis=1, keepdims=True) + 1e-5) * f64(gamma)
        h = h + (f64(b) if beta else 0.0)
        xs = x.cuda()
        given = ops.NormedInput(xs, gamma.cuda(), b.cuda() if beta else None, 1e-5, torch.bfloat16, rows=None if rows is None else rows.cuda())
        got = f64(ops.linear_q4(given, weight, out_dtype=torch.float32))
        # mean and variance: k roundings at most, of entries up to five times a row's deviation
        off = product_bound(h, w, torch.float32, 2) + (2.0 ** -8 + (k + 16) * 2.0 ** -24) * (np.abs(h) + 1.0) @ np.abs(w).T
        assert got.shape == h[:, :1].shape[:1] + (n,) and (np.abs(got - h @ w.T) <= off).all()
        # bit by bit what the same rows give one at a time
        one = ops.linear_q4(ops.NormedInput(xs, given.gamma, given.beta, 1e-5, torch.bfloat16,
                                            rows=torch.tensor([0 if rows is None else int(rows[0])], dtype=torch.int32, device="cuda")), weight,
                            out_dtype=torch.float32)
        if given.n_rows <= 8:
            assert np.array_equal(got[:1], f64(one))
    ops.check_status()


@gpu
def test_products_give_the_same_bits_again_and_for_a_row_among_others():
    x, w = rough((16, 1600), 1).cuda(), ops.quantize_q4(normal((500, 1600), 2, 0.05).cuda())
    first = ops.linear_q4(x, w, out_dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(first, ops.linear_q4(x, w, out_dtype=torch.float32))
    assert torch.equal(first[3:4], ops.linear_q4(x[3:4], w, out_dtype=torch.float32))


@gpu
@pytest.mark.parametrize("m", [3, 8, 20, 64, 200])
def test_what_the_two_pieces_of_a_row_hold(m):
    """Weights of a unit matrix give each entry by itself, the group's largest among those that meet only zeros: entries down to 2^-13
    of it come back as they are, smaller ones within half the second piece's least step, 2^-14 of the scale, which the largest
    entry is more than 224 of."""
    k = 256
    gen = torch.Generator().manual_seed(m)
    x = (1.0 + torch.rand((m, k), generator=gen)) * torch.exp2(-torch.randint(0, 30, (m, k), generator=gen).float())
    x = (x * torch.where(torch.rand((m, k), generator=gen) < 0.5, -1.0, 1.0)).bfloat16()
    x[:, ::32] = ((1.0 + torch.rand((m, k // 32), generator=gen)) * 8.0).bfloat16()
    got = f64(ops.linear_q4(x.cuda(), ops.quantize_q4(torch.eye(k).cuda()), out_dtype=torch.float32)).reshape(m, -1, 32)
    want = f64(x).reshape(m, -1, 32)
    top = np.abs(want).max(axis=2, keepdims=True)
    exact = np.abs(want) >= 2.0 ** -13 * top
    assert exact.any() and not exact.all() and np.array_equal(got[exact], want[exact])
    assert (np.abs(got - want) <= 2.0 ** -14 / 224 * top).all() and 2.0 ** -14 / 224 < 2.0 ** -21


@gpu
def test_a_row_that_is_no_number_leaves_the_others():
    x = normal((5, 256), 1).bfloat16()
    x[1, 7], x[3, 200] = float("inf"), float("nan")
    w = ops.quantize_q4(normal((140, 256), 2).cuda())
    y = f64(ops.linear_q4(x.cuda(), w, out_dtype=torch.float32))
    assert np.isnan(y[[1, 3]]).all() and np.isfinite(y[[0, 2, 4]]).all()


@gpu
def test_no_rows():
    w = ops.quantize_q4(normal((140, 256), 2).cuda())
    assert ops.linear_q4(torch.empty(0, 256, dtype=torch.bfloat16, device="cuda"), w).shape == (0, 140)
    rows = ops.quantize_q8(torch.empty(0, 256, device="cuda"))
    assert ops.linear_q4(rows, w).shape == (0, 140)
    x = torch.empty(0, 256, device="cuda")
    assert ops.residual_add_norm_q8(x, None, 1.0, torch.ones(256, device="cuda"), 1e-5).codes.shape == (0, 256)


# ------------------------------------------------------------------------------------------------ the norm
def check_norm(x0, y, mult, y2, mult2, scale, weight, eps, x, rows):
    added = 0.0 if y is None else mult * f64(y) + (0.0 if y2 is None else mult2 * f64(y2))
    size = 0.0 if y is None else abs(mult) * np.abs(f64(y)) + (0.0 if y2 is None else abs(mult2) * np.abs(f64(y2)))
    if scale is not None:
        added, size = added * f64(scale), size * np.abs(f64(scale))
    stream = f64(x0) + added
    # at most four roundings of 2^-24 on the way to the stream, of what is added and of the stream itself
    assert (np.abs(f64(x) - stream) <= 4 * 2.0 ** -24 * (np.abs(f64(x0)) + size)).all()
    stream = f64(x)
    h = stream / np.sqrt((stream ** 2).mean(axis=1, keepdims=True) + eps) * f64(weight)
    m, k = h.shape
    # the row's sum of squares is off by at most k roundings, half of that in the root, and a few more behind it
    rel = (k / 2 + 8) * 2.0 ** -24
    g = plain.groups_of(h)
    top = np.abs(g).max(axis=2)
    e = plain.scale_bytes(u8(rows.scales), m) - 127.0
    assert (e >= plain.smallest_exponent(top * (1 - rel), 448.0)).all() and (e <= plain.smallest_exponent(top * (1 + rel), 448.0)).all()
    got = plain.q8_values(u8(rows.codes), u8(rows.scales)).reshape(g.shape)
    half = np.maximum(2.0 ** -4 * np.abs(g), 2.0 ** (e[..., None] - 10))           # half a step of e4m3, subnormal numbers included
    assert (np.abs(got - g) <= half * (1 + 2 * rel) + 2 * rel * np.abs(g)).all()
    assert (got.reshape(m, -1)[:, k:] == 0).all()


@gpu
@pytest.mark.parametrize("m,k", [(1, 1), (1, 31), (3, 128), (2, 1000), (129, 1600), (5, 2051), (4, 4096), (3, 8192), (2, 10001), (2, 20000)])
def test_norm_with_rows_in_eight_bits(m, k):
    for case in range(4):
        x, y, y2 = normal((m, k), 1, 2.0), normal((m, k), 2), normal((m, k), 3)
        weight, scale = 1.0 + 0.3 * normal((k,), 4), normal((k,), 5)
        y, y2, scale = (None if case == 0 else y, y2 if case >= 2 else None, scale if case == 3 else None)
        dev = lambda t: None if t is None else t.cuda()
        xs = x.cuda()
        rows = ops.residual_add_norm_q8(xs, dev(y), 0.7, weight.cuda(), 1e-5, y2=dev(y2), mult2=-0.4, scale=dev(scale))
        check_norm(x, y, 0.7, y2, -0.4, scale, weight, 1e-5, xs, rows)


@gpu
@pytest.mark.parametrize("k", [1024, 2048, 4096, 8192, 8200, 16384])
def test_norm_of_rows_with_a_few_large_entries(k):
    """Every eighth entry of the first 2,048 is 4,096, the rest are 1: a sum of squares in 32 bits that runs over all of a thread's
    entries loses each 1 beside 2^24.  Entries lie 4e-7, less their weight's rounding of 2^-24, above and below the middle of two
    codes; the row's factor may be off by 2^-23 (the squares of eight and their sum: four roundings of 2^-24, half of that in the
    root) and the entry's one rounding is 2^-24: 1.8e-7 of 3.4e-7, so every code has to be the 64-bit formula's."""
    x = torch.ones(3, k)
    x[:, 8 * torch.arange(min(k // 8, 256))] = 4096.0
    h0 = f64(x) / np.sqrt((f64(x) ** 2).mean(axis=1, keepdims=True) + 1e-5)
    # middles of two codes between 256 and 416 at a scale of 1, in turn above and below; each group's first entry is 430
    middles = np.array([272.0, 304.0, 336.0, 368.0, 400.0])
    column = np.arange(k)
    want = middles[column % 5] * np.where(column // 5 % 2 == 0, 1 + 4e-7, 1 - 4e-7)
    want[::32] = 430.0
    weight = torch.from_numpy(want / h0[0]).float()
    xs = x.cuda()
    rows = ops.residual_add_norm_q8(xs, None, 1.0, weight.cuda(), 1e-5)
    values, e = plain.q8_of(h0 * f64(weight))
    assert np.array_equal(plain.scale_bytes(u8(rows.scales), 3) - 127.0, e)
    assert np.array_equal(plain.e4m3(u8(rows.codes)), values)


@gpu
def test_norm_of_strided_and_unaligned_rows():
    buf, other = normal((7, 700), 1).cuda(), normal((7, 700), 2).cuda()
    weight = 1.0 + 0.3 * normal((512,), 4)
    for at in (0, 8, 3):
        x, y = buf[:, at:at + 512], other[:, at + 1:at + 513]
        x0, around = x.clone(), buf.clone()
        rows = ops.residual_add_norm_q8(x, y, 0.5, weight.cuda(), 1e-6)
        check_norm(x0, y, 0.5, None, 0.0, None, weight, 1e-6, x, rows)
        assert torch.equal(buf[:, :at], around[:, :at]) and torch.equal(buf[:, at + 512:], around[:, at + 512:])


@gpu
def test_norm_of_zeros_and_of_rows_that_are_no_numbers():
    x = normal((4, 256), 1)
    x[1] = 0.0
    x[2, 9] = float("nan")
    xs = x.cuda()
    rows = ops.residual_add_norm_q8(xs, None, 1.0, torch.ones(256).cuda(), 1e-5)
    v = plain.q8_values(u8(rows.codes), u8(rows.scales))
    assert (v[1] == 0).all() and np.isnan(v[2]).all() and np.isfinite(v[[0, 3]]).all()


# ------------------------------------------------------------------------------------------------ drafted tokens
def verify_case(b, g, v, seed, near=0.6, spread=2.0):
    gen = torch.Generator().manual_seed(seed)
    logits = torch.randn((b, g + 1, v), generator=gen) * spread
    draft_logits = logits[:, :g] + near * torch.randn((b, g, v), generator=gen)
    draws = torch.rand((b, g + 1), generator=gen, dtype=torch.float64)
    drafts = torch.multinomial(torch.softmax(draft_logits.reshape(b * g, v), 1), 1, generator=gen).reshape(b, g).int() if g else torch.empty(b, 0, dtype=torch.int32)
    return logits, draft_logits, drafts, draws


def check_verify(logits, draft_logits, drafts, draws, temperature, top_k):
    dev = [t.cuda() for t in (logits, draft_logits, drafts, draws)]
    tokens, kept = ops.verify_drafts(*dev, temperature, top_k)
    again = ops.verify_drafts(*dev, temperature, top_k)
    assert torch.equal(tokens, again[0]) and torch.equal(kept, again[1])
    assert tokens.dtype == kept.dtype == torch.int32
    seen = 0
    for i in range(logits.shape[0]):
        want, n, margin = plain.verify(logits[i].numpy(), draft_logits[i].numpy(), drafts[i].tolist(), draws[i].numpy(), temperature, top_k)
        # sums of 32-bit exponentials decide about a draft (each within 2^-22, arguments up to 20 off by 2^-24 of themselves)
        # and 64-bit ones about the token: a decision nearer than 1e-5 says nothing
        if margin < 1e-5 and (tokens[i].tolist(), int(kept[i])) != (want, n):
            continue
        assert tokens[i].tolist() == want and int(kept[i]) == n, f"sequence {i}: {tokens[i].tolist()} for {want}"
        seen += 1
    assert seen >= logits.shape[0] * 0.9


@gpu
@pytest.mark.parametrize("b,g,v", [(1, 1, 1), (3, 2, 5), (40, 4, 33), (17, 0, 200), (9, 3, 1031), (6, 5, 5000), (3, 4, 50257), (2, 70, 300)])
@pytest.mark.parametrize("temperature,top_k", [(0.0, 0), (1.0, 0), (0.7, 40), (1.3, 5), (0.5, 1), (0.9, -3), (1.0, 700)])
def test_verification(b, g, v, temperature, top_k):
    check_verify(*verify_case(b, g, v, b + 7 * g + v), temperature, top_k)


@gpu
def test_verification_of_equal_logits():
    """Rows of equal logits, of a few values only, and a cut among equals: ties go to the lowest index."""
    logits, draft_logits, drafts, draws = verify_case(24, 3, 4000, 5)
    logits[:8], draft_logits[:8] = 1.25, 1.25
    logits[8:16] = logits[8:16].round()
    draft_logits[8:16] = draft_logits[8:16].round()
    logits[16:] = (logits[16:] > 3).float()
    for temperature, top_k in ((1.0, 0), (1.0, 40), (0.8, 1500), (0.0, 0)):
        check_verify(logits, draft_logits, drafts, draws, temperature, top_k)


@gpu
@pytest.mark.parametrize("vocab,top_k", [(517, 0), (6000, 0), (6000, 50)])
def test_verification_of_logits_far_from_zero(vocab, top_k):
    """Only differences of logits count: at logits of 1,000 and a temperature of 0.01 a draw a ten-thousandth below or above the
    border is still decided right."""
    b = 128
    logits, draft_logits, drafts, draws = verify_case(b, 1, vocab, 3)
    logits, draft_logits = (1000.0 + 0.01 * t for t in (logits, draft_logits))
    want = []
    for i in range(b):
        p, q = (plain.softmax_kept(t[i, 0].numpy(), 0.01, top_k) for t in (logits, draft_logits))
        x = int(np.argmax(q)) if q[drafts[i, 0]] == 0 or p[drafts[i, 0]] == 0 else int(drafts[i, 0])
        drafts[i, 0] = x
        ratio = p[x] / q[x]
        draws[i, 0] = min(ratio * (1 + (1e-4 if i % 2 else -1e-4)), 0.999)
        want.append(int(draws[i, 0] * q[x] < p[x]))
    assert 30 < sum(want) < 120
    _, kept = ops.verify_drafts(logits.cuda(), draft_logits.cuda(), drafts.cuda(), draws.cuda(), 0.01, top_k)
    assert kept.tolist() == want


@gpu
@pytest.mark.parametrize("b,g,vocab,temperature,top_k", [(15, 4, 50257, 1.0, 0), (60, 4, 50257, 0.7, 0), (6, 2, 50257, 0.3, 40), (30, 4, 1031, 1.3, 0),
                                                         (6, 2, 40000, 0.01, 0), (3, 1, 50257, 1.0, 1000), (41, 40, 300, 1.0, 0)])
def test_verification_decides_in_64_bits(b, g, vocab, temperature, top_k):
    """Draws a thousand-millionth below the border take a draft, as far above it refuse it, several in a sequence.  The kernel's
    exponentials are within 1e-13 (and a sum of n of them within n 2^-53), the statement's within a few 2^-53: an error of 1e-11 at most."""
    logits, draft_logits, drafts, draws = verify_case(b, g, vocab, 21)
    if temperature < 0.1:
        logits, draft_logits = (500.0 + 0.01 * t for t in (logits, draft_logits))
    for i in range(b):
        for j in range(g):
            p, q = (plain.softmax_kept(t[i, j].numpy(), temperature, top_k) for t in (logits, draft_logits))
            x = int(np.argmax(np.where(q > 1.1 * p, p, -1.0)))               # the target's likeliest among those the draft has too much of
            assert 0 < p[x] < q[x]
            drafts[i, j] = x
            draws[i, j] = p[x] / q[x] * (1 + (-1e-9 if j < i % (g + 1) else 1e-9))
    _, kept = ops.verify_drafts(logits.cuda(), draft_logits.cuda(), drafts.cuda(), draws.cuda(), temperature, top_k)
    assert kept.tolist() == [i % (g + 1) for i in range(b)]


@gpu
@pytest.mark.parametrize("temperature", [1e-37, 1e-42, 5e-324])
@pytest.mark.parametrize("top_k", [0, 40, 700])
def test_verification_at_the_lowest_temperatures(temperature, top_k):
    """All of a row's mass lies on its maximum."""
    logits, draft_logits, drafts, draws = verify_case(6, 3, 5000, 5, near=0.1)
    drafts = draft_logits.argmax(dim=2).int()
    tokens, kept = ops.verify_drafts(logits.cuda(), draft_logits.cuda(), drafts.cuda(), draws.cuda(), temperature, top_k)
    want = ops.verify_drafts(logits.cuda(), None, drafts.cuda(), draws.cuda(), 0.0, 0)
    assert torch.equal(tokens, want[0]) and torch.equal(kept, want[1])


@gpu
def test_verification_with_masked_logits():
    """-inf and the type's lowest value take a token out; a row that is masked whole, or holds an infinity, gives its first
    maximum, and the rows of other sequences are as ever."""
    logits, draft_logits, drafts, draws = verify_case(12, 3, 300, 6)
    low = torch.finfo(torch.float32).min
    logits[0:4, :, 50:] = -float("inf")
    logits[4:8, :, :290] = low
    draft_logits[2:6, :, 100:] = -float("inf")
    logits[8] = -float("inf")
    logits[9, :, 17] = float("inf")
    for temperature, top_k in ((1.0, 0), (0.7, 20), (0.0, 0)):
        tokens, kept = ops.verify_drafts(logits.cuda(), draft_logits.cuda(), drafts.cuda(), draws.cuda(), temperature, top_k)
        assert kept[8].item() == 0 and tokens[8].tolist() == [0, -1, -1, -1] or int(drafts[8, 0]) == 0
        if temperature > 0:
            assert kept[9].item() == 0 and tokens[9].tolist() == [17, -1, -1, -1]
        sound = [0, 1, 2, 3, 4, 5, 6, 7, 10, 11]
        check_verify(logits[sound], draft_logits[sound], drafts[sound], draws[sound], temperature, top_k)


@gpu
@pytest.mark.parametrize("vocab", [300, 5000, 50257])
def test_verification_of_rows_without_a_distribution(vocab):
    """Rows with a NaN somewhere, with an infinity, masked whole: the token is the row's first maximum, a NaN above every number, as the
    sampler's ``argmax`` has it, wherever it lies; rows beside them are as ever."""
    rng = np.random.default_rng(vocab)
    rows = normal((60, vocab), 5)
    for i in range(40):
        for at in rng.integers(0, vocab, size=1 + i % 3):
            rows[i, at] = float("nan")
    rows[36:40] = torch.where(rows[36:40].isnan(), rows[36:40], torch.tensor(1.25))          # more equal ones than a block ranks
    rows[39, 5:] = float("nan")
    rows[40:44, 7], rows[44:48] = float("inf"), -float("inf")
    rows = rows.cuda()
    want = ops.argmax(rows)
    assert torch.equal(want.long(), rows.argmax(dim=1))
    rows.view(torch.int32)[20:40][rows[20:40].isnan()] = -4194304            # a NaN with its sign set
    drafts = torch.zeros(60, 0, dtype=torch.int32, device="cuda")
    draws = torch.rand((60, 1), dtype=torch.float64).cuda()
    for temperature, top_k in ((0.0, 0), (1.0, 0), (0.7, 20), (0.7, 600)):
        tokens, kept = ops.verify_drafts(rows[:, None], None, drafts, draws, temperature, top_k)
        upto = 48 if temperature > 0 else 60
        assert torch.equal(tokens[:upto, 0], want[:upto]) and (kept == 0).all()
    check_verify(rows[48:, None].cpu(), torch.zeros(12, 0, vocab), drafts[48:].cpu(), draws[48:].cpu(), 0.7, 20)


@gpu
def test_verification_where_the_draft_is_the_target():
    """p and q equal: every draft is taken; where a draft that is not the row's own is refused, the token comes from p."""
    logits, _, drafts, draws = verify_case(30, 4, 500, 7)
    tokens, kept = ops.verify_drafts(logits.cuda(), logits[:, :4].contiguous().cuda(), drafts.cuda(), draws.cuda(), 1.0, 0)
    assert (kept == 4).all()
    check_verify(logits, logits[:, :4].contiguous(), drafts, draws, 1.0, 0)


@gpu
def test_verification_ends_at_a_missing_draft():
    logits, draft_logits, drafts, draws = verify_case(20, 4, 200, 8, near=0.05)
    for i in range(20):
        drafts[i, i % 5:] = -1
    drafts[7, 1] = 200                                     # no token of the vocabulary ends them too
    for temperature, top_k in ((1.0, 0), (0.7, 30), (0.0, 0)):
        check_verify(logits, draft_logits, drafts, draws, temperature, top_k)
    _, kept = ops.verify_drafts(logits.cuda(), draft_logits.cuda(), drafts.cuda(), draws.cuda(), 1.0, 0)
    assert all(int(kept[i]) <= i % 5 for i in range(20))


@gpu
def test_verification_of_strided_logits():
    logits, draft_logits, drafts, draws = verify_case(5, 3, 700, 9)
    wide = torch.randn(8, 5, 900)
    wide[1:6, 1:5, 100:800] = logits
    other = torch.randn(3, 5, 750)
    other[:, :, 33:733] = draft_logits.transpose(0, 1)
    got = ops.verify_drafts(wide.cuda()[1:6, 1:5, 100:800], other.cuda()[:, :, 33:733].transpose(0, 1), drafts.cuda(), draws.cuda(), 0.8, 50)
    want = ops.verify_drafts(logits.cuda(), draft_logits.cuda(), drafts.cuda(), draws.cuda(), 0.8, 50)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
@pytest.mark.parametrize("top_k", [700, 2 ** 31 - 1, 2 ** 31, 2 ** 40, -2 ** 40])
def test_verification_with_a_top_k_past_the_vocabulary(top_k):
    dev = [t.cuda() for t in verify_case(6, 3, 700, 11)]
    got, want = ops.verify_drafts(*dev, 0.9, top_k), ops.verify_drafts(*dev, 0.9, 0)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@gpu
def test_verified_tokens_are_distributed_as_the_target():
    """The first token of 20,000 independent sequences of one draft, over a vocabulary of 6: frequencies against the target's
    probabilities (a binomial count is within 5 of its standard deviations but for one in a million)."""
    n, v = 20000, 6
    gen = torch.Generator().manual_seed(3)
    row, q_row = torch.randn(2, v, generator=gen)[0], torch.randn(v, generator=gen)
    logits, draft_logits = row.expand(n, 2, v).contiguous(), q_row.expand(n, 1, v).contiguous()
    drafts = torch.multinomial(torch.softmax(q_row, 0), n, replacement=True, generator=gen).reshape(n, 1).int()
    draws = torch.rand((n, 2), generator=gen, dtype=torch.float64)
    tokens, _ = ops.verify_drafts(logits.cuda(), draft_logits.cuda(), drafts.cuda(), draws.cuda(), 1.0, 0)
    p = torch.softmax(row.double(), 0).numpy()
    count = np.bincount(tokens[:, 0].cpu().numpy(), minlength=v)
    assert (np.abs(count - n * p) <= 5 * np.sqrt(n * p * (1 - p))).all()


# ------------------------------------------------------------------------------------------------ streams and graphs
@gpu
def test_calls_on_two_streams_at_once_and_in_graphs():
    """Two chains (norm, product, verification) on streams of their own, then recorded and replayed with other inputs."""
    def chain(x, y, w, q4, logits, draft_logits, drafts, draws):
        rows = ops.residual_add_norm_q8(x, y, 0.5, w, 1e-5)
        a = ops.linear_q4(rows, q4)
        b = ops.linear_q4(a, q4, out_dtype=torch.float32)
        return a, b, *ops.verify_drafts(logits, draft_logits, drafts, draws, 0.7, 40)

    def inputs(seed):
        return [normal((40, 256), seed).cuda(), normal((40, 256), seed + 1).cuda(), torch.ones(256).cuda()], \
            [t.cuda() for t in verify_case(4, 3, 2000, seed)]

    q4 = ops.quantize_q4(normal((256, 256), 1, 0.1).cuda())
    sets = [inputs(s) for s in (10, 20)]
    want = [[t.clone() for t in chain(*[t.clone() for t in s[0]], q4, *s[1])] for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for i, (s, stream) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(stream):
                got[i] = chain(s[0][0].clone(), *s[0][1:], q4, *s[1])
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(g, w))
    held = [[t.clone() for t in s[0]] + [t.clone() for t in s[1]] for s in sets]
    graphs, outs = [], []
    for h in held:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            x = h[0].clone()
            outs.append(chain(x, *h[1:3], q4, *h[3:]))
        graphs.append(g)
    for h, s in zip(held, reversed(sets)):                  # each graph gets the other's inputs
        for a, b in zip(h, s[0] + s[1]):
            a.copy_(b)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, reversed(want)):
        assert all(torch.equal(a, b) for a, b in zip(o, w))
    ops.check_status()


def test_only_fixed_weights_are_fetched_early(monkeypatch):
    """What the kernels are told: a weight is fetched ahead of the work in front of the call where its type says that nothing writes
    it any more, as a loaded model's does, and not otherwise."""
    from math_utils_b200.parts.linear import Linear
    records = []

    class Library:
        @staticmethod
        def mu_linear_q4(record):
            records.append(ops._LINEAR_Q4_ARGS.unpack(record))
            return 0

    monkeypatch.setattr(ops, "library", Library)
    monkeypatch.setattr(ops, "_on_current_device", lambda *t: None)
    monkeypatch.setattr(ops, "_stream", lambda: 0)
    monkeypatch.setattr(ops, "status_word", lambda device: torch.zeros(1, dtype=torch.int32))
    w = fake_weight(200, 300)
    monkeypatch.setattr(ops, "quantize_q4", lambda given: w)
    for x in (torch.zeros(4, 300, dtype=torch.bfloat16), torch.zeros(40, 300, dtype=torch.bfloat16), fake_rows(4, 300)):
        ops.linear_q4(x, w)
        ops.linear_q4(x, ops.FixedQ4Weight(*w))
    assert [r[-1] for r in records] == [0, 1] * 3

    class Runtime:
        weight_bits, row_bits, saved_bytes = 4, 16, 0
    Runtime.ops = ops
    Linear(torch.zeros(200, 300, dtype=torch.bfloat16), None, Runtime)(torch.zeros(4, 300, dtype=torch.bfloat16))
    assert records[-1][-1] == 1


@gpu
@pytest.mark.parametrize("m", [1, 8, 20, 200])
def test_products_of_weights_written_right_before(m):
    """Codes, exponents and bias that the kernel in front of the call writes, eagerly and in a recorded graph, and whatever ran in front of
    that (the product before lets its successor in early)."""
    x = normal((m, 1300), 1).bfloat16().cuda()
    sets = [(ops.quantize_q4(normal((700, 1300), s, 0.05).cuda()), normal((700,), s + 50).cuda()) for s in (2, 3)]
    want = [ops.linear_q4(x, w, bias=b, out_dtype=torch.float32) for w, b in sets]
    held, bias = Q4Weight(*(t.clone() for t in sets[0][0])), sets[0][1].clone()

    def write(i):                                           # kernels, not copies: a copy would order everything after it
        codes, scales = (t.view(torch.uint8) for t in sets[i][0])
        torch.bitwise_or(codes, 0, out=held.codes)
        torch.bitwise_or(scales, 0, out=held.scales.view(torch.uint8))
        torch.add(sets[i][1], 0.0, out=bias)
        return ops.linear_q4(x, held, bias=bias, out_dtype=torch.float32)

    for turn in range(20):
        assert torch.equal(write(turn % 2), want[turn % 2])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = [write(turn % 2) for turn in range(10)]
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[turn % 2]) for turn, g in enumerate(got))
    ops.check_status()


# ------------------------------------------------------------------------------------------------ refusals
def fake_weight(n, k):
    kp = plain.padded(k)
    return Q4Weight(torch.zeros(n, kp // 2, dtype=torch.uint8),
                    torch.zeros(-(-n // 128), kp // 128, 32, 4, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu))


def fake_rows(m, k):
    kp = plain.padded(k)
    return Q8Rows(torch.zeros(m, kp, dtype=torch.uint8).view(torch.float8_e4m3fn),
                  torch.zeros(-(-m // 128), kp // 128, 32, 4, 4, dtype=torch.uint8).view(torch.float8_e8m0fnu))


def test_refusals_of_products():
    """What a product cannot take is refused before anything is launched, wherever the tensors lie."""
    w, x = fake_weight(200, 300), torch.zeros(4, 300, dtype=torch.bfloat16)
    bad = [
        (dict(x=x.float()), "bfloat16"), (dict(x=x.half()), "bfloat16"), (dict(x=x[0]), "bfloat16"),
        (dict(x=torch.zeros(4, 256, dtype=torch.bfloat16)), "rounded up to 128"), (dict(x=torch.zeros(300, 4, dtype=torch.bfloat16).t()), "unit stride"),
        (dict(x=fake_rows(4, 200)), "float8_e4m3fn"), (dict(x=Q8Rows(fake_rows(4, 300).codes, fake_rows(4, 200).scales)), "scales"),
        (dict(x=Q8Rows(fake_rows(200, 300).codes, fake_rows(4, 300).scales)), "scales"),
        (dict(weight=Q4Weight(w.codes.float(), w.scales)), "uint8"), (dict(weight=Q4Weight(w.codes[:, :100], w.scales)), "multiple of 128"),
        (dict(weight=Q4Weight(w.codes, w.scales[:1])), "scales"), (dict(weight=Q4Weight(w.codes, w.scales.view(torch.uint8))), "scales"),
        (dict(weight=Q4Weight(torch.zeros(200, 400, dtype=torch.uint8)[:, :192], w.scales)), "contiguous"),
        (dict(act="silu"), "activation"), (dict(bias=torch.zeros(199)), "bias"), (dict(bias=torch.zeros(200).double()), "bias"),
        (dict(residual=torch.zeros(4, 199)), "residual"), (dict(residual=torch.zeros(4, 200).bfloat16()), "residual"),
        (dict(out=torch.zeros(5, 200)), "output"), (dict(out=torch.zeros(200, 4).t()), "output"), (dict(out=torch.zeros(4, 200).half()), "bfloat16 or float32"),
        (dict(), "CUDA"),
    ]
    for given, words in bad:
        args = dict(x=x, weight=w)
        args.update(given)
        with pytest.raises(KernelError, match=words):
            ops.linear_q4(**args)


def test_refusals_of_the_quantisers_and_the_norm():
    x = torch.zeros(4, 300)
    for call, words in (
            (lambda: ops.quantize_q4(x.half()), "bfloat16 or float32"), (lambda: ops.quantize_q4(x[0]), "matrix"), (lambda: ops.quantize_q4(x.t()), "unit stride"),
            (lambda: ops.quantize_q4(x[:0]), "matrix"), (lambda: ops.quantize_q4(x), "CUDA"),
            (lambda: ops.quantize_q8(x.double()), "bfloat16 or float32"), (lambda: ops.quantize_q8(x.t()), "unit stride"), (lambda: ops.quantize_q8(x), "CUDA"),
            (lambda: ops.residual_add_norm_q8(x.bfloat16(), None, 1.0, torch.ones(300), 1e-5), "float32"),
            (lambda: ops.residual_add_norm_q8(x, x[:3], 1.0, torch.ones(300), 1e-5), "shaped like the stream"),
            (lambda: ops.residual_add_norm_q8(x, x, 1.0, torch.ones(299), 1e-5), "weight"),
            (lambda: ops.residual_add_norm_q8(x, None, 1.0, torch.ones(300), 1e-5, y2=x), "first branch"),
            (lambda: ops.residual_add_norm_q8(x, None, 1.0, torch.ones(300), 1e-5, scale=torch.ones(300)), "first branch"),
            (lambda: ops.residual_add_norm_q8(x, x, 1.0, torch.ones(300), 1e-5, scale=torch.ones(299)), "scale"),
            (lambda: ops.residual_add_norm_q8(x[:1].expand(4, 300), x, 1.0, torch.ones(300), 1e-5), "apart"),
            (lambda: ops.residual_add_norm_q8(x, x, 1.0, torch.ones(300), 1e-5), "CUDA")):
        with pytest.raises(KernelError, match=words):
            call()


def test_refusals_of_verification():
    logits, draft_logits, drafts, draws = verify_case(2, 3, 20, 1)
    good = dict(logits=logits, draft_logits=draft_logits, drafts=drafts, draws=draws, temperature=1.0, top_k=0)
    for given, words in (
            (dict(logits=logits.double()), "float32"), (dict(logits=logits[0]), "float32"), (dict(logits=logits.transpose(1, 2)), "unit inner stride"),
            (dict(draft_logits=draft_logits[:, :2]), "draft's logits"), (dict(draft_logits=draft_logits.bfloat16()), "draft's logits"),
            (dict(draft_logits=None), "are needed"), (dict(drafts=drafts.long()), "int32"), (dict(drafts=drafts[:1]), "drafts are int32"),
            (dict(draws=draws.float()), "float64"), (dict(draws=draws[:, :3]), "float64"), (dict(temperature=float("nan")), "finite"),
            (dict(temperature=float("inf")), "finite"), (dict(), "CUDA")):
        with pytest.raises(KernelError, match=words):
            ops.verify_drafts(**{**good, **given})


@gpu
def test_refusals_on_the_device():
    x, w = normal((4, 256), 1).bfloat16().cuda(), ops.quantize_q4(normal((130, 256), 2).cuda())
    with pytest.raises(KernelError, match="CUDA"):
        ops.linear_q4(x.cpu(), w)
    with pytest.raises(KernelError, match="CUDA"):
        ops.linear_q4(x, w, bias=torch.zeros(130))
    shifted = torch.zeros(130 * 128 + 16, dtype=torch.uint8, device="cuda")[16:].view(130, 128)
    with pytest.raises(KernelError, match="alignment"):
        ops.linear_q4(x, Q4Weight(shifted, w.scales))
    with pytest.raises(KernelError, match="bad argument"):          # output rows that overlap
        ops.linear_q4(x, w, out=torch.zeros(200, device="cuda").as_strided((4, 130), (1, 1)))
