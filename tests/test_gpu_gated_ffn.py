"""The gated feed-forward block against its 64-bit form, forward and backward."""

import importlib
import math

import pytest
import torch

from tests import product_ref as ref
from tilefusion_amd import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
_one = importlib.import_module("tilefusion_amd.ops.gated_ffn")._backward   # of some gradients, as autograd asks for them
TYPES = [torch.float16, torch.bfloat16]
ACTIVATIONS = ["silu", "gelu", "gelu_tanh"]


def _randn(g, *shape, dtype, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def _block(m, f, k, dtype, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed + m * 5 + f * 3 + k)
    return _randn(g, m, k, dtype=dtype), _randn(g, f, k, dtype=dtype, scale=k ** -0.5), _randn(g, f, k, dtype=dtype, scale=k ** -0.5), g


def _check_forward(x, w_gate, w_up, activation):
    want, bounds = ref.gated_ffn(x.reshape(-1, x.shape[-1]), w_gate, w_up, activation)
    shape = (*x.shape[:-1], w_gate.shape[0])
    kept = ops.gated_ffn(x, w_gate, w_up, activation, keep=True)
    alone = ops.gated_ffn(x, w_gate, w_up, activation)
    assert alone.shape == shape and torch.equal(alone, kept[0])
    for name, got, w, b in zip(("h", "gate", "up"), kept, want, bounds):
        assert got.shape == shape and got.dtype == x.dtype
        ref.assert_within(got.reshape(w.shape), w, b, f"{name} {tuple(x.shape)} F={w_gate.shape[0]} {x.dtype} {activation}")


SIZES = [
    (1, 1, 1), (1, 1, 8), (1, 16, 64), (1, 512, 4096), (2, 33, 40), (3, 257, 1000), (7, 100, 33), (16, 64, 256), (17, 96, 72), (32, 1000, 512), (64, 64, 64),
    (65, 63, 127), (128, 64, 128), (129, 65, 136), (128, 256, 1024), (200, 128, 64), (255, 129, 264), (256, 128, 256), (257, 300, 520), (300, 1544, 1032),
    (513, 1030, 96), (1111, 770, 328),
]


# sizes that reach the kernels which those do not (tests/test_products_cpu.py looks)
KERNELS = [
    (35, 350, 64), (17, 1, 64), (37, 3004, 1984), (42, 3635, 728), (226, 2781, 448), (358, 1620, 72), (567, 5492, 64), (271, 5523, 64), (396, 5528, 72),
    (658, 5679, 64), (34, 14236, 72), (127, 10001, 520), (33, 25751, 72), (100, 25801, 65),
]


@pytest.mark.parametrize("m,f,k", SIZES + KERNELS)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward_sizes(m, f, k, dtype):
    x, w_gate, w_up, _ = _block(m, f, k, dtype)
    _check_forward(x, w_gate, w_up, "silu")


@pytest.mark.parametrize("m,f,k", [(1, 200, 128), (40, 136, 72), (150, 200, 264), (300, 256, 512), (9, 31, 15)])
@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward_activations(m, f, k, activation, dtype):
    x, w_gate, w_up, _ = _block(m, f, k, dtype, seed=1)
    _check_forward(x * 3, w_gate, w_up, activation)


def test_forward_shapes_strides_alignment():
    g = torch.Generator(device=DEV).manual_seed(2)
    base = _randn(g, 6, 5, 80, dtype=torch.float16)
    w = _randn(g, 64, 100, dtype=torch.float16, scale=0.1)
    _check_forward(base, w[:, :80], w[:, 20:], "silu")              # leading dimensions, strided weights
    _check_forward(base.transpose(0, 1), w[:, :80], w[:, 20:], "silu")
    _check_forward(base[0, 0], w[:, :80], w[:, 20:], "silu")         # one token, no leading dimension
    flat = _randn(g, 70 * 128 + 1, dtype=torch.float16)
    _check_forward(flat[1:].view(70, 128), flat[1:64 * 128 + 1].view(64, 128), flat[:64 * 128].view(64, 128), "gelu")   # odd addresses
    both = _randn(g, 2 * 96, 128, dtype=torch.bfloat16, scale=0.1)   # one tensor that holds both weights
    _check_forward(_randn(g, 130, 128, dtype=torch.bfloat16), both[:96], both[96:], "silu")
    _check_forward(_randn(g, 130, 128, dtype=torch.bfloat16), both[96:], both[:96], "silu")
    _check_forward(_randn(g, 130, 128, dtype=torch.bfloat16), both[:96], both[:96], "silu")   # the same weight twice


def test_forward_infinities_and_nan_stay_in_their_rows():
    x, w_gate, w_up, _ = _block(200, 160, 136, torch.bfloat16)
    clean = ops.gated_ffn(x, w_gate, w_up)
    x[3, 7] = float("nan")
    x[150, 0] = float("inf")
    x[199, 135] = -float("inf")
    h = ops.gated_ffn(x, w_gate, w_up)
    rows = torch.ones(200, dtype=torch.bool, device=DEV)
    rows[[3, 150, 199]] = False
    assert torch.equal(h[rows], clean[rows]) and h[3].isnan().all() and not h[[150, 199]].isfinite().all()


def test_large_gates():
    # far out on both sides the activations are 0 and the identity
    x = torch.tensor([[1.0], [-1.0]], device=DEV, dtype=torch.bfloat16)
    w_gate = torch.tensor([[50.0], [1e4], [1e20], [3e38]], device=DEV).bfloat16()
    w_up = torch.ones(4, 1, device=DEV).bfloat16()
    for activation in ACTIVATIONS:
        h, gate, up = ops.gated_ffn(x, w_gate, w_up, activation, keep=True)
        # (silu(-50) = -50 exp(-50) = -9.64e-21, the others' are smaller)
        assert torch.equal(h[0], w_gate[:, 0]) and (h[1].abs() <= 9.7e-21).all()
        one = torch.ones_like(h)
        grads = ops.gated_ffn_backward(one, x, w_gate, w_up, gate, up, activation)
        # (x[0]'s gradient is the sum of w_gate and of act(w_gate), 6e38, which is infinite in the type)
        assert all(t.isfinite().all() for t in (grads[0][1], grads[1], grads[2])) and grads[0][0] == float("inf")


def _far(g, activation):
    """How far an activation in fp32 may be off, relative to its terms: a few roundings, and exp's argument, which is off by its own rounding."""
    return 2.0 ** -20 + 2.0 ** -21 * {"silu": g.abs(), "gelu": g * g / 2, "gelu_tanh": 1.6 * (g + 0.044715 * g ** 3).abs()}[activation]


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", TYPES)
def test_activations_are_right_in_their_leading_digits(dtype, activation):
    # every number of the type from -14 to 14 as a gate that is no sum, far out on the left as well, where the activation is small
    values = torch.arange(0, 0x8000, device=DEV, dtype=torch.int16).view(dtype)
    values = values[values.abs() <= 14]
    values = torch.cat([values, -values])
    step, tiny, g = ref.half_step(dtype), ref.TINY[dtype], values.double()
    up = 1024.0 if dtype == torch.float16 else 1.0   # (h reaches further down in fp16 so)
    x = torch.zeros(len(values), 8, device=DEV, dtype=dtype)
    x[:, 0], x[:, 1] = values, 1.0
    w_gate, w_up = torch.zeros(2, 1, 8, device=DEV, dtype=dtype)
    w_gate[0, 0], w_up[0, 1] = 1.0, up
    h = ops.gated_ffn(x, w_gate, w_up, activation)[:, 0].double()
    far = _far(g, activation)
    # (torch.special.ndtr is (1 + erf) / 2, without leading digits from -8 on)
    phi = torch.special.erfc(-g / math.sqrt(2)) / 2 if activation == "gelu" else ref.phi(g, activation)
    rest = ref.act_slope(g, activation) - ref.phi(g, activation)   # g * phi'(g)
    if activation == "gelu":
        rest = g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    want, small = up * g * phi, 2.0 ** -120 * up   # (fp32 below its normal numbers)
    assert ((h - want).abs() <= (far + step * (1 + far)) * want.abs() + tiny + small).all()
    # the gradients of gate and up, each through a weight of one number
    gate, ones = values[:, None], torch.ones(len(values), 1, device=DEV, dtype=dtype)
    one, none = torch.ones(1, 8, device=DEV, dtype=dtype), torch.zeros(1, 8, device=DEV, dtype=dtype)
    grad_gate = ops.gated_ffn_backward(ones * up, x, one, none, gate, ones, activation)[0][:, 3].double()
    grad_up = ops.gated_ffn_backward(ones * up, x, none, one, gate, ones, activation)[0][:, 3].double()
    assert ((grad_up - want).abs() <= (far + step * (1 + far)) * want.abs() + tiny + small).all()
    slope, terms = up * (phi + rest), up * (phi + rest.abs())
    assert ((grad_gate - slope).abs() <= far * terms + step * (slope.abs() + far * terms) + tiny + small * 16).all()


@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_gates_beyond_the_largest_number_of_fp16(activation):
    # kept as infinities, they still say which side of the activation they are on: 0 with a slope of 0, the identity with a slope of 1
    x = torch.tensor([[256.0], [-256.0], [1.0]], device=DEV).half()
    w_gate, w_up = torch.tensor([[512.0]], device=DEV).half(), torch.tensor([[0.25]], device=DEV).half()
    h, gate, up = ops.gated_ffn(x, w_gate, w_up, activation, keep=True)
    assert gate[:2, 0].tolist() == [float("inf"), -float("inf")] and h[1:, 0].tolist() == [0.0, 128.0]
    grad_h = torch.tensor([[0.0], [0.5], [0.25]], device=DEV).half()
    grad_x, grad_gate, grad_up = ops.gated_ffn_backward(grad_h[1:], x[1:], w_gate, w_up, gate[1:], up[1:], activation)
    # token 1: nothing; token 2: dg = 0.25 * 0.25 and du = 0.25 * 512
    assert grad_x[:, 0].tolist() == [0.0, 0.0625 * 512 + 128 * 0.25] and grad_gate.item() == 0.0625 and grad_up.item() == 128.0
    # the other side: dg = 0.5 * 64 of a gate that is infinite, in the gradient of the gate's weight
    one = torch.ones(1, 1, device=DEV).half()
    grads = ops.gated_ffn_backward(one * 0.5, x[:1], w_gate * 0, w_up * 0, gate[:1], up[:1], activation)
    assert grads[1].item() == 0.5 * 64 * 256 and grads[2].item() == float("inf")
    assert ops.gated_ffn_backward(one, one, one, one, one * float("nan"), one, activation)[0].isnan().all()


# ---- backward ------------------------------------------------------------------------------
def _check_backward(grad_h, x, w_gate, w_up, gate, up, activation, alone=False):
    results = [(ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up, activation), (0, 1, 2))]
    if alone:   # gradients that are asked for without the others: what runs is chosen for each
        results += [(_one(grad_h, x, w_gate, w_up, gate, up, activation, of == (0,), of != (0,)), of) for of in ((0,), (1, 2))]
    f, k = w_gate.shape
    want, bounds = ref.gated_ffn_backward(grad_h.reshape(-1, f), x.reshape(-1, k), w_gate, w_up, gate.reshape(-1, f), up.reshape(-1, f), activation)
    for got, of in results:
        for i, (name, g, w, b, like) in enumerate(zip(("grad_x", "grad_w_gate", "grad_w_up"), got, want, bounds, (x, w_gate, w_up))):
            if i not in of:
                assert g is None
                continue
            assert g.shape == like.shape and g.dtype == x.dtype
            what = f"{name} {tuple(x.shape)} F={f} {x.dtype} {activation} of {of}"
            ref.assert_within(g.reshape(w.shape), w, b, what)
            # errors of many roundings are independent: in all far less than every one at its largest
            assert (g.reshape(w.shape).double() - w).norm() <= 2 * ref.half_step(x.dtype) * w.norm(), what


BACKWARD_SIZES = [(1, 1, 1), (1, 64, 64), (3, 17, 9), (31, 100, 33), (64, 64, 64), (65, 127, 72), (130, 96, 200), (257, 136, 264), (400, 513, 104), (1000, 160, 1032)]


# sizes that reach the tiles, and sums in parts, which those do not (tests/test_products_cpu.py looks)
BACKWARD_KERNELS = [
    (3667, 1, 2320), (2442, 1, 1592), (3214, 3946, 8), (1810, 409, 2304), (130, 8700, 5936), (1, 6720, 1296), (1, 2186, 1800), (2, 3339, 520), (3951, 2907, 8),
    (1, 3238, 1184), (26477, 548, 8), (34566, 1353, 144),
]
# both products in one launch: every tile, with neither, either and both sums in parts
BACKWARD_PAIRS = [
    (960, 513, 3992), (4466, 497, 1056), (2, 2501, 3504), (5558, 4584, 152), (580, 200, 3880), (3057, 1, 2928), (1, 462, 3424), (2842, 2564, 8),
    (836, 1, 8), (1, 385, 8), (964, 784, 8), (525, 271, 3536), (2493, 1, 3568), (1, 718, 2880), (4121, 5190, 8),
]


@pytest.mark.parametrize("m,f,k", BACKWARD_SIZES + BACKWARD_KERNELS + BACKWARD_PAIRS)
@pytest.mark.parametrize("dtype", TYPES)
def test_backward_sizes(m, f, k, dtype):
    x, w_gate, w_up, g = _block(m, f, k, dtype, seed=4)
    _check_backward(*(_randn(g, m, f, dtype=dtype) for _ in range(1)), x, w_gate, w_up, _randn(g, m, f, dtype=dtype), _randn(g, m, f, dtype=dtype), "silu", alone=True)


def _scaled_backward(grad_h, x, w_gate, w_up, gate, up, activation):
    """The gradients and their bounds in fp16.  Where the largest of dg and du is below 2^-6 or above 65504 they have a power of two in common by which
    it is 2^14 to 2^15.  What fp16's smallest numbers leave out of one is 2^-25, 2^-39 of the largest then."""
    d, g, u = grad_h.double(), gate.double(), up.double()
    grads = d * u * ref.act_slope(g, activation), d * ref.act(g, activation)
    top = max(t.abs().max() for t in grads)
    most = 2.0 ** -25 if 2.0 ** -6 <= top <= 65504 else 2.0 ** -39 * top
    offs = [ref.FN * size + ref.half_step(x.dtype) * t.abs() + most for t, size in zip(grads, ((d * u).abs() * (1 + g.abs()), (d * g).abs()))]
    (dg, du), (off_g, off_u) = grads, offs
    return ref._products([(torch.cat([dg, du], 1), torch.cat([off_g, off_u], 1), torch.cat([w_gate, w_up]).t()), (dg.t(), off_g.t(), x.t()),
                          (du.t(), off_u.t(), x.t())], x.dtype)


# grad_h, up, weights and tokens: dg and du beyond 65504, and below fp16's smallest number, where the gradients that they add up to are not
RANGES = {"large": (300.0, 300.0, 2.0 ** -10, 2.0 ** -10), "small": (2.0 ** -13, 2.0 ** -9, 1024.0, 1024.0)}


@pytest.mark.parametrize("m,f,k", [(1, 64, 64), (70, 40, 24), (130, 96, 200), (257, 136, 264), (31, 100, 33), (2, 2501, 3504), (2493, 1, 3568)])
@pytest.mark.parametrize("span", list(RANGES))
@pytest.mark.parametrize("activation", ACTIVATIONS)
def test_backward_beyond_the_range_of_fp16(m, f, k, span, activation):
    of_h, of_up, of_w, of_x = RANGES[span]
    g = torch.Generator(device=DEV).manual_seed(16 + m + f + k)
    dtype = torch.float16
    grad_h, gate, up = _randn(g, m, f, dtype=dtype, scale=of_h), _randn(g, m, f, dtype=dtype), _randn(g, m, f, dtype=dtype, scale=of_up)
    x, w_gate, w_up = _randn(g, m, k, dtype=dtype, scale=of_x), *(_randn(g, f, k, dtype=dtype, scale=of_w) for _ in range(2))
    if span == "small":   # (du has no part of up, and would be the largest)
        w_up.zero_()
        gate *= 2.0 ** -9
    want, bounds = _scaled_backward(grad_h, x, w_gate, w_up, gate, up, activation)
    assert (want[0].abs() < 65504).all() and (want[0].abs().max() > 2.0 ** -14)
    got = ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up, activation)
    some = [_one(grad_h, x, w_gate, w_up, gate, up, activation, of, not of) for of in (True, False)]
    for grads, of in ((got, (0, 1, 2)), (some[0], (0,)), (some[1], (1, 2))):
        for i in of:
            ref.assert_within(grads[i], want[i], bounds[i], f"{i} of {of}")
            floor = want[i].numel() ** 0.5 * ref.TINY[dtype]
            assert (grads[i].double() - want[i]).norm() <= 2 * ref.half_step(dtype) * want[i].norm() + floor


@pytest.mark.parametrize("power", list(range(-22, 14)))
def test_backward_at_every_size_of_its_gradients(power):
    m, f, k = 60, 72, 40
    x, w_gate, w_up, g = _block(m, f, k, torch.float16, seed=23)
    grad_h, gate, up = (_randn(g, m, f, dtype=torch.float16) for _ in range(3))
    grad_h *= 2.0 ** power
    by = 2.0 ** max(0, -power // 2 - 4)   # (results within the type)
    x, w_gate, w_up = (t * by if power < 0 else t * 2.0 ** -6 for t in (x, w_gate, w_up))
    want, bounds = _scaled_backward(grad_h, x, w_gate, w_up, gate, up, "silu")
    for got, a, bound in zip(ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up), want, bounds):
        ref.assert_within(got, a, bound, str(power))
        assert (got.double() - a).norm() <= 2 * ref.half_step(torch.float16) * a.norm() + a.numel() ** 0.5 * ref.TINY[torch.float16]


def test_an_infinite_gradient_does_not_take_the_others_range():
    # one token's grad_h is infinite (a step that a loss scaler leaves out): the other tokens' gradients are as without it
    m, f, k = 200, 72, 96
    x, w_gate, w_up, g = _block(m, f, k, torch.float16, seed=17)
    grad_h, gate, up = (_randn(g, m, f, dtype=torch.float16, scale=s) for s in (300.0, 1.0, 300.0))
    w_gate, w_up = w_gate * 2.0 ** -8, w_up * 2.0 ** -8
    grad_h[7] = 0
    clean = ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up)
    assert clean[0].isfinite().all()
    grad_h[7, 5], grad_h[7, 6] = float("inf"), float("nan")
    grads = ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up)
    others = torch.arange(m, device=DEV) != 7
    assert torch.equal(grads[0][others], clean[0][others]) and not grads[0][7].isfinite().any()


def test_ranges_that_change_between_replays():
    m, f, k = 140, 72, 96
    x, w_gate, w_up, g = _block(m, f, k, torch.float16, seed=18)
    grad_h, gate, up = (_randn(g, m, f, dtype=torch.float16) for _ in range(3))
    start = grad_h.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up)
    for by in (1.0, 2.0 ** 14, 2.0 ** -9, 1.0, 0.0):
        grad_h.copy_(start * by)
        want = [t.clone() for t in ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up)]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), by


@pytest.mark.parametrize("activation", ACTIVATIONS)
@pytest.mark.parametrize("dtype", TYPES)
def test_backward_activations(activation, dtype):
    x, w_gate, w_up, g = _block(150, 200, 88, dtype, seed=5)
    grad_h = _randn(g, 150, 200, dtype=dtype)
    _, gate, up = ops.gated_ffn(x * 2, w_gate, w_up, activation, keep=True)
    _check_backward(grad_h, x * 2, w_gate, w_up, gate, up, activation)


@pytest.mark.parametrize("f", [128, 130])
def test_backward_of_some(f):
    # what is not asked for is not computed, and changes nothing of what is
    x, w_gate, w_up, g = _block(100, f, 72, torch.bfloat16, seed=11)
    grad_h = _randn(g, 100, f, dtype=torch.bfloat16)
    _, gate, up = ops.gated_ffn(x, w_gate, w_up, keep=True)
    want = ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up)
    for asked in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.clone().requires_grad_(i in asked) for i, t in enumerate((x, w_gate, w_up))]
        ops.gated_ffn(*leaves).backward(grad_h)
        for i, leaf in enumerate(leaves):
            assert torch.equal(leaf.grad, want[i]) if i in asked else leaf.grad is None


def test_offsets_that_pass_32_bits():
    # h, gate and up of more than 4 GiB each, and gradients that are sums over them
    m, f, k = 70000, 32768, 64
    g = torch.Generator(device=DEV).manual_seed(12)
    x, w = _randn(g, m, k, dtype=torch.bfloat16), _randn(g, 2, f, k, dtype=torch.bfloat16, scale=0.125)
    h, gate, up = ops.gated_ffn(x, w[0], w[1], keep=True)
    for rows in (slice(0, 200), slice(m - 200, m)):
        want, bounds = ref.gated_ffn(x[rows], w[0], w[1], "silu")
        for got, a, b in zip((h, gate, up), want, bounds):
            ref.assert_within(got[rows], a, b)
    # all but the last rows have no gradient: theirs is that of a small problem
    h.zero_()
    h[-200:] = _randn(g, 200, f, dtype=torch.bfloat16)
    grad_x, grad_gate, grad_up = ops.gated_ffn_backward(h, x, w[0], w[1], gate, up)
    want, bounds = ref.gated_ffn_backward(h[-200:], x[-200:], w[0], w[1], gate[-200:], up[-200:], "silu")
    assert (grad_x[:-200] == 0).all()
    for got, a, b in zip((grad_x[-200:], grad_gate, grad_up), want, bounds):
        ref.assert_within(got, a, b)


def test_more_tiles_than_a_launch_has():
    # 2^23 + 1024 tiles of 64 x 32, the only ones for so few columns
    m, f, k = (1 << 19) + 5, 1 << 15, 8
    x, w_gate, w_up, _ = _block(m, f, k, torch.bfloat16, seed=19)
    h = ops.gated_ffn(x, w_gate, w_up)
    for at in (0, 8191 * 64 - 40, m - 60):
        rows = slice(at, at + 60)
        want, bounds = ref.gated_ffn(x[rows], w_gate, w_up, "silu")
        ref.assert_within(h[rows], want[0], bounds[0], f"{at}")


def test_backward_shapes_strides_and_empty():
    g = torch.Generator(device=DEV).manual_seed(6)
    dtype = torch.float16
    x, w = _randn(g, 3, 11, 48, dtype=dtype), _randn(g, 2, 72, 48, dtype=dtype, scale=0.2)
    tall = _randn(g, 3, 72, 11, dtype=dtype)
    _check_backward(tall.transpose(1, 2), x, w[0], w[1], tall.transpose(1, 2) * 2, tall.flip(0).transpose(1, 2), "silu")
    flat = _randn(g, 33 * 72 + 1, dtype=dtype)
    odd = flat[1:].view(33, 72)
    _check_backward(odd, x.reshape(33, 48), w[0], w[1], odd * 0.5, odd + 1, "gelu")
    one = torch.ones(1, device=DEV, dtype=dtype)
    _check_backward(one.expand(33, 72), x.reshape(33, 48), w[0], w[1], odd * 0.5, odd + 1, "gelu")   # the gradient of a sum: one number for all
    empty = torch.empty(0, 72, device=DEV, dtype=dtype)
    grads = ops.gated_ffn_backward(empty, torch.empty(0, 48, device=DEV, dtype=dtype), w[0], w[1], empty, empty)
    assert grads[0].shape == (0, 48) and (grads[1] == 0).all() and (grads[2] == 0).all()
    assert ops.gated_ffn(torch.empty(2, 0, 48, device=DEV, dtype=dtype), w[0], w[1]).shape == (2, 0, 72)


@pytest.mark.parametrize("asked", [(0,), (1,), (2,), (0, 1, 2)])
def test_autograd_of_no_tokens(asked):
    leaves = [torch.randn(*s, device=DEV).half().requires_grad_(i in asked) for i, s in enumerate(((0, 48), (72, 48), (72, 48)))]
    ops.gated_ffn(*leaves).sum().backward()
    for i, leaf in enumerate(leaves):
        assert (leaf.grad == 0).all() and leaf.grad.shape == leaf.shape if i in asked else leaf.grad is None


def test_backward_with_any_workspace_and_gradients_apart():
    # a workspace that holds NaN, one that is just large enough, and gradients of the weights that lie anywhere
    m, f, k = 70, 40, 24
    x, w_gate, w_up, g = _block(m, f, k, torch.bfloat16, seed=7)
    grad_h, gate, up = (_randn(g, m, f, dtype=torch.bfloat16) for _ in range(3))
    want = ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up)
    lib = _capi.load()
    size = lib.tf_gated_ffn_backward_workspace_bytes(m, f, k)
    room = torch.full((size + 64,), 0xFF, device=DEV, dtype=torch.uint8)
    got = [torch.full_like(t, float("nan")) for t in (x, w_gate, w_up)]
    _capi.check(lib.tf_gated_ffn_backward(*(t.data_ptr() for t in (grad_h, x, w_gate, w_up, gate, up, *got)), _capi.TF_DTYPE_BF16, _capi.TF_ACT_SILU,
                                          m, f, k, room.data_ptr(), size, torch.cuda.current_stream().cuda_stream), "tf_gated_ffn_backward")
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert (room[size:] == 0xFF).all()


def test_autograd_is_the_explicit_backward():
    x, w_gate, w_up, g = _block(90, 72, 56, torch.bfloat16, seed=8)
    grad_h = _randn(g, 90, 72, dtype=torch.bfloat16)
    h0, gate, up = ops.gated_ffn(x, w_gate, w_up, "gelu", keep=True)
    want = ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up, "gelu")
    leaves = [t.clone().requires_grad_() for t in (x, w_gate, w_up)]
    h = ops.gated_ffn(*leaves, "gelu")
    assert torch.equal(h, h0)
    h.backward(grad_h)
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w)
    # some leaves only, and a copy of x that is used twice
    x2 = x.clone().requires_grad_()
    h, gate, up = ops.gated_ffn(x2, w_gate, w_up, "gelu", keep=True)
    assert not gate.requires_grad and not up.requires_grad
    (grad,) = torch.autograd.grad(h, x2, grad_h)
    assert torch.equal(grad, want[0])
    with pytest.raises(RuntimeError):
        torch.autograd.grad(torch.autograd.grad(ops.gated_ffn(x2, w_gate, w_up).sum(), x2, create_graph=True)[0].sum(), x2)
    with torch.no_grad():
        assert not ops.gated_ffn(*leaves).requires_grad


def test_replayed_and_on_two_streams():
    x, w_gate, w_up, g = _block(140, 200, 96, torch.float16, seed=9)
    grad_h = _randn(g, 140, 200, dtype=torch.float16)

    def step():
        h, gate, up = ops.gated_ffn(x, w_gate, w_up, keep=True)
        return (h, *ops.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up))

    want = [t.clone() for t in step()]
    sides = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for side in sides:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                results.append(step())
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        x.mul_(0.5 if n % 2 else 2.0)
        want = [t.clone() for t in step()]
        for t in out:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n
    leaf = w_gate.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.gated_ffn(x, leaf, w_up)


def test_compiled_call():
    x, w_gate, w_up, _ = _block(20, 48, 32, torch.bfloat16)
    want = ops.gated_ffn(x, w_gate, w_up)
    assert torch.equal(torch.compile(lambda *t: ops.gated_ffn(*t), backend="eager")(x, w_gate, w_up), want)


def test_refusals():
    x, w_gate, w_up, _ = _block(4, 16, 32, torch.float16)
    h = torch.zeros(4, 16, device=DEV).half()
    for bad in ((x, w_gate, w_up.bfloat16()), (x, w_gate, w_up[:8]), (x[:, :16], w_gate, w_up), (x, w_gate.cpu(), w_up), (x.float(), w_gate.float(), w_up.float()),
                (x, w_gate, w_up, "relu"), (x, w_gate[0], w_up), (x[..., :0], w_gate[:, :0], w_up[:, :0])):
        with pytest.raises(RuntimeError):
            ops.gated_ffn(*bad)
    for bad in ((h[:3], x, w_gate, w_up, h, h), (h, x, w_gate, w_up, h.float(), h), (h, x, w_gate, w_up, h, h[:, :8]), (h, x, w_gate, w_up, h, h, "tanh")):
        with pytest.raises(RuntimeError):
            ops.gated_ffn_backward(*bad)
