"""The cross entropy of a linear head against its 64-bit form, forward and backward."""

import importlib

import pytest
import torch

from tests import product_ref as ref
from tilefusion_amd import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
_one = importlib.import_module("tilefusion_amd.ops.linear_cross_entropy")._backward   # of some gradients, as autograd asks for them
TYPES = [torch.float16, torch.bfloat16]


def _head(t, v, k, dtype, seed=0, ignored=True):
    g = torch.Generator(device=DEV).manual_seed(seed + t * 5 + v * 3 + k)
    hidden = torch.randn(t, k, device=DEV, generator=g).to(dtype)
    weight = (torch.randn(v, k, device=DEV, generator=g) * 2 * k ** -0.5).to(dtype)
    target = torch.randint(0, v, (t,), device=DEV, generator=g)
    if ignored:
        target[torch.rand(t, device=DEV, generator=g) < 0.2] = -100
    return hidden, weight, target, g


def _check_forward(hidden, weight, target, ignore_index=-100):
    loss, lse = ops.linear_cross_entropy(hidden, weight, target, ignore_index)
    (want_loss, want_lse), (b_loss, b_lse) = ref.linear_cross_entropy(hidden.reshape(-1, hidden.shape[-1]), weight, target.reshape(-1), ignore_index)
    assert loss.shape == target.shape == lse.shape and loss.dtype == lse.dtype == torch.float32
    what = f"{tuple(hidden.shape)} V={weight.shape[0]} {hidden.dtype}"
    ref.assert_within(lse.reshape(-1), want_lse, b_lse, "lse " + what)
    ref.assert_within(loss.reshape(-1), want_loss, b_loss, "loss " + what)
    assert (loss[target == ignore_index] == 0).all()
    return lse


def _check_backward(grad_loss, hidden, weight, target, ignore_index=-100, alone=False):
    lse = ops.linear_cross_entropy(hidden, weight, target, ignore_index)[1]
    got = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse, ignore_index)
    want, bounds = ref.linear_cross_entropy_backward(grad_loss.reshape(-1), hidden.reshape(-1, hidden.shape[-1]), weight, target.reshape(-1), ignore_index)
    results = [(got, (0, 1))]
    if alone:   # gradients that are asked for without the other: what runs is chosen for each
        results += [(_one(grad_loss, hidden, weight, target, lse, ignore_index, of == 0, of == 1), (of,)) for of in (0, 1)]
    for grads, of in results:
        for i, (name, g, w, b, like) in enumerate(zip(("grad_hidden", "grad_weight"), grads, want, bounds, (hidden, weight))):
            if i not in of:
                assert g is None
                continue
            assert g.shape == like.shape and g.dtype == like.dtype
            what = f"{name} {tuple(hidden.shape)} V={weight.shape[0]} {hidden.dtype} of {of}"
            number = ref.assert_within(g.reshape(w.shape), w, b, what)
            if w.norm() > 0:
                floor = w.numel() ** 0.5 * ref.TINY[hidden.dtype]   # results too small for the type
                assert (g.reshape(w.shape).double() - w)[number].norm() <= 2 * ref.half_step(hidden.dtype) * w.norm() + floor, what
    return got


SIZES = [
    (1, 1, 1), (1, 2, 8), (1, 1000, 64), (1, 5003, 256), (2, 63, 40), (5, 65, 33), (16, 1000, 128), (37, 4099, 72), (64, 64, 64), (100, 129, 136), (128, 128, 128),
    (130, 1000, 1000), (255, 2049, 96), (256, 256, 64), (257, 777, 264), (300, 3001, 520), (700, 300, 128), (1025, 513, 88),
]


# sizes that reach the kernels which those do not (tests/test_products_cpu.py looks)
KERNELS = [
    (1, 1, 264), (1883, 67, 72), (1752, 50, 64), (2319, 49, 72), (354, 855, 2048), (2411, 173, 712), (480, 2674, 448), (197, 5649, 72), (2891, 5564, 80),
    (898, 4350, 64), (2865, 2786, 64), (967, 5420, 72), (2925, 3106, 64), (2206, 5545, 64), (65, 17495, 80), (127, 30001, 264), (38, 54305, 72),
    (100, 54305, 65),
]
# and the tiles, and sums in parts, of gradients
BACKWARD_KERNELS = [
    (3599, 1, 2208), (2522, 1, 1544), (1, 903, 8), (1849, 886, 2288), (130, 17395, 5936), (1175, 15938, 8), (1, 13431, 1296), (1, 3567, 2328), (1, 3263, 1168),
    (898, 1, 8), (791, 3609, 1104), (22312, 129, 5776), (15938, 1175, 8), (33847, 1059, 8),
]
# both products in one launch: every tile, with neither, either and both sums in parts
BACKWARD_PAIRS = [
    (1069, 1055, 3728), (5423, 1379, 928), (133, 8627, 2456), (5318, 9225, 152), (534, 464, 3624), (2989, 1, 3256), (1, 969, 3344), (2689, 5305, 8),
    (839, 1, 8), (1, 835, 8), (1001, 1741, 8), (385, 579, 3608), (4635, 1, 3616), (1, 1421, 2712), (5816, 7434, 8),
]


@pytest.mark.parametrize("t,v,k", SIZES + KERNELS)
@pytest.mark.parametrize("dtype", TYPES)
def test_forward_sizes(t, v, k, dtype):
    hidden, weight, target, _ = _head(t, v, k, dtype)
    _check_forward(hidden, weight, target)


@pytest.mark.parametrize("t,v,k", SIZES + KERNELS + BACKWARD_KERNELS + BACKWARD_PAIRS)
@pytest.mark.parametrize("dtype", TYPES)
def test_backward_sizes(t, v, k, dtype):
    hidden, weight, target, g = _head(t, v, k, dtype, seed=1)
    scale = 4096.0 if dtype == torch.float16 else 1.0
    _check_backward(torch.full((t,), scale / t, device=DEV), hidden, weight, target, alone=True)
    _check_backward((torch.rand(t, device=DEV, generator=g) - 0.5) * scale, hidden, weight, target)


@pytest.mark.parametrize("dtype", TYPES)
def test_pieces_of_the_vocabulary(dtype):
    # 40000 tokens: pieces of 4096 columns, the last one of an odd width
    hidden, weight, target, g = _head(40000, 8195, 24, dtype, seed=2)
    lib = _capi.load()
    assert lib.tf_linear_cross_entropy_backward_workspace_bytes(40000, 8195, 24) < 2 * 40000 * 8195 * 2
    _check_backward(torch.rand(40000, device=DEV, generator=g) / 40000 * (4096 if dtype == torch.float16 else 1), hidden, weight, target)


def test_backward_of_some():
    hidden, weight, target, g = _head(100, 500, 72, torch.bfloat16, seed=11)
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    want = ops.linear_cross_entropy_backward(torch.ones(100, device=DEV), hidden, weight, target, lse)
    for asked in (0, 1):
        leaves = [t.clone().requires_grad_(i == asked) for i, t in enumerate((hidden, weight))]
        ops.linear_cross_entropy(*leaves, target)[0].sum().backward()
        assert torch.equal(leaves[asked].grad, want[asked]) and leaves[1 - asked].grad is None


def test_offsets_that_pass_32_bits():
    # a table of more than 4 GiB and its gradient; the targets are its last words
    t, v, k = 70, 600000, 4096
    g = torch.Generator(device=DEV).manual_seed(12)
    hidden = torch.randn(t, k, device=DEV, generator=g, dtype=torch.bfloat16)
    weight = torch.zeros(v, k, device=DEV, dtype=torch.bfloat16)
    weight[-500:] = torch.randn(500, k, device=DEV, generator=g) * 0.03
    target = v - 1 - torch.arange(t, device=DEV)
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    z, off = ref.product(hidden, weight[-500:])
    zeros = torch.full((t, 1), float(torch.tensor(float(v - 500)).double().log()), device=DEV, dtype=torch.float64)   # exp(0), v - 500 times
    want_lse = torch.logsumexp(torch.cat([z, zeros], 1), 1)
    bound = off.amax(1) + ref.FN * (1 + want_lse.abs())
    ref.assert_within(lse, want_lse, bound)
    ref.assert_within(loss, want_lse - z.gather(1, (target - v + 500)[:, None])[:, 0], 2 * bound)
    grad_hidden, grad_weight = ops.linear_cross_entropy_backward(torch.ones(t, device=DEV), hidden, weight, target, lse)
    p = torch.exp(z - want_lse[:, None]) - torch.nn.functional.one_hot(target - v + 500, 500).double()
    for got, want in ((grad_hidden, p @ weight[-500:].double()), (grad_weight[-500:], p.t().contiguous() @ hidden.double()),
                      (grad_weight[:3], torch.exp(-want_lse).sum(0) * 0 + (torch.exp(-want_lse)[:, None] * hidden.double()).sum(0).expand(3, k))):
        assert (got.double() - want).norm() <= 2 * ref.half_step(torch.bfloat16) * want.norm() * 1.5


@pytest.mark.parametrize("t", [1, 2, 3])
def test_few_tokens_and_a_table_of_very_many_words(t):
    # rows of softmax gradients that 32-bit offsets would not reach 63 of: pieces of the vocabulary
    v, k, some = 34_100_001, 8, 500
    assert _capi.load().tf_linear_cross_entropy_backward_piece(t, v, k) < v
    g = torch.Generator(device=DEV).manual_seed(14)
    hidden = torch.randn(t, k, device=DEV, generator=g, dtype=torch.bfloat16)
    weight = torch.randn(v, k, device=DEV, generator=g, dtype=torch.bfloat16)
    target = torch.tensor([v - 1, 7, 1 << 25], device=DEV)[:t]   # the last word, one in front, the first of the second piece
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    grad_hidden, grad_weight = ops.linear_cross_entropy_backward(torch.ones(t, device=DEV), hidden, weight, target, lse)
    z, off = ref.product(hidden, weight)
    want_lse = torch.logsumexp(z, 1)
    bound = off.amax(1) + ref.FN * (1 + want_lse.abs())
    ref.assert_within(lse, want_lse, bound)
    ref.assert_within(loss, want_lse - z.gather(1, target[:, None])[:, 0], 2 * bound)
    p = torch.exp(z - want_lse[:, None])
    p[torch.arange(t, device=DEV), target] -= 1
    want = p @ weight.double()
    assert (grad_hidden.double() - want).norm() <= 3 * ref.half_step(torch.bfloat16) * want.norm()
    for words in (slice(0, some), slice((1 << 25) - some, (1 << 25) + some), slice(v - some, v)):
        want = p[:, words].t().contiguous() @ hidden.double()
        assert (grad_weight[words].double() - want).norm() <= 3 * ref.half_step(torch.bfloat16) * want.norm()


def test_more_tiles_than_a_launch_has():
    # 2^24 tiles of 64 x 64, the only ones for so few columns: 511 rows of them at a time
    t, v, k = 65530, 1 << 20, 8
    hidden, weight, target, _ = _head(t, v, k, torch.bfloat16, seed=19)
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    for at in (0, 511 * 64 - 20, 2 * 511 * 64 - 20, t - 40):
        rows = slice(at, at + 40)
        (want_loss, want_lse), bounds = ref.linear_cross_entropy(hidden[rows], weight, target[rows], -100)
        ref.assert_within(lse[rows], want_lse, bounds[1], f"lse {at}")
        ref.assert_within(loss[rows], want_loss, bounds[0], f"loss {at}")


def test_shapes_strides_and_alignment():
    hidden, weight, target, g = _head(60, 300, 80, torch.float16, seed=3)
    _check_forward(hidden.view(3, 20, 80), weight, target.view(3, 20))
    _check_forward(hidden.view(3, 20, 80).transpose(0, 1), weight, target.view(3, 20).t())
    wide = torch.randn(300, 100, device=DEV, generator=g).half()
    _check_forward(hidden, wide[:, 20:], target)
    flat = torch.randn(300 * 80 + 1, device=DEV, generator=g).half()
    _check_forward(flat[1:60 * 80 + 1].view(60, 80), flat[1:].view(300, 80), target)
    _check_backward(torch.rand(3, 20, device=DEV, generator=g), hidden.view(3, 20, 80), wide[:, 20:], target.view(3, 20))
    _check_backward(torch.rand(60, device=DEV, generator=g), flat[1:60 * 80 + 1].view(60, 80), flat[1:].view(300, 80), target)
    _check_backward(torch.ones(1, device=DEV).expand(60), hidden, weight, target)   # the gradient of a sum
    one = hidden[0], weight, target[0] * 0
    assert ops.linear_cross_entropy(*one)[0].shape == ()


def test_ignored_and_invalid_targets():
    hidden, weight, target, g = _head(200, 500, 64, torch.bfloat16, seed=4, ignored=False)
    grad_loss = torch.rand(200, device=DEV, generator=g)
    target[::3] = 7
    _check_forward(hidden, weight, target, ignore_index=7)      # a word of the vocabulary may be the ignored one
    _check_backward(grad_loss, hidden, weight, target, ignore_index=7)
    # nothing of an ignored token's gradient is looked at
    bad = grad_loss.clone()
    bad[::3] = float("nan")
    lse = ops.linear_cross_entropy(hidden, weight, target, 7)[1]
    for a, b in zip(ops.linear_cross_entropy_backward(bad, hidden, weight, target, lse, 7),
                    ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse, 7)):
        assert torch.equal(a, b)
    everything = torch.full_like(target, -100)
    loss, lse = ops.linear_cross_entropy(hidden, weight, everything)
    assert (loss == 0).all() and lse.isfinite().all()
    for grad in ops.linear_cross_entropy_backward(grad_loss, hidden, weight, everything, lse):
        assert (grad == 0).all()
    for word in (-1, 500, 1 << 40, -(1 << 40)):
        target[5] = word
        loss, lse = ops.linear_cross_entropy(hidden, weight, target, 7)
        assert loss.isnan().nonzero().flatten().tolist() == [5] and lse.isfinite().all()
        grad_hidden, grad_weight = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse, 7)
        assert grad_weight.isnan().all() and grad_hidden[5].isnan().all() and grad_hidden[:5].isfinite().all() and grad_hidden[6:].isfinite().all()


@pytest.mark.parametrize("t,v,k", [(1, 100, 64), (37, 1000, 72), (200, 513, 65), (613, 3001, 128), (1100, 700, 264)])
@pytest.mark.parametrize("dtype", TYPES)
def test_whatever_stands_in_an_ignored_tokens_row(t, v, k, dtype):
    # a padded batch: rows that nothing was ever written to
    hidden, weight, target, g = _head(t, v, k, dtype, seed=15, ignored=False)
    grad_loss = torch.rand(t, device=DEV, generator=g)
    target[::3] = -100
    clean = hidden.clone()
    clean[::3] = 0
    hidden[::3, ::2], hidden[::3, 1::2] = float("nan"), float("inf")
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    want_loss, want_lse = ops.linear_cross_entropy(clean, weight, target)
    counted = target != -100
    assert torch.equal(loss, want_loss) and torch.equal(lse[counted], want_lse[counted]) and (loss[::3] == 0).all()
    want = ops.linear_cross_entropy_backward(grad_loss, clean, weight, target, want_lse)
    for of_hidden, of_weight in ((True, True), (True, False), (False, True)):
        got = _one(grad_loss, hidden, weight, target, lse, -100, of_hidden, of_weight)
        for a, b in zip(got, want if of_hidden and of_weight else _one(grad_loss, clean, weight, target, want_lse, -100, of_hidden, of_weight)):
            assert b is None if a is None else a.isfinite().all() and torch.equal(a, b)
    assert (want[0][::3] == 0).all()


def test_infinite_logits_and_nan_stay_with_their_token():
    hidden, weight, target, _ = _head(150, 300, 64, torch.float16, seed=5, ignored=False)
    clean = ops.linear_cross_entropy(hidden, weight, target)
    bad = hidden.clone()
    bad[4, 0] = float("nan")
    bad[100] = 0
    bad[100, 1] = float("inf")    # logits of both infinities
    loss, lse = ops.linear_cross_entropy(bad, weight, target)
    rows = torch.ones(150, dtype=torch.bool, device=DEV)
    rows[[4, 100]] = False
    assert torch.equal(loss[rows], clean[0][rows]) and torch.equal(lse[rows], clean[1][rows])
    assert loss[4].isnan() and not lse[100].isfinite()
    # words that cannot occur: logits of -inf take no part
    weight[::2] = 0
    weight[::2, 0] = -float("inf")
    hidden[:, 0] = 1.0
    target = target // 2 * 2 + 1
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    (want_loss, want_lse), bounds = ref.linear_cross_entropy(hidden, weight[1::2].contiguous(), target // 2, -100)
    ref.assert_within(lse, want_lse, bounds[1])
    ref.assert_within(loss, want_loss, bounds[0])
    weight[:] = 0
    weight[:, 0] = -float("inf")
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    assert (lse == -float("inf")).all()


def test_large_logits_do_not_overflow():
    hidden, weight, target, _ = _head(64, 200, 128, torch.bfloat16, seed=6)
    _check_forward(hidden * 64, weight * 64, target)
    _check_backward(torch.ones(64, device=DEV), hidden * 16, weight * 16, target)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [1e-30, 1e-7, 1.0, 1e4])
def test_the_size_of_grad_loss_does_not_matter(dtype, size):
    # exact powers of two apart, results are exact powers of two apart (bf16; fp16 as far as its results reach)
    hidden, weight, target, g = _head(90, 400, 64, dtype, seed=7)
    grad_loss = torch.rand(90, device=DEV, generator=g)
    lse = ops.linear_cross_entropy(hidden, weight, target)[1]
    by = 2.0 ** round(__import__("math").log2(size))
    base = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse)
    got = ops.linear_cross_entropy_backward(grad_loss * by, hidden, weight, target, lse)
    for a, b in zip(got, base):
        assert (a.double() - b.double() * by).abs().max() <= (ref.TINY[dtype] if dtype == torch.bfloat16 or by <= 1 else float("inf"))+ (
            0 if dtype == torch.bfloat16 else 2 * ref.half_step(dtype) * (b.double() * by).abs().max())


@pytest.mark.parametrize("size", [2.0 ** -20, 1.0, 4096.0])
@pytest.mark.parametrize("dtype", TYPES)
def test_an_infinite_grad_loss_does_not_take_the_others_range(dtype, size):
    hidden, weight, target, g = _head(90, 400, 64, dtype, seed=21, ignored=False)
    grad_loss = (torch.rand(90, device=DEV, generator=g) + 0.25) * size
    lse = ops.linear_cross_entropy(hidden, weight, target)[1]
    want, bounds = ref.linear_cross_entropy_backward(grad_loss, hidden, weight, target, -100)
    others = torch.arange(90, device=DEV) != 7
    for bad in (float("inf"), -float("inf"), float("nan")):
        grad_loss[7] = bad
        grad_hidden, grad_weight = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse)
        ref.assert_within(grad_hidden[others], want[0][others], bounds[0][others], str(bad))
        assert not grad_hidden[7].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("size", [2.0 ** -40, 2.0 ** -10, 1.0, 2.0 ** 13, 2.0 ** 15])
def test_backward_within_bounds_at_any_size_of_grad_loss(dtype, size):
    # large ones in fp16 as well, up to results beyond the type, which are infinities of their sign and nothing else
    hidden, weight, target, g = _head(90, 400, 64, dtype, seed=22)
    grad_loss = (torch.rand(90, device=DEV, generator=g) - 0.5) * size
    lse = ops.linear_cross_entropy(hidden, weight, target)[1]
    grads = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse)
    want, bounds = ref.linear_cross_entropy_backward(grad_loss, hidden, weight, target, -100)
    for got, a, bound in zip(grads, want, bounds):
        number = ref.assert_within(got, a, bound, str(size))
        rest = torch.where(number, got.double() - a, torch.zeros_like(a))
        assert rest.norm() <= 2 * ref.half_step(dtype) * a.norm() + a.numel() ** 0.5 * ref.TINY[dtype]
        assert number.float().mean() > 0.5


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", ["mean", "sequences"])
def test_one_weight_for_many_tokens_is_not_rounded_as_one(dtype, kind):
    """The largest term of a gradient is a token's grad_loss itself: rounded to 16 bits it would be off by the same for all tokens of the same
    grad_loss, here just over halfway between two numbers of the type and just over a power of two, where that is most."""
    t, v, k = 512, 4096, 256
    hidden, weight, target, g = _head(t, v, k, dtype, seed=13, ignored=False)
    step = 2 * ref.half_step(dtype)
    grad_loss = torch.full((t,), 1 + step * 0.52, device=DEV)
    if kind == "sequences":   # the last one's is another
        grad_loss[-64:] = 0.8
    lse = ops.linear_cross_entropy(hidden, weight, target)[1]
    grads = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse)
    want, _ = ref.linear_cross_entropy_backward(grad_loss, hidden, weight, target, -100)
    # Errors that are independent from element to element: of rounding the result (1), of m * hidden (1, for the weight where m is not 1), and of softmax
    # gradients, p - 1 at the target, p up to a few hundredths (under 0.6): at most sqrt(1 + 1 + 0.36) = 1.54 times the result's alone.  Rounded
    # as one number: half a step over 1 is 2.4 times that (uniform errors: sqrt(3) times over their mean square, 1.4 for the binade), 2.6 in all.
    for got, a in zip(grads, want):
        alone = (a.to(dtype).double() - a).norm()
        assert (got.double() - a).norm() <= 1.75 * alone, (got.double() - a).norm() / alone


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("padding", [1, 3, 4, 64, 255, 256, 257, 700])
def test_one_weight_for_the_tokens_of_a_padded_batch(dtype, padding):
    # as above, of a mean, with tokens behind the last one that counts: nothing is rounded with hidden, whose part would be 1.4 times the result's
    t, v, k = 512, 4096, 256
    hidden, weight, target, g = _head(t + padding, v, k, dtype, seed=20, ignored=False)
    target[t:] = -100
    grad_loss = torch.full((t + padding,), 1 + 2 * ref.half_step(dtype) * 0.52, device=DEV)
    lse = ops.linear_cross_entropy(hidden, weight, target)[1]
    grads = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse)
    want, _ = ref.linear_cross_entropy_backward(grad_loss, hidden, weight, target, -100)
    for got, a in zip(grads, want):
        # the result's rounding, and that of the softmax gradients (0.6 of it at most): sqrt(1 + 0.36) = 1.17
        alone = (a.to(dtype).double() - a).norm()
        assert (got.double() - a).norm() <= 1.25 * alone, (got.double() - a).norm() / alone
    alike = ops.linear_cross_entropy_backward(grad_loss[:t], hidden[:t], weight, target[:t], lse[:t])
    assert (grads[0][t:] == 0).all()
    for got, a in zip((grads[0][:t], grads[1]), alike):   # (sums may be cut otherwise)
        assert (got.double() - a.double()).norm() <= 2 * ref.half_step(dtype) * a.double().norm()


def test_gradient_against_differences():
    # the loss itself along a direction: central differences of step 2^-4 on values that are multiples of it (exact in fp16)
    g = torch.Generator(device=DEV).manual_seed(8)
    t, v, k = 40, 96, 48
    grid = lambda *s: (torch.randint(-8, 9, s, device=DEV, generator=g) / 16).half()   # noqa: E731
    hidden, weight, target = grid(t, k), grid(v, k), torch.randint(0, v, (t,), device=DEV, generator=g)
    lse = ops.linear_cross_entropy(hidden, weight, target)[1]
    grad_hidden, grad_weight = ops.linear_cross_entropy_backward(torch.ones(t, device=DEV), hidden, weight, target, lse)
    step = 1.0 / 16
    total = lambda h, w: ops.linear_cross_entropy(h, w, target)[0].double().sum().item()   # noqa: E731
    for k_at in (0, 17, 47):
        e = torch.zeros_like(hidden)
        e[:, k_at] = step
        along = grad_hidden[:, k_at].double().sum().item()
        # the third derivative of lse along a coordinate is at most the largest |weight|^3 = 1/8, times step^2 / 6, each of t tokens
        assert abs((total(hidden + e, weight) - total(hidden - e, weight)) / (2 * step) - along) <= t * (step ** 2 / 48 + 2.0 ** -11 + FAR / step)
        e = torch.zeros_like(weight)
        e[:5, k_at] = step
        along = grad_weight[:5, k_at].double().sum().item()
        assert abs((total(hidden, weight + e) - total(hidden, weight - e)) / (2 * step) - along) <= t * (step ** 2 / 48 + 2.0 ** -11 + FAR / step)


FAR = 2.0 ** -19   # of a loss near 5: its fp32 error


def test_any_workspace():
    t, v, k = 150, 1000, 40
    hidden, weight, target, g = _head(t, v, k, torch.bfloat16, seed=9)
    grad_loss = torch.rand(t, device=DEV, generator=g)
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    grads = ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse)
    lib, st = _capi.load(), torch.cuda.current_stream().cuda_stream
    size = lib.tf_linear_cross_entropy_workspace_bytes(t, v, k)
    room = torch.full((size + 64,), 0xFF, device=DEV, dtype=torch.uint8)
    got = [torch.full((t,), float("nan"), device=DEV) for _ in range(2)]
    _capi.check(lib.tf_linear_cross_entropy(*(x.data_ptr() for x in (hidden, weight, target, *got)), _capi.TF_DTYPE_BF16, t, v, k, -100, room.data_ptr(),
                                            size, st), "tf_linear_cross_entropy")
    assert torch.equal(got[0], loss) and torch.equal(got[1], lse) and (room[size:] == 0xFF).all()
    size = lib.tf_linear_cross_entropy_backward_workspace_bytes(t, v, k)
    room = torch.full((size + 64,), 0xFF, device=DEV, dtype=torch.uint8)
    got = [torch.full_like(x, float("nan")) for x in (hidden, weight)]
    _capi.check(lib.tf_linear_cross_entropy_backward(*(x.data_ptr() for x in (grad_loss, hidden, weight, target, lse, *got)), _capi.TF_DTYPE_BF16, t, v, k,
                                                     -100, room.data_ptr(), size, st), "tf_linear_cross_entropy_backward")
    assert torch.equal(got[0], grads[0]) and torch.equal(got[1], grads[1]) and (room[size:] == 0xFF).all()


def test_autograd_replay_streams_and_empty():
    hidden, weight, target, g = _head(120, 900, 72, torch.bfloat16, seed=10)
    leaves = [hidden.clone().requires_grad_(), weight.clone().requires_grad_()]
    loss, lse = ops.linear_cross_entropy(*leaves, target)
    assert not lse.requires_grad
    valid = int((target != -100).sum())
    (loss.sum() / valid).backward()
    want = ops.linear_cross_entropy_backward(torch.full((120,), 1.0 / valid, device=DEV), hidden, weight, target, lse)
    assert torch.equal(leaves[0].grad, want[0]) and torch.equal(leaves[1].grad, want[1])

    grad_loss = torch.rand(120, device=DEV, generator=g)

    def step():
        loss, lse = ops.linear_cross_entropy(hidden, weight, target)
        return (loss, *ops.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse))

    want = [x.clone() for x in step()]
    results = []
    for side in [torch.cuda.Stream() for _ in range(2)]:
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):
                results.append(step())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for got in results for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for n in range(4):
        hidden.mul_(0.5 if n % 2 else 2.0)
        grad_loss.mul_(3.0)
        want = [x.clone() for x in step()]
        for x in out:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.linear_cross_entropy(leaves[0], weight, target)

    none = hidden[:0], weight, target[:0]
    loss, lse = ops.linear_cross_entropy(*none)
    assert loss.shape == (0,) == lse.shape
    grad_hidden, grad_weight = ops.linear_cross_entropy_backward(loss, *none, lse)
    assert grad_hidden.shape == (0, 72) and (grad_weight == 0).all()


@pytest.mark.parametrize("asked", [(0,), (1,), (0, 1)])
def test_autograd_of_no_tokens(asked):
    leaves = [torch.randn(*s, device=DEV).bfloat16().requires_grad_(i in asked) for i, s in enumerate(((0, 24), (100, 24)))]
    ops.linear_cross_entropy(*leaves, torch.empty(0, device=DEV, dtype=torch.int64))[0].sum().backward()
    for i, leaf in enumerate(leaves):
        assert (leaf.grad == 0).all() and leaf.grad.shape == leaf.shape if i in asked else leaf.grad is None


def test_refusals():
    hidden, weight, target, _ = _head(8, 32, 16, torch.float16)
    for bad in ((hidden, weight.bfloat16(), target), (hidden, weight[:, :8], target), (hidden, weight, target[:4]), (hidden, weight, target.int()),
                (hidden.float(), weight.float(), target), (hidden, weight.cpu(), target), (hidden, weight[0], target), (hidden[:, :0], weight[:, :0], target),
                (hidden, weight[:0], target)):
        with pytest.raises(RuntimeError):
            ops.linear_cross_entropy(*bad)
    loss, lse = ops.linear_cross_entropy(hidden, weight, target)
    for bad in ((loss.half(), hidden, weight, target, lse), (loss[:4], hidden, weight, target, lse), (loss, hidden, weight, target, lse.double()),
                (loss, hidden, weight, target, lse[:2])):
        with pytest.raises(RuntimeError):
            ops.linear_cross_entropy_backward(*bad)
