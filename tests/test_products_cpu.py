"""CPU-only checks of gemm_int8, quantize_rows, gated_ffn and linear_cross_entropy: what the C ABI refuses before it touches the device, and
the 64-bit forms that the GPU tests compare with, their gradients against differences."""

import ctypes

import pytest
import torch

from tests import product_ref as ref
from tilefusion_amd import _capi, ops

P = 0x1000   # never dereferenced: validation fails first
F16, BF16, F32 = _capi.TF_DTYPE_F16, _capi.TF_DTYPE_BF16, _capi.TF_DTYPE_F32
BAD, UNSUPPORTED, OK = _capi.TF_ERR_INVALID_ARG, _capi.TF_ERR_UNSUPPORTED, _capi.TF_OK


def test_gemm_int8_arguments():
    lib = _capi.load()
    f, none = lib.tf_gemm_int8, (None, 0, None)
    assert f(P, P, P, P, P, F32, 4, 4, 0, *none) == BAD and f(P, P, P, P, P, F32, -1, 4, 16, *none) == BAD
    assert f(P, P, P, P, P, 3, 4, 4, 16, *none) == UNSUPPORTED
    assert f(P, P, P, P, P, F16, 4, 4, 131072, *none) == BAD and b"131071" in lib.tf_last_error()
    assert f(P, P, P, P, P, F16, 1 << 30, 4, 16, *none) == BAD
    for at in range(5):
        pointers = [P] * 5
        pointers[at] = None
        assert f(*pointers, F16, 4, 4, 16, *none) == BAD
    assert f(None, None, None, None, None, F16, 0, 4, 4, *none) == OK == f(None, None, None, None, None, F16, 4, 0, 4, *none)
    # rows that 16-byte requests cannot walk: room for copies of them
    size = lib.tf_gemm_int8_workspace_bytes
    assert size(7, 9, 160) == 0 == size(0, 9, 17) == size(7, 9, 131072) and size(7, 9, 17) == 16 * 128
    assert f(P, P, P, P, P, F16, 7, 9, 17, P, size(7, 9, 17) - 1, None) == BAD and b"workspace" in lib.tf_last_error()
    assert f(P, P, P, P, P, F16, 7, 9, 17, P + 8, size(7, 9, 17), None) == BAD == f(P, P, P, P, P, F16, 7, 9, 17, None, size(7, 9, 17), None)
    assert f(P + 8, P, P, P, P, F16, 7, 9, 160, *none) == BAD == f(P, P + 1, P, P, P, F16, 7, 9, 160, *none)


def test_quantize_rows_arguments():
    f = _capi.load().tf_quantize_rows
    assert f(P, P, P, F32, 4, 4, None) == UNSUPPORTED and f(P, P, P, F16, 4, 0, None) == BAD and f(P, P, P, F16, 1 << 24, 4, None) == BAD
    assert f(None, P, P, F16, 4, 4, None) == BAD == f(P, None, P, F16, 4, 4, None) == f(P, P, None, F16, 4, 4, None) == f(P, P, P, F16, -1, 4, None)
    assert f(None, None, None, F16, 0, 4, None) == OK


def test_gated_ffn_arguments():
    lib = _capi.load()
    f, none = lib.tf_gated_ffn, (None, 0, None)
    assert f(P, P, P, P, None, None, F32, 0, 4, 4, 8, *none) == UNSUPPORTED
    assert f(P, P, P, P, None, None, F16, 3, 4, 4, 8, *none) == BAD and b"activation" in lib.tf_last_error()
    assert f(P, P, P, P, P, None, F16, 0, 4, 4, 8, *none) == BAD and f(P, P, P, None, P, P, F16, 0, 4, 4, 8, *none) == BAD
    for m, n, k in ((-1, 4, 8), (4, 0, 8), (4, 4, 0), (1 << 22, 4, 8), (4, 1 << 21, 8), (4, 4, 1 << 22)):
        assert f(P, P, P, P, None, None, F16, 0, m, n, k, *none) == BAD
    assert f(None, None, None, None, None, None, F16, 0, 0, 4, 4, *none) == OK
    for at in range(3):
        pointers = [P] * 4
        pointers[at] = P + 2
        assert f(*pointers, None, None, F16, 0, 4, 4, 8, *none) == BAD and b"boundaries" in lib.tf_last_error()
    size = lib.tf_gated_ffn_workspace_bytes
    assert size(4, 5, 8) == 0 == size(0, 5, 9) and size(4, 5, 9) == (4 + 10) * 128
    assert f(P, P, P, P, None, None, F16, 0, 4, 5, 9, P, size(4, 5, 9) - 1, None) == BAD and b"workspace" in lib.tf_last_error()
    size = lib.tf_gated_ffn_backward_workspace_bytes
    assert size(0, 4, 4) == 0 == size(4, 0, 4) == size(1 << 22, 4, 4) and size(64, 64, 64) > 0
    b = lib.tf_gated_ffn_backward
    want = size(64, 64, 64)
    assert b(*[P] * 9, F16, 0, 64, 64, 64, P, want - 1, None) == BAD and b"workspace" in lib.tf_last_error()
    assert b(*[P] * 9, F16, 0, 64, 64, 64, P + 8, want, None) == BAD and b(*[P] * 9, F16, 0, 64, 64, 64, None, want, None) == BAD
    for gone in ([0], [1], [2], [3], [4], [5], [7], [8], [6, 7, 8], [6, 7]):   # (no gradient, or that of one weight)
        pointers = [None if at in gone else P for at in range(9)]
        assert b(*pointers, F16, 0, 64, 64, 64, P, want, None) == BAD, gone
    assert b(*[P + 2] * 9, F16, 0, 64, 64, 64, P, want, None) == BAD and b"boundaries" in lib.tf_last_error()


def test_linear_cross_entropy_arguments():
    lib = _capi.load()
    for f, size, n in ((lib.tf_linear_cross_entropy, lib.tf_linear_cross_entropy_workspace_bytes, 5),
                       (lib.tf_linear_cross_entropy_backward, lib.tf_linear_cross_entropy_backward_workspace_bytes, 7)):
        want = size(8, 100, 64)
        assert want > 0 and size(0, 100, 64) == 0 == size(8, 0, 64) == size(8, 100, 0) == size(1 << 22, 100, 64)
        assert f(*[P] * n, F32, 8, 100, 64, -100, P, want, None) == UNSUPPORTED
        assert f(*[P] * n, F16, 8, 100, 64, -100, P, want - 1, None) == BAD and b"workspace" in lib.tf_last_error()
        assert f(*[P] * n, F16, 8, 100, 64, -100, P + 4, want, None) == BAD == f(*[P] * n, F16, 8, 100, 64, -100, None, want, None)
        for sizes in ((-1, 100, 64), (8, 0, 64), (8, 100, 0), (8, 1 << 28, 64), (8, 100, 1 << 22)):
            assert f(*[P] * n, F16, *sizes, -100, P, want, None) == BAD
        for gone in [[at] for at in range(5)] + ([[5, 6]] if n == 7 else []):
            pointers = [None if at in gone else P for at in range(n)]
            assert f(*pointers, F16, 8, 100, 64, -100, P, want, None) == BAD, gone
        assert f(*[P + 2] * n, F16, 8, 100, 64, -100, P, want, None) == BAD and b"boundaries" in lib.tf_last_error()
    assert lib.tf_linear_cross_entropy(*[None] * 5, F16, 0, 100, 64, -100, None, 0, None) == OK


def test_gradients_of_no_tokens_alone():
    # a tensor without elements has no address: that of grad_x, asked for without the weights' (as where they are frozen), is null
    lib = _capi.load()
    for f in (F16, BF16):
        assert lib.tf_gated_ffn_backward(*[None] * 9, f, 0, 0, 64, 64, None, 0, None) == OK
        assert lib.tf_linear_cross_entropy_backward(*[None] * 7, f, 0, 100, 64, -100, None, 0, None) == OK
    assert lib.tf_gated_ffn_backward(*[None] * 8, P, F16, 0, 0, 64, 64, None, 0, None) == BAD   # of one weight


def test_workspace_of_the_backward_pass_is_a_piece_of_the_vocabulary():
    size = _capi.load().tf_linear_cross_entropy_backward_workspace_bytes
    # 8192 tokens x 131072 words: the logits are 2 GiB in 16 bits; and it does not grow with the vocabulary from some size on
    assert size(8192, 131072, 1024) < 2 ** 30 and size(8192, 131072, 1024) == size(8192, 1 << 20, 1024)


def test_wrappers_refuse_on_the_cpu():
    x, w = torch.zeros(4, 8).half(), torch.zeros(6, 8).half()
    for call in (lambda: ops.gated_ffn(x, w, w), lambda: ops.quantize_rows(x), lambda: ops.linear_cross_entropy(x, w, torch.zeros(4, dtype=torch.long)),
                 lambda: ops.gemm_int8(x.char(), w.char(), torch.ones(4), torch.ones(6), torch.zeros(4, 6))):
        with pytest.raises((NotImplementedError, RuntimeError)):
            call()
    with pytest.raises(RuntimeError, match="must be"):
        ops.gated_ffn(x, w[:, :4], w[:, :4])
    with pytest.raises(RuntimeError, match="target"):
        ops.linear_cross_entropy(x, w, torch.zeros(5, dtype=torch.long))


def test_schemas():
    want = {
        "quantize_rows": "(Tensor x, Tensor(a!) q, Tensor(b!) scale) -> ()",
        "gemm_int8": "(Tensor A, Tensor B, Tensor scale_a, Tensor scale_b, Tensor(a!) C) -> ()",
        "gated_ffn": "(Tensor x, Tensor w_gate, Tensor w_up, str activation, Tensor(a!) h, Tensor(b!)? gate, Tensor(c!)? up) -> ()",
        "gated_ffn_backward": "(Tensor grad_h, Tensor x, Tensor w_gate, Tensor w_up, Tensor gate, Tensor up, str activation, Tensor(a!)? grad_x, Tensor(b!)? grad_w) -> ()",
        "linear_cross_entropy": "(Tensor hidden, Tensor weight, Tensor target, int ignore_index, Tensor(a!) loss, Tensor(b!) lse) -> ()",
        "linear_cross_entropy_backward": "(Tensor grad_loss, Tensor hidden, Tensor weight, Tensor target, Tensor lse, int ignore_index, Tensor(a!)? grad_hidden, Tensor(b!)? grad_weight) -> ()",
    }
    for name, schema in want.items():
        assert str(getattr(torch.ops.tilefusion, name).default._schema) == f"tilefusion::{name}{schema}"
        assert callable(getattr(ops, name))


# ---- the formulas --------------------------------------------------------------------------
@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_activation_slope_against_differences(activation):
    g = torch.linspace(-9, 9, 1801, dtype=torch.float64)
    step = 1e-5
    differences = (ref.act(g + step, activation) - ref.act(g - step, activation)) / (2 * step)
    assert (ref.act_slope(g, activation) - differences).abs().max() < 1e-9   # step^2 and 1e-16 / step
    assert ref.act_slope(g, activation).abs().max() < 1.13                   # (what the bounds count with)
    plain = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu,
             "gelu_tanh": lambda x: torch.nn.functional.gelu(x, approximate="tanh")}[activation]
    assert (ref.act(g, activation) - plain(g)).abs().max() < 1e-13


@pytest.mark.parametrize("activation", ["silu", "gelu", "gelu_tanh"])
def test_gated_ffn_gradients_against_autograd(activation):
    gen = torch.Generator().manual_seed(1)
    x, w_gate, w_up, grad_h = (torch.randn(*s, generator=gen).bfloat16() for s in ((7, 5), (6, 5), (6, 5), (7, 6)))
    leaves = [t.double().requires_grad_() for t in (x, w_gate, w_up)]
    gate, up = leaves[0] @ leaves[1].t(), leaves[0] @ leaves[2].t()
    want = torch.autograd.grad((ref.act(gate, activation) * up * grad_h.double()).sum(), leaves)
    got, bounds = ref.gated_ffn_backward(grad_h, x, w_gate, w_up, gate.detach(), up.detach(), activation)
    for a, b, bound in zip(got, want, bounds):
        assert (a - b).abs().max() < 1e-12 and (bound > 0).all()


def test_linear_cross_entropy_gradients_against_autograd():
    gen = torch.Generator().manual_seed(2)
    hidden, weight = (torch.randn(*s, generator=gen).half() for s in ((9, 5), (11, 5)))
    target, grad_loss = torch.randint(0, 11, (9,), generator=gen), torch.rand(9, generator=gen)
    target[::4] = -100
    leaves = [t.double().requires_grad_() for t in (hidden, weight)]
    loss = torch.nn.functional.cross_entropy(leaves[0] @ leaves[1].t(), target, reduction="none")
    (want_loss, _), _ = ref.linear_cross_entropy(hidden, weight, target, -100)
    assert (loss - want_loss).abs().max() < 1e-12
    want = torch.autograd.grad((loss * grad_loss.double()).sum(), leaves)
    got, bounds = ref.linear_cross_entropy_backward(grad_loss, hidden, weight, target, -100)
    for a, b, bound in zip(got, want, bounds):
        assert (a - b).abs().max() < 1e-12 and (bound > 0).all()


def test_the_comparison_sees_a_planted_mistake():
    want, bounds = ref.gated_ffn(torch.randn(8, 64).half(), torch.randn(16, 64).half() / 8, torch.randn(16, 64).half() / 8, "silu")
    good = want[0].to(torch.float16)
    ref.assert_within(good, want[0], bounds[0])
    for at, by in (((3, 5), 1.02), ((0, 0), 0.98)):
        bad = good.clone()
        bad[at] = (want[0][at] * by).half()
        with pytest.raises(AssertionError, match="out of bounds"):
            ref.assert_within(bad, want[0], bounds[0] + 0 * want[0])


# ---- what a call runs, decided on the host ---------------------------------------------------
def test_cases_reach_every_kernel():
    """Every kernel that a call can run is run by a case of the GPU tests."""
    import tests.test_gpu_gated_ffn as ffn
    import tests.test_gpu_gemm_int8 as int8
    import tests.test_gpu_linear_cross_entropy as loss
    lib = _capi.load()

    def padded(k, to, lines):
        return k if k % to == 0 else -(-k // lines) * lines

    one = set(range(17))
    assert {lib.tf_product_kernel_index(m, n, padded(k, 16, 128) // 2, 0) for m, n, k in int8.SIZES + int8.KERNELS} == one
    assert {lib.tf_product_kernel_index(t, v, padded(k, 8, 64), 0) for t, v, k in loss.SIZES + loss.KERNELS} == one
    two = {0, 3, 4, 5, 6, 7, 8, 9, 10, 12, 14, 15, 16}
    assert {lib.tf_product_kernel_index(m, f, padded(k, 8, 64), 1) for m, f, k in ffn.SIZES + ffn.KERNELS} == two


def _cols(m, n, rows):
    parts = ctypes.c_int(0)
    shape = _capi.load().tf_product_cols_plan(m, n, rows, ctypes.byref(parts))
    return shape, parts.value > 1


def _pair(one, other):
    parts = ctypes.c_int(0), ctypes.c_int(0)
    shape = _capi.load().tf_product_pair_plan(*one, *other, *(ctypes.byref(p) for p in parts))
    return None if shape < 0 else (shape, parts[0].value > 1, parts[1].value > 1)


def test_cases_reach_every_form_of_a_gradient():
    import tests.test_gpu_gated_ffn as ffn
    import tests.test_gpu_linear_cross_entropy as loss

    def up(x):
        return -(-x // 64) * 64

    every = {(shape, cut) for shape in range(4) for cut in (False, True)}
    ffn_cases = ffn.BACKWARD_SIZES + ffn.BACKWARD_KERNELS + ffn.BACKWARD_PAIRS   # (each runs with both gradients and with one)
    assert {_cols(m, k, 2 * up(f)) for m, f, k in ffn_cases} == every
    assert {_cols(up(f) + f, k, m) for m, f, k in ffn_cases} == every
    loss_cases = loss.SIZES + loss.BACKWARD_KERNELS + loss.BACKWARD_PAIRS
    assert {_cols(t, k, up(v)) for t, v, k in loss_cases} == every
    assert {_cols(up(v), k, t) for t, v, k in loss_cases} == every

    pairs = {(shape, one, other) for shape in range(4) for one in (False, True) for other in (False, True)}
    assert {_pair((m, k, 2 * up(f)), (up(f) + f, k, m)) for m, f, k in ffn_cases} - {None} == pairs
    assert {_pair((t, k, up(v)), (up(v), k, t)) for t, v, k in loss_cases} - {None} == pairs
    parts = ctypes.byref(ctypes.c_int())
    assert _capi.load().tf_product_pair_plan(4, 4, 0, 4, 4, 4, parts, parts) == -1 == _capi.load().tf_product_pair_plan(4, 4, 4, 4, 4, 4, None, parts)
    plan = _capi.load().tf_product_cols_plan
    assert plan(0, 4, 4, ctypes.byref(ctypes.c_int())) == -1 == plan(4, 4, 4, None) and _capi.load().tf_product_kernel_index(4, 4, 1 << 22, 0) == -1


def test_no_plan_has_more_tiles_than_a_launch():
    lib = _capi.load()
    tile = [(16, 16), (16, 16), (32, 16), (32, 32), (32, 32), (64, 32), (64, 64)] + [(128, 128)] * 3 + [(192, 128), (192, 192), (256, 128), (256, 192), (256, 256), (128, 128), (128, 128)]
    for m, n in ((1, (1 << 28) - 64), (16, (1 << 28) - 64), (100, (1 << 28) - 64), (1 << 20, 16), ((1 << 22) - 64, 64)):
        bm, bn = tile[lib.tf_product_kernel_index(m, n, 64, 0)]
        assert -(-m // bm) * -(-n // bn) < 1 << 23, (m, n)


def test_columns_of_tiles_fit_a_launch():
    """Rows of tiles may take several launches, a row of them may not."""
    lib = _capi.load()
    width = [16, 16, 16, 32, 32, 32, 64, 128, 128, 128, 128, 192, 128, 192, 256, 128, 128]
    for n in ((1 << 28) - 64, (1 << 29) - 64):
        for m in (1, 16, 17, 64, 65, 100, 128, 1000, 1 << 16, 1 << 22, (1 << 30) - 1):
            for k in (8, 32, 64, 72, 1024):
                assert -(-n // width[lib.tf_product_kernel_index(m, n, k, 0)]) < 1 << 23, (m, n, k)
    for m in (1, 17, 1 << 16, (1 << 22) - 64):
        assert lib.tf_product_kernel_index(m, (1 << 21) - 64, 8, 1) in (0, 3, 4, 5, 6)
    assert lib.tf_gemm_int8(P, P, P, P, P, F16, 1, (1 << 29) - 63, 16, None, 0, None) == BAD and b"too large" in lib.tf_last_error()
    assert lib.tf_gemm_int8_workspace_bytes(1, (1 << 29) - 63, 17) == 0


def test_offsets_of_a_gradient_stay_within_32_bits():
    """Lanes walk 64 rows of an operand that is summed over its rows, and up to 256 of one that is not, by 32-bit offsets: from kLead bytes
    in front of the first row on, to its farthest 16 bytes of 512."""
    piece = _capi.load().tf_linear_cross_entropy_backward_piece

    def farthest(rows, pitch):
        return 2 * (rows - 1) * pitch + 512 + 4096

    most = (1 << 28) - 64
    for t in (1, 2, 3, 4, 5, 31, 32, 33, 63, 64, 100, 256, 1000, 32768, (1 << 22) - 64):
        for v in (1, 64, 65, 34_100_000, 34_100_224, 1 << 25, 1 << 26, 1 << 27, most):
            columns = piece(t, v, 8)   # P's pitch
            assert 0 < columns <= -(-v // 64) * 64 and columns % 64 == 0
            assert farthest(64, columns) < 1 << 32 and farthest(min(t, 256), columns) < 1 << 32, (t, v)
    # the gated block's: rows of [dg | du], of weights and of tokens
    f, k = (1 << 21) - 64, (1 << 22) - 64
    assert farthest(256, 2 * f) < 1 << 32 and farthest(64, k) < 1 << 32
    assert piece(0, 4, 4) == -1 == piece(4, 0, 4) == piece(4, 4, 0) == piece(4, 1 << 28, 4)


def test_neither_a_recorded_call_nor_its_backward_pass_is_captured(monkeypatch):
    import importlib
    import types

    leaf = torch.zeros(1, requires_grad=True)
    autograd = importlib.import_module("tilefusion_amd.ops._autograd")
    assert autograd.records("op", leaf) and not autograd.records("op", leaf.detach())
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    assert not autograd.records("op", leaf.detach())
    with pytest.raises(RuntimeError, match="op: .*captured"):
        autograd.records("op", leaf)
    for name, function in (("gated_ffn", "_GatedFfn"), ("linear_cross_entropy", "_LinearCrossEntropy")):
        backward = getattr(importlib.import_module("tilefusion_amd.ops." + name), function).backward
        with pytest.raises(RuntimeError, match=name + ": .*captured"):
            backward(types.SimpleNamespace(needs_input_grad=(True,) * 4), leaf.detach(), None)


# ---- derivatives that there are not ---------------------------------------------------------
def _differentiable():
    gen = torch.Generator().manual_seed(3)
    x, w, grad = (torch.randn(*s, generator=gen).bfloat16() for s in ((4, 8), (6, 8), (4, 6)))
    target, one = torch.tensor([0, 5, 2, -100]), torch.ones(4)
    return x, {
        "gated_ffn": lambda x: ops.gated_ffn(x, w, w),
        "gated_ffn_backward": lambda x: ops.gated_ffn_backward(grad, x, w, w, grad, grad)[0],
        "linear_cross_entropy": lambda x: ops.linear_cross_entropy(x, w, target)[0],
        "linear_cross_entropy_backward": lambda x: ops.linear_cross_entropy_backward(one, x, w, target, one)[0],
    }


@pytest.mark.parametrize("name", list(_differentiable()[1]))
def test_forward_mode_and_transforms_are_refused(name):
    # (their results are written into fresh tensors, whose tangent would be zero)
    x, calls = _differentiable()
    call = calls[name]
    with pytest.raises(RuntimeError, match=f"{name}: there are no forward-mode"):
        torch.func.jvp(call, (x,), (torch.ones_like(x),))
    with pytest.raises(RuntimeError, match=f"{name}: there are no forward-mode"):
        torch.func.jacfwd(call)(x)
    with torch.autograd.forward_ad.dual_level(), torch.no_grad():
        with pytest.raises(RuntimeError, match=f"{name}: there are no forward-mode"):
            call(torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)))
    with pytest.raises(RuntimeError, match=f"{name}: does not work under torch.func"):
        torch.func.grad(lambda x: call(x).float().sum())(x)
    with pytest.raises(RuntimeError, match=f"{name}: does not work under torch.func"):
        torch.func.vmap(call)(torch.stack([x, x]))
    # inside a dual level or a transform, on tensors that have no part in it, the call goes on (to an op that has no kernel on the CPU)
    with torch.autograd.forward_ad.dual_level(), pytest.raises(NotImplementedError):
        call(x)
    with pytest.raises(NotImplementedError):
        torch.func.grad(lambda y: (y * call(x).float().sum()).sum())(torch.ones(3))
