"""gemm_int8 and quantize_rows against 64-bit arithmetic: whole numbers exactly, scaled sums within three roundings and the result's."""

import pytest
import torch

from tests.product_ref import TINY, half_step
from tilefusion_amd import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _ints(g, *shape):
    return torch.randint(-128, 128, shape, device=DEV, dtype=torch.int8, generator=g)


def _expect(a, b, sa, sb):
    return (a.double() @ b.double().t().contiguous()) * sa.double()[:, None] * sb.double()


def _check(a, b, sa, sb, out):
    c = torch.full((a.shape[0], b.shape[0]), float("nan"), device=DEV, dtype=out)
    ops.gemm_int8(a, b, sa, sb, c)
    want = _expect(a, b, sa, sb)
    # int32 -> fp32 and two products, each rounded once; then the result's rounding
    bound = want.abs() * (4 * 2.0 ** -24 + half_step(out) * (out != torch.float32)) + TINY[out]
    # what rounds beyond the largest number of the type is infinite
    most = torch.finfo(out).max * (1 + half_step(out) * 0.5) if out != torch.float32 else float("inf")
    beyond = want.abs() > most * (1 - 2.0 ** -20)
    within = torch.where(beyond, (c.double() == torch.sign(want) * float("inf")) | (want.abs() < most * (1 + 2.0 ** -20)), (c.double() - want).abs() <= bound)
    assert within.all(), f"{tuple(a.shape)} x {tuple(b.shape)} {out}"


SIZES = [
    (1, 1, 1), (1, 1, 16), (1, 64, 64), (1, 4096, 128), (2, 17, 33), (16, 4096, 256), (15, 129, 80), (33, 65, 1040), (64, 64, 128), (63, 257, 144),
    (128, 128, 128), (129, 255, 272), (200, 300, 1000), (256, 256, 512), (257, 511, 1024), (700, 130, 2064), (1000, 1544, 1032), (97, 1999, 4096),
]


# sizes that reach the kernels which those do not (tests/test_products_cpu.py looks)
KERNELS = [
    (1, 1, 528), (889, 172, 144), (179, 583, 128), (334, 438, 144), (381, 792, 3968), (162, 2558, 1824), (746, 1748, 896), (358, 3187, 144), (2835, 5627, 192),
    (1670, 2341, 128), (2120, 3587, 144), (1018, 5500, 128), (1974, 4508, 128), (2103, 5383, 144),
    (108, 12711, 144), (127, 20000, 1040), (33, 55674, 144), (100, 55673, 17),
]


@pytest.mark.parametrize("m,n,k", SIZES + KERNELS)
@pytest.mark.parametrize("out", [torch.float32, torch.float16, torch.bfloat16])
def test_sizes(m, n, k, out):
    g = torch.Generator(device=DEV).manual_seed(m * 7 + n * 3 + k)
    a, b = _ints(g, m, k), _ints(g, n, k)
    sa = torch.rand(m, device=DEV, generator=g) / k
    sb = torch.rand(n, device=DEV, generator=g) - 0.5
    _check(a, b, sa, sb, out)


def test_the_largest_sum_fits():
    # every product 2^14, 131071 of them: 16384 below 2^31
    k = 131071
    a, b = (torch.full((n, k), -128, device=DEV, dtype=torch.int8) for n in (3, 5))
    c = torch.empty(3, 5, device=DEV)
    one = torch.ones(5, device=DEV)
    ops.gemm_int8(a, b, one[:3].clone(), one, c)
    assert (c.double() == float(torch.tensor(k * 16384, dtype=torch.float32))).all()


def test_offsets_that_pass_32_bits():
    # operands and a result of more than 4 GiB each: the last rows
    g = torch.Generator(device=DEV).manual_seed(4)
    m, n, k = 70000, 33000, 65536
    a = torch.randint(-128, 128, (m, k), device=DEV, dtype=torch.int8, generator=g)
    b = torch.randint(-128, 128, (300, k), device=DEV, dtype=torch.int8, generator=g)
    one = torch.ones(m, device=DEV)
    c = torch.empty(m, 300, device=DEV)
    ops.gemm_int8(a, b, one, one[:300], c)
    assert torch.equal(c[-200:].double(), _expect(a[-200:], b, one[-200:], one[:300]).float().double())
    c = torch.empty(300, m, device=DEV)
    ops.gemm_int8(b, a, one[:300], one, c)
    assert torch.equal(c[:, -200:].double(), _expect(b, a[-200:], one[:300], one[-200:]).float().double())
    a, b = a[:, :64].contiguous(), a[:n, :64].contiguous()
    c = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
    ops.gemm_int8(a, b, one, one[:n], c)
    for rows in (slice(0, 300), slice(m // 2, m // 2 + 300), slice(m - 300, m)):
        want = _expect(a[rows], b, one[rows], one[:n])
        assert ((c[rows].double() - want).abs() <= want.abs() * half_step(torch.bfloat16)).all()
    x = torch.randn(40000, 64000, device=DEV, generator=g, dtype=torch.bfloat16)
    q, scale = ops.quantize_rows(x)
    for rows in (slice(0, 4), slice(39990, 40000)):
        want_q, want_scale = _quantized(x[rows])
        assert torch.equal(q[rows], want_q) and torch.equal(scale[rows], want_scale)


def test_more_tiles_than_a_launch_has():
    # more than 2^23 tiles of 64 x 64, the largest for so few columns
    g = torch.Generator(device=DEV).manual_seed(5)
    m, n, k = (1 << 18) + 3, (1 << 17) + 1, 16
    a, b = _ints(g, m, k), _ints(g, n, k)
    sa, sb = torch.rand(m, device=DEV, generator=g), torch.rand(n, device=DEV, generator=g)
    c = torch.empty(m, n, device=DEV, dtype=torch.bfloat16)
    ops.gemm_int8(a, b, sa, sb, c)
    for at in (0, 4093 * 64 - 50, 4094 * 64 - 50, 4095 * 64 - 50, m - 100):
        want = _expect(a[at:at + 100], b, sa[at:at + 100], sb)
        assert ((c[at:at + 100].double() - want).abs() <= want.abs() * (4 * 2.0 ** -24 + half_step(torch.bfloat16)) + TINY[torch.bfloat16]).all(), at


def test_strides_alignment_and_empty():
    g = torch.Generator(device=DEV).manual_seed(3)
    wide = _ints(g, 130, 400)
    a, b = wide[:70, 1:257], _ints(g, 256, 90).t()           # rows that start anywhere, a transposed weight
    sa, sb = torch.rand(140, device=DEV, generator=g)[::2], torch.rand(90, device=DEV, generator=g)
    _check(a, b, sa, sb, torch.float32)
    flat = _ints(g, 64 * 256 + 8)
    _check(flat[3:3 + 64 * 256].view(64, 256), flat[8:].view(64, 256), sa[:64], sb[:64], torch.float16)   # contiguous, at odd addresses
    for m, n in ((0, 8), (8, 0)):
        ops.gemm_int8(torch.empty(m, 16, device=DEV, dtype=torch.int8), torch.empty(n, 16, device=DEV, dtype=torch.int8),
                      torch.empty(m, device=DEV), torch.empty(n, device=DEV), torch.empty(m, n, device=DEV))


def _quantized(x):
    x = x.double()
    scale = (x.abs().amax(dim=-1) / 127).float()
    step = scale.double()[..., None]
    q = torch.where(step > 0, torch.round(x / torch.where(step > 0, step, torch.ones_like(step))), torch.zeros_like(x))
    return q.to(torch.int8), scale


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 7), (3, 8), (5, 64), (2, 255), (16, 4096), (9, 4104), (300, 1032), (1, 20000), (2, 65536), (1025, 33)])
def test_quantize_rows(rows, k, dtype):
    g = torch.Generator(device=DEV).manual_seed(rows + k)
    x = torch.randn(rows, k, device=DEV, generator=g).to(dtype)
    q, scale = ops.quantize_rows(x)
    want_q, want_scale = _quantized(x)
    assert torch.equal(scale, want_scale) and torch.equal(q, want_q)


def test_quantize_rows_every_fp16_value_against_many_steps():
    # all finite positive fp16 numbers up to a row's largest: every middle of two whole numbers among them
    values = torch.arange(0, 31744, device=DEV, dtype=torch.int16).view(torch.float16)
    for top in (31743, 20000, 16000, 15361, 14999, 12345, 3000, 1024, 1000, 254, 127, 5, 1):
        x = torch.cat([values[:top + 1], -values[:top + 1]]).view(1, -1)
        q, scale = ops.quantize_rows(x)
        want_q, want_scale = _quantized(x)
        assert torch.equal(scale, want_scale) and torch.equal(q, want_q), top


def test_quantize_rows_special_rows():
    x = torch.randn(6, 100, device=DEV).half()
    x[1] = 0
    x[2, 50] = float("inf")
    x[3, 99] = float("nan")
    x[4, 0] = -float("inf")
    q, scale = ops.quantize_rows(x.view(2, 3, 100))
    assert q.shape == (2, 3, 100) and scale.shape == (2, 3)
    q, scale = q.view(6, 100), scale.view(6)
    assert scale[1] == 0 and (q[1:5] == 0).all() and scale[2:5].isnan().all() and scale[[0, 5]].isfinite().all()
    c = torch.empty(6, 4, device=DEV)
    ops.gemm_int8(q, torch.ones(4, 100, device=DEV, dtype=torch.int8), scale, torch.ones(4, device=DEV), c)
    assert c[2:5].isnan().all() and (c[1] == 0).all() and c[[0, 5]].isfinite().all()
    q, scale = ops.quantize_rows(torch.empty(0, 5, device=DEV).half())
    assert q.shape == (0, 5) and scale.shape == (0,)
    # rows that start anywhere
    base = torch.randn(10 * 65 + 1, device=DEV).bfloat16()
    for x in (base[1:].view(10, 65), base[:650].view(10, 65)[:, 3:40]):
        q, scale = ops.quantize_rows(x)
        want_q, want_scale = _quantized(x)
        assert torch.equal(scale, want_scale) and torch.equal(q, want_q)


def test_on_another_stream_and_replayed():
    g = torch.Generator(device=DEV).manual_seed(9)
    x = torch.randn(40, 512, device=DEV, generator=g).bfloat16()
    w, sb = _ints(g, 300, 512), torch.rand(300, device=DEV, generator=g)
    c = torch.empty(40, 300, device=DEV, dtype=torch.bfloat16)

    def layer():
        q, scale = ops.quantize_rows(x)
        ops.gemm_int8(q, w, scale, sb, c)

    layer()
    want = c.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.zero_()
        layer()
    side.synchronize()
    assert torch.equal(c, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer()
    for _ in range(4):
        c.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, want)
        x.copy_(torch.randn(40, 512, device=DEV, generator=g))
        layer()
        want = c.clone()


def test_refusals():
    a, b = (torch.zeros(4, 32, device=DEV, dtype=torch.int8) for _ in range(2))
    s, c = torch.ones(4, device=DEV), torch.zeros(4, 4, device=DEV)
    for bad in ((a.half(), b, s, s, c), (a, b[:, :16], s, s, c), (a, b, s[:3], s, c), (a, b, s, s.double(), c), (a, b, s, s, c.double()),
                (a, b, s, s, c[:3]), (a, b.cpu(), s, s, c), (a, b, s, s, torch.zeros(4, 8, device=DEV)[:, ::2]), (a[0], b, s, s, c)):
        with pytest.raises(RuntimeError):
            ops.gemm_int8(*bad)
    for x in (torch.zeros(2, 3, device=DEV), torch.zeros((), device=DEV).half(), torch.zeros(2, 0, device=DEV).half()):
        with pytest.raises(RuntimeError):
            ops.quantize_rows(x)
    assert (c == 0).all()
    assert _capi.load().tf_gemm_int8(a.data_ptr(), b.data_ptr(), s.data_ptr(), s.data_ptr(), c.data_ptr(), 0, 1, 1, 131072, None, 0, None) == _capi.TF_ERR_INVALID_ARG
