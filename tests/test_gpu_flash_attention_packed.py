"""Attention over packed sequences, against the formula in 64 bits."""

import math

import pytest
import torch

from tests import attention_ref as ref
from tilefusion_amd import _capi, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _offsets(lengths, first=0):
    return torch.tensor([first] + (first + torch.tensor(lengths).cumsum(0)).tolist(), dtype=torch.int32, device=DEV)


def _rows(t, s, h, hkv, d, dtype, seed=5):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(n, heads, d, generator=g).to(dtype).to(DEV) for n, heads in ((t, h), (s, hkv), (s, hkv))]


def _want(q, k, v, lq, lkv, scale, causal):
    """Formula and bounds; a weight is rounded once to the type, whose smallest number (fp16) is 2^-24."""
    dtype, group = q.dtype, q.shape[1] // k.shape[1]
    out, bound = (torch.zeros(q.shape, dtype=torch.float64, device=DEV) for _ in range(2))
    lse, lse_bound = torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64, device=DEV), torch.zeros(q.shape[1], q.shape[0], device=DEV)
    floor = 2.0 ** -25 if dtype == torch.float16 else 0.0
    a = b = 0
    for m, n in zip(lq, lkv):
        masked = torch.arange(n, device=DEV)[None] > torch.arange(m, device=DEV)[:, None] + n - m if causal else None
        for head in range(q.shape[1]):
            rows = (slice(a, a + m), head)
            out[rows], lse[head, a:a + m], bound[rows], lse_bound[head, a:a + m] = ref.attend(
                q[rows], k[b:b + n, head // group], v[b:b + n, head // group], scale, masked, ref.half_step(dtype) + 2.0 ** -20, floor)
        a, b = a + m, b + n
    none = lse == -math.inf
    out.masked_fill_(none.t()[:, :, None], 0.0)
    bound.masked_fill_(none.t()[:, :, None], 0.0)
    return out, bound, lse, lse_bound


def _check(lq, lkv=None, h=4, hkv=2, d=64, dtype=torch.bfloat16, causal=True, scale=None, tail=0, rows=None):
    q, k, v = rows or _rows(sum(lq) + tail, sum(lkv or lq) + tail, h, hkv, d, dtype)
    out, lse = ops.flash_attention_packed(q, k, v, _offsets(lq), _offsets(lkv) if lkv else None, scale, causal, True)
    scale = d ** -0.5 if scale is None else scale
    t = sum(lq)
    want, bound, want_lse, lse_bound = _want(q[:t], k, v, lq, lkv or lq, scale, causal)
    ref.assert_within(out[:t], want, bound, "out")
    ref.assert_within(lse[:, :t], want_lse, lse_bound, "lse")
    assert (out[t:] == 0).all() and (lse[:, t:] == -math.inf).all()
    assert torch.equal(ops.flash_attention_packed(q, k, v, _offsets(lq), _offsets(lkv) if lkv else None, scale, causal), out)
    return out, lse


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[1], [2], [15, 16, 17], [0, 31, 0, 0, 33, 64, 65], [127, 1, 129, 200], [513], [1000, 3]])
def test_lengths(dtype, d, causal, lengths):
    _check(lengths, d=d, dtype=dtype, causal=causal, tail=5)


# rows of a workgroup for D = 64 and 128
@pytest.mark.parametrize("rows,lengths,h,hkv", [((64, 64), [100, 31], 4, 2), ((64, 128), [500, 300, 41], 32, 8), ((256, 256), [700, 300, 41, 200], 32, 8),
                                                ((256, 256), [1500, 4, 1200], 32, 8), ((256, 256), [4100], 16, 16), ((128, 128), [130] * 40, 8, 8),
                                                ((256, 256), [2049, 2047], 40, 8)])
@pytest.mark.parametrize("causal", [False, True])
def test_every_kernel(rows, lengths, h, hkv, causal):
    for d, n in zip((64, 128), rows):
        assert _capi.load().tf_flash_attention_packed_rows(sum(lengths), len(lengths), h, hkv, d) == n
        for dtype in (torch.float16, torch.bfloat16):
            _check(lengths, h=h, hkv=hkv, d=d, dtype=dtype, causal=causal)


@pytest.mark.parametrize("h,hkv", [(1, 1), (8, 8), (3, 1), (5, 5), (12, 4), (7, 1), (48, 8), (64, 1), (100, 1)])
def test_groups(h, hkv):
    for causal in (False, True):
        _check([70, 1, 200, 13], h=h, hkv=hkv, causal=causal)
        _check([70, 1, 200, 13], h=h, hkv=hkv, causal=causal, d=128, dtype=torch.float16)


@pytest.mark.parametrize("lq,lkv", [([1, 1, 1], [100, 1, 2000]), ([5, 64, 3], [69, 64, 1000]), ([100, 30, 7, 300], [10, 0, 7, 299]),
                                    ([0, 4, 0], [50, 0, 0]), ([128, 16], [8000, 3])])
@pytest.mark.parametrize("causal", [False, True])
def test_keys_of_another_number(lq, lkv, causal):
    for d, dtype in ((64, torch.bfloat16), (128, torch.float16)):
        _check(lq, lkv, d=d, dtype=dtype, causal=causal, tail=2)
        _check(lq, lkv, h=16, hkv=1, d=d, dtype=dtype, causal=causal)


def test_more_queries_than_keys_in_large_tiles():
    _check([3000, 1500], [700, 1], h=16, hkv=8, d=128)
    _check([3000, 1500], [2999, 1499], h=16, hkv=8, d=64)


@pytest.mark.parametrize("n", [63, 64, 65, 200, 1000])
def test_many_sequences(n):
    g = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 60, (n,), generator=g).tolist()
    _check(lengths, h=2, hkv=1)
    lengths = [x * (20 if i % 17 == 0 else 1) for i, x in enumerate(lengths)]
    _check(lengths, h=4, hkv=1, causal=False)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-4])
def test_scales(scale):
    _check([300, 40], scale=scale)


def test_scores_that_fall_and_rise_along_the_keys():
    # references that are set low and raised late, and sets whose first tiles weigh nothing in the end
    for slope in (-0.5, 0.5):
        q, k, v = _rows(400, 400, 2, 1, 64, torch.float16)
        k[:, 0, 0] = torch.arange(400, device=DEV) * slope
        q[:, :, 0] = 2.0
        _check([400], h=2, hkv=1, dtype=torch.float16, scale=1.0, rows=(q, k, v))


def test_masked_and_unused_rows_are_not_seen():
    # whatever stands behind a row's last key, in other sequences and behind the last one
    for d, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        lengths = [100, 33, 260]
        for h, hkv in ((2, 2), (8, 1), (32, 8)):
            q, k, v = _rows(sum(lengths) + 7, sum(lengths) + 7, h, hkv, d, dtype)
            first = ops.flash_attention_packed(q, k, v, _offsets(lengths))
            for bad in (math.inf, -math.inf, math.nan):
                k2, v2 = k.clone(), v.clone()
                at = 133 + 150   # a token of the last sequence, in the middle of a tile
                k2[at:], v2[at:] = bad, bad
                got = ops.flash_attention_packed(q, k2, v2, _offsets(lengths))
                assert torch.equal(got[:at], first[:at])
                v2 = v.clone()
                v2[at, :, 3] = bad
                got = ops.flash_attention_packed(q, k, v2, _offsets(lengths))
                assert torch.equal(got[:at], first[:at])
                seen = got[at:393, :, 3]
                assert (seen.isnan() if bad != bad else seen == bad).all()
                others = [c for c in range(d) if c != 3]
                assert torch.equal(got[at:393][:, :, others], first[at:393][:, :, others])


def test_slices_of_one_projection_and_turned_layouts():
    lengths, h, hkv, d = [70, 131], 8, 2, 64
    t = sum(lengths)
    wide = _rows(t, t, h + 2 * hkv, hkv, d, torch.bfloat16)[0].flatten(1)
    q, k, v = (x.unflatten(1, (-1, d)) for x in wide.split([h * d, hkv * d, hkv * d], dim=1))
    want = ops.flash_attention_packed(*(x.contiguous() for x in (q, k, v)), _offsets(lengths))
    assert torch.equal(ops.flash_attention_packed(q, k, v, _offsets(lengths)), want)
    turned = [x.permute(1, 0, 2).contiguous().permute(1, 0, 2) for x in (q, k, v)]
    assert torch.equal(ops.flash_attention_packed(*turned, _offsets(lengths)), want)
    odd = [torch.zeros(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x) for x in (q, k, v)]
    assert torch.equal(ops.flash_attention_packed(*odd, _offsets(lengths)), want)
    one_head = k[:, :1].expand(t, hkv, d)
    assert torch.equal(ops.flash_attention_packed(q, one_head, one_head, _offsets(lengths)),
                       ops.flash_attention_packed(q, one_head.contiguous(), one_head.contiguous(), _offsets(lengths)))


def test_offsets_that_begin_late_and_reach_too_far():
    q, k, v = _rows(100, 100, 4, 2, 64, torch.float16)
    want = ops.flash_attention_packed(q[10:90].contiguous(), k[10:90].contiguous(), v[10:90].contiguous(), _offsets([30, 50]))
    got, lse = ops.flash_attention_packed(q, k, v, _offsets([30, 50], first=10), keep=True)
    assert torch.equal(got[10:90], want) and (got[:10] == 0).all() and (got[90:] == 0).all() and (lse[:, :10] == -math.inf).all()
    far = torch.tensor([0, 40, 10 ** 9], dtype=torch.int32, device=DEV)
    assert torch.equal(ops.flash_attention_packed(q, k, v, far), ops.flash_attention_packed(q, k, v, _offsets([40, 60])))
    # (what does not ascend is no error either)
    for odd in ([0, 60, 20, 100], [-50, 30, -2, 2 ** 31 - 1], [100, 0, 100, 0]):
        ops.flash_attention_packed(q, k, v, torch.tensor(odd, dtype=torch.int32, device=DEV))
    torch.cuda.synchronize()
    nothing = ops.flash_attention_packed(q, k, v, torch.zeros(1, dtype=torch.int32, device=DEV))
    assert (nothing == 0).all()


def test_replayed_with_other_offsets_and_on_other_streams():
    q, k, v = _rows(900, 900, 8, 2, 128, torch.bfloat16)
    offsets = _offsets([100, 500, 300])
    ops.flash_attention_packed(q, k, v, offsets)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse = ops.flash_attention_packed(q, k, v, offsets, keep=True)
    for lengths in ([100, 500, 300], [0, 899, 1], [300, 300, 200], [1, 1, 1]):
        offsets.copy_(_offsets(lengths))
        want = ops.flash_attention_packed(q, k, v, offsets, keep=True)
        out.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[0]) and torch.equal(lse, want[1])
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for n in range(9):
        with torch.cuda.stream(streams[n % 3]):
            outs.append(ops.flash_attention_packed(q, k, v, offsets))
    torch.cuda.synchronize()
    assert all(torch.equal(o, out) for o in outs)


def test_refusals():
    q, k, v = _rows(50, 50, 4, 2, 64, torch.float16)
    offsets = _offsets([20, 30])

    def bad(message, *args, **kw):
        with pytest.raises(RuntimeError, match=message):
            ops.flash_attention_packed(*args, **kw)

    bad("float16 or bfloat16", q.float(), k.float(), v.float(), offsets)
    bad("dtype", q, k.bfloat16(), v, offsets)
    bad("value must be", q, k, v[:, :1], offsets)
    bad("multiple of kv_heads", q[:, :3], k, v, offsets)
    bad("need kv_offsets", q, k[:40], v[:40], offsets)
    bad("shape of offsets", q, k, v, offsets, offsets[:2])
    bad("int32", q, k, v, offsets.long())
    bad("int32", q, k, v, offsets, offsets.long())
    bad("CUDA", q, k, v, offsets.cpu())
    bad("CUDA", q, k.cpu(), v.cpu(), offsets)
    bad("head dim", *_rows(50, 50, 4, 2, 96, torch.float16), offsets)
    bad("finite", q, k, v, offsets, softmax_scale=math.inf)
    bad("query must be", q[0], k, v, offsets)
    assert ops.flash_attention_packed(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device=DEV)).shape == (0, 4, 64)
    out = ops.flash_attention_packed(q, k[:0], v[:0], offsets, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert (out == 0).all()


@pytest.mark.parametrize("ahead,n", [(20.6, 60001), (25.5, 200001)])
@pytest.mark.parametrize("m,h,hkv,d", [(1, 1, 1, 64), (5, 6, 1, 128), (2500, 8, 8, 128), (4200, 8, 8, 64), (4200, 8, 8, 128)])
def test_weights_far_below_the_largest_count_in_fp16(ahead, n, m, h, hkv, d):
    # one key ahead of equal ones by 20.6 or 25.5 (in units of log2), whose weights are together 4% or 0.4% of the sum: among those of a row whose
    # largest is 1 fp16 has 2^-20.6 only to 4%, and nothing for 2^-25.5
    rows = _capi.load().tf_flash_attention_packed_rows(m, 1, h, hkv, d)
    assert rows == {1: 64, 5: 64, 2500: 128, 4200: 256}[m]
    key, value = torch.zeros(n, hkv, d), torch.ones(n, hkv, d)
    key[n // 3, :, 0], value[n // 3] = ahead, -1.0
    q = torch.zeros(m, h, d)
    q[..., 0] = 1.0
    q, key, value = (x.half().to(DEV) for x in (q, key, value))
    out, lse = ops.flash_attention_packed(q, key, value, _offsets([m]), _offsets([n]), math.log(2.0), False, True)
    # all rows, heads and columns are one number
    score = key[:, 0, 0].double() * math.log(2.0)
    p = torch.softmax(score, 0)
    v = value[:, 0, 0].double()
    want, want_lse = (p * v).sum(), torch.logsumexp(score, 0)
    # Relative errors of weights move the result by their part of sum p |v - out|: a rounding of 2^-11, exp2 and its argument 2^-20, the score's (one product that is not
    # zero, scaled) 2^-22 of it.  Below fp16's normal numbers a rounding is of 2^-25, with the largest at 2^7 or more 2^-32 of that.  Sums in fp32: a tile of 64
    # after the other, whose parts are added as a tree or by the product in two steps, so n / 32 + 64 roundings of 2^-24 at most.
    distance = (v - want).abs()
    sums = (n / 32 + 64) * 2.0 ** -24
    bound = 2.0 ** -11 * want.abs() + 2.01 * ((2.0 ** -11 + 2.0 ** -20 + ahead * 2.0 ** -22) * (p * distance).sum() + 2.0 ** -32 * p.max() * distance.sum() + sums)
    ref.assert_within(out, want.expand_as(out), bound.expand_as(out), "out")
    ref.assert_within(lse, want_lse.expand_as(lse), torch.full_like(lse, sums + (1.0 + ahead) * 2.0 ** -21), "lse")


def test_weights_far_above_the_first_in_fp16():
    # the first keys' scores set a reference that those behind them exceed by up to 8, which does not raise it, and by more: weights stay within the type
    for rise in (1.0, 7.9, 8.0, 8.1, 15.0, 40.0):
        q, k, v = _rows(300, 300, 2, 1, 64, torch.float16)
        k.mul_(0.01)
        k[200:, 0, 0] = rise
        q[:, :, 0] = 1.0
        v[250:, 0, 1] = 60000.0
        for causal in (False, True):
            _check([300], h=2, hkv=1, dtype=torch.float16, causal=causal, scale=math.log(2.0), rows=(q, k, v))
