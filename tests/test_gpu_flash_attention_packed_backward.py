"""Gradients of attention over packed sequences, against the formula in 64 bits, against differences, and through autograd."""

import math

import pytest
import torch

from tests import attention_ref as ref
from tilefusion_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _offsets(lengths, first=0):
    return torch.tensor([first] + (first + torch.tensor(lengths).cumsum(0)).tolist(), dtype=torch.int32, device=DEV)


def _rows(t, s, h, hkv, d, dtype, seed=5, grad=1.0):
    g = torch.Generator().manual_seed(seed)
    q, k, v, do = (torch.randn(n, heads, d, generator=g) for n, heads in ((t, h), (s, hkv), (s, hkv), (t, h)))
    return [x.to(dtype).to(DEV) for x in (q, k, v, do * grad)]


def _want(q, k, v, do, out, lse, lq, lkv, scale, causal):
    """The gradients from out and lse as they are, and bounds: of P = exp(s - lse) the relative error (its score's, that of exp2 and one rounding), of
    dS = P (dP - delta) that and the errors of dP and delta (sums of D products in fp32) and one rounding, all of them weighed with what they
    multiply; sums over n rows (a group's heads) or keys in fp32."""
    dtype, d = q.dtype, q.shape[-1]
    group = q.shape[1] // k.shape[1]
    grads = [torch.zeros(x.shape, dtype=torch.float64, device=DEV) for x in (q, k, v)]
    bounds = [torch.zeros_like(x) for x in grads]
    step = ref.half_step(dtype)
    a = b = 0
    for m, n in zip(lq, lkv):
        masked = torch.arange(n, device=DEV)[None] > torch.arange(m, device=DEV)[:, None] + n - m if causal else None
        for head in range(q.shape[1]):
            rows, keys = (slice(a, a + m), head), (slice(b, b + n), head // group)
            qd, kd, vd, gd, od = (x.double() for x in (q[rows], k[keys], v[keys], do[rows], out[rows]))
            s = qd @ kd.t().contiguous() * scale
            size = qd.abs() @ kd.abs().t().contiguous() * abs(scale) * (d + 8) * 2.0 ** -24
            l = lse[head, a:a + m].double()[:, None]
            p = torch.exp(s - l)
            off_p = size + 2.0 ** -20 + l.abs() * 2.0 ** -22 + s.abs() * 2.0 ** -22
            if masked is not None:
                p, off_p = p.masked_fill(masked, 0.0), off_p.masked_fill(masked, 0.0)
            dp, delta = gd @ vd.t().contiguous(), (gd * od).sum(1, keepdim=True)
            off_d = (d + 4) * 2.0 ** -24 * (gd.abs() @ vd.abs().t().contiguous() + (gd * od).abs().sum(1, keepdim=True))
            ds = p * (dp - delta)
            err = p * off_d + (off_p + step) * ds.abs()
            if masked is not None:   # (no part of the sum, also where an infinite gradient would make 0 * inf of it)
                ds, err = ds.masked_fill(masked, 0.0), err.masked_fill(masked, 0.0)
            grads[0][rows] += scale * (ds @ kd)
            bounds[0][rows] += abs(scale) * (err @ kd.abs() + n * 2.0 ** -24 * (ds.abs() @ kd.abs()))
            grads[1][keys] += scale * (ds.t().contiguous() @ qd)
            bounds[1][keys] += abs(scale) * (err.t().contiguous() @ qd.abs() + m * group * 2.0 ** -24 * (ds.abs().t().contiguous() @ qd.abs()))
            finite = gd.masked_fill(~gd.isfinite(), 0.0)
            grads[2][keys] += p.t().contiguous() @ finite
            for i, c in (~gd.isfinite()).nonzero().tolist():   # (to the keys that row i sees, and not 0 * inf to the others)
                to = ~masked[i] if masked is not None else torch.ones(n, dtype=torch.bool, device=DEV)
                grads[2][keys][:, c] += torch.where(to, gd[i, c], 0.0)
            bounds[2][keys] += ((off_p + step) * p).t().contiguous() @ finite.abs() + m * group * 2.0 ** -24 * (p.t().contiguous() @ finite.abs())
        a, b = a + m, b + n
    # (what is below 2^-29 of a lane's largest dS, or below 2^-39, has no part in fp16: far less than a rounding of the sums)
    return grads, [1.01 * e + step * x.abs() + torch.finfo(dtype).tiny * step * 2 for e, x in zip(bounds, grads)]


def _check(lq, lkv=None, h=4, hkv=2, d=64, dtype=torch.bfloat16, causal=True, scale=None, tail=0, grad=1.0, rows=None):
    q, k, v, do = rows or _rows(sum(lq) + tail, sum(lkv or lq) + tail, h, hkv, d, dtype, grad=grad)
    of, kv = _offsets(lq), _offsets(lkv) if lkv else None
    out, lse = ops.flash_attention_packed(q, k, v, of, kv, scale, causal, True)
    got = ops.flash_attention_packed_backward(do, q, k, v, out, lse, of, kv, scale, causal)
    lse0 = lse.masked_fill(lse == -math.inf, 0.0)   # (rows without a key: all masked)
    want, bound = _want(q, k, v, do, out, lse0, lq, lkv or lq, d ** -0.5 if scale is None else scale, causal)
    for name, a, b, c in zip(("grad_query", "grad_key", "grad_value"), got, want, bound):
        ref.assert_within(a, b, c, name)
    assert all((x[n:] == 0).all() for x, n in zip(got, (sum(lq), sum(lkv or lq), sum(lkv or lq))))
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", [[1], [2], [15, 16, 17], [0, 31, 0, 0, 33, 64, 65], [127, 1, 129, 200], [513], [1000, 3]])
def test_lengths(dtype, d, causal, lengths):
    _check(lengths, d=d, dtype=dtype, causal=causal, tail=5)


@pytest.mark.parametrize("h,hkv", [(1, 1), (8, 8), (3, 1), (5, 5), (12, 4), (7, 1), (48, 8), (64, 1), (100, 1)])
def test_groups(h, hkv):
    for causal in (False, True):
        _check([70, 1, 200, 13], h=h, hkv=hkv, causal=causal)
        _check([70, 1, 200, 13], h=h, hkv=hkv, causal=causal, d=128, dtype=torch.float16)


@pytest.mark.parametrize("lq,lkv", [([1, 1, 1], [100, 1, 2000]), ([5, 64, 3], [69, 64, 1000]), ([100, 30, 7, 300], [10, 0, 7, 299]),
                                    ([0, 4, 0], [50, 0, 0]), ([128, 16], [3000, 3])])
@pytest.mark.parametrize("causal", [False, True])
def test_keys_of_another_number(lq, lkv, causal):
    for d, dtype in ((64, torch.bfloat16), (128, torch.float16)):
        _check(lq, lkv, d=d, dtype=dtype, causal=causal, tail=2)
        _check(lq, lkv, h=16, hkv=1, d=d, dtype=dtype, causal=causal)


@pytest.mark.parametrize("n", [63, 65, 300])
def test_many_sequences(n):
    g = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 60, (n,), generator=g).tolist()
    lengths = [x * (10 if i % 17 == 0 else 1) for i, x in enumerate(lengths)]
    _check(lengths, h=4, hkv=1)
    _check(lengths, h=2, hkv=2, causal=False, d=128)


@pytest.mark.parametrize("grad", [1e-6, 1e-4, 3000.0, 60000.0])
def test_gradients_at_the_ends_of_fp16(grad):
    _check([200, 70], dtype=torch.float16, grad=grad / 4)
    _check([200, 70], dtype=torch.float16, grad=grad / 4, d=128, causal=False, h=8)


def test_gradients_of_different_sizes_in_one_call():
    # tokens that count 2^-20 as much as others, before them and behind them, and tokens that do not count
    q, k, v, do = _rows(400, 400, 4, 2, 64, torch.float16)
    for order in (1, -1):
        weight = torch.ones(400, device=DEV)
        weight[:150], weight[150:200], weight[200:] = 2.0 ** -10, 0.0, 2.0 ** 10
        _check([400], dtype=torch.float16, rows=(q, k, v, do * (weight if order == 1 else weight.flip(0))[:, None, None].half()))


@pytest.mark.parametrize("causal", [False, True])
def test_an_infinite_gradient_beside_large_ones_in_fp16(causal):
    # small ones, by which the powers of two are chosen, then one that is infinite among ones that are 2^18 times as large
    for d in (64, 128):
        q, k, v, do = _rows(64, 64, 2, 1, d, torch.float16, seed=d)
        do[:32] *= 2.0 ** -8
        do[32:] *= 2.0 ** 10
        do[33, 1, 5] = math.inf
        _check([64], h=2, hkv=1, d=d, causal=causal, rows=(q, k, v, do))


def test_long_rows_of_small_weights_in_fp16():
    # weights of 2^-13, of which fp16 alone keeps ten bits less than of larger ones
    _check([4], [9000], dtype=torch.float16, causal=False, scale=0.01)


@pytest.mark.parametrize("scale", [0.0, -0.2, 1.0, 1e-4])
def test_scales(scale):
    _check([300, 40], scale=scale)
    _check([300, 40], scale=scale, dtype=torch.float16)


def test_differences():
    # (the loss is linear in out: differences of the formula in 64 bits around 16-bit inputs)
    q, k, v, do = _rows(40, 40, 2, 1, 64, torch.bfloat16)
    of = _offsets([25, 15])
    out, lse = ops.flash_attention_packed(q, k, v, of, keep=True)
    grads = ops.flash_attention_packed_backward(do, q, k, v, out, lse, of)

    def loss(q, k, v):
        total = 0.0
        for a, b in ((0, 25), (25, 40)):
            s = torch.einsum("ihd,jd->hij", q[a:b], k[a:b, 0]) / 8.0
            s = s.masked_fill(torch.ones(b - a, b - a, device=DEV).triu(1).bool(), -math.inf)
            total = total + (torch.einsum("hij,jd->ihd", torch.softmax(s, -1), v[a:b, 0]) * do[a:b].double()).sum()
        return total

    g = torch.Generator().manual_seed(1)
    inputs = [x.double() for x in (q, k, v)]
    for n, grad in enumerate(grads):
        for _ in range(4):
            way = torch.randn(grad.shape, generator=g, dtype=torch.float64).to(DEV)
            h = 1e-4
            ahead, behind = ([x + (h * way if i == n else 0.0) * sign for i, x in enumerate(inputs)] for sign in (1.0, -1.0))
            slope = (loss(*ahead) - loss(*behind)) / (2 * h)
            # roundings of 2^-9 of the gradient's elements, of P, dS, out and delta: eight of them, each off by chance at worst all one way
            assert abs((grad.double() * way).sum() - slope) <= 8 * 2.0 ** -9 * (grad.double().abs() * way.abs()).sum()


def test_autograd_and_slices():
    lengths, h, hkv, d = [70, 131], 8, 2, 64
    t = sum(lengths)
    of = _offsets(lengths)
    wide = _rows(t, t, h + 2 * hkv, hkv, d, torch.bfloat16)[0].flatten(1).requires_grad_()
    q, k, v = (x.unflatten(1, (-1, d)) for x in wide.split([h * d, hkv * d, hkv * d], dim=1))
    do = _rows(t, t, h, hkv, d, torch.bfloat16)[3]
    out = ops.flash_attention_packed(q, k, v, of)
    out.backward(do)
    with torch.no_grad():
        o, lse = ops.flash_attention_packed(q, k, v, of, keep=True)
        want = ops.flash_attention_packed_backward(do, q, k, v, o, lse, of)
    assert torch.equal(out, o)
    assert torch.equal(wide.grad, torch.cat([x.flatten(1) for x in want], dim=1))
    # one gradient alone, one head of keys for all, an expanded gradient
    k1 = k.detach().clone().requires_grad_()
    ops.flash_attention_packed(q.detach(), k1, v.detach(), of).backward(do)
    assert torch.equal(k1.grad, want[1])
    q1 = q.detach().clone().requires_grad_()
    ops.flash_attention_packed(q1, k.detach(), v.detach(), of).backward(do)
    assert torch.equal(q1.grad, want[0])
    one = k.detach()[:, :1].clone().requires_grad_()
    ops.flash_attention_packed(q.detach(), one.expand(t, hkv, d), v.detach(), of).backward(do)
    ref_k = k.detach()[:, :1].expand(t, hkv, d).contiguous().requires_grad_()
    ops.flash_attention_packed(q.detach(), ref_k, v.detach(), of).backward(do)
    assert torch.equal(one.grad, ref_k.grad.sum(1, keepdim=True))
    q2 = q.detach().clone().requires_grad_()
    ops.flash_attention_packed(q2, k.detach(), v.detach(), of).sum().backward()
    with torch.no_grad():
        want = ops.flash_attention_packed_backward(torch.ones_like(o), q, k, v, o, lse, of)
    assert torch.equal(q2.grad, want[0])


def test_masked_and_unused_rows_are_not_seen():
    for d, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        lengths = [100, 33, 260]
        n = sum(lengths)
        for h, hkv in ((2, 2), (8, 1)):
            q, k, v, do = _rows(n + 7, n + 7, h, hkv, d, dtype)
            of = _offsets(lengths)
            out, lse = ops.flash_attention_packed(q, k, v, of, keep=True)
            first = ops.flash_attention_packed_backward(do, q, k, v, out, lse, of)
            at = 133 + 150
            for bad in (math.inf, -math.inf, math.nan):
                # rows of no sequence
                spoilt = [x.clone() for x in (do, q, k, v, out, lse.t())]
                for x in spoilt:
                    x[n:] = bad
                got = ops.flash_attention_packed_backward(*spoilt[:5], spoilt[5].t(), of)
                assert all(torch.equal(a, b) for a, b in zip(got, first))
                # a gradient in the middle of a sequence: queries before and behind it, keys behind it and other sequences see nothing of it
                do2 = do.clone()
                do2[at, :, 3] = bad
                gq, gk, gv = ops.flash_attention_packed_backward(do2, q, k, v, out, lse, of)
                keep = [i for i in range(n) if i != at]
                assert torch.equal(gq[keep], first[0][keep]) and not gq[at].isfinite().any()
                clear = [i for i in range(n) if not 133 <= i <= at]
                assert torch.equal(gk[clear], first[1][clear]) and torch.equal(gv[clear], first[2][clear])
                # (dP and delta are infinities, of one sign or of two: their difference is NaN or an infinity)
                assert not gk[133:at + 1].isfinite().any()
                assert (gv[133:at + 1, :, 3].isnan() if bad != bad else gv[133:at + 1, :, 3] == bad).all()
                others = [c for c in range(d) if c != 3]
                assert torch.equal(gv[133:at + 1][:, :, others], first[2][133:at + 1][:, :, others])
                # keys and values that rows in front of them do not see
                k2, v2 = k.clone(), v.clone()
                k2[at:n], v2[at:n] = bad, bad
                out2, lse2 = ops.flash_attention_packed(q, k2, v2, of, keep=True)
                gq, gk, gv = ops.flash_attention_packed_backward(do, q, k2, v2, out2, lse2, of)
                assert torch.equal(gq[:at], first[0][:at]) and torch.equal(gk[:133], first[1][:133]) and torch.equal(gv[:133], first[2][:133])
                # queries that keys behind them are not seen by
                q2 = q.clone()
                q2[at] = bad
                out2, lse2 = ops.flash_attention_packed(q2, k, v, of, keep=True)
                gq, gk, gv = ops.flash_attention_packed_backward(do, q2, k, v, out2, lse2, of)
                assert torch.equal(gq[keep], first[0][keep])
                assert torch.equal(gk[clear], first[1][clear]) and torch.equal(gv[clear], first[2][clear])
                assert gk[133:at + 1].isnan().all() and gv[133:at + 1].isnan().all()


def test_the_same_bits_every_time_and_replayed():
    q, k, v, do = _rows(900, 900, 8, 2, 128, torch.bfloat16)
    offsets = _offsets([100, 500, 300])
    out, lse = ops.flash_attention_packed(q, k, v, offsets, keep=True)
    first = ops.flash_attention_packed_backward(do, q, k, v, out, lse, offsets)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(first, ops.flash_attention_packed_backward(do, q, k, v, out, lse, offsets)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        o, l = ops.flash_attention_packed(q, k, v, offsets, keep=True)
        grads = ops.flash_attention_packed_backward(do, q, k, v, o, l, offsets)
    for lengths in ([100, 500, 300], [0, 899, 1], [300, 300, 200], [1, 1, 1]):
        offsets.copy_(_offsets(lengths))
        out, lse = ops.flash_attention_packed(q, k, v, offsets, keep=True)
        want = ops.flash_attention_packed_backward(do, q, k, v, out, lse, offsets)
        for x in grads:
            x.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, want))


def test_refusals():
    q, k, v, do = _rows(50, 50, 4, 2, 64, torch.float16)
    of = _offsets([20, 30])
    out, lse = ops.flash_attention_packed(q, k, v, of, keep=True)

    def bad(message, *args):
        with pytest.raises(RuntimeError, match=message):
            ops.flash_attention_packed_backward(*args)

    bad("grad_out must be", do[:, :2], q, k, v, out, lse, of)
    bad("dtype", do.bfloat16(), q, k, v, out, lse, of)
    bad("out must be", do, q, k, v, out[:40], lse, of)
    bad("lse must be", do, q, k, v, out, lse.t(), of)
    bad("lse must be", do, q, k, v, out, lse.double(), of)
    bad("need kv_offsets", do, q, k[:40], v[:40], out, lse, of)
    q1 = q.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="autograd does not record"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.flash_attention_packed(q1, k, v, of)
    torch.cuda.synchronize()
    loss = ops.flash_attention_packed(q1, k, v, of).sum()
    (grad,) = torch.autograd.grad(loss, q1, create_graph=True)
    with pytest.raises(RuntimeError):
        grad.sum().backward()
    with pytest.raises(RuntimeError, match="torch.func"):
        torch.func.grad(lambda x: ops.flash_attention_packed(x, k, v, of).sum())(q)
    nothing = ops.flash_attention_packed_backward(do[:0], q[:0], k, v, out[:0], lse[:, :0], torch.zeros(3, dtype=torch.int32, device=DEV), of)
    assert nothing[0].shape == (0, 4, 64) and (nothing[1] == 0).all() and (nothing[2] == 0).all()
    nothing = ops.flash_attention_packed_backward(do, q, k[:0], v[:0], out, lse, of, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert (nothing[0] == 0).all() and nothing[1].shape == (0, 2, 64)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_no_queries_or_no_keys_at_all(dtype):
    q, k, v, do = _rows(0, 50, 4, 2, 64, dtype)
    of, kv = _offsets([0, 0]), _offsets([20, 30])
    out, lse = ops.flash_attention_packed(q, k, v, of, kv, keep=True)
    assert out.shape == (0, 4, 64) and lse.shape == (4, 0)
    grads = ops.flash_attention_packed_backward(do, q, k, v, out, lse, of, kv)
    assert grads[0].shape == q.shape and (grads[1] == 0).all() and (grads[2] == 0).all()
    q, k, v, do = _rows(50, 0, 4, 2, 64, dtype)
    for causal in (False, True):
        out, lse = ops.flash_attention_packed(q, k, v, kv, of, None, causal, True)
        assert (out == 0).all() and (lse == -math.inf).all()
        grads = ops.flash_attention_packed_backward(do, q, k, v, out, lse, kv, of, None, causal)
        assert (grads[0] == 0).all() and grads[1].shape == k.shape == grads[2].shape
    # no sequence: rows of none
    out, lse = ops.flash_attention_packed(q, q[:, :2], q[:, :2], _offsets([]), keep=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    for g in ops.flash_attention_packed_backward(do, q, q[:, :2], q[:, :2], out, lse, _offsets([])):
        assert (g == 0).all()


def _spread(x, token, head):
    """x with rows `token` and heads `head` elements apart, in memory that is not touched otherwise."""
    n, h, d = x.shape
    y = torch.empty((n - 1) * token + (h - 1) * head + d, dtype=x.dtype, device=DEV).as_strided(x.shape, (token, head, 1))
    return y.copy_(x)


# heads of keys as far apart as those of 2^17 tokens x 128, beyond 32 bits, and heads of queries that are copied (2^31 elements in a group)
@pytest.mark.parametrize("h,hkv,of_query,of_keys", [(4, 2, 1 << 24, 1 << 24), (4, 4, 1 << 30, 1 << 30), (4, 2, 1 << 30, 1 << 31), (2, 2, 64, 1 << 32)])
def test_heads_far_from_each_other(h, hkv, of_query, of_keys):
    for d, dtype in ((64, torch.float16), (128, torch.bfloat16)):
        q, k, v, do = _rows(170, 170, h, hkv, d, dtype)
        of = _offsets([100, 70])
        far = _spread(q, d, max(of_query, 170 * d)), _spread(k, d, of_keys), _spread(v, d, of_keys)
        out, lse = ops.flash_attention_packed(q, k, v, of, keep=True)
        for own in (far, (far[0], k, v), (q, *far[1:])):
            assert all(torch.equal(a, b) for a, b in zip(ops.flash_attention_packed(*own, of, keep=True), (out, lse)))
            got = ops.flash_attention_packed_backward(do, *own, out, lse, of)
            assert all(torch.equal(a, b) for a, b in zip(got, ops.flash_attention_packed_backward(do, q, k, v, out, lse, of)))
        leaves = [x.detach().requires_grad_() for x in far]
        ops.flash_attention_packed(*leaves, of).backward(do)
        assert all(torch.equal(x.grad, g) for x, g in zip(leaves, got))
        del far, own, leaves


def test_tokens_far_from_each_other():
    # further apart than 32-bit offsets reach within a tile: copied
    q, k, v, do = _rows(40, 40, 2, 1, 64, torch.bfloat16)
    of = _offsets([25, 15])
    want = ops.flash_attention_packed(q, k, v, of)
    assert torch.equal(ops.flash_attention_packed(_spread(q, 1 << 24, 64), _spread(k, 1 << 25, 64), _spread(v, 1 << 24, 64), of), want)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths,h,hkv,d", [([25, 15], 2, 1, 64), ([25, 15], 4, 2, 128), ([130, 47, 1], 4, 2, 64), ([200], 6, 2, 128)])
def test_gradients_of_the_loss_by_autograd_and_by_differences(dtype, causal, lengths, h, hkv, d):
    # (from the definition of the forward pass alone, in 64 bits)
    q, k, v, do = _rows(sum(lengths), sum(lengths), h, hkv, d, dtype)
    of = _offsets(lengths)
    out, lse = ops.flash_attention_packed(q, k, v, of, None, None, causal, True)
    got = ops.flash_attention_packed_backward(do, q, k, v, out, lse, of, None, None, causal)
    want, bounds = ref.gradients(q, k, v, do, out, lse, lengths, d ** -0.5, causal)
    for name, a, b, c in zip(("grad_query", "grad_key", "grad_value"), got, want, bounds):
        ref.assert_within(a, b, c, name)
    ref.assert_slopes(got, q, k, v, do, lengths, d ** -0.5, causal, bounds)


def test_offsets_beyond_32_bits():
    # tokens that lie 2^20 elements apart: the last of them 10 GiB behind the first
    lengths, h, hkv, d = [100, 4000, 900], 4, 2, 64
    t = sum(lengths)
    q, k, v, do = _rows(t, t, h, hkv, d, torch.float16)
    of = _offsets(lengths)
    out, lse = ops.flash_attention_packed(q, k, v, of, keep=True)
    want = ops.flash_attention_packed_backward(do, q, k, v, out, lse, of)
    far = [_spread(x, 1 << 20, d) for x in (q, k, v)]
    assert all(torch.equal(a, b) for a, b in zip(ops.flash_attention_packed(*far, of, keep=True), (out, lse)))
    assert all(torch.equal(a, b) for a, b in zip(ops.flash_attention_packed_backward(do, *far, out, lse, of), want))


def test_results_beyond_32_bits():
    # 2^32 elements of queries, results and gradients: sequences at both ends and around the middle, a head from each end and one between
    tokens, h, d, n = 1 << 18, 128, 128, 128
    g = torch.Generator(device=DEV).manual_seed(1)
    q, do = (torch.randn(tokens, h, d, dtype=torch.bfloat16, device=DEV, generator=g) for _ in range(2))
    k, v = (torch.randn(tokens, 1, d, dtype=torch.bfloat16, device=DEV, generator=g) for _ in range(2))
    of = _offsets([n] * (tokens // n))
    out, lse = ops.flash_attention_packed(q, k, v, of, keep=True)
    grads = ops.flash_attention_packed_backward(do, q, k, v, out, lse, of)
    for a in (0, tokens // 2 - n, tokens // 2, tokens - n):
        s = slice(a, a + n)
        want, bound = _want(q[s], k[s], v[s], do[s], out[s], lse[:, s], [n], [n], d ** -0.5, True)
        for name, x, b, c in zip(("grad_query", "grad_key", "grad_value"), grads, want, bound):
            ref.assert_within(x[s], b, c, f"{name} from {a}")
        masked = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
        for head in (0, 63, 127):
            o, l, off, off_l = ref.attend(q[s, head], k[s, 0], v[s, 0], d ** -0.5, masked, ref.half_step(torch.bfloat16) + 2.0 ** -20)
            ref.assert_within(out[s, head], o, off, f"out from {a}")
            ref.assert_within(lse[head, s], l, off_l, f"lse from {a}")


def test_offsets_at_the_ends_of_their_type():
    # ends far in front of their beginnings name no rows, and those far behind the last row all there are
    low, high = -2 ** 31, 2 ** 31 - 1
    for dtype, d in ((torch.float16, 64), (torch.bfloat16, 128)):
        q, k, v, do = _rows(100, 100, 4, 2, d, dtype)
        for odd, even in (([60, low], [60, 60]), ([30, low, low + 1, -1], [30, 30, 30, 30]), ([40, high], [40, 100]), ([100, low], [100, 100]), ([low, 70], [0, 70])):
            odd, even = (torch.tensor(x, dtype=torch.int32, device=DEV) for x in (odd, even))
            for causal in (False, True):
                want = ops.flash_attention_packed(q, k, v, even, None, None, causal, True)
                assert all(torch.equal(a, b) for a, b in zip(ops.flash_attention_packed(q, k, v, odd, None, None, causal, True), want))
                got, wanted = (ops.flash_attention_packed_backward(do, q, k, v, *want, x, None, None, causal) for x in (odd, even))
                assert all(torch.equal(a, b) for a, b in zip(got, wanted))
                # (with keys of their own; what does not ascend gives some numbers)
                ops.flash_attention_packed_backward(do, q, k, v, *ops.flash_attention_packed(q, k, v, even, odd, None, causal, True), even, odd, None, causal)
    torch.cuda.synchronize()
