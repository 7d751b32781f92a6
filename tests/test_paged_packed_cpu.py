"""CPU-only checks of append_paged_kv, flash_decode_paged and flash_attention_packed: what the C ABI refuses before it touches the device, where a
position lies in a paged cache, and that the comparisons of the GPU tests see mistakes."""

import ctypes
import math
import os
import subprocess

import pytest
import torch

from tests import attention_ref as ref
from tilefusion_amd import _capi, ops

P = 0x1000   # never dereferenced: validation fails first
F16, BF16, F32 = _capi.TF_DTYPE_F16, _capi.TF_DTYPE_BF16, _capi.TF_DTYPE_F32
BAD, UNSUPPORTED, OK = _capi.TF_ERR_INVALID_ARG, _capi.TF_ERR_UNSUPPORTED, _capi.TF_OK
CPP = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")


def _i64(*values):
    return (ctypes.c_int64 * len(values))(*values)


def _cache(**changed):
    """8 pages of 16 tokens, 2 heads x 64; 3 sequences of up to 4 pages."""
    fields = dict(key=P, value=P, key_strides=_i64(2048, 64, 1024), value_strides=_i64(2048, 64, 1024), pages=8, page_size=16, kv_heads=2, D=64,
                  page_table=P, table_width=4, table_stride=4, lengths=P, sequences=3, dtype=F16)
    return ctypes.byref(_capi.PagedCache(**{**fields, **changed}))


BAD_CACHES = [dict(key=None), dict(value=None), dict(page_table=None), dict(lengths=None), dict(pages=0), dict(pages=1 << 31), dict(kv_heads=0),
              dict(kv_heads=65537), dict(page_size=0), dict(page_size=65537), dict(sequences=-1), dict(sequences=(1 << 20) + 1), dict(table_width=-1),
              dict(table_width=1 << 31), dict(table_stride=-4), dict(key=P + 8), dict(value=P + 2), dict(key_strides=_i64(2048, 60, 1024)),
              dict(value_strides=_i64(-2048, 64, 1024)), dict(key_strides=_i64(2048, 32, 1024)), dict(value_strides=_i64(2048, 64, 8))]


def test_append_arguments():
    lib = _capi.load()

    def call(cache=None, query=P, key=P, value=P, strides=_i64(256, 64, 128, 64, 128, 64), cos=P, sin=P, positions=100, rotated=64, offsets=None, tokens=3,
             heads=4, query_out=P, key_out=P):
        return lib.tf_append_paged_kv(cache or _cache(), query, key, value, strides, cos, sin, positions, rotated, 0, offsets, tokens, heads, query_out,
                                      key_out, None)

    for changed in BAD_CACHES:
        assert call(_cache(**changed)) == BAD, changed
    assert call(_cache(dtype=F32)) == UNSUPPORTED == call(_cache(D=96)) and b"head dim" in lib.tf_last_error()
    assert lib.tf_append_paged_kv(None, P, P, P, _i64(*[64] * 6), P, P, 100, 64, 0, None, 3, 4, P, P, None) == BAD
    for changed in (dict(query=None), dict(key=None), dict(value=None), dict(strides=None), dict(cos=None), dict(sin=None), dict(query_out=None),
                    dict(query=P + 2), dict(key_out=P + 8), dict(rotated=0), dict(rotated=33), dict(rotated=66), dict(positions=-1), dict(tokens=-1),
                    dict(tokens=1 << 24), dict(heads=0), dict(heads=65537), dict(strides=_i64(256, 64, 128, 60, 128, 64)),
                    dict(strides=_i64(256, 64, 128, 64, 128, -64))):
        assert call(**changed) == BAD, changed
    assert call(tokens=0, query=None, key=None, value=None, query_out=None, key_out=None) == OK


def test_decode_arguments():
    lib = _capi.load()
    size = lib.tf_flash_decode_paged_workspace_bytes
    want = size(3, 4, 2, 64)
    assert want > 0 and size(0, 4, 2, 64) == 0 == size(3, 5, 2, 64) == size(3, 4, 0, 64) == size(3, 0, 2, 64) == size(3, 4, 2, 96)
    # beside the words of the items it does not grow with the sequences
    assert size(1003, 4, 2, 64) - size(1002, 4, 2, 64) == 2 * 256 == size(1003, 64, 2, 64) - size(1002, 64, 2, 64) - 2 * 256

    def call(cache=None, query=P, strides=_i64(256, 64), out=P, heads=4, scale=0.125, workspace=P, workspace_bytes=want):
        return lib.tf_flash_decode_paged(cache or _cache(), query, strides, out, heads, scale, workspace, workspace_bytes, None)

    for changed in BAD_CACHES:
        assert call(_cache(**changed)) == BAD, changed
    assert call(_cache(dtype=F32)) == UNSUPPORTED == call(_cache(D=32))
    assert call(_cache(page_size=24)) == UNSUPPORTED and b"multiple of 16" in lib.tf_last_error()
    assert call(_cache(key_strides=_i64(2048, 1 << 26, 1024))) == UNSUPPORTED
    assert call(_cache(table_width=(1 << 31) // 16)) == BAD == call(_cache(sequences=1 << 20, table_width=1 << 20)) and b"2^31" in lib.tf_last_error()
    assert call(_cache(sequences=1 << 20), heads=64) == BAD
    for changed in (dict(query=None), dict(strides=None), dict(out=None), dict(workspace=None), dict(query=P + 2), dict(out=P + 8), dict(workspace=P + 4),
                    dict(heads=0), dict(heads=3), dict(heads=65538), dict(scale=math.nan), dict(scale=math.inf), dict(strides=_i64(256, 60)),
                    dict(strides=_i64(-256, 64)), dict(workspace_bytes=want - 1)):
        assert call(**changed) == BAD, changed
    assert call(_cache(sequences=0), query=None, out=None, workspace=None, workspace_bytes=0) == OK


def _packed(**changed):
    fields = dict(query=P, key=P, value=P, query_strides=_i64(256, 64), key_strides=_i64(128, 64), value_strides=_i64(128, 64), tokens=70, kv_tokens=70,
                  sequences=3, heads=4, kv_heads=2, D=64, offsets=P, kv_offsets=None, softmax_scale=0.125, causal=1, dtype=BF16)
    return ctypes.byref(_capi.PackedAttention(**{**fields, **changed}))


def test_packed_arguments():
    lib = _capi.load()
    size = lib.tf_flash_attention_packed_backward_workspace_bytes
    want = size(_packed())

    def forward(p, out=P, lse=P):
        return lib.tf_flash_attention_packed(p, out, lse, None)

    def backward(p, grad_out=P, out=P, lse=P, grad_query=P, grad_key=P, grad_value=P, workspace=P, workspace_bytes=want):
        return lib.tf_flash_attention_packed_backward(p, grad_out, out, lse, grad_query, grad_key, grad_value, workspace, workspace_bytes, None)

    assert want == (70 * 4 * 16 + 255) // 256 * 256 and size(None) == 0 == size(_packed(tokens=-1)) == size(_packed(heads=1))
    for call in (forward, backward):
        assert call(None) == BAD
        assert call(_packed(dtype=F32)) == UNSUPPORTED == call(_packed(D=96))
        for changed in (dict(query=None), dict(key=None), dict(value=None), dict(offsets=None), dict(query=P + 2), dict(key=P + 8), dict(value=P + 4),
                        dict(tokens=-1), dict(tokens=1 << 24), dict(kv_tokens=-1), dict(kv_tokens=71), dict(sequences=-1), dict(sequences=65537),
                        dict(heads=0), dict(heads=3), dict(heads=2048), dict(kv_heads=0), dict(softmax_scale=math.nan), dict(softmax_scale=-math.inf),
                        dict(query_strides=_i64(256, 60)), dict(key_strides=_i64(-128, 64)), dict(value_strides=_i64(1 << 24, 64)),
                        dict(heads=256, query_strides=_i64(256, (1 << 24) - 8)), dict(heads=1024, kv_heads=1, tokens=1 << 21, kv_offsets=P)):
            assert call(_packed(**changed)) == BAD, changed
        nothing = dict(tokens=0, kv_tokens=0, query=None, key=None, value=None, offsets=None)
        assert call(_packed(**nothing)) == OK
    assert forward(_packed(), out=None) == BAD == forward(_packed(), out=P + 8)
    for changed in (dict(grad_out=None), dict(out=None), dict(lse=None), dict(grad_out=P + 2), dict(grad_query=P + 8), dict(grad_value=P + 4),
                    dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=want - 1), dict(grad_key=None), dict(grad_value=None)):
        assert backward(_packed(), **changed) == BAD, changed


def test_parts_of_the_gradients_rows():
    # where tiles of keys are few their rows are cut, and the sums of the parts need room of their own
    size = _capi.load().tf_flash_attention_packed_backward_workspace_bytes
    sums = lambda **c: size(_packed(**c)) - (c["tokens"] * c.get("heads", 4) * 16 + 255) // 256 * 256
    one = lambda tokens, heads=2: 2 * tokens * heads * 64 * 4
    assert sums(tokens=70, kv_tokens=70) == 0
    assert sums(tokens=2000, kv_tokens=2000, sequences=1) == 8 * one(2000)     # 4000 rows, 30 tiles
    assert sums(tokens=2000, kv_tokens=2000, sequences=8) == 0                  # 500 of each
    assert sums(tokens=9000, kv_tokens=9000, sequences=1, heads=16, kv_heads=8) == 0   # 568 tiles


def test_rows_of_a_workgroup():
    rows = _capi.load().tf_flash_attention_packed_rows
    for d in (64, 128):
        assert rows(100, 4, 4, 2, d) == 64 and rows(2000, 14, 32, 8, d) == 256 == rows(16384, 1, 32, 8, d) and rows(5200, 40, 8, 8, d) == 128
        # short texts leave most of a large tile empty
        assert rows(3000, 1000, 8, 8, d) == 64 and rows(30000, 300, 8, 8, d) == 128
    # one round of workgroups: 64 rows for two on a CU (D = 64) or one
    assert rows(800, 1, 32, 8, 64) == 64 and rows(800, 1, 32, 8, 128) == 128 and rows(512, 1, 32, 8, 128) == 64
    assert rows(-1, 1, 4, 2, 64) == 0 == rows(10, 1, 3, 2, 64) == rows(10, 1, 4, 0, 64) == rows(10, 1, 4, 2, 96) and rows(0, 0, 4, 2, 64) == 64


def test_pages_and_divisions():
    subprocess.check_call(["make", "-C", CPP, "test_paged_cache_host"], stdout=subprocess.DEVNULL)
    out = subprocess.run([os.path.join(CPP, "test_paged_cache_host")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_rotation_tables():
    cos, sin = ops.rotation_tables(1000, 64, device="cpu")
    assert cos.shape == (1000, 32) == sin.shape and cos.dtype == torch.float32
    for p, i in ((0, 0), (1, 0), (999, 0), (999, 31), (500, 7)):
        angle = p * 10000.0 ** (-2 * i / 64)
        assert abs(cos[p, i].item() - math.cos(angle)) < 2.0 ** -24 and abs(sin[p, i].item() - math.sin(angle)) < 2.0 ** -24
    assert ops.rotation_tables(0, 8, device="cpu")[0].shape == (0, 4)
    for arguments in ((-1, 8), (4, 0), (4, 7)):
        with pytest.raises(RuntimeError, match="rotation_tables"):
            ops.rotation_tables(*arguments, device="cpu")


def _calls():
    g = torch.Generator().manual_seed(3)
    q, out = (torch.randn(2, 4, 64, generator=g).bfloat16() for _ in range(2))
    k, v = (torch.randn(2, 2, 64, generator=g).bfloat16() for _ in range(2))
    cache = [torch.zeros(4, 16, 2, 64).bfloat16() for _ in range(2)]
    table, lengths, offsets = torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32)
    cos, sin = ops.rotation_tables(8, 64, device="cpu")
    return q, {
        "append_paged_kv": lambda q: ops.append_paged_kv(q, k, v, cos, sin, *cache, table, lengths),
        "flash_decode_paged": lambda q: ops.flash_decode_paged(q, *cache, table, lengths),
        "flash_attention_packed": lambda q: ops.flash_attention_packed(q, k, v, offsets),
        "flash_attention_packed_backward": lambda q: ops.flash_attention_packed_backward(out, q, k, v, out, torch.zeros(4, 2), offsets)[0],
    }


@pytest.mark.parametrize("name", list(_calls()[1]))
def test_wrappers_refuse_what_there_is_not(name):
    q, calls = _calls()
    call = calls[name]
    with pytest.raises(NotImplementedError):   # no kernel on the CPU
        call(q)
    with pytest.raises(RuntimeError, match=f"{name}: "):
        call(q[0])
    if name in ("append_paged_kv", "flash_decode_paged"):
        with pytest.raises(RuntimeError, match=f"{name}: there is no gradient"):
            call(q.clone().requires_grad_())
        with torch.no_grad(), pytest.raises(NotImplementedError):
            call(q.clone().requires_grad_())
    # (results are written into fresh tensors, whose tangent would be zero)
    with pytest.raises(RuntimeError, match=f"{name}: there are no forward-mode"):
        torch.func.jvp(call, (q,), (torch.ones_like(q),))
    with torch.autograd.forward_ad.dual_level(), torch.no_grad(), pytest.raises(RuntimeError, match=f"{name}: there are no forward-mode"):
        call(torch.autograd.forward_ad.make_dual(q, torch.ones_like(q)))
    with pytest.raises(RuntimeError, match=f"{name}: does not work under torch.func"):
        torch.func.grad(lambda x: call(x).float().sum())(q)
    with pytest.raises(RuntimeError, match=f"{name}: does not work under torch.func"):
        torch.func.vmap(call)(torch.stack([q, q]))


def test_a_recorded_call_is_not_captured(monkeypatch):
    q, calls = _calls()
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    with pytest.raises(RuntimeError, match="flash_attention_packed: .*captured"):
        calls["flash_attention_packed"](q.clone().requires_grad_())


def test_schemas():
    want = {
        "append_paged_kv": "(Tensor query, Tensor key, Tensor value, Tensor cos, Tensor sin, Tensor(a!) key_cache, Tensor(b!) value_cache, "
                           "Tensor page_table, Tensor lengths, Tensor? offsets, bool interleaved, Tensor(c!) query_out, Tensor(d!)? key_out) -> ()",
        "flash_decode_paged": "(Tensor query, Tensor key_cache, Tensor value_cache, Tensor page_table, Tensor lengths, float softmax_scale, "
                              "Tensor(a!) out) -> ()",
        "flash_attention_packed": "(Tensor query, Tensor key, Tensor value, Tensor offsets, Tensor? kv_offsets, float softmax_scale, bool causal, "
                                  "Tensor(a!) out, Tensor(b!)? lse) -> ()",
        "flash_attention_packed_backward": "(Tensor grad_out, Tensor query, Tensor key, Tensor value, Tensor out, Tensor lse, Tensor offsets, "
                                           "Tensor? kv_offsets, float softmax_scale, bool causal, Tensor(a!)? grad_query, Tensor(b!)? grad_key, "
                                           "Tensor(c!)? grad_value) -> ()",
    }
    for name, schema in want.items():
        assert str(getattr(torch.ops.tilefusion, name).default._schema) == f"tilefusion::{name}{schema}"
        assert callable(getattr(ops, name))


# ---- the comparisons ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_the_comparison_passes_its_own_rounding_and_sees_mistakes(dtype):
    g = torch.Generator().manual_seed(8)
    q, k, v = (torch.randn(n, 64, generator=g).to(dtype) for n in (33, 40, 40))
    masked = torch.arange(40)[None] > torch.arange(33)[:, None] + 7
    step, floor = ref.half_step(dtype) + 2.0 ** -20, 2.0 ** -25 if dtype == torch.float16 else 0.0
    want, lse, bound, lse_bound = ref.attend(q, k, v, 0.125, masked, step, floor)
    ref.assert_within(want.to(dtype), want, bound)
    ref.assert_within(lse.float(), lse, lse_bound)
    # (the mistakes are planted in the oracle)
    wrong = {"mask": ref.attend(q, k, v, 0.125, masked.roll(1, dims=1), step, floor), "scale": ref.attend(q, k, v, 0.127, masked, step, floor),
             "key": ref.attend(q, torch.cat([k[:-1], k[:1]]), v, 0.125, masked, step, floor)}
    for name, (out, l, _, _) in wrong.items():
        with pytest.raises(AssertionError):
            ref.assert_within(out.to(dtype), want, bound, name)
    x, position = torch.randn(5, 2, 64, generator=g).to(dtype), torch.arange(5) + 90
    cos, sin = ops.rotation_tables(100, 32, device="cpu")
    turned, bound = ref.rotate(x, position, cos, sin, False)
    ref.assert_within(turned.to(dtype), turned, bound)
    assert torch.equal(turned[..., 32:], x[..., 32:].double())
    for other in (ref.rotate(x, position + 1, cos, sin, False)[0], ref.rotate(x, position, cos, sin, True)[0], ref.rotate(x, position, cos, -sin, False)[0]):
        with pytest.raises(AssertionError):
            ref.assert_within(other.to(dtype), turned, bound)
    # a turn keeps a pair's length, and the product of two turned by one angle
    pairs = lambda y: y[..., :16] ** 2 + y[..., 16:32] ** 2
    torch.testing.assert_close(pairs(turned), pairs(x.double()), rtol=1e-6, atol=1e-6)


def test_heads_of_packed_operands_lie_anywhere():
    # a [heads, tokens, D] of 2^17 tokens x 128, turned: heads 2^24 elements apart.  (What is refused in these calls is another argument, so that none runs.)
    lib = _capi.load()
    size = lib.tf_flash_attention_packed_backward_workspace_bytes

    def refused(message, **changed):
        p = _packed(**changed)
        for status in (lib.tf_flash_attention_packed(p, P + 8, P, None),
                       lib.tf_flash_attention_packed_backward(p, P, P, P, P + 8, P, P, P, size(p), None)):
            assert status == BAD and message in lib.tf_last_error(), (changed, lib.tf_last_error())

    far = 1 << 24
    for name in ("query_strides", "key_strides", "value_strides"):
        refused(b"boundar", **{name: _i64(128, far)})
        refused(b"boundar", **{name: _i64(128, far)}, D=128)
        refused(b"strides", **{name: _i64(far, 128)})
        refused(b"strides", **{name: _i64(128, far + 4)})
        refused(b"strides", **{name: _i64(128, -far)})
        refused(b"strides", **{name: _i64(128, 1 << 40)})
    for name in ("key_strides", "value_strides"):
        refused(b"boundar", **{name: _i64(128, 1 << 34)})
    # the heads of a group are reached from one another in 32 bits, one head alone is not
    refused(b"within 2^31", query_strides=_i64(128, 1 << 30))
    refused(b"boundar", query_strides=_i64(128, 1 << 30), heads=2)
    refused(b"boundar", query_strides=_i64(128, 1 << 34), heads=2)


def test_the_wrapper_copies_what_the_kernels_do_not_reach():
    from tilefusion_amd.ops.flash_attention_packed import _within_reach

    def rows(n, heads, token, head):
        return torch.empty((n - 1) * token + (heads - 1) * head + 64, dtype=torch.float16).as_strided((n, heads, 64), (token, head, 1))

    near = rows(2, 2, 128, 64)
    for q, k, copied in ((near, near, (False, False)), (rows(2, 2, 64, 1 << 24), near, (False, False)), (rows(2, 2, 64, 1 << 24), rows(2, 2, 64, 1 << 24), (False, False)),
                         (rows(2, 2, 1 << 24, 64), near, (True, False)), (near, rows(2, 2, 1 << 24, 64), (False, True)), (rows(1, 2, 1 << 24, 64), near, (False, False)),
                         (rows(2, 2, 64, 1 << 30), rows(2, 1, 64, 64), (True, False)), (rows(2, 2, 64, 1 << 30), rows(2, 2, 64, 64), (False, False))):
        got_q, got_k, got_v = _within_reach(q, k, k)
        assert [got_q is not q, got_k is not k, got_v is not k] == [copied[0], copied[1], copied[1]]
        assert not copied[0] or (got_q.is_contiguous() and got_q.shape == q.shape)
        assert not copied[1] or (got_k.is_contiguous() and got_k.shape == k.shape)


def test_new_tokens_have_places_of_their_own():
    # rows of the cache that would lie on each other in part: two tokens' rows would be written to one place, in no order
    lib = _capi.load()

    def call(**changed):   # (refused in any case: half of an odd number is turned)
        status = lib.tf_append_paged_kv(_cache(**changed), P, P, P, _i64(256, 64, 128, 64, 128, 64), P, P, 100, 33, 0, None, 3, 4, P, P, None)
        assert status == BAD
        return b"on each other" in lib.tf_last_error()

    # 8 pages of 16 tokens, 2 heads x 64, strides of page, token and head
    for strides in ((2048, 64, 1024), (2048, 128, 64), (64, 1024, 512), (64, 512, 1 << 20), (1 << 33, 64, 1024), (4096, 128, 2048), (1 << 62, 64, 1024)):
        assert not call(key_strides=_i64(*strides)) and not call(value_strides=_i64(*strides)), strides
    for strides in ((1024, 64, 1024), (2048, 64, 64), (2040, 128, 64), (64, 64, 64), (64, 504, 1 << 20), (2048, 0, 1024), (0, 64, 1024), (2048, 64, 0),
                    (2048, 64, 960), (128, 64, 1 << 20)):
        assert call(key_strides=_i64(*strides)) and call(value_strides=_i64(*strides)), strides
    # the stride of one alone says nothing
    assert not call(kv_heads=1, key_strides=_i64(1024, 64, 0)) and not call(pages=1, key_strides=_i64(64, 64, 1024))
    assert not call(page_size=1, key_strides=_i64(128, 0, 64), value_strides=_i64(128, 64, 64))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("causal", [False, True])
def test_the_comparisons_of_gradients_see_factors(dtype, causal):
    g = torch.Generator().manual_seed(5)
    lengths = [25, 15]
    q, do = (torch.randn(40, 4, 64, generator=g).to(dtype) for _ in range(2))
    k, v = (torch.randn(40, 2, 64, generator=g).to(dtype) for _ in range(2))
    problem = (q, k, v, do, lengths, 0.125, causal)
    out, lse = torch.empty_like(q), torch.empty(4, 40)
    for a, b in ((0, 25), (25, 40)):
        masked = torch.ones(b - a, b - a).triu(1).bool() if causal else None
        for head in range(4):
            o, l, _, _ = ref.attend(q[a:b, head], k[a:b, head // 2], v[a:b, head // 2], 0.125, masked)
            out[a:b, head], lse[head, a:b] = o.to(dtype), l.float()
    want, bounds = ref.gradients(q, k, v, do, out, lse, lengths, 0.125, causal)
    right = [x.to(dtype) for x in want]
    for a, b, c in zip(right, want, bounds):
        ref.assert_within(a, b, c)
    ref.assert_slopes(right, *problem, bounds)
    # (the mistakes are planted in the oracle: a factor in one gradient, and a head that is left out of a group's sum)
    for n in range(3):
        for factor in (0.7, 0.9, 1.1, 1.3, 2.0, 0.125, -1.0):
            wrong = [x * factor if i == n else x for i, x in enumerate(want)]
            with pytest.raises(AssertionError):
                ref.assert_within(wrong[n].to(dtype), want[n], bounds[n])
            with pytest.raises(AssertionError):
                ref.assert_slopes([x.to(dtype) for x in wrong], *problem, bounds)
    less = do.clone()
    less[:, 1] = 0.0
    wrong = ref.gradients(q, k, v, less, out, lse, lengths, 0.125, causal)[0]
    for n in (1, 2):
        with pytest.raises(AssertionError):
            ref.assert_within(wrong[n].to(dtype), want[n], bounds[n])


def test_ranges_and_tiles_of_packed_sequences():
    subprocess.check_call(["make", "-C", CPP, "test_packed_sequences_host"], stdout=subprocess.DEVNULL)
    out = subprocess.run([os.path.join(CPP, "test_packed_sequences_host")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


def test_ranges_of_equal_cost():
    subprocess.check_call(["make", "-C", CPP, "test_equal_ranges_host"], stdout=subprocess.DEVNULL)
    out = subprocess.run([os.path.join(CPP, "test_equal_ranges_host")], capture_output=True, text=True, timeout=60)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout + out.stderr


@pytest.mark.parametrize("scale", [1e39, -1e39, 1e300, 2.4e38, -2.4e38])
def test_scales_beyond_fp32_are_refused(scale):
    # (the kernels scale by softmax_scale log2(e) in fp32, of which these make an infinity; the alignment of out is refused where the scale is not)
    lib = _capi.load()

    def statuses(scale):
        p = _packed(softmax_scale=scale)
        calls = [lambda: lib.tf_flash_attention_packed(p, P + 8, P, None),
                 lambda: lib.tf_flash_attention_packed_backward(p, P, P, P, P + 8, P, P, P, 1 << 20, None),
                 lambda: lib.tf_flash_decode_paged(_cache(), P, _i64(256, 64), P + 8, 4, scale, P, 1 << 30, None)]
        return [(call(), lib.tf_last_error()) for call in calls]

    assert all(status == BAD and b"softmax_scale" in error for status, error in statuses(scale))
    assert all(status == BAD and b"boundar" in error for status, error in statuses(math.copysign(2.3e38, scale)))


@pytest.mark.parametrize("name", ["flash_decode_paged", "flash_attention_packed", "flash_attention_packed_backward"])
def test_a_head_dimension_of_zero_is_refused_by_name(name):
    q, calls = _calls()
    with pytest.raises(RuntimeError, match=f"{name}: query must be"):
        calls[name](q[..., :0])
