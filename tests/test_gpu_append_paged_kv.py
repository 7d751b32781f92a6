"""New tokens enter a paged cache with their positions rotated in, against the formula in 64 bits."""

import math

import pytest
import torch

from tests import attention_ref as ref
from tilefusion_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _rows(t, h, hkv, d, dtype, seed=3):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(t, n, d, generator=g).to(dtype).to(DEV) for n in (h, hkv, hkv)]


def _offsets(new):
    return torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


def _check(lengths, new, page=16, h=4, hkv=2, d=64, rotated=None, interleaved=False, dtype=torch.float16, layout="heads", tail=0, with_offsets=True):
    cache = ref.Cache(lengths, page, hkv, d, dtype, layout)
    before = cache.key.clone(), cache.value.clone()
    cos, sin = ops.rotation_tables(max(lengths) + 1, rotated or d, device=DEV)
    t = sum(new)
    q, k, v = _rows(t + tail, h, hkv, d, dtype)
    got_q, got_k = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths, _offsets(new) if with_offsets else None,
                                       interleaved, True)
    at = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        if n == 0:
            continue
        position = torch.arange(length - n, length, device=DEV)
        rows = slice(at, at + n)
        pages, places = cache.places(b, length - n, length)
        for got, x in ((got_q, q), (got_k, k)):
            want, bound = ref.rotate(x[rows], position, cos, sin, interleaved)
            ref.assert_within(got[rows], want, bound, f"sequence {b}")
        assert torch.equal(cache.key[pages, places], got_k[rows])
        assert torch.equal(cache.value[pages, places], v[rows])
        # ... and nothing else in the cache has changed
        cache.key[pages, places], cache.value[pages, places] = before[0][pages, places], before[1][pages, places]
        at += n
    for a, b in zip((cache.key, cache.value), before):
        assert torch.equal(a.nan_to_num(nan=-9.0), b.nan_to_num(nan=-9.0))
    assert (got_q[t:] == 0).all() and (got_k[t:] == 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("lengths,new", [([1], [1]), ([16, 17, 100, 33], [16, 1, 70, 0]), ([5, 5, 5], [5, 0, 5]), ([2000, 1, 129], [1999, 1, 128])])
def test_prompts(dtype, d, interleaved, lengths, new):
    _check(lengths, new, dtype=dtype, d=d, interleaved=interleaved, tail=3)


@pytest.mark.parametrize("n", [1, 63, 64, 65, 200, 4100, 5000])
def test_a_token_each(n):
    g = torch.Generator().manual_seed(n)
    lengths = torch.randint(1, 40, (n,), generator=g).tolist()
    _check(lengths, [1] * n, h=2, hkv=1)
    _check(lengths, [1] * n, h=2, hkv=1, with_offsets=False)


@pytest.mark.parametrize("rotated", [2, 6, 16, 24, 32, 48, 64])
@pytest.mark.parametrize("interleaved", [False, True])
def test_part_of_a_head(rotated, interleaved):
    _check([50, 3], [20, 3], rotated=rotated, interleaved=interleaved)
    _check([50, 3], [20, 3], rotated=rotated, interleaved=interleaved, d=128, dtype=torch.bfloat16)


@pytest.mark.parametrize("page", [1, 7, 16, 48, 256])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_pages_and_layouts(page, layout):
    _check([300, 1, 49], [260, 1, 48], page=page, layout=layout, h=3, hkv=3)
    _check([300, 1, 49], [260, 1, 48], page=page, layout=layout, h=40, hkv=8, d=128)


def test_empty_sequences_between():
    new = [0] * 70 + [3] + [0] * 100 + [2, 0, 0, 1] + [0] * 5
    _check([max(n, 9) for n in new], new, h=1, hkv=1, tail=1)


def test_far_positions():
    # the tables hold the angle's cosine to the last bit of fp32 wherever the position is
    cos, sin = ops.rotation_tables(300000, 128, device=DEV)
    p, i = 299999, torch.arange(64, dtype=torch.float64, device=DEV)
    angle = p * 10000.0 ** (-i / 64)
    assert (cos[p].double() - angle.cos()).abs().max() <= 2.0 ** -24 and (sin[p].double() - angle.sin()).abs().max() <= 2.0 ** -24
    _check([290001], [5], page=256, d=128)


def test_slices_of_one_projection():
    lengths = [40, 3, 77]
    cache = ref.Cache(lengths, 16, 2, 64, torch.bfloat16)
    cos, sin = ops.rotation_tables(100, 64, device=DEV)
    wide = _rows(3, 12, 2, 64, torch.bfloat16)[0].flatten(1)
    q, k, v = (x.unflatten(1, (-1, 64)) for x in wide.split([8 * 64, 2 * 64, 2 * 64], dim=1))
    assert not q.is_contiguous()
    first = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths)
    stored = cache.key.clone(), cache.value.clone()
    second = ops.append_paged_kv(q.contiguous(), k.contiguous(), v.contiguous(), cos, sin, cache.key, cache.value, cache.table, cache.lengths)
    assert torch.equal(first, second)
    assert all(torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in zip(stored, (cache.key, cache.value)))


def test_tokens_without_a_place():
    lengths, new = [40, 33, 20], [4, 3, 2]
    q, k, v = _rows(9, 4, 2, 64, torch.float16)
    cos, sin = ops.rotation_tables(41, 64, device=DEV)

    def run(change):
        cache = ref.Cache(lengths, 16, 2, 64, torch.float16)
        tables = [cos, sin]
        change(cache, tables)
        before = cache.key.clone(), cache.value.clone()
        out = ops.append_paged_kv(q, k, v, *tables, cache.key, cache.value, cache.table, cache.lengths, _offsets(new), False, True)
        changed = [(a.nan_to_num(nan=-9.0) != b.nan_to_num(nan=-9.0)).any(dim=(2, 3)) for a, b in zip((cache.key, cache.value), before)]
        assert torch.equal(*changed)
        return cache, out, changed[0]

    _, good, changed = run(lambda cache, tables: None)
    assert changed.sum() == 9
    for bad in (-1, 10 ** 6, 2 ** 31 - 1):
        # positions 30 .. 32 of sequence 1: the last one's page is missing
        _, out, changed = run(lambda cache, tables: cache.table.__setitem__((1, 2), bad))
        assert changed.sum() == 8
        for x, y in zip(out, good):
            assert x[6].isnan().all() and torch.equal(x[:6], y[:6]) and torch.equal(x[7:], y[7:])
    # longer than its row of the table
    _, out, changed = run(lambda cache, tables: cache.lengths.__setitem__(1, 16 * cache.table.shape[1] + 1))
    assert out[0][6].isnan().all() and not out[0][:4].isnan().any()
    _, out, changed = run(lambda cache, tables: cache.lengths.__setitem__(1, 2 ** 31 - 1))
    assert changed.sum() == 6 and out[0][4:7].isnan().all() and not out[0][7:].isnan().any()
    # tables of 38 positions: the last two of sequence 0
    _, out, changed = run(lambda cache, tables: tables.__setitem__(slice(None), [cos[:38].contiguous(), sin[:38].contiguous()]))
    assert changed.sum() == 7 and out[0][2:4].isnan().all() and torch.equal(out[0][:2], good[0][:2]) and torch.equal(out[0][4:], good[0][4:])
    # a sequence that is shorter than its new tokens, an idle slot
    for short in (1, 0, -3, -2 ** 31):
        _, out, changed = run(lambda cache, tables: cache.lengths.__setitem__(2, short))
        assert changed.sum() == 7 and (out[0][7:] == 0).all() and (out[1][7:] == 0).all()


def test_offsets_that_do_not_begin_at_zero():
    cache = ref.Cache([30, 20], 16, 2, 64, torch.float16)
    q, k, v = _rows(9, 4, 2, 64, torch.float16)
    cos, sin = ops.rotation_tables(64, 64, device=DEV)
    offsets = torch.tensor([2, 5, 7], dtype=torch.int32, device=DEV)
    out = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths, offsets)
    assert (out[:2] == 0).all() and (out[7:] == 0).all()
    want, bound = ref.rotate(q[2:5], torch.arange(27, 30, device=DEV), cos, sin, False)
    ref.assert_within(out[2:5], want, bound)


def test_replayed():
    lengths = [40, 3, 77]
    cache = ref.Cache(lengths, 16, 2, 128, torch.bfloat16)
    q, k, v = _rows(3, 4, 2, 128, torch.bfloat16)
    cos, sin = ops.rotation_tables(100, 128, device=DEV)
    ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths)
    for step in range(3):
        cache.lengths.copy_(torch.tensor([n - step for n in lengths], dtype=torch.int32))
        q.add_(0.5)
        graph.replay()
        torch.cuda.synchronize()
        other = ref.Cache(lengths, 16, 2, 128, torch.bfloat16)
        other.lengths.copy_(cache.lengths)
        assert torch.equal(out, ops.append_paged_kv(q, k, v, cos, sin, other.key, other.value, other.table, other.lengths))
        for b, n in enumerate(cache.lengths.tolist()):
            if n > 0:
                place = cache.places(b, n - 1, n)
                assert torch.equal(cache.key[place], other.key[place]) and torch.equal(cache.value[place], other.value[place])


def test_refusals():
    cache = ref.Cache([40, 3], 16, 2, 64, torch.float16)
    q, k, v = _rows(2, 4, 2, 64, torch.float16)
    cos, sin = ops.rotation_tables(64, 64, device=DEV)
    names = ["query", "key", "value", "cos", "sin", "key_cache", "value_cache", "page_table", "lengths", "offsets"]
    args = dict(zip(names, [q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths, None]))

    def bad(message, **changed):
        with pytest.raises(RuntimeError, match=message):
            ops.append_paged_kv(**{**args, **changed})

    bad("float16 or bfloat16", query=q.float())
    bad("dtype", key=k.bfloat16())
    bad("key must be", key=k[:, :1])
    bad("value must be", value=v[:1])
    bad("query must be", query=q[0])
    bad("one token for each", lengths=cache.lengths[:1], page_table=cache.table[:1])
    bad("float32", cos=cos.double())
    bad("rotated / 2", sin=sin[:, :8])
    bad("rotated must be", cos=torch.zeros(8, 33, device=DEV), sin=torch.zeros(8, 33, device=DEV))
    bad("rotated must be", cos=torch.zeros(8, 0, device=DEV), sin=torch.zeros(8, 0, device=DEV))
    bad("offsets must be", offsets=torch.zeros(2, dtype=torch.int32, device=DEV))
    bad("int32", offsets=torch.zeros(3, dtype=torch.int64, device=DEV))
    bad("CUDA", offsets=torch.zeros(3, dtype=torch.int32))
    bad("CUDA", page_table=cache.table.cpu())
    bad("places of their own", key_cache=cache.key[:1].expand(cache.key.shape))
    bad("shape of key_cache", value_cache=cache.value[1:])
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.append_paged_kv(q.clone().requires_grad_(), *list(args.values())[1:])
    for positions, rotated in ((-1, 64), (8, 0), (8, 3)):
        with pytest.raises(RuntimeError, match="rotation_tables"):
            ops.rotation_tables(positions, rotated, device=DEV)
    empty = ops.append_paged_kv(q[:0], k[:0], v[:0], cos, sin, cache.key, cache.value, cache.table, cache.lengths, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert empty.shape == (0, 4, 64)


@pytest.mark.parametrize("through_the_dispatcher", [False, True])
def test_autograd_sees_that_the_cache_has_changed(through_the_dispatcher):
    # what was saved of the cache for a backward pass is not what it was: that raises, as for any change in place
    g = torch.Generator().manual_seed(4)
    lengths = [40, 33]
    cache = ref.Cache(lengths, 16, 2, 64, torch.float16)
    q, k, v = _rows(2, 4, 2, 64, torch.float16)
    cos, sin = ops.rotation_tables(41, 64, device=DEV)
    if through_the_dispatcher:   # (tables in pieces are made whole, which the direct call leaves to the wrapper)
        cos, sin = (torch.cat([x, x], dim=1)[:, :32] for x in (cos, sin))

    def append():
        return ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths, None, False, True)

    for saved in (cache.key, cache.value):
        x = torch.randn(saved[0].shape, generator=g).half().to(DEV).requires_grad_()
        loss = (x * saved[0]).sum()
        loss.backward(retain_graph=True)
        append()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()
    # a sequence's pages, attended to where they lie
    rows = cache.table[0, :1].long()
    one = slice(int(rows), int(rows) + 1)
    q1 = torch.randn(16, 4, 64, generator=g).half().to(DEV).requires_grad_()
    offsets = _offsets([16])
    out = ops.flash_attention_packed(q1, cache.key[one].squeeze(0), cache.value[one].squeeze(0), offsets)
    append()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.sum().backward()
    # the inputs have not changed, and a call without tokens changes nothing
    versions = [x._version for x in (q, k, v, cache.table, cache.lengths, cache.key, cache.value)]
    ops.append_paged_kv(q[:0], k[:0], v[:0], cos, sin, cache.key, cache.value, cache.table, cache.lengths, torch.zeros(3, dtype=torch.int32, device=DEV))
    assert versions == [x._version for x in (q, k, v, cache.table, cache.lengths, cache.key, cache.value)]
    append()
    assert versions[:5] == [x._version for x in (q, k, v, cache.table, cache.lengths)]


def test_a_cache_of_inference_tensors():
    # (they count no changes, inside inference mode and outside)
    with torch.inference_mode():
        cache = ref.Cache([40, 33], 16, 2, 64, torch.float16)
        q, k, v = _rows(2, 4, 2, 64, torch.float16)
        cos, sin = ops.rotation_tables(41, 64, device=DEV)
        want = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths)
        stored = cache.key.clone()
    got = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths)
    assert torch.equal(got, want) and torch.equal(cache.key.nan_to_num(), stored.nan_to_num())


def test_results_that_a_program_hands_in_count_as_changed():
    # torch.ops.tilefusion: the results are arguments, which may be anyone's
    lengths = [5, 3]
    cache = ref.Cache(lengths, 16, 2, 64, torch.float16)
    q, k, v = _rows(2, 4, 2, 64, torch.float16)
    cos, sin = ops.rotation_tables(41, 64, device=DEV)
    offsets, direct = _offsets([1, 1]), torch.ops.tilefusion
    outs = {name: torch.zeros(shape, dtype=dtype, device=DEV) for name, shape, dtype in
            [("q", q.shape, q.dtype), ("k", k.shape, k.dtype), ("decoded", q.shape, q.dtype), ("out", q.shape, q.dtype), ("lse", (4, 2), torch.float32),
             ("dq", q.shape, q.dtype), ("dk", k.shape, k.dtype), ("dv", k.shape, k.dtype)]}
    before = {name: x._version for name, x in outs.items()}
    direct.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths, offsets, False, outs["q"], outs["k"])
    direct.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths, 0.125, outs["decoded"])
    direct.flash_attention_packed(q, k, v, offsets, None, 0.125, True, outs["out"], outs["lse"])
    after_forward = {name: outs[name]._version for name in ("out", "lse")}
    direct.flash_attention_packed_backward(q, q, k, v, outs["out"], outs["lse"], offsets, None, 0.125, True, outs["dq"], outs["dk"], outs["dv"])
    assert all(outs[name]._version > n for name, n in before.items())
    assert after_forward == {name: outs[name]._version for name in ("out", "lse")}


def test_caches_whose_rows_lie_on_each_other_are_refused():
    cache = ref.Cache([40, 3], 16, 2, 64, torch.float16)
    q, k, v = _rows(2, 4, 2, 64, torch.float16)
    cos, sin = ops.rotation_tables(64, 64, device=DEV)
    pages = cache.key.shape[0]
    # each page half of the one in front of it
    half = torch.zeros((pages + 1) * 1024, dtype=torch.float16, device=DEV).as_strided((pages, 16, 2, 64), (1024, 128, 64, 1))
    for caches in ((half, cache.value), (cache.key, half)):
        with pytest.raises(RuntimeError, match="on each other"):
            ops.append_paged_kv(q, k, v, cos, sin, *caches, cache.table, cache.lengths)
    assert (half == 0).all()
    # (read it may be)
    ops.flash_decode_paged(q, half, half, cache.table, cache.lengths)
    # keys and values side by side, of two layers in one tensor, in an order of dimensions that is neither of the usual ones
    both = torch.zeros(2, 16, pages, 2, 2, 64, dtype=torch.float16, device=DEV)
    key, value = (both[1, :, :, i].transpose(0, 1) for i in range(2))
    got = ops.append_paged_kv(q, k, v, cos, sin, key, value, cache.table, cache.lengths)
    want = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths)
    assert torch.equal(got, want) and (both[0] == 0).all()
    for b, n in enumerate([40, 3]):
        place = cache.places(b, n - 1, n)
        assert torch.equal(key[place], cache.key[place]) and torch.equal(value[place], cache.value[place])


def test_offsets_beyond_32_bits():
    # 8 GiB of keys, of which three pages are written, the last one among them
    d, page = 128, 16
    pages = 2 ** 33 // (page * d * 2)
    key, value = (torch.empty(pages, page, 1, d, dtype=torch.float16, device=DEV) for _ in range(2))
    cache = ref.Cache([40], page, 1, d, torch.float16)
    where = [pages - 1, 0, pages // 2 + 3]
    q, k, v = _rows(40, 4, 1, d, torch.float16)
    cos, sin = ops.rotation_tables(41, d, device=DEV)
    got = ops.append_paged_kv(q, k, v, cos, sin, key, value, torch.tensor([where], dtype=torch.int32, device=DEV), cache.lengths, _offsets([40]))
    want = ops.append_paged_kv(q, k, v, cos, sin, cache.key, cache.value, cache.table, cache.lengths, _offsets([40]))
    assert torch.equal(got, want)
    for i, p in enumerate(where):
        rows, own = min(page, 40 - i * page), cache.table[0, i].long()
        assert torch.equal(key[p, :rows], cache.key[own, :rows]) and torch.equal(value[p, :rows], cache.value[own, :rows])
