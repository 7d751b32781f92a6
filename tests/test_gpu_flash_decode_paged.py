"""One new token of every sequence over a paged cache, against the formula in 64 bits."""

import math

import pytest
import torch

from tests import attention_ref as ref
from tilefusion_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _query(b, h, d, dtype, seed=1, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(b, h, d, generator=g) * spread).to(dtype).to(DEV)


def _check(q, cache, scale=None):
    got = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths, scale)
    want, bound = ref.decode(q, cache.keys, cache.values, scale)
    ref.assert_within(got, want, bound)
    return got


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lengths", [[1], [0, 1, 2, 15, 16, 17, 31, 32, 33], [127, 128, 129, 0, 0, 255, 257], [1000, 3, 5003], [40000]])
def test_lengths(dtype, d, lengths):
    cache = ref.Cache(lengths, 16, 2, d, dtype)
    _check(_query(len(lengths), 8, d, dtype), cache)


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (8, 8), (3, 1), (24, 8), (16, 1), (17, 1), (40, 2), (64, 1), (12, 4)])
def test_groups(heads, kv_heads):
    for d in (64, 128):
        cache = ref.Cache([77, 600, 0, 2049], 32, kv_heads, d, torch.bfloat16)
        _check(_query(4, heads, d, torch.bfloat16), cache)


@pytest.mark.parametrize("page", [16, 32, 48, 64, 128, 256, 1008])
@pytest.mark.parametrize("layout", ["heads", "tokens"])
def test_pages_and_layouts(page, layout):
    for d in (64, 128):
        cache = ref.Cache([1500, 16, 1, 1008, 1009], page, 4, d, torch.float16, layout)
        _check(_query(5, 8, d, torch.float16), cache)


@pytest.mark.parametrize("n", [1, 64, 65, 300, 1030])
def test_many_sequences(n):
    g = torch.Generator().manual_seed(n)
    lengths = torch.randint(0, 200, (n,), generator=g).tolist()
    cache = ref.Cache(lengths, 16, 1, 64, torch.float16)
    _check(_query(n, 2, 64, torch.float16), cache)


@pytest.mark.parametrize("scale", [0.0, 1.0, -0.3, 1e-3, 4.0])
def test_scales(scale):
    cache = ref.Cache([513, 70], 16, 2, 64, torch.bfloat16)
    _check(_query(2, 4, 64, torch.bfloat16), cache, scale)


def test_weights_far_below_the_largest_count_in_fp16():
    # one key ahead of 30000 equal ones by 20 (in units of log2), whose weights are together 3% of the result
    d, n = 64, 30001
    cache = ref.Cache([n], 16, 1, d, torch.float16)
    key, value = torch.zeros(n, 1, d), torch.ones(n, 1, d)
    key[12345, 0, 0], value[12345] = 20.0, -1.0
    pages, rows = cache.places(0, 0, n)
    cache.keys, cache.values = [key.half().to(DEV)], [value.half().to(DEV)]
    cache.key[pages, rows], cache.value[pages, rows] = cache.keys[0], cache.values[0]
    q = torch.zeros(1, 1, d)
    q[..., 0] = 1.0
    _check(q.half().to(DEV), cache, math.log(2.0))


def test_large_scores():
    for spread in (30.0, 300.0):
        cache = ref.Cache([2000, 100], 16, 2, 128, torch.bfloat16)
        got = ops.flash_decode_paged(_query(2, 4, 128, torch.bfloat16, spread=spread), cache.key, cache.value, cache.table, cache.lengths, 1.0)
        # (nearly all weight on one key: between values that are there)
        assert got.isfinite().all() and got.abs().max() <= cache.values[0].abs().max().maximum(cache.values[1].abs().max())


def test_rows_behind_a_sequence_are_not_seen():
    # (the cache's unused rows are NaN already: here infinities, and of the kind that a zero weight would turn to NaN)
    for d in (64, 128):
        cache = ref.Cache([5, 130, 47], 64, 2, d, torch.float16, extra=0)
        q = _query(3, 8, d, torch.float16)
        first = _check(q, cache)
        for fill in (math.inf, -math.inf, 0.0):
            cache.key[cache.key.isnan() | cache.key.isinf()] = fill
            cache.value[cache.value.isnan() | cache.value.isinf()] = fill
            assert torch.equal(ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths), first)
            cache.key[cache.key == fill] = math.inf
            cache.value[cache.value == fill] = math.inf


def test_an_infinite_value_stays_in_its_column():
    cache = ref.Cache([300, 300], 16, 1, 64, torch.bfloat16)
    q = _query(2, 2, 64, torch.bfloat16)
    first = _check(q, cache)
    page, row = cache.places(0, 299, 300)
    cache.value[page, row, 0, 5] = math.inf
    got = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
    assert (got[0, :, 5] == math.inf).all()
    got[0, :, 5] = first[0, :, 5]
    assert torch.equal(got, first)


def test_pages_that_the_cache_does_not_have():
    lengths = [100, 50, 40, 0, 33]
    for bad in (-1, 10 ** 6, 2 ** 31 - 1):
        cache = ref.Cache(lengths, 16, 2, 64, torch.float16)
        q = _query(5, 4, 64, torch.float16)
        first = _check(q, cache)
        cache.table[0, 3] = bad
        got = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
        assert got[0].isnan().all() and torch.equal(got[1:], first[1:])


def test_lengths_beyond_the_table_and_below_zero():
    cache = ref.Cache([100, 50, 40, 0, 33], 16, 2, 64, torch.float16)
    q = _query(5, 4, 64, torch.float16)
    first = _check(q, cache)
    width = cache.table.shape[1]
    for bad in (16 * width + 1, 2 ** 31 - 1):
        cache.lengths[1] = bad
        got = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
        keep = [0, 2, 3, 4]
        assert got[1].isnan().all() and torch.equal(got[keep], first[keep])
    cache.lengths[1] = -5
    got = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
    assert (got[1] == 0).all()


def test_two_sequences_share_pages():
    cache = ref.Cache([200, 200], 16, 2, 128, torch.bfloat16)
    cache.table[1, :10] = cache.table[0, :10]
    cache.keys[1][:160], cache.values[1][:160] = cache.keys[0][:160], cache.values[0][:160]
    _check(_query(2, 8, 128, torch.bfloat16), cache)


def test_queries_and_tables_with_strides():
    cache = ref.Cache([200, 17, 900], 16, 2, 128, torch.bfloat16)
    wide = _query(3, 12, 128, torch.bfloat16)
    want = ops.flash_decode_paged(wide[:, 2:10].contiguous(), cache.key, cache.value, cache.table, cache.lengths)
    assert torch.equal(ops.flash_decode_paged(wide[:, 2:10], cache.key, cache.value, cache.table, cache.lengths), want)
    turned = wide[:, 2:10].permute(1, 0, 2).contiguous().permute(1, 0, 2)
    assert torch.equal(ops.flash_decode_paged(turned, cache.key, cache.value, cache.table, cache.lengths), want)
    odd = torch.zeros(3 * 8 * 128 + 1, dtype=torch.bfloat16, device=DEV)[1:].view(3, 8, 128)
    odd.copy_(wide[:, 2:10])
    assert torch.equal(ops.flash_decode_paged(odd, cache.key, cache.value, cache.table, cache.lengths), want)
    table = torch.full((3, cache.table.shape[1] + 5), -1, dtype=torch.int32, device=DEV)
    table[:, 2:-3] = cache.table
    assert torch.equal(ops.flash_decode_paged(wide[:, 2:10], cache.key, cache.value, table[:, 2:-3], cache.lengths), want)


def test_the_same_bits_every_time():
    cache = ref.Cache([5000, 1, 3333, 100, 0, 2047], 16, 4, 128, torch.float16)
    q = _query(6, 16, 128, torch.float16)
    first = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
    for _ in range(20):
        assert torch.equal(ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths), first)


def test_replayed_with_other_lengths_and_on_other_streams():
    lengths = [700, 64, 3000, 1]
    cache = ref.Cache(lengths, 16, 2, 128, torch.bfloat16)
    q = _query(4, 8, 128, torch.bfloat16)
    ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
        graphs.append((graph, out))
    for cut in (0, 10, 63, 0, 500):
        now = [max(0, n - cut) for n in lengths]
        cache.lengths.copy_(torch.tensor(now, dtype=torch.int32))
        want = ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths)
        for graph, out in graphs:
            out.zero_()
            graph.replay()
        torch.cuda.synchronize()
        exact, bound = ref.decode(q, [k[:n] for k, n in zip(cache.keys, now)], [v[:n] for v, n in zip(cache.values, now)])
        for _, out in graphs:
            assert torch.equal(out, want)
        ref.assert_within(want, exact, bound)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    outs = []
    for n in range(12):
        with torch.cuda.stream(streams[n % 3]):
            outs.append(ops.flash_decode_paged(q, cache.key, cache.value, cache.table, cache.lengths))
    torch.cuda.synchronize()
    for out in outs:
        assert torch.equal(out, want)


def test_offsets_beyond_32_bits():
    # pages of 2 GiB between the first and the last that are used
    d, page = 128, 16
    pages = 2 ** 33 // (page * d * 2)   # 8 GiB of keys, of which three pages are touched
    key, value = (torch.empty(pages, page, 1, d, dtype=torch.float16, device=DEV) for _ in range(2))
    cache = ref.Cache([40], page, 1, d, torch.float16)
    where = [pages - 1, 0, pages // 2 + 3]
    for i, p in enumerate(where):
        key[p], value[p] = cache.key[cache.table[0, i].long()], cache.value[cache.table[0, i].long()]
    q = _query(1, 4, d, torch.float16)
    got = ops.flash_decode_paged(q, key, value, torch.tensor([where], dtype=torch.int32, device=DEV), cache.lengths)
    assert torch.equal(got, _check(q, cache))


def test_refusals():
    cache = ref.Cache([40, 3], 16, 2, 64, torch.float16)
    q = _query(2, 4, 64, torch.float16)
    args = [q, cache.key, cache.value, cache.table, cache.lengths]
    def bad(message, scale=None, **changed):
        call = [changed.get(str(i), a) for i, a in enumerate(args)]
        with pytest.raises(RuntimeError, match=message):
            ops.flash_decode_paged(*call, scale)
    def at(i, t):
        return {str(i): t}
    bad("must be float16 or bfloat16", **at(0, q.float()))
    bad("dtype", **at(1, cache.key.bfloat16()))
    bad("shape of key_cache", **at(2, cache.value[:1]))
    bad("int32", **at(3, cache.table.long()))
    bad("int32", **at(4, cache.lengths.long()))
    bad("CUDA", **at(4, cache.lengths.cpu()))
    bad("CUDA", **at(1, cache.key.cpu()))
    bad("page_table", **at(3, cache.table[:1]))
    bad("multiple", **at(0, _query(2, 3, 64, torch.float16)))
    bad("query must be", **at(0, q[0]))
    bad("query must be", **at(0, _query(2, 4, 128, torch.float16)))
    bad("finite", scale=math.inf)
    bad("finite", scale=math.nan)
    small = ref.Cache([40, 3], 8, 2, 64, torch.float16)
    bad("multiple of 16", **{"1": small.key, "2": small.value, "3": small.table})
    narrow = ref.Cache([40, 3], 16, 2, 32, torch.float16)
    bad("head dim", **{"0": _query(2, 4, 32, torch.float16), "1": narrow.key, "2": narrow.value})
    bad("places of their own", **at(1, cache.key[:1].expand(cache.key.shape)))
    with pytest.raises(RuntimeError, match="no gradient"):
        ops.flash_decode_paged(q.clone().requires_grad_(), *args[1:])
    with torch.no_grad():
        ops.flash_decode_paged(q.clone().requires_grad_(), *args[1:])
    assert ops.flash_decode_paged(q[:0], cache.key, cache.value, cache.table[:0], cache.lengths[:0]).shape == (0, 4, 64)
