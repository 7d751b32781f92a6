"""The operators of a paged cache and of packed sequences as programs use them together: prompts that enter a cache while they are attended to,
further pieces of a prompt, tokens one by one out of a captured graph; and a layer's attention under autograd in front of its gated block."""

import pytest
import torch

from tests import attention_ref as ref
from tests.test_gpu_flash_attention_packed import _want
from tilefusion_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
H, HKV, D, PAGE, SLOTS, PAGES = 8, 2, 128, 16, 4, 20


def _offsets(lengths):
    return torch.tensor([0] + torch.tensor(lengths).cumsum(0).tolist(), dtype=torch.int32, device=DEV)


class _Server:
    """Slots with what they hold kept aside, to compare with."""

    def __init__(self, dtype, interleaved):
        g = torch.Generator().manual_seed(11)
        self.g, self.dtype, self.interleaved = g, dtype, interleaved
        self.cos, self.sin = ops.rotation_tables(PAGES * PAGE, 64 if interleaved else D, device=DEV)
        # (unused rows hold NaN, pages are of any slot)
        self.key, self.value = (torch.full((SLOTS * PAGES, HKV, PAGE, D), float("nan"), dtype=dtype, device=DEV).permute(0, 2, 1, 3) for _ in range(2))
        self.table = torch.randperm(SLOTS * PAGES, generator=g).to(torch.int32).view(SLOTS, PAGES).to(DEV)
        self.lengths = torch.zeros(SLOTS, dtype=torch.int32, device=DEV)
        self.keys, self.values = ([torch.zeros(0, HKV, D, dtype=dtype, device=DEV) for _ in range(SLOTS)] for _ in range(2))

    def projection(self, tokens):
        """Queries, keys and values of new tokens: slices of one tensor."""
        x = torch.randn(tokens, H + 2 * HKV, D, generator=self.g).to(self.dtype).to(DEV)
        return x, (x[:, :H], x[:, H:H + HKV], x[:, H + HKV:])

    def remember(self, new, q, k, v, got_q, got_k):
        """The new tokens' rotation and their places, checked; what the slots hold from now on is what is in the cache."""
        at = 0
        for b, n in enumerate(new):
            if n == 0:
                continue
            first, rows = self.keys[b].shape[0], slice(at, at + n)
            position = torch.arange(first, first + n, device=DEV)
            pages, places = self.table[b].long()[position // PAGE], position % PAGE
            for got, x in ((got_q[rows], q[rows]), (self.key[pages, places], k[rows])):
                want, bound = ref.rotate(x, position, self.cos, self.sin, self.interleaved)
                ref.assert_within(got, want, bound, f"slot {b}")
            assert got_k is None or torch.equal(self.key[pages, places], got_k[rows])
            assert torch.equal(self.value[pages, places], v[rows])
            self.keys[b] = torch.cat([self.keys[b], self.key[pages, places]])
            self.values[b] = torch.cat([self.values[b], self.value[pages, places]])
            at += n

    def prompts(self, new):
        _, (q, k, v) = self.projection(sum(new))
        self.lengths += torch.tensor(new, dtype=torch.int32, device=DEV)
        before = [x.shape[0] for x in self.keys]
        got_q, got_k = ops.append_paged_kv(q, k, v, self.cos, self.sin, self.key, self.value, self.table, self.lengths, _offsets(new), self.interleaved, True)
        self.remember(new, q, k, v, got_q, got_k)
        if any(before):   # a further piece: its slot's keys up to here
            keys, values = torch.cat(self.keys), torch.cat(self.values)
            out = ops.flash_attention_packed(got_q, keys, values, _offsets(new), _offsets([x.shape[0] for x in self.keys]))
        else:
            keys, values = got_k, v
            out = ops.flash_attention_packed(got_q, keys, values, _offsets(new))
        want, bound, _, _ = _want(got_q, keys, values, new, [x.shape[0] for x in self.keys], D ** -0.5, True)
        ref.assert_within(out, want, bound, "prompts")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("interleaved", [False, True])
def test_conversations(dtype, interleaved):
    server = _Server(dtype, interleaved)
    server.prompts([70, 0, 133, 16])
    server.prompts([31, 0, 1, 64])
    # a step of all slots, of which one is idle, captured: the lengths grow on the device
    active = torch.tensor([1, 0, 1, 1], dtype=torch.int32, device=DEV)
    x, (q, k, v) = server.projection(SLOTS)

    def step():
        server.lengths.add_(active)
        turned = ops.append_paged_kv(q, k, v, server.cos, server.sin, server.key, server.value, server.table, server.lengths, None, interleaved)
        return turned, ops.flash_decode_paged(turned, server.key, server.value, server.table, server.lengths)

    ops.flash_decode_paged(q, server.key, server.value, server.table, server.lengths)   # (what a first call sets up)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, out = step()
    for n in range(20):   # over the ends of pages
        x.copy_(server.projection(SLOTS)[0])
        if n % 5 == 4:
            now, got = step()
        else:
            out.fill_(7.0)
            graph.replay()
            now, got = turned, out
        torch.cuda.synchronize()
        used = active.bool()
        server.remember(active.tolist(), q[used], k[used], v[used], now[used], None)
        assert server.lengths.tolist() == [y.shape[0] for y in server.keys] and (now[~used] == 0).all()
        want, bound = ref.decode(now, server.keys, server.values)
        ref.assert_within(got, want, bound, f"step {n}")
        assert torch.equal(ops.flash_decode_paged(now, server.key, server.value, server.table, server.lengths), got)
    # one slot's text again, as one piece: its last token's row is that of the decoding, within both bounds
    keys, values = server.keys[2], server.values[2]
    one = ops.flash_attention_packed(now[2:3], keys, values, _offsets([1]), _offsets([keys.shape[0]]))
    want, bound, _, _ = _want(now[2:3], keys, values, [1], [keys.shape[0]], D ** -0.5, True)
    ref.assert_within(one, want, bound, "one piece")


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_a_layer_under_autograd_is_its_calls_one_by_one(dtype):
    g = torch.Generator().manual_seed(2)
    lengths, f = [130, 1, 64, 77], 264
    t = sum(lengths)
    x = torch.randn(t + 3, H + 2 * HKV, D, generator=g).to(dtype).to(DEV).requires_grad_()
    w = [(torch.randn(f, H * D, generator=g) * (H * D) ** -0.5).to(dtype).to(DEV).requires_grad_() for _ in range(2)]
    grad = torch.randn(t + 3, f, generator=g).to(dtype).to(DEV)
    offsets = _offsets(lengths)

    out = ops.flash_attention_packed(x[:, :H], x[:, H:H + HKV], x[:, H + HKV:], offsets)
    ops.gated_ffn(out.flatten(1), *w).backward(grad)

    with torch.no_grad():
        q, k, v = x[:, :H], x[:, H:H + HKV], x[:, H + HKV:]
        out, lse = ops.flash_attention_packed(q, k, v, offsets, keep=True)
        _, gate, up = ops.gated_ffn(out.flatten(1), *w, keep=True)
        grad_out, *grad_w = ops.gated_ffn_backward(grad, out.flatten(1), *w, gate, up)
        grads = ops.flash_attention_packed_backward(grad_out.view(out.shape), q, k, v, out, lse, offsets)
    assert torch.equal(x.grad, torch.cat(grads, dim=1))
    for a, b in zip(w, grad_w):
        assert torch.equal(a.grad, b)


def test_compiled_calls_are_the_eager_ones():
    server = _Server(torch.bfloat16, False)
    server.prompts([40, 3, 0, 18])
    _, (q, k, v) = server.projection(SLOTS)
    lengths = server.lengths + torch.tensor([1, 1, 0, 1], dtype=torch.int32, device=DEV)

    def step(q, k, v, key, value):
        turned = ops.append_paged_kv(q, k, v, server.cos, server.sin, key, value, server.table, lengths)
        return turned, ops.flash_decode_paged(turned, key, value, server.table, lengths)

    def texts(q, k, v):
        return ops.flash_attention_packed(q, k, v, torch.tensor([0, 1, 4], dtype=torch.int32, device=DEV))

    caches = [[x.clone(memory_format=torch.preserve_format) for x in (server.key, server.value)] for _ in range(2)]
    with torch.no_grad():
        want, got = step(q, k, v, *caches[0]), torch.compile(step, backend="eager")(q, k, v, *caches[1])
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        assert all(torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) for a, b in zip(*caches))
        assert torch.equal(texts(q, k, v), torch.compile(texts, backend="eager")(q, k, v))
