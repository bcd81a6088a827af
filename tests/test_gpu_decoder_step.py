"""The decoder operators as they are used together: prompts of ragged lengths through one layer's projections, cache and
attention, then steps of one token each.  Every stage is held against its 64-bit form over what the stage before it
left on the device, so each keeps the bound that it has alone."""
import numpy as np
import pytest
import torch

from iconnx_amd import ops
from tests import decoder_ref as ref

pytestmark = pytest.mark.gpu
TERMS = {torch.bfloat16: 1, torch.float16: 2, torch.float32: 3}
E, HQ, HKV, D, PAGE = 200, 6, 2, 64, 16


class Layer:
    def __init__(self, bits, dtype, lengths, room):
        g = torch.Generator().manual_seed(5)
        self.dtype, self.bits, self.lengths = dtype, bits, list(lengths)
        self.host = {}
        for name, (K, N) in dict(q=(E, HQ * D), kv=(E, 2 * HKV * D), out=(HQ * D, E)).items():
            w = torch.randint(-127, 128, (K, N), generator=g, dtype=torch.int8)
            s = (torch.rand(N, generator=g) + 0.5) * (K ** -0.5 / 73.0)  # (outputs about as large as the inputs)
            b = torch.randn(N, generator=g) * 0.1
            self.host[name] = (w.numpy(), s.numpy(), b.numpy())
            setattr(self, name, (ops.TokenWeight(w.cuda(), s.cuda()), b.cuda()))
        width = -(-(max(lengths) + room) // PAGE)
        self.cache = ops.KvCache(len(lengths) * width + 1, PAGE, HKV, D, bits=bits)
        self.table = torch.randperm(len(lengths) * width, generator=g).view(len(lengths), width).int().cuda()
        self.k, self.v = [[] for _ in lengths], [[] for _ in lengths]

    def slots(self, b, first, n):
        j = torch.arange(first, first + n).cuda()
        return self.table[b].long()[j // PAGE] * PAGE + j % PAGE

    def run(self, x, slots, lengths, starts=None):
        """(quantized x, its scales, q, keys and values, attention, y)"""
        qx, sx = ops.gpu_quantize_tokens(x)
        q = ops.gpu_token_qlinear(qx, self.q[0], x_scale=sx, bias=self.q[1], dtype=self.dtype).view(-1, HQ, D)
        kv = ops.gpu_token_qlinear(qx, self.kv[0], x_scale=sx, bias=self.kv[1], dtype=self.dtype).view(-1, 2 * HKV, D)
        ops.gpu_kv_cache_write(self.cache, kv[:, :HKV], kv[:, HKV:], slots)
        a = ops.gpu_kv_cache_attention(q, self.cache, self.table, lengths, q_starts=starts)
        y = ops.gpu_token_qlinear(a.view(-1, HQ * D), self.out[0], bias=self.out[1])
        return qx, sx, q, kv, a, y

    def product(self, name, q, s, y):
        want, p = ref.token_qlinear(q, s, *self.host[name])
        assert (np.abs(ref.f64(y).reshape(want.shape) - want) <= ref.token_qlinear_bound(want, p, self.dtype)).all(), name

    def check(self, x, stages, rows):
        """rows: of each sequence, whose last tokens they are; what it cached before is in self.k, self.v."""
        qx, sx, q, kv, a, y = stages
        wq, ws = ref.quantize_tokens(x)
        assert (ref.f64(qx) == wq).all() and (ref.f64(sx).astype(np.float32) == ws).all()
        self.product("q", wq, ws, q)
        self.product("kv", wq, ws, kv)
        starts = np.cumsum([0] + list(rows))
        for b, n in enumerate(rows):
            self.k[b].append(ref.cached(kv[starts[b]:starts[b + 1], :HKV], self.bits))
            self.v[b].append(ref.cached(kv[starts[b]:starts[b + 1], HKV:], self.bits))
        k, v = [np.concatenate(t) for t in self.k], [np.concatenate(t) for t in self.v]
        for b, n in enumerate(self.lengths):
            assert len(k[b]) == n
            rk, rv = ops.gpu_kv_cache_read(self.cache, self.slots(b, 0, n))
            assert (ref.f64(rk) == k[b]).all() and (ref.f64(rv) == v[b]).all()
        want, bound = ref.attention(q, k, v, self.lengths, starts, D ** -0.5, terms=TERMS[self.dtype], dtype=self.dtype)
        assert (np.abs(ref.f64(a) - want) <= bound).all()
        self.product("out", *ref.quantize_tokens(a.view(-1, HQ * D)), y)


def tokens(n, dtype, seed):
    return torch.randn(n, E, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


def ints(v):
    return torch.tensor(v, dtype=torch.int32).cuda()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bits", [4, 8])
def test_prompts_then_steps(bits, dtype):
    lengths = [1, 37, 64, 90]
    layer = Layer(bits, dtype, lengths, room=20)
    x = tokens(sum(lengths), dtype, 1)
    slots = torch.cat([layer.slots(b, 0, n) for b, n in enumerate(lengths)])
    layer.check(x, layer.run(x, slots, ints(lengths), ints(np.cumsum([0] + lengths).tolist())), lengths)
    for step in range(3):
        x = tokens(4, dtype, 10 + step)
        slots = torch.cat([layer.slots(b, n, 1) for b, n in enumerate(layer.lengths)])
        layer.lengths = [n + 1 for n in layer.lengths]
        layer.check(x, layer.run(x, slots, ints(layer.lengths)), [1] * 4)


def test_prompts_beside_steps():
    """A new prompt, a piece of one and decoding sequences in one call."""
    layer = Layer(4, torch.bfloat16, [1, 70, 64, 90], room=100)
    before = [0, 70, 64, 89]
    x = tokens(sum(before), torch.bfloat16, 2)
    layer.lengths = before
    slots = torch.cat([layer.slots(b, 0, n) for b, n in enumerate(before)])
    layer.check(x, layer.run(x, slots, ints(before), ints(np.cumsum([0] + before).tolist())), before)
    rows = [40, 1, 30, 1]
    x = tokens(sum(rows), torch.bfloat16, 3)
    slots = torch.cat([layer.slots(b, before[b], n) for b, n in enumerate(rows)])
    layer.lengths = [m + n for m, n in zip(before, rows)]
    layer.check(x, layer.run(x, slots, ints(layer.lengths), ints(np.cumsum([0] + rows).tolist())), rows)


def test_a_captured_step_replayed_as_the_sequences_grow():
    lengths = [5, 16, 33, 64]
    eager, replayed = (Layer(8, torch.bfloat16, lengths, room=20) for _ in range(2))
    x = tokens(sum(lengths), torch.bfloat16, 1)
    starts = ints(np.cumsum([0] + lengths).tolist())
    for layer in (eager, replayed):
        layer.run(x, torch.cat([layer.slots(b, 0, n) for b, n in enumerate(lengths)]), ints(lengths), starts)
    spare = (eager.cache.pages - 1) * PAGE  # (a page that no sequence has: where the warming run writes)
    x, slots, counts = tokens(4, torch.bfloat16, 9), torch.arange(spare, spare + 4).cuda(), ints(lengths)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        replayed.run(x, slots, counts)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = replayed.run(x, slots, counts)[-1]
    for step in range(4):
        x.copy_(tokens(4, torch.bfloat16, 20 + step))
        slots.copy_(torch.cat([eager.slots(b, n + step, 1) for b, n in enumerate(lengths)]))
        counts.copy_(ints([n + step + 1 for n in lengths]))
        want = eager.run(x, slots, counts)[-1]
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), step
