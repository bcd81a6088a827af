"""Int8 products with a scale for each token and each channel, against 64 bits."""
import numpy as np
import pytest
import torch

from iconnx_amd import ops
from tests import decoder_ref as ref

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def inputs(M, K, N, dtype, seed=0, bias=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g)
    x[:, :: max(1, K // 7)] *= 12.0
    w = torch.randint(-128, 128, (K, N), generator=g, dtype=torch.int8)
    ws = 0.001 + torch.rand(N, generator=g) * 0.01
    return x.to(dtype).cuda(), w.cuda(), ws.cuda(), (torch.randn(N, generator=g).cuda() if bias else None)


def check(y, q, s, w, ws, bias, dtype):
    want, mag = ref.token_qlinear(q, s, w.cpu().numpy(), ws.cpu().numpy(), None if bias is None else bias.cpu().numpy())
    err = np.abs(ref.f64(y).reshape(want.shape) - want)
    bound = ref.token_qlinear_bound(want, mag, dtype)
    assert (err <= bound).all(), "off by %g where %g is allowed" % (err.max(), bound[np.unravel_index((err - bound).argmax(), err.shape)])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K", [(1, 1), (1, 128), (3, 7), (5, 64), (17, 130), (4, 1000), (2, 4096), (1, 9001), (33, 20000)])
def test_quantized_tokens_are_the_definitions_bits(M, K, dtype):
    x = inputs(M, K, 1, dtype, seed=K)[0]
    q, s = ops.gpu_quantize_tokens(x)
    wq, wsc = ref.quantize_tokens(x)
    assert np.array_equal(s.cpu().numpy(), wsc)
    assert np.array_equal(q.cpu().numpy(), wq)


def test_values_half_way_between_bytes_go_to_the_even_one():
    # max 127 * 2^k: the scale is 2^k, the quotients are exact halves
    x = torch.stack([torch.cat([torch.tensor([127.0]), torch.arange(-126, 127) + 0.5]) * 2.0 ** k for k in (-130, -20, 0, 40)]).cuda()
    # and neighbours of halves under scales that are no powers of two
    y = torch.empty(64, 512)
    for r in range(64):
        s = np.float32(1.0 + r / 77.0)
        half = (np.arange(511) % 252 - 126 + 0.5) * np.float64(s)
        near = half.astype(np.float32)
        y[r, 0] = float(np.float32(127.0) * s)
        y[r, 1:] = torch.from_numpy(np.where(np.arange(511) % 3 == 0, near, np.nextafter(near, np.float32(0 if r % 2 else 1e9))))
    for t in (x, y.cuda()):
        q, s = ops.gpu_quantize_tokens(t)
        wq, wsc = ref.quantize_tokens(t)
        assert np.array_equal(s.cpu().numpy(), wsc) and np.array_equal(q.cpu().numpy(), wq)


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_of_zeros_tiny_values_and_not_finite_ones(dtype):
    x = torch.randn(8, 200)
    x[1] = 0
    x[2] = 1e-45 if dtype == torch.float32 else 0
    x[3, 17] = float("inf")
    x[4, 199] = float("nan")
    x[5, 0] = -float("inf")
    x[6] *= 1e-38 if dtype != torch.float16 else 1e-7
    x[7] *= 1e37 if dtype != torch.float16 else 1e4
    x = x.to(dtype).cuda()
    q, s = ops.gpu_quantize_tokens(x)
    wq, wsc = ref.quantize_tokens(x)
    assert np.array_equal(s.cpu().numpy(), wsc, equal_nan=True) and np.array_equal(q.cpu().numpy(), wq)
    w = torch.randint(-127, 128, (200, 40), dtype=torch.int8).cuda()
    y = ops.gpu_token_qlinear(x[:7], ops.TokenWeight(w, torch.full((40,), 0.01).cuda()))
    bad = torch.isnan(y).all(1).cpu()
    assert bad.tolist() == [False, False, False, True, True, True, False]
    assert not torch.isnan(y[~bad.cuda()]).any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 768, 768), (2, 100, 37), (7, 4096, 256), (16, 129, 65), (31, 1000, 500), (64, 512, 192),
                                   (65, 256, 129), (100, 3000, 77), (129, 640, 384), (257, 200, 300), (300, 1111, 263), (1025, 384, 520),
                                   (2049, 128, 1000), (3, 4096, 4096), (3, 4096, 4100), (3, 4097, 64), (5, 1024, 8192), (5, 1000, 8200),
                                   (9, 20000, 48), (16, 8200, 40), (1, 6145, 33), (2, 131071, 20), (24, 40000, 17)])
def test_product(M, K, N, dtype):
    x, w, ws, bias = inputs(M, K, N, dtype, seed=M + N, bias=(M + N) % 3 != 0)
    tw = ops.TokenWeight(w, ws)
    assert tw.shape == (K, N)
    y = ops.gpu_token_qlinear(x, tw, bias=bias)
    assert y.dtype == dtype and tuple(y.shape) == (M, N)
    q, s = ref.quantize_tokens(x)
    check(y, q, s, w, ws, bias, dtype)
    # over tokens quantized once: the same
    qx, sx = ops.gpu_quantize_tokens(x)
    z = ops.gpu_token_qlinear(qx, tw, x_scale=sx, bias=bias, dtype=dtype)
    assert torch.equal(y, z)


@pytest.mark.parametrize("M", [4096, 4500])
@pytest.mark.parametrize("K,N", [(640, 4096), (700, 4222)])
def test_large_product_by_rows_of_it(M, K, N):
    x, w, ws, bias = inputs(M, K, N, torch.bfloat16, seed=M)
    y = ops.gpu_token_qlinear(x, ops.TokenWeight(w, ws), bias=bias)
    rows = torch.cat([torch.arange(0, 64), torch.arange(M // 2, M // 2 + 40), torch.arange(M - 70, M)]).cuda()
    q, s = ref.quantize_tokens(x[rows])
    check(y[rows], q, s, w, ws, bias, torch.bfloat16)
    # every row, against one that is computed alone
    assert torch.equal(y[rows[:3]], ops.gpu_token_qlinear(x[rows[:3]].contiguous(), ops.TokenWeight(w, ws), bias=bias))


@pytest.mark.parametrize("M,K,N", [(6, 256, 64), (6, 250, 64), (200, 250, 130), (200, 384, 96)])
def test_rows_with_a_stride_an_offset_and_leading_axes(M, K, N):
    x, w, ws, bias = inputs(M, K + 9, N, torch.bfloat16)
    tw = ops.TokenWeight(w[:K].contiguous(), ws)
    part = x[:, 5:5 + K]
    want = ops.gpu_token_qlinear(part.contiguous(), tw)
    assert torch.equal(ops.gpu_token_qlinear(part, tw), want)
    assert torch.equal(ops.gpu_token_qlinear(part.contiguous().view(2, M // 2, K), tw).view(M, N), want)
    qa, sa = ops.gpu_quantize_tokens(part)
    qb, sb = ops.gpu_quantize_tokens(part.contiguous())
    assert torch.equal(qa, qb) and torch.equal(sa, sb)
    wide = torch.zeros(M, K + 3, dtype=torch.int8, device="cuda")
    wide[:, 3:] = qa
    assert torch.equal(ops.gpu_token_qlinear(wide[:, 3:], tw, x_scale=sa, dtype=torch.bfloat16), want)
    # int8 rows whose storage ends with the last of them, and goes on behind it
    for tail in (0, 5, 128):
        flat = torch.full(((M - 1) * 512 + K + tail + 16,), 77, dtype=torch.int8, device="cuda")
        rows = torch.as_strided(flat, (M, K), (512, 1), 16)
        rows.copy_(qa)
        assert torch.equal(ops.gpu_token_qlinear(rows, tw, x_scale=sa, dtype=torch.bfloat16), want)
    # ... and whose distance passes what a tile's offsets hold
    far = torch.zeros(3 * (1 << 24), dtype=torch.int8, device="cuda").view(3, 1 << 24)[:, :K]
    far.copy_(qa[:3])
    assert torch.equal(ops.gpu_token_qlinear(far, tw, x_scale=sa[:3].contiguous(), dtype=torch.bfloat16), want[:3])
    three, s3 = ops.gpu_quantize_tokens(part.contiguous().view(2, M // 2, K))
    assert three.shape == (2, M // 2, K) and torch.equal(three.reshape(M, K), qa)
    assert torch.equal(ops.gpu_token_qlinear(three, tw, x_scale=s3, dtype=torch.bfloat16).view(M, N), want)
    out = torch.empty_like(want)
    assert ops.gpu_token_qlinear(part, tw, out=out) is out and torch.equal(out, want)


def test_no_tokens_and_no_channels():
    tw = ops.TokenWeight(torch.zeros(64, 32, dtype=torch.int8).cuda(), torch.ones(32).cuda())
    assert ops.gpu_token_qlinear(torch.empty(0, 64).cuda(), tw).shape == (0, 32)
    none = ops.TokenWeight(torch.zeros(64, 0, dtype=torch.int8).cuda(), torch.ones(0).cuda())
    assert ops.gpu_token_qlinear(torch.randn(3, 64).cuda(), none).shape == (3, 0)
    q, s = ops.gpu_quantize_tokens(torch.empty(0, 7).cuda())
    assert q.shape == (0, 7) and s.shape == (0,)


@pytest.mark.parametrize("M", [1, 8, 40, 600])
def test_captured_and_replayed(M):
    x, w, ws, bias = inputs(M, 512, 384, torch.bfloat16)
    tw = ops.TokenWeight(w, ws)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.gpu_token_qlinear(x, tw, bias=bias)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = ops.gpu_token_qlinear(x, tw, bias=bias)
    for n in range(4):
        x.copy_(torch.randn(M, 512))
        want = ops.gpu_token_qlinear(x, tw, bias=bias)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want), n


def test_refusals():
    x, w, ws, bias = inputs(4, 64, 32, torch.float32)
    tw = ops.TokenWeight(w, ws)
    q, s = ops.gpu_quantize_tokens(x)
    bad = [lambda: ops.gpu_token_qlinear(x[:, :63], tw), lambda: ops.gpu_token_qlinear(x, tw, x_scale=s),
           lambda: ops.gpu_token_qlinear(q, tw), lambda: ops.gpu_token_qlinear(q, tw, x_scale=s[:3]),
           lambda: ops.gpu_token_qlinear(x.double(), tw), lambda: ops.gpu_token_qlinear(x, tw, bias=bias.half()),
           lambda: ops.gpu_token_qlinear(x, tw, bias=bias[:31]), lambda: ops.gpu_token_qlinear(x, tw, dtype=torch.int32),
           lambda: ops.gpu_token_qlinear(x, w), lambda: ops.gpu_token_qlinear(x.cpu(), tw), lambda: ops.gpu_quantize_tokens(w),
           lambda: ops.gpu_quantize_tokens(x[0, 0]), lambda: ops.gpu_quantize_tokens(x[:, :0]), lambda: ops.TokenWeight(w, ws[:5]),
           lambda: ops.TokenWeight(w.view(torch.uint8), ws), lambda: ops.TokenWeight(w.cpu(), ws.cpu()),
           lambda: ops.gpu_token_qlinear(x, tw, out=torch.empty(4, 33, device="cuda"))]
    for f in bad:
        with pytest.raises(ops.IconnxError):
            f()
    with pytest.raises(AttributeError):
        tw.scale = s
