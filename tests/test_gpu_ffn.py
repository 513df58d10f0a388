"""The dense gated FFN (gated_ffn) and the int8 operators on the GPU against
plain 64-bit forms (_ffn_oracle), within bounds derived there."""
import pytest
import torch

from tests import _ffn_oracle as O
from warp_route import functional as F

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.float16, torch.bfloat16]
# (tokens, hidden, intermediate): single tokens, whole tiles, one past and one
# short of tiles and steps, sizes of one, K shorter than a step.
SHAPES = [(1, 64, 64), (1, 2048, 1408), (1, 1, 1), (2, 1, 7), (5, 9, 1), (3, 33, 65), (16, 512, 256),
          (17, 129, 191), (64, 256, 512), (100, 101, 37), (127, 264, 136), (257, 520, 264),
          (130, 1000, 24), (300, 72, 1030), (1025, 136, 72)]


def tokens(seed, rows, cols, dtype, device, std=1.0):
    gen = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(rows, cols, generator=gen, device=device) * std).to(dtype)


def layer(T, h, I, dtype, device, seed=0):
    std = h ** -0.5
    return (tokens(seed, T, h, dtype, device), tokens(seed + 1, I, h, dtype, device, std),
            tokens(seed + 2, I, h, dtype, device, std),
            tokens(seed + 3, h, I, dtype, device, I ** -0.5))


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T,h,I", SHAPES)
def test_forward_and_gradients(cuda, T, h, I, dtype):
    print(f"[gpu] gated_ffn {T} {h} {I} {dtype}", flush=True)
    args = layer(T, h, I, dtype, cuda)
    dy = tokens(9, T, h, dtype, cuda)
    want, bound = O.ffn(*args)
    O.assert_within(F.gated_ffn(*args), want, bound, "y without gradients")
    for t in args:
        t.requires_grad_(True)
    y = F.gated_ffn(*args)
    O.assert_within(y.detach(), want, bound, "y")
    got = torch.autograd.grad(y, args, dy)
    args = [t.detach() for t in args]
    for name, g, (w, b) in zip(("dx", "dw_gate", "dw_up", "dw_down"), got, O.ffn_grads(*args, dy)):
        assert g.dtype == dtype
        O.assert_within(g, w, b, name)


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("rows,cols", [(1, 1), (1, 7), (3, 16), (5, 255), (2, 4096), (130, 1001),
                                       (7, 16384)])
def test_quantize_int8(cuda, rows, cols, dtype):
    x = tokens(3, rows, cols, dtype, cuda)
    q, s = F.quantize_int8(x)
    wq, ws = O.codes(x)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    assert torch.equal(q.double(), wq)
    O.assert_within(s, ws, 1.01 * O.E * ws, "scales")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("M,K,N", [(1, 1, 1), (1, 4096, 512), (3, 17, 5), (16, 128, 64), (33, 255, 300),
                                   (64, 1504, 260), (129, 640, 1000), (300, 2048, 100),
                                   (2, 131071, 3), (1030, 96, 70)])
def test_int8_matmul(cuda, M, K, N, dtype):
    print(f"[gpu] int8_matmul {M} {K} {N} {dtype}", flush=True)
    gen = torch.Generator(device=cuda).manual_seed(1)
    q, w = (torch.randint(-128, 128, (r, K), generator=gen, device=cuda).to(torch.int8)
            for r in (M, N))
    q[0] = -128  # the largest sum there is
    w[0] = -128
    s = torch.rand(M, generator=gen, device=cuda) + 0.5
    sw = torch.rand(N, generator=gen, device=cuda) + 0.5
    if dtype == torch.float16:
        s *= 2.0 ** -16  # sums of up to 2^31 into its range
    want, bound = O.int8_product(q, s, w, sw, dtype)
    O.assert_within(F.int8_matmul(q, s, w, sw, dtype), want, bound, "out")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("T,h,I", SHAPES)
def test_gated_ffn_int8(cuda, T, h, I, dtype):
    print(f"[gpu] gated_ffn_int8 {T} {h} {I} {dtype}", flush=True)
    x, *w = layer(T, h, I, dtype, cuda)
    qw = [t for m in w for t in F.quantize_int8(m)]
    want, bound = O.ffn_int8(x, *qw, dtype)
    O.assert_within(F.gated_ffn_int8(x, *qw), want, bound, "y")


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
@pytest.mark.parametrize("need", [(1, 0, 0, 0), (0, 1, 0, 0), (0, 0, 1, 0), (0, 0, 0, 1), (0, 1, 0, 1),
                                  (1, 0, 1, 0)])
def test_some_gradients_only(cuda, need, dtype):
    """What is not needed is not computed and changes nothing of the rest (within
    the bounds: products are split as their own sizes ask)."""
    args = layer(700, 264, 520, dtype, cuda)
    dy = tokens(9, 700, 264, dtype, cuda)
    for t, n in zip(args, need):
        t.requires_grad_(bool(n))
    y = F.gated_ffn(*args)
    got = torch.autograd.grad(y, [t for t, n in zip(args, need) if n], dy)
    ref = O.ffn_grads(*(t.detach() for t in args), dy)
    for g, (w, b) in zip(got, [r for r, n in zip(ref, need) if n]):
        O.assert_within(g, w, b, str(need))
