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
          (130, 1000, 24), (300, 72, 1030), (1025, 136, 72),
          # few ragged rows; K split over slices; whole rounds and a split last one
          (48, 1500, 515), (65, 512, 4096), (40, 4096, 256), (2048, 256, 4096), (1111, 2050, 1034),
          (2500, 1024, 520)]


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
                                   (2, 131071, 3), (1030, 96, 70), (64, 8191, 33), (2300, 1024, 4100)])
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


def test_no_tokens(cuda):
    x, *w = layer(0, 24, 40, torch.bfloat16, cuda)
    for t in [x] + w:
        t.requires_grad_(True)
    y = F.gated_ffn(x, *w)
    assert y.shape == (0, 24)
    grads = torch.autograd.grad(y, [x] + w, torch.zeros_like(y))
    assert grads[0].shape == (0, 24) and all(not g.any() for g in grads[1:])
    qw = [t for m in w for t in F.quantize_int8(m.detach())]
    assert F.gated_ffn_int8(x, *qw).shape == (0, 24)
    q, s = F.quantize_int8(x.detach())
    assert q.shape == (0, 24) and s.shape == (0,)
    assert F.int8_matmul(q, s, *qw[:2]).shape == (0, 40)


@pytest.mark.parametrize("shape", [(24,), (1, 24), (2, 3, 24), (2, 0, 24), (2, 1, 5, 24)], ids=str)
def test_leading_dimensions(cuda, shape):
    x, *w = layer(30, 24, 40, torch.float16, cuda)
    rows = x[:torch.Size(shape[:-1]).numel()].contiguous()
    x = rows.view(shape)
    assert torch.equal(F.gated_ffn(x, *w), F.gated_ffn(rows, *w).view(shape))
    q, s = F.quantize_int8(x)
    assert q.shape == shape and s.shape == shape[:-1]
    qw = [t for m in w for t in F.quantize_int8(m)]
    assert F.int8_matmul(q, s, *qw[:2]).shape == shape[:-1] + (40,)
    assert torch.equal(F.gated_ffn_int8(x, *qw), F.gated_ffn_int8(rows, *qw).view(shape))


@pytest.mark.parametrize("T", [3, 70])
def test_tensors_that_start_anywhere(cuda, T):
    """Views at an element that is not 16-byte aligned give what aligned copies
    give, gradients too, and the elements around outputs stay (outputs are new)."""
    args = layer(T, 40, 72, torch.bfloat16, cuda) + (tokens(9, T, 40, torch.bfloat16, cuda),)

    def shifted(t):
        buf = torch.empty(t.numel() + 3, dtype=t.dtype, device=cuda)
        buf[3:] = t.reshape(-1)
        return buf[3:].view(t.shape)

    def step(x, wg, wu, wd, dy):
        leaves = [t.detach().requires_grad_(True) for t in (x, wg, wu, wd)]
        y = F.gated_ffn(*leaves)
        return [y.detach(), *torch.autograd.grad(y, leaves, dy)]

    for a, b in zip(step(*args), step(*(shifted(t) for t in args))):
        assert torch.equal(a, b)
    x, *w = args[:4]
    qw = [t for m in w for t in F.quantize_int8(m)]
    assert torch.equal(F.gated_ffn_int8(x, *qw), F.gated_ffn_int8(shifted(x), *map(shifted, qw)))
    for a, b in zip(F.quantize_int8(x), F.quantize_int8(shifted(x))):
        assert torch.equal(a, b)


def test_gradient_of_any_layout(cuda):
    """The gradient that arrives may be expanded or transposed."""
    args = [t.requires_grad_(True) for t in layer(9, 40, 72, torch.float32, cuda)]
    y = F.gated_ffn(*args)
    one = torch.autograd.grad(y, args, torch.ones_like(y), retain_graph=True)
    sums = torch.autograd.grad(y.sum(), args, retain_graph=True)
    base = tokens(4, 40, 9, torch.float32, cuda)
    turned = torch.autograd.grad(y, args, base.t(), retain_graph=True)
    plain = torch.autograd.grad(y, args, base.t().contiguous())
    for a, b, c, d in zip(one, sums, turned, plain):
        assert torch.equal(a, b) and torch.equal(c, d)


def test_refusals(cuda):
    x, wg, wu, wd = layer(4, 32, 48, torch.float16, cuda)
    for args, match in [((x.t(), wg, wu, wd), "contiguous"), ((x, wg.t(), wu, wd), "shape|contig"),
                        ((x, wg, wu[:-1], wd), "shape"), ((x, wg, wu, wu), "shape"),
                        ((x, wg.float(), wu, wd), "w_gate must be"), ((x, wg, wu, wd.cpu()), "CUDA"),
                        ((x.double(), wg, wu, wd), "float32, float16 or bfloat16"),
                        ((x[:, :0], wg, wu, wd), "shape|contiguous")]:
        with pytest.raises(RuntimeError, match=match):
            F.gated_ffn(*args)
    q, s = F.quantize_int8(x)
    w, sw = F.quantize_int8(wg)
    for args, match in [((q, s, w, sw[:-1]), "w_scale"), ((q.float(), s, w, sw), "x must be"),
                        ((q, s.half(), w, sw), "x_scale must be"), ((q, s, w[:, :-1], sw), "w must"),
                        ((q, s, w, sw, torch.float8_e4m3fn), "out_dtype")]:
        with pytest.raises(RuntimeError, match=match):
            F.int8_matmul(*args)
    big = torch.zeros(1, 131072, dtype=torch.int8, device=cuda)
    with pytest.raises(RuntimeError, match="in_features"):
        F.int8_matmul(big, s[:1], big, sw[:1])


@pytest.mark.parametrize("T", [5, 200])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("h,I", [(64, 96), (50, 75)])
def test_non_finite_token_leaves_the_others(cuda, T, bad, h, I):
    x, *w = layer(T, h, I, torch.bfloat16, cuda)
    qw = [t for m in w for t in F.quantize_int8(m)]
    broken = x.clone()
    broken[2, 7] = bad
    rest = torch.arange(T, device=cuda) != 2
    for f, ws in ((F.gated_ffn, w), (F.gated_ffn_int8, qw)):
        y, z = f(x, *ws), f(broken, *ws)
        assert torch.equal(y[rest], z[rest])
        assert not torch.isfinite(z[2]).all()
    assert F.gated_ffn_int8(broken, *qw)[2].isnan().all()
    q, s = F.quantize_int8(broken)
    assert s[2].isnan() and not q[2].any() and torch.isfinite(s[rest]).all()
    leaf = broken.clone().requires_grad_(True)
    dx, = torch.autograd.grad(F.gated_ffn(leaf, *w), leaf, torch.ones_like(x))
    leaf = x.clone().requires_grad_(True)
    want, = torch.autograd.grad(F.gated_ffn(leaf, *w), leaf, torch.ones_like(x))
    assert torch.equal(dx[rest], want[rest])


@pytest.mark.parametrize("dtype", DTYPES, ids=str)
def test_quantize_extremes(cuda, dtype):
    """Zero rows, the type's largest and smallest values, exact ties, and values
    around half-integers of a code."""
    f = torch.finfo(dtype)
    rows = [[0.0] * 8, [f.max, -f.max, f.max / 2, f.max / 254, 0, 1, -1, f.tiny],
            [f.smallest_normal * v for v in (1, -1, 0.5, 0.25, 0, 0.75, -0.5, 0)],
            [127, 0.5, 1.5, 2.5, -0.5, -1.5, 63.5, -126.5],
            [254, 1, 3, 5, -1, -3, 127, -253], [1e-3, 5e-4, -1e-3, 3e-4, 0, 0, 2.5e-4, 7e-4]]
    x = torch.tensor(rows, dtype=torch.float64, device=cuda).to(dtype)
    gen = torch.Generator(device=cuda).manual_seed(0)
    near = torch.randint(-127, 127, (64, 8), generator=gen, device=cuda).double() + 0.5
    near[:, 0] = 127
    near = near * (1 + torch.randint(-2, 3, near.shape, generator=gen, device=cuda) * f.eps)
    x = torch.cat([x, near.to(dtype)])
    q, s = F.quantize_int8(x)
    wq, ws = O.codes(x)
    assert torch.equal(q.double(), wq)
    O.assert_within(s, ws, 1.01 * O.E * ws + O.step(torch.float32), "scales")


def test_quantize_more_rows_than_one_launch_holds(cuda):
    """2^26 rows of 64 threads are 2^32 threads, more than a launch holds.  One column:
    codes are the sign times 127, 0 for a zero, which any row can be held against."""
    rows = (1 << 26) + 5
    x = torch.arange(rows, device=cuda, dtype=torch.int32).remainder_(3).sub_(1).to(torch.float16)
    q, s = F.quantize_int8(x.view(rows, 1))
    assert torch.equal(q.view(-1), x.to(torch.int8) * 127)
    one = torch.tensor(1.0 / 127.0, device=cuda)  # 1 / 127 rounded to fp32, as a division is
    assert torch.equal(s, torch.where(x == 0, torch.ones_like(one), one))


def test_same_bits_every_time(cuda):
    for T, h, I in [(1, 512, 256), (16, 4096, 1024), (48, 515, 515), (65, 512, 4096), (700, 512, 520)]:
        args = layer(T, h, I, torch.float16, cuda)
        dy = tokens(9, T, h, torch.float16, cuda)
        qw = [t for m in args[1:] for t in F.quantize_int8(m)]

        def once():
            leaves = [t.detach().requires_grad_(True) for t in args]
            y = F.gated_ffn(*leaves)
            return [y.detach(), *torch.autograd.grad(y, leaves, dy), F.gated_ffn_int8(args[0], *qw)]

        first = once()
        for _ in range(3):
            for a, b in zip(first, once()):
                assert torch.equal(a, b), (T, h, I)


def test_two_streams_at_once(cuda):
    """Calls on different streams have workspaces of their own."""
    sets = [layer(T, 512, 1024, torch.bfloat16, cuda, seed=T) for T in (96, 100)]
    want = [F.gated_ffn(*a) for a in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(10):
        for a, st, out in zip(sets, streams, got):
            with torch.cuda.stream(st):
                out.append(F.gated_ffn(*a))
    torch.cuda.synchronize()
    for w, outs in zip(want, got):
        assert all(torch.equal(w, o) for o in outs)


@pytest.mark.parametrize("T,h,I,dtype", [(1, 512, 256, torch.float16), (65, 512, 4096, torch.bfloat16),
                                         (300, 330, 515, torch.float32)])
def test_captured_training_step_replays(cuda, T, h, I, dtype):
    """Forward and backward in one graph; every replay, with eager work between,
    equals the eager step on the same inputs."""
    *args, dy = layer(T, h, I, dtype, cuda) + (tokens(9, T, h, dtype, cuda),)
    for t in args:
        t.requires_grad_(True)

    def step():
        y = F.gated_ffn(*args)
        return [y.detach(), *torch.autograd.grad(y, args, dy)]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        with torch.no_grad():
            args[0].copy_(tokens(20 + i, T, h, dtype, cuda))
            dy.copy_(tokens(30 + i, T, h, dtype, cuda))
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(eager, captured):
            assert torch.equal(a, b)


def test_capture_beside_a_live_eager_graph_is_refused(cuda):
    args = [t.requires_grad_(True) for t in layer(4, 64, 96, torch.float16, cuda)]
    alive = F.gated_ffn(*args)
    with pytest.raises(RuntimeError, match="eager autograd graph"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            F.gated_ffn(*args)
    with torch.no_grad(), torch.cuda.graph(torch.cuda.CUDAGraph()):
        F.gated_ffn(*args)  # no graph of its own: allowed
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = F.gated_ffn(*args)
        grads = torch.autograd.grad(y, args, torch.ones_like(y))
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.isfinite(g).all() for g in grads)


def test_two_calls_of_the_same_weights(cuda):
    """Weights used twice, eagerly and within one capture: gradients add up."""
    x, *w = layer(6, 64, 96, torch.float32, cuda)
    for t in w:
        t.requires_grad_(True)

    def step():
        y = F.gated_ffn(F.gated_ffn(x, *w), *w)
        return [y.detach(), *torch.autograd.grad(y, w, torch.ones_like(y))]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for _ in range(3):
        eager = step()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, captured))
    mid = F.gated_ffn(x, *(t.detach() for t in w))
    inner = mid.clone().requires_grad_(True)
    gin, *second = torch.autograd.grad(F.gated_ffn(inner, *w), [inner, *w], torch.ones_like(mid))
    first = torch.autograd.grad(F.gated_ffn(x, *w), w, gin)
    for a, b, c in zip(eager[1:], first, second):
        assert torch.equal(a, b + c)


def test_differentiable_once(cuda):
    args = [t.requires_grad_(True) for t in layer(3, 32, 48, torch.float32, cuda)]
    y = F.gated_ffn(*args)
    grads = torch.autograd.grad(y, args, torch.ones_like(y), create_graph=True)
    with pytest.raises(RuntimeError, match="differentiable once"):
        grads[0].sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y = F.gated_ffn(*args)
        with torch.no_grad():
            args[1].mul_(2)
        torch.autograd.grad(y, args, torch.ones_like(y))


def test_rows_past_32_bit_offsets(cuda):
    """150000 x 16384 activations: 2.5e9 elements.  The last rows, which lie past
    2^32 bytes, are those of a call on these rows alone, and their own oracle."""
    T, h, I = 150000, 64, 16384
    x, *w = layer(T, h, I, torch.bfloat16, cuda)
    tail = x[-40:].contiguous()
    want, bound = O.ffn(tail, *w)
    x.requires_grad_(True)
    y = F.gated_ffn(x, *w)
    O.assert_within(y[-40:].detach(), want, bound, "y")
    dy = tokens(9, T, h, torch.bfloat16, cuda)
    dx, = torch.autograd.grad(y, x, dy)
    want, bound = O.ffn_grads(tail, *w, dy[-40:])[0]
    O.assert_within(dx[-40:], want, bound, "dx")
    del y, dx
    qw = [t for m in w for t in F.quantize_int8(m)]
    want, bound = O.ffn_int8(tail, *qw, torch.bfloat16)
    O.assert_within(F.gated_ffn_int8(x.detach(), *qw)[-40:], want, bound, "int8")


def test_directional_difference(cuda):
    """The fp32 step's gradients against a central difference of its own outputs
    along a direction: L = sum(dy y) in 64 bits, step 2^-7.  The truncation is
    step^2 / 6 times the third derivative, which is 64 times smaller again at a
    step 8 times as short, so that half the change between steps 2^-7 and 2^-4
    bounds it; the rounding is at most the forward bound over the step."""
    args = layer(33, 64, 80, torch.float32, cuda)
    dy = tokens(9, 33, 64, torch.float32, cuda)
    v = [tokens(40 + i, *t.shape, torch.float32, cuda) * t.abs().mean() for i, t in enumerate(args)]
    leaves = [t.clone().requires_grad_(True) for t in args]
    grads = torch.autograd.grad(F.gated_ffn(*leaves), leaves, dy)
    want = sum((g.double() * d.double()).sum() for g, d in zip(grads, v)).item()

    def diff(eps):
        ends, err = [], 0.0
        for sign in (1, -1):
            moved = [t + sign * eps * d for t, d in zip(args, v)]
            _, bound = O.ffn(*moved)
            # the moved inputs are rounded too: 2^-24 of each, through the gradients
            ends.append((F.gated_ffn(*moved).double() * dy.double()).sum().item())
            err += (bound * dy.double().abs()).sum().item()
            err += sum((g.double().abs() * m.double().abs()).sum().item() * O.E * 2
                       for g, m in zip(grads, moved))
        return (ends[0] - ends[1]) / (2 * eps), err / (2 * eps)

    fine, rounding = diff(2.0 ** -7)
    coarse, _ = diff(2.0 ** -4)
    assert abs(fine - want) <= rounding + 0.5 * abs(fine - coarse)


def test_modules_and_stack(cuda):
    """Train one step of a GatedFFN, quantise it, and run it as the shared expert
    of a two-layer MoE stack, eager and captured."""
    from warp_route import GatedFFN
    from warp_route.stack import MoEStack
    from warp_route.synthetic import make_layer
    E, h, I, k = 4, 128, 256, 2
    torch.manual_seed(0)
    ffn = GatedFFN(h, 192, torch.float16).to(cuda)
    x = tokens(1, 6, h, torch.float16, cuda)
    y = ffn(x)
    y.float().pow(2).sum().backward()
    for p in ffn.parameters():
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any()
        with torch.no_grad():
            p -= 1e-3 * p.grad
        p.grad = None
    del y
    served = ffn.quantized()
    assert torch.equal(served(x), F.gated_ffn_int8(x, *(t for n in ("gate", "up", "down") for t in
                       F.quantize_int8(getattr(ffn, n + "_proj").detach()))))
    assert set(served.state_dict()) == {f"{n}_{s}" for n in ("gate", "up", "down")
                                        for s in ("codes", "scales")}
    layers = [make_layer(E, h, I, torch.float16, seed=s, device=cuda, batch=6,
                         x_dtype=torch.float16)[1:] for s in (1, 2)]
    stack = MoEStack(layers, E, h, I, k, shared=[ffn, served])
    plain = MoEStack(layers, E, h, I, k)
    for rows in (x, x[0].contiguous()):
        a = rows + (plain._moe(rows, *layers[0]) + ffn(rows).detach())
        want = a + (plain._moe(a, *layers[1]) + served(a))
        got = stack(rows)
        assert torch.equal(got, want) and not got.requires_grad
        step = stack.capture(rows)
        for _ in range(3):
            assert torch.equal(step(rows), want)
            stack(rows)
        assert torch.equal(MoEStack(layers, E, h, I, k, shared=[None, None])(rows), plain(rows))


@pytest.mark.parametrize("T,h,I", [(3, 50, 75), (40, 33, 129), (257, 130, 71)])
def test_c_abi_writes_its_outputs_only(cuda, T, h, I):
    """Direct calls of the C-ABI with a canary behind every buffer it writes,
    the workspace of exactly the size asked for."""
    import ctypes
    from warp_route import capi
    lib, guard = capi.lib(), 4096
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    x, *w = layer(T, h, I, torch.float16, cuda)
    dy = tokens(9, T, h, torch.float16, cuda)
    kept = []

    def buffer(nbytes):
        t = torch.full((nbytes + guard,), 0xA5, dtype=torch.uint8, device=cuda)
        kept.append((t, nbytes))
        return t

    row = lib.wr_ffn_saved_row(I)
    a = capi.WrFfnArgs()
    a.dtype, a.batch_size, a.hidden_dim, a.intermediate_dim = capi.WR_F16, T, h, I
    for name, t in zip(("x", "w_gate", "w_up", "w_down", "dout"), (x, *w, dy)):
        setattr(a, name, t.data_ptr())
    bufs = {n: buffer(b) for n, b in (
        ("out", 2 * T * h), ("saved_gate", 4 * T * row), ("saved_up", 4 * T * row),
        ("saved_act", 2 * T * row), ("dx", 2 * T * h), ("dw_gate", 2 * I * h), ("dw_up", 2 * I * h),
        ("dw_down", 2 * I * h))}
    for n, t in bufs.items():
        setattr(a, n, t.data_ptr())
    for entry, back in (("wr_ffn_forward", 0), ("wr_ffn_backward", 1)):
        a.workspace_bytes = lib.wr_ffn_workspace_bytes(back, a.dtype, h, I, T)
        a.workspace = buffer(a.workspace_bytes).data_ptr()
        assert getattr(lib, entry)(ctypes.byref(a), stream) == capi.WR_OK

    def shaped(n, r, c):
        return bufs[n][:2 * r * c].view(torch.float16).view(r, c)

    torch.cuda.synchronize()
    O.assert_within(shaped("out", T, h), *O.ffn(x, *w), "y")
    shapes = {"dx": (T, h), "dw_gate": (I, h), "dw_up": (I, h), "dw_down": (h, I)}
    for (n, s), ref in zip(shapes.items(), O.ffn_grads(x, *w, dy)):
        O.assert_within(shaped(n, *s), *ref, n)

    (q, sx), (p, sp), (d, sd) = (F.quantize_int8(t) for t in w)
    m = capi.WrFfnInt8Args()
    m.dtype, m.batch_size, m.hidden_dim, m.intermediate_dim = capi.WR_F16, T, h, I
    for name, t in zip(("x", "w_gate", "s_gate", "w_up", "s_up", "w_down", "s_down"),
                       (x, q, sx, p, sp, d, sd)):
        setattr(m, name, t.data_ptr())
    m.out = buffer(2 * T * h).data_ptr()
    m.workspace_bytes = lib.wr_ffn_int8_workspace_bytes(h, I, T)
    m.workspace = buffer(m.workspace_bytes).data_ptr()
    assert lib.wr_ffn_int8(ctypes.byref(m), stream) == capi.WR_OK
    codes, scales = buffer(T * h), buffer(4 * T)
    assert lib.wr_quantize_int8(x.data_ptr(), capi.WR_F16, T, h, codes.data_ptr(),
                                scales.data_ptr(), stream) == capi.WR_OK
    k = capi.WrInt8Args()
    k.out_dtype, k.rows, k.out_features, k.in_features = capi.WR_F32, T, I, h
    for name, t in zip(("x", "x_scale", "w", "w_scale"), (codes, scales, q, sx)):
        setattr(k, name, t.data_ptr())
    k.out = buffer(4 * T * I).data_ptr()
    k.workspace_bytes = lib.wr_int8_workspace_bytes(T, I, h)
    k.workspace = buffer(k.workspace_bytes).data_ptr()
    assert lib.wr_int8_matmul(ctypes.byref(k), stream) == capi.WR_OK
    torch.cuda.synchronize()
    for t, n in kept:
        assert (t[n:] == 0xA5).all()
