"""Measured cases of the dense gated feed-forward operators: the work that
callers have them do, in the package's kernels (``own``) or in plain torch.

Operators ("op" of a case):

  ffn       ``gated_ffn``: y = (silu(x Wg^T) * (x Wu^T)) Wd^T for T tokens, the
            dense FFN or shared expert beside a routed MoE layer
  train     the same with its backward pass: y and the gradients of x and of
            the three matrices for a given gradient of y
  int8      ``quantize_int8`` of T tokens, then ``int8_matmul`` with int8
            weights that have a scale per output channel
  ffn8      ``gated_ffn_int8``: the gated FFN on int8 weights, x and the
            activations quantised per token

Sizes ("T" tokens, hidden size "h", intermediate size "I"; for int8 the
product is [T, h] x [I, h]^T) are those of the package's configurations
(``synthetic.CONFIGS``), their tensor-parallel shards, and generic ragged ones.
"dtype" is that of x and the output (and of the weights where they are not
int8).  Tokens are N(0, 1), weights N(0, 0.02) as in the package's synthetic
layers, the gradient of y N(0, 1), as a loss scaled into range gives.
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STD = 0.02
# Widest integer sum of a product of int8 codes that fp32 holds exactly:
# 1024 * 128 * 128 = 2^24.
EXACT_COLUMNS = 1024


def _functional():
    """The package's entry points (imported only where its kernels run)."""
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "warp-route_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    from warp_route import functional
    return functional


def _case(op, T, h, I, dtype, **named):
    return dict(named, op=op, T=T, h=h, I=I, dtype=dtype)


def listed():
    return [
        # One decode token through two shared experts of a layer of many small
        # experts: the smallest call, where launches and latency count.
        _case("ffn", 1, 2048, 2816, "bf16", name="ffn token of shared experts bf16"),
        # A decode batch through a large dense FFN: the weights' bytes count.
        _case("ffn", 16, 4096, 14336, "f16", name="ffn decode batch f16"),
        # A prompt through the same layer: the matrix cores count.
        _case("ffn", 2048, 4096, 14336, "bf16", name="ffn prompt bf16"),
        # A training step of the shared experts over a micro-batch.
        _case("train", 4096, 2048, 2816, "bf16", name="train shared experts bf16"),
        # A training step of a large dense FFN: the largest case.
        _case("train", 4096, 4096, 14336, "bf16", name="train large layer bf16"),
        # Sizes that are multiples of nothing, a packed batch of odd length.
        _case("train", 777, 1500, 2051, "f16", name="train ragged f16"),
        # Full-precision training of a small layer.
        _case("train", 1024, 2048, 1408, "f32", name="train small experts f32"),
        # One decode token through an int8 projection.
        _case("int8", 1, 4096, 14336, "f16", name="int8 token f16"),
        # A small ragged batch, fp32 in and out.
        _case("int8", 45, 1500, 2051, "f32", name="int8 ragged batch f32"),
        # A prompt through an int8 projection of gate and up together.
        _case("int8", 4096, 4096, 28672, "bf16", name="int8 prompt bf16"),
        # A decode batch and a prompt through the int8 FFN.
        _case("ffn8", 16, 4096, 14336, "f16", name="ffn8 decode batch f16"),
        _case("ffn8", 2048, 4096, 14336, "bf16", name="ffn8 prompt bf16"),
    ]


# A drawn case costs no more than the largest listed one; fp32 products run at
# a sixteenth of the 16-bit rate, so that they get a sixteenth of its work.
MAX_FLOPS = 18.0 * 4096 * 4096 * 14336
SHAPES = [(4096, 14336), (2048, 1408), (2048, 2816), (6144, 10752), (256, 512)]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        op = rng.choice(["ffn", "ffn", "train", "train", "train", "int8", "int8", "ffn8"])
        # ffn8 takes fp32 too, but its second rounding to int8 makes steps
        # of a code from differences of an ulp, which fp32 outputs show.
        dtype = rng.choice(["f16", "bf16", "f16", "bf16", "f32"][:4 if op == "ffn8" else 5])
        T = _log_int(rng, 1, 4096)
        kind = rng.choice(["config", "aligned", "ragged"])
        if kind == "config":
            h, I = rng.choice(SHAPES)
            I //= rng.choice([1, 1, 2, 4])
        elif kind == "aligned":
            h, I = (64 * _log_int(rng, 1, 128) for _ in range(2))
        else:
            h, I = (_log_int(rng, 33, 4096) for _ in range(2))
        c = _case(op, T, h, I, dtype)
        if work(c)["flops"] <= MAX_FLOPS / (16 if dtype == "f32" else 1):
            return c


def work(case):
    """Bytes: each input read once, each output written once.  Operations: the
    matrix products (three in an FFN, each with two more in its backward)."""
    op, T, h, I = case["op"], case["T"], case["h"], case["I"]
    es = DTYPES[case["dtype"]].itemsize
    if op == "ffn":
        return {"bytes": es * (3.0 * h * I + 2 * T * h), "flops": 6.0 * T * h * I}
    if op == "train":  # x, dy and the weights in; y, dx and the weights' gradients out
        return {"bytes": es * (6.0 * h * I + 4 * T * h), "flops": 18.0 * T * h * I}
    if op == "int8":
        return {"bytes": 1.0 * h * I + 4 * I + es * T * (h + I), "flops": 2.0 * T * h * I}
    return {"bytes": 3.0 * h * I + 4 * (2 * I + h) + 2.0 * es * T * h, "flops": 6.0 * T * h * I}


def _round_codes(w):
    """int8 codes and fp32 scales of w's rows: scale = max|row| / 127, codes
    the nearest integers of 127 w / max|row|, ties to even (in 64 bits: a code
    is a value next to a border)."""
    w = w.double()
    amax = w.abs().amax(dim=1, keepdim=True)
    amax = torch.where(amax > 0, amax, torch.full_like(amax, 127.0))
    return torch.round(127.0 * w / amax).to(torch.int8), (amax / 127.0).reshape(-1)


def prepare(case, seed):
    """Tokens and weights; for the int8 operators the quantised weights that a
    serving program keeps, for training the gradient of y."""
    dev = torch.device("cuda:0")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    T, h, I = case["T"], case["h"], case["I"]

    def normal(rows, cols, std):
        return (torch.randn(rows, cols, generator=gen, device=dev) * std).to(dt)

    s = dict(op=case["op"], x=normal(T, h, 1.0))
    shapes = [(I, h)] if case["op"] == "int8" else [(I, h), (I, h), (h, I)]
    s["w"] = [normal(r, c, STD) for r, c in shapes]
    if case["op"] == "train":
        s["dy"] = normal(T, h, 1.0)
        for t in [s["x"]] + s["w"]:
            t.requires_grad_(True)
    if case["op"] in ("int8", "ffn8"):
        coded = [_round_codes(w) for w in s["w"]]
        s["w"] = [(q, sc.float()) for q, sc in coded]
    return s


def _code_product(a, b):
    """a b^T of int8 codes as exact whole numbers (fp64 holds them)."""
    acc = torch.zeros(a.shape[0], b.shape[0], dtype=torch.int32, device=a.device)
    for k in range(0, a.shape[1], EXACT_COLUMNS):
        part = a[:, k:k + EXACT_COLUMNS].float() @ b[:, k:k + EXACT_COLUMNS].float().t()
        acc += part.to(torch.int32)
    return acc


def _plain_int8(x, w):
    q, sx = _round_codes(x)
    return _code_product(q, w[0]).float() * sx.float().unsqueeze(1) * w[1]


def _plain(s):
    x = s["x"].detach()
    dt = x.dtype
    if s["op"] == "int8":
        return _plain_int8(x, s["w"][0]).to(dt)
    if s["op"] == "ffn8":
        g, u = (_plain_int8(x, w) for w in s["w"][:2])
        return _plain_int8(g / (1 + torch.exp(-g)) * u, s["w"][2]).to(dt)
    x = x.float()
    wg, wu, wd = (w.detach().float() for w in s["w"])
    g, u = x @ wg.t(), x @ wu.t()
    sig = 1 / (1 + torch.exp(-g))
    act = g * sig * u
    y = act @ wd.t()
    if s["op"] == "ffn":
        return y.to(dt)
    dy = s["dy"].float()
    da = dy @ wd
    du = da * g * sig
    dg = da * u * sig * (1 + g * (1 - sig))
    out = [y, dg @ wg + du @ wu, dg.t() @ x, du.t() @ x, dy.t() @ act]
    return [t.to(dt) for t in out]


def run(state):
    s = state
    if not own:
        return _plain(s)
    F = _functional()
    if s["op"] == "int8":
        q, sx = F.quantize_int8(s["x"])
        return F.int8_matmul(q, sx, *s["w"][0], out_dtype=s["x"].dtype)
    if s["op"] == "ffn8":
        return F.gated_ffn_int8(s["x"], *(t for w in s["w"] for t in w))
    y = F.gated_ffn(s["x"], *s["w"])
    if s["op"] == "ffn":
        return y
    return [y.detach(), *torch.autograd.grad(y, [s["x"], *s["w"]], s["dy"])]


def exact(case, seed):
    """The definition in 64 bits."""
    s = prepare(case, seed)
    x = s["x"].detach().double()

    def coded(v, w):
        m = v.abs().max(dim=1).values.clamp_min(torch.finfo(torch.float64).tiny)
        codes = (v * 127.0 / m[:, None]).round()
        return codes @ w[0].double().t() * (m[:, None] / 127.0 * w[1].double()[None, :])

    if case["op"] == "int8":
        return coded(x, s["w"][0])
    if case["op"] == "ffn8":
        g, u = coded(x, s["w"][0]), coded(x, s["w"][1])
        return coded(g * torch.sigmoid(g) * u, s["w"][2])
    wg, wu, wd = (w.detach().double() for w in s["w"])
    g, u = x @ wg.t(), x @ wu.t()
    if case["op"] == "ffn":
        return (torch.nn.functional.silu(g) * u) @ wd.t()
    sig = torch.sigmoid(g)
    act = g * sig * u
    dy = s["dy"].double()
    da = dy @ wd
    dg, du = da * u * (sig + g * sig * (1 - sig)), da * g * sig
    return [act @ wd.t(), torch.cat([dg, du], 1) @ torch.cat([wg, wu]),
            dg.t().contiguous() @ x, du.t().contiguous() @ x, dy.t().contiguous() @ act]
