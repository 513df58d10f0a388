"""Plain 64-bit dense FFN and int8 products, with bounds of how far a result in
fewer bits may be off, term by term.

u(t) = torch.finfo(t).eps / 2 is the relative error of a rounding to type t, E
= 2^-24 that of fp32.  A sum of n fp32 products in any order is off by at most
(n + 8) E times the sum of the products' magnitudes (one rounding per product
and addition; the 8 covers joins of partial sums).  expf, the division and
the products around them in silu and its derivative are off by a few ulp: 16 E.
fp16 results below its normal range are off by half its smallest step."""
import torch

E = 2.0 ** -24


def u(dtype):
    return torch.finfo(dtype).eps / 2


def step(dtype):
    """Half the smallest step of a type (its subnormals)."""
    f = torch.finfo(dtype)
    return f.smallest_normal * f.eps / 2


def fsum(n):
    return (n + 8) * E


def gate_parts(x, wg, wu, dtype):
    """g, u, a = silu(g) u in 64 bits and their errors as fp32 values."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, uu = x @ wg.t(), x @ wu.t()
    k = fsum(x.shape[1])
    dg = k * (x.abs() @ wg.abs().t())
    du = k * (x.abs() @ wu.abs().t())
    silu = g * torch.sigmoid(g)
    a = silu * uu
    # |silu'| <= 1.1
    da = 1.1 * dg * (uu.abs() + du) + silu.abs() * du + 16 * E * a.abs()
    return g, uu, a, dg, du, da


def ffn(x, wg, wu, wd):
    """y of gated_ffn and its bound."""
    dt = x.dtype
    _, _, a, _, _, da = gate_parts(x, wg, wu, dt)
    wd = wd.double()
    da = da + u(dt) * (a.abs() + da) + step(dt)  # a stored in x's dtype
    y = a @ wd.t()
    dy = (da @ wd.abs().t()) + fsum(a.shape[1]) * ((a.abs() + da) @ wd.abs().t())
    return y, dy + u(dt) * (y.abs() + dy) + step(dt)


def ffn_grads(x, wg, wu, wd, dy):
    """[dx, dWg, dWu, dWd] and their bounds."""
    dt = x.dtype
    g, uu, a, eg, eu, ea = gate_parts(x, wg, wu, dt)
    x, wg, wu, wd, dy = (t.double() for t in (x, wg, wu, wd, dy))
    # a is kept in x's dtype, g and u in fp32
    ea = ea + u(dt) * (a.abs() + ea) + step(dt)
    s = torch.sigmoid(g)
    silu, f = g * s, s * (1 + g * (1 - s))  # f = silu', |f| <= 1.1, |f'| <= 0.5
    da = dy @ wd
    eda = fsum(dy.shape[1]) * (dy.abs() @ wd.abs())
    du, dg = da * silu, da * uu * f
    fda = da.abs() + eda
    # f is s + silu (1 - s): its terms' magnitudes stay below 1.3
    edu = eda * silu.abs() + fda * 1.1 * eg + 16 * E * du.abs()
    edg = (eda * (uu.abs() + eu) * f.abs() + fda * 1.1 * eu + fda * (uu.abs() + eu) * 0.5 * eg +
           16 * E * 1.3 * fda * (uu.abs() + eu))
    edu = edu + u(dt) * (du.abs() + edu) + step(dt)
    edg = edg + u(dt) * (dg.abs() + edg) + step(dt)

    def out(v, e, magnitude, n):
        e = e + fsum(n) * (magnitude + e)
        return v, e + u(dt) * (v.abs() + e) + step(dt)

    T, I = x.shape[0], wg.shape[0]
    return [
        out(dg @ wg + du @ wu, edg @ wg.abs() + edu @ wu.abs(),
            dg.abs() @ wg.abs() + du.abs() @ wu.abs(), 2 * I),
        out(dg.t() @ x, edg.t() @ x.abs(), dg.abs().t() @ x.abs(), T),
        out(du.t() @ x, edu.t() @ x.abs(), du.abs().t() @ x.abs(), T),
        out(dy.t() @ a, dy.abs().t() @ ea, dy.abs().t() @ a.abs(), T),
    ]


def codes(x):
    """(codes, scales) of quantize_int8 in 64 bits, finite rows."""
    x = x.double()
    m = x.abs().amax(-1, keepdim=True)
    safe = torch.where(m > 0, m, torch.ones_like(m))
    return torch.round(x * 127.0 / safe), torch.where(m > 0, m / 127.0, safe).squeeze(-1)


def int8_product(q, s, w, sw, dtype):
    """int8_matmul of codes and scales, and its bound: one rounding of the sum, one
    per scale, one to dtype."""
    y = (q.double() @ w.double().t()) * s.double()[:, None] * sw.double()
    e = 3.01 * E * y.abs() + step(torch.float32)
    return y, e + u(dtype) * (y.abs() + e) + step(dtype)


def ffn_int8(x, wg, sg, wu, su, wd, sd, dtype):
    """gated_ffn_int8 and its bound: a code of the activations may be the other
    neighbour where the quotient is within its own error of a half-integer."""
    q, s = codes(x)
    s = s.float()
    g, eg = int8_product(q, s, wg, sg, torch.float32)
    uu, eu = int8_product(q, s, wu, su, torch.float32)
    silu = g * torch.sigmoid(g)
    a = silu * uu
    ea = 1.1 * eg * (uu.abs() + eu) + silu.abs() * eu + 16 * E * a.abs()
    m = a.abs().amax(-1, keepdim=True)
    em = ea.amax(-1, keepdim=True)
    safe = torch.where(m > 0, m, torch.ones_like(m))
    t = a * 127.0 / safe
    et = 127.0 * (ea + a.abs() * em / safe) / safe
    qa = torch.round(t)
    flip = ((t - torch.floor(t) - 0.5).abs() <= et).double()
    sa = safe / 127.0
    y = (qa @ wd.double().t()) * sa * sd.double()
    # The kernel's sum is (sum (qa + f) w) sa (1 + d) sd with codes off by f, |f| <= flip, and
    # its scale and roundings off by |d| <= em / safe + 4 E: it differs from y by at most
    # |sum f w| sa sd (1 + |d|) + |y| |d|.
    d = em / safe + 4 * E
    e = (flip @ wd.double().abs().t()) * sa * sd.double() * (1 + d) + y.abs() * d
    return y, e + u(dtype) * (y.abs() + e) + step(dtype)


def assert_within(got, want, bound, label):
    got = got.double()
    assert got.shape == want.shape, (label, got.shape, want.shape)
    bad = ~((got - want).abs() <= bound)
    if bad.any():
        i = bad.nonzero()[0].tolist()
        worst = ((got - want).abs() / bound.clamp_min(1e-300)).max().item()
        raise AssertionError(f"{label}: {int(bad.sum())} of {bad.numel()} values out of bounds, first "
                             f"at {i}: {got[tuple(i)].item()} against {want[tuple(i)].item()} "
                             f"+- {bound[tuple(i)].item():.3g}; worst {worst:.2f} bounds")
