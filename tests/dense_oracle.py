"""64-bit values of the dense operators and the tolerances of their tests.

A 16-bit rounding is off by at most h = eps / 2 of the value.  What a test allows is counted from the roundings that the
operator makes: `close` bounds the 2-norm of the difference over the whole result, over every row and over every column by
(number of 16-bit roundings on the way) * h * (2-norm of the exact result): independent roundings add up in squares to less
than that, and inputs are drawn so that sums do not cancel as a whole.  A single row or column of few elements may be
unluckier than the whole, so it gets twice that, and it is held to the larger of its own norm and the mean one: an element
y = sum_i a_i b_i whose a_i are rounded is off by a sum of terms of up to h |a_i b_i|, in squares h^2 sum (a_i b_i)^2, which
is h times the size that such sums have on average, however far this one happens to cancel.
"""
import torch

ROWS_AND_COLS = 2.0


def half(dtype):
    return torch.finfo(dtype).eps / 2


def close(got, want, roundings, what=""):
    g, w = got.detach().double().cpu(), want.detach().double().cpu()
    assert g.shape == w.shape, (what, g.shape, w.shape)
    if g.numel() == 0:
        return
    assert torch.isfinite(g).all(), f"{what}: not finite"
    g, w = g.reshape(-1, g.shape[-1]), w.reshape(-1, w.shape[-1])
    d = g - w
    tol = roundings * half(got.dtype)
    tiny = torch.finfo(got.dtype).smallest_normal      # below it a rounding is not relative
    err = float(d.norm() / (w.norm() + tiny))
    assert err <= tol, f"{what}: {err:.3e} off, {tol:.3e} allowed"
    for dim, name in ((1, "row"), (0, "column")):
        n = w.norm(dim=dim)
        ref = torch.maximum(n, n.square().mean().sqrt()) + tiny
        e = d.norm(dim=dim) / ref
        k = int(e.argmax())
        assert float(e[k]) <= ROWS_AND_COLS * tol, f"{what}: {name} {k} is {float(e[k]):.3e} off, {ROWS_AND_COLS * tol:.3e} allowed"


def quantize(x):
    """Codes and scale of each row, from the definition, in 64 bits."""
    x = x.detach().double().cpu()
    top = x.abs().amax(dim=-1, keepdim=True)
    codes = torch.where(top > 0, torch.round(127 * x / torch.where(top > 0, top, 1.0)), 0.0)
    return codes, (top / 127).squeeze(-1)


def silu(g):
    return g * torch.sigmoid(g)


def ffn(x, wg, wu, wd):
    x, wg, wu, wd = (t.detach().double().cpu() for t in (x, wg, wu, wd))
    g, u = x @ wg.t(), x @ wu.t()
    h = silu(g) * u
    return g, u, h, h @ wd.t()


def ffn_grads(x, wg, wu, wd, dy):
    g, u, h, _ = ffn(x, wg, wu, wd)
    x, wg, wu, wd, dy = (t.detach().double().cpu() for t in (x, wg, wu, wd, dy))
    s = torch.sigmoid(g)
    dh = dy @ wd
    dg, du = dh * u * s * (1 + g * (1 - s)), dh * g * s
    return {"dx": dg @ wg + du @ wu, "dw_gate": dg.t() @ x, "dw_up": du.t() @ x, "dw_down": dy.t() @ h}
