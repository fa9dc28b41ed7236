"""64-bit references and error bounds of the dense products and their gradients."""
import math

import torch

from tests._util import TOL

F = torch.nn.functional
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
# |act'| <= 1.13 for all of them (gelu's maximum is 1.129)
SLOPE = 1.13


def act64(v, act):
    return {"none": lambda u: u * 1.0, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
            "gelu_tanh": lambda u: F.gelu(u, approximate="tanh")}[act](v)


def act_grad64(z, act):
    z = z.double().requires_grad_()
    return torch.autograd.grad(act64(z, act).sum(), z)[0]


def half_step(dtype, v):
    """Rounding to dtype: half a step, at least half the smallest subnormal (smallest normal * eps)."""
    f = torch.finfo(dtype)
    return torch.clamp(v.abs() * (f.eps / 2), min=f.smallest_normal * f.eps / 2)


def product_bound(a, b):
    """f32 sums of products: TOL sum |a b| (a [n, k], b [m, k] in f64)."""
    return TOL * (a.abs() @ b.abs().t())


def check(got, ref, bound, what=""):
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    err = (got.double() - ref).abs()
    ok = (err <= bound) | (got.double() == ref)
    if not bool(ok.all()):
        i = int((~ok).reshape(-1).nonzero()[0])
        raise AssertionError(f"{what}: {int((~ok).sum())} of {ok.numel()} beyond the bound; first at {i}: got "
                             f"{got.reshape(-1)[i].item()!r}, want {ref.reshape(-1)[i].item()!r}, error "
                             f"{err.reshape(-1)[i].item():.3e}, bound {bound.reshape(-1)[i].item():.3e}")


def linear_ref(x, w, bias, act, residual, ydt):
    """(z, its bound, y, its bound).  An f32 epilogue adds a rounding of 2^-24
    of each intermediate; the activation is good to 8 of them."""
    X, W = x.double(), w.double()
    z = X @ W.t()
    zb = product_bound(X, W)
    if bias is not None:
        z = z + bias.double()
        zb = zb + 2.0 ** -23 * (z.abs() + bias.double().abs())
    a = act64(z, act)
    yb = SLOPE * zb + 8 * 2.0 ** -24 * (a.abs() + z.abs())
    y = a
    if residual is not None:
        y = a + residual.double()
        yb = yb + 2.0 ** -23 * (y.abs() + residual.double().abs())
    return z, zb + half_step(ydt, z), y, yb + half_step(ydt, y)


def backward_ref(dy, x, w, z, act, dw_dtype, base_dw=None, base_db=None):
    """{name: (gradient, bound)}; dz is rounded to dy's type where that has 16
    bits and dw is not f32."""
    DY, X, W = dy.double(), x.double(), w.double()
    if act == "none":
        dz, dzb = DY, torch.zeros_like(DY)
        rounded = dzb
    else:
        g = act_grad64(z, act)
        dz = DY * g
        # act' to 16 roundings of its terms, which are below 1 + |z|
        dzb = 16 * 2.0 ** -24 * DY.abs() * (1 + z.double().abs())
        rounded = dzb + (half_step(dy.dtype, dz) if dy.dtype != torch.float32 and dw_dtype != torch.float32 else 0)
    dx = dz @ W
    dw = dz.t() @ X
    db = dz.sum(0)
    out = {"dx": (dx, product_bound(dz, W.t()) + rounded @ W.abs() + half_step(x.dtype, dx))}
    wb = product_bound(dz.t(), X.t()) + rounded.t() @ X.abs()
    bb = TOL * dz.abs().sum(0) + dzb.sum(0)
    if base_dw is not None:
        dw = dw + base_dw.double()
        db = db + base_db.double()
        wb = wb + 2.0 ** -23 * (dw.abs() + base_dw.double().abs())
        bb = bb + 2.0 ** -23 * (db.abs() + base_db.double().abs())
    out["dw"] = (dw, wb + half_step(dw_dtype, dw))
    out["db"] = (db, bb + half_step(torch.float32, db))
    return out


def randn(shape, dtype=torch.float32, scale=1.0, seed=0, device="cuda"):
    g = torch.Generator(device=device).manual_seed(seed)
    return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype)


def strided(t, extra, offset=0):
    """The same values with `extra` elements behind each row, the first row
    `offset` elements into its buffer; the gaps hold NaN."""
    r, c = t.shape
    buf = torch.full((r * (c + extra) + offset,), math.nan, dtype=t.dtype, device=t.device)
    v = buf[offset:offset + r * (c + extra)].view(r, c + extra)[:, :c]
    v.copy_(t)
    return v
