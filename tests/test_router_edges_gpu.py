"""The router's losses and gradients where scores leave f32's range or
precision, against 64-bit definitions."""
import math

import pytest

torch = pytest.importorskip("torch")

from tests import _dense_util as U  # noqa: E402
from tests.test_router_train_gpu import SIGMOID, SOFTMAX, SQRT_SOFTPLUS, reference  # noqa: E402

pytestmark = pytest.mark.gpu
LOWEST = torch.finfo(torch.float32).min


@pytest.mark.parametrize("E,masked", [(40, 20), (200, 3), (1500, 700)])
@pytest.mark.parametrize("bad", [-math.inf, LOWEST, -100.0])
def test_masked_experts_of_sqrt_softplus(cuda_device, bad, E, masked):
    """Logits whose gate score overflows: no share and no gradient there, the
    other experts as if they were alone."""
    from objeta_b200.router import balance_loss, router_backward
    T, k = 12, 3
    l = U.randn((T, E), seed=5)
    ids = torch.topk(l[:, masked:], k, dim=1).indices.to(torch.int32) + masked
    l[:, :masked] = bad
    dw = U.randn((T, k), seed=6)
    b = balance_loss(l, ids, score_func=SQRT_SOFTPLUS)
    dl = router_backward(l, ids, dw, score_func=SQRT_SOFTPLUS, renormalize=True, balance=b, balance_grad=0.5,
                         z_grad=0.1)
    assert not dl[:, :masked].any()
    sub = l[:, masked:].contiguous()
    n = sub.shape[1]
    # f has E in place of the n experts that are left
    _, _, rb, rz, rdl, mag = reference(sub, ids - masked, SQRT_SOFTPLUS, None, None, dw, True, 1.0, 0.5 * E / n, 0.1)
    assert abs(float(b.balance) - rb * E / n) <= 64 * 2.0 ** -24 * rb * E / n
    assert abs(float(b.z) - rz) <= 64 * 2.0 ** -24 * (rz + math.sqrt(rz))
    U.check(dl[:, masked:].contiguous(), rdl, 64 * 2.0 ** -24 * mag + 1e-37)


@pytest.mark.parametrize("func", [SOFTMAX, SIGMOID, SQRT_SOFTPLUS])
def test_row_of_minus_infinity(cuda_device, func):
    """Such a token counts, and adds nothing to a loss or a gradient; the others' results are theirs alone."""
    from objeta_b200.router import balance_loss, router_backward
    l = U.randn((5, 40), seed=5)
    ids = torch.topk(l, 3, dim=1).indices.to(torch.int32)
    dw = U.randn((5, 3), seed=6)
    l[2] = -math.inf
    b = balance_loss(l, ids, score_func=func)
    dl = router_backward(l, ids, dw, score_func=func, renormalize=True, balance=b, balance_grad=0.5, z_grad=0.1)
    assert int(b.tokens[0]) == 5 and not dl[2].any() and bool(torch.isfinite(dl).all())
    rest = torch.tensor([0, 1, 3, 4], device="cuda")
    z = torch.logsumexp(l[rest].double(), 1).square().sum() / 5
    assert abs(float(b.z) - float(z)) <= 64 * 2.0 ** -24 * (float(z) + math.sqrt(float(z)))
    s = [torch.softmax, lambda v, _: torch.sigmoid(v), lambda v, _: sqrt_softplus(v)][func](l[rest].double(), 1)
    counts = torch.bincount(ids.reshape(-1).long(), minlength=40).double()
    bal = (counts * 40 / (3 * 5) * (s / s.sum(1, keepdim=True)).sum(0) / 5).sum()
    assert abs(float(b.balance) - float(bal)) <= 64 * 2.0 ** -24 * float(bal)


def sqrt_softplus(v):
    return torch.sqrt(torch.nn.functional.softplus(v, threshold=20.0))


@pytest.mark.parametrize("l", [-19.9, -20.1, -40.0, -88.0])
def test_sqrt_softplus_far_branch(cuda_device, l):
    """Down to -88 the score is the gate's log1p(exp(-l)) branch."""
    from objeta_b200.router import balance_loss, router_backward
    v = U.randn((9, 24), seed=3)
    v[:, 7] = l
    v[4] = l
    ids = torch.topk(v, 2, dim=1).indices.to(torch.int32)
    dw = U.randn((9, 2), seed=4)
    b = balance_loss(v, ids, score_func=SQRT_SOFTPLUS)
    dl = router_backward(v, ids, dw, score_func=SQRT_SOFTPLUS, renormalize=True, balance=b, balance_grad=0.5)
    _, _, rb, _, rdl, mag = reference(v, ids, SQRT_SOFTPLUS, None, None, dw, True, 1.0, 0.5, 0.0)
    assert abs(float(b.balance) - rb) <= 64 * 2.0 ** -24 * rb
    U.check(dl, rdl, 64 * 2.0 ** -24 * mag + 1e-37)


@pytest.mark.parametrize("func", [SOFTMAX, SIGMOID])
@pytest.mark.parametrize("E,k", [(16, 3), (60, 8), (120, 12), (256, 8), (600, 3), (600, 40), (1500, 40)])
def test_renormalised_weights_of_far_ids(cuda_device, func, E, k):
    """Given ids (a hash layer's) whose scores underflow beside the others':
    the renormalised weights are still a share of one another.  Ordinary
    tokens between them, and the losses' gradients beside."""
    from objeta_b200.router import balance_loss, router_backward
    far = [0.0, 60.0, 69.5, 86.0, 87.5, 0.0, 88.5, 90.0, 95.0, 100.0, 101.0, 0.0]
    T = len(far)
    l = U.randn((T, E), seed=E)
    l[:, E - 1] = 1.0
    gen = torch.Generator().manual_seed(E)
    ids = torch.stack([torch.randperm(E - 1, generator=gen)[:k] for _ in range(T)]).to(torch.int32).cuda()
    down = torch.tensor(far, device="cuda")[:, None] + math.log(E) * (func == SIGMOID)
    l.scatter_(1, ids.long(), (l.gather(1, ids.long()).clamp(min=-1.5, max=1.5) - down).float())
    dw = U.randn((T, k), seed=6)
    b = balance_loss(l, ids, score_func=func)
    for kw, bg, zg in ((dict(), 0.0, 0.0), (dict(balance=b, balance_grad=0.3, z_grad=0.02), 0.3, 0.02)):
        dl = router_backward(l, ids, dw, score_func=func, renormalize=True, route_scale=2.5, **kw)
        *_, rdl, mag = reference(l, ids, func, None, None, dw, True, 2.5, bg, zg)
        # a weight's q is off by its exponent's rounding, at most 12 in size once relative to the largest
        U.check(dl, rdl, (64 + 24) * 2.0 ** -24 * mag + 1e-37, f"{func} {E} {k}")


@pytest.mark.parametrize("func", [SOFTMAX, SIGMOID, SQRT_SOFTPLUS])
@pytest.mark.parametrize("E,k", [(16, 3), (600, 40), (1500, 40)])
@pytest.mark.parametrize("bad", [-math.inf, LOWEST, -300.0])
def test_renormalised_weights_of_nothing(cuda_device, func, E, k, bad):
    """Selected scores that are all 0 (masked ids): a sum of 0 divides nothing, and nothing flows back."""
    from objeta_b200.router import router_backward
    T = 6
    l = U.randn((T, E), seed=E)
    ids = torch.arange(k, dtype=torch.int32, device="cuda").expand(T, k).contiguous()
    l[:, :k] = bad
    l[3, :k] = 0.5  # an ordinary token among them
    dw = U.randn((T, k), seed=6)
    dl = router_backward(l, ids, dw, score_func=func, renormalize=True)
    rest = torch.arange(T, device="cuda") != 3
    assert not dl[rest].any() and bool(torch.isfinite(dl).all()) and bool(dl[3].any())


@pytest.mark.parametrize("func", [SOFTMAX, SIGMOID])
def test_far_ids_of_long_runs(cuda_device, func):
    """More tokens than the teams of one round hold, every seventh with far ids."""
    from objeta_b200.router import router_backward
    T, E, k = 6000, 1100, 3
    l = U.randn((T, E), seed=1)
    l[::7, :k] -= 95.0
    ids = torch.topk(l, k, dim=1).indices.to(torch.int32)
    ids[::7] = torch.arange(k, dtype=torch.int32, device="cuda")
    dw = U.randn((T, k), seed=2)
    dl = router_backward(l, ids, dw, score_func=func, renormalize=True)
    *_, rdl, mag = reference(l, ids, func, None, None, dw, True, 1.0, 0.0, 0.0)
    U.check(dl, rdl, (64 + 24) * 2.0 ** -24 * mag + 1e-37)
    inplace = l.clone()
    router_backward(inplace, ids, dw, score_func=func, renormalize=True, d_dlogits=inplace)
    assert torch.equal(inplace, dl)


@pytest.mark.parametrize("func,offsets", [(SOFTMAX, (0.0, 11.0, 60.0, -60.0)), (SIGMOID, (0.0, 11.0, -60.0))])
@pytest.mark.parametrize("E", [24, 64, 256, 400, 1500])
def test_common_offset_of_the_logits(cuda_device, func, offsets, E):
    """Scores stay as exact as f32 scores where all logits of a token lie far from 0."""
    from objeta_b200.router import balance_loss, router_backward
    T, k = 600, 4
    for off in offsets:
        l = U.randn((T, E), scale=1.5, seed=E) + off
        ids = torch.topk(l, k, dim=1).indices.to(torch.int32)
        dw = U.randn((T, k), seed=2)
        b = balance_loss(l, ids, score_func=func)
        for renorm in (True, False):
            L = l.double().requires_grad_()
            s = torch.softmax(L, 1) if func == SOFTMAX else torch.exp(torch.nn.functional.logsigmoid(L))
            w = s.gather(1, ids.long())
            if renorm:
                w = w / w.sum(1, keepdim=True)
            f = torch.bincount(ids.reshape(-1).long(), minlength=E).double() * E / (k * T)
            bal = (f * (s / s.sum(1, keepdim=True)).mean(0)).sum()
            for weights, grad in ((dw, 0.0), (None, 1.0)):
                ref = torch.autograd.grad((w * dw.double()).sum() if weights is not None else bal, L, retain_graph=True)[0]
                dl = router_backward(l, ids, weights, score_func=func, renormalize=renorm,
                                     balance=b if grad else None, balance_grad=grad)
                # an exponent below 16.6 is rounded by 2^-21 on average at most (2.7e-7 of its exponential), another
                # few roundings of 2^-24 follow: 10 of those over all.  (Of the balance loss a difference is left, of
                # terms a few times its size.)
                rel = float((dl.double() - ref).norm() / ref.norm())
                assert rel <= (40 if grad else 10) * 2.0 ** -24, (off, renorm, grad, rel)
