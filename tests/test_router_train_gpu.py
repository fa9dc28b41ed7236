"""Counts, balance and z losses, the gradient of the router's logits and of the
combine's weights, against 64-bit definitions differentiated by autograd, and
a run of them together as a router is trained."""
import math

import pytest

torch = pytest.importorskip("torch")

from tests import _dense_util as U  # noqa: E402

pytestmark = pytest.mark.gpu
SOFTMAX, SIGMOID, SQRT_SOFTPLUS = 0, 1, 2


def scores64(l, func):
    if func == SOFTMAX:
        return torch.softmax(l, 1)
    if func == SIGMOID:
        return torch.sigmoid(l)
    # the gate's branches (log1p(exp(-l)) below -20)
    low = l < -20
    return torch.sqrt(torch.where(l > 20, l, torch.log1p(torch.exp(torch.where(low, -l, torch.clamp(l, max=20.0))))))


def reference(l32, ids, func, off, mask, dw, renorm, scale, bg, zg):
    """(counts, tokens, balance, z, dlogits, magnitude of dlogits' terms)."""
    T, E = l32.shape
    k = ids.shape[1]
    l = l32.double().requires_grad_()
    off = [0, T] if off is None else off.tolist()
    S = len(off) - 1
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask.bool().cpu()
    s = scores64(l, func)
    p = s / s.sum(1, keepdim=True)
    counts = torch.zeros(S, E, dtype=torch.int32)
    tokens = torch.zeros(S, dtype=torch.int32)
    terms, rows = [], []
    idc = ids.cpu().long()
    for q in range(S):
        r = torch.arange(off[q], off[q + 1])
        r = r[keep[r]]
        tokens[q] = r.numel()
        sel = idc[r].reshape(-1)
        sel = sel[(sel >= 0) & (sel < E)]
        counts[q] = torch.bincount(sel, minlength=E).to(torch.int32)
        if r.numel():
            terms.append((p[r.cuda()].mean(0) * counts[q].cuda().double() * E / (k * r.numel())).sum())
            rows.append(r)
    if not rows:
        zero = torch.zeros(T, E, dtype=torch.double, device="cuda")
        return counts, tokens, 0.0, 0.0, zero, zero
    balance = torch.stack(terms).mean()
    r = torch.cat(rows).cuda()
    z = torch.logsumexp(l[r], 1).square().mean()
    loss = bg * balance + zg * z
    good = (ids >= 0) & (ids < E)
    if dw is not None:
        w = torch.where(good, torch.gather(s, 1, torch.where(good, ids, torch.zeros_like(ids)).long()), 0.0)
        if renorm:
            w = w / w.sum(1, keepdim=True).clamp(min=1e-300)
        loss = loss + (scale * w * dw.double() * good)[r].sum()
    dl = torch.autograd.grad(loss, l)[0]
    # how large the terms are that a gradient is made of: each is a chain of at most 64 roundings
    with torch.no_grad():
        N = r.numel()
        B = torch.zeros(T, E, dtype=torch.double, device="cuda")
        for q, rr in enumerate([torch.arange(off[q], off[q + 1]) for q in range(S)]):
            n = int(tokens[q])
            if n:
                B[rr.cuda()] = abs(bg) * counts[q].cuda().double() * E / (k * n * n * len(terms))
        G = torch.zeros(T, E, dtype=torch.double, device="cuda")
        if dw is not None:
            a = torch.where(good, torch.gather(s, 1, torch.where(good, ids, torch.zeros_like(ids)).long()), 0.0)
            Q = a.sum(1, keepdim=True).clamp(min=1e-300) if renorm else torch.ones(T, 1, device="cuda")
            g = dw.double().abs()
            gq = abs(scale) / Q * (g + ((g * a).sum(1, keepdim=True) / Q if renorm else 0)) * good
            G.scatter_add_(1, torch.where(good, ids, torch.zeros_like(ids)).long(), gq)
        soft = torch.softmax(l, 1)
        if func == SOFTMAX:
            mag = soft * (B + G + ((B + G) * soft).sum(1, keepdim=True))
        else:
            tot = s.sum(1, keepdim=True)
            d = s * 1.0  # |s'| <= s for the sigmoid; for sqrt-softplus s' = sigma / (2 s)
            if func == SQRT_SOFTPLUS:
                d = torch.sigmoid(l.abs()) / (2 * s)
            mag = d * ((B + (B * p).sum(1, keepdim=True)) / tot + G)
        mag = mag + abs(zg) * 2 / N * torch.logsumexp(l, 1, keepdim=True).abs() * soft
        counted = torch.zeros(T, 1, dtype=torch.double, device="cuda")
        counted[r] = 1
    return counts, tokens, float(balance.detach()), float(z.detach()), dl, mag * counted


def run_case(T, E, k, S, func, renorm=True, masked=False, dropped=False, seed=0, scale=1.0, bg=0.3, zg=0.02,
             weights=True, spread=1.5, stride=0):
    from objeta_b200.router import balance_loss, router_backward
    l = U.randn((T, E), scale=spread, seed=seed) + U.randn((E,), seed=seed + 1)
    ids = torch.topk(l, k, dim=1).indices.to(torch.int32) if T else torch.zeros(0, k, dtype=torch.int32, device="cuda")
    g = torch.Generator().manual_seed(seed)
    if dropped:
        ids[torch.rand(T, k, generator=g).cuda() < 0.3] = -1
    off = None
    if S > 1:
        off = torch.sort(torch.randint(0, T + 1, (S + 1,), generator=g))[0].to(torch.int32)  # gaps before and behind
        off[S // 2] = off[S // 2 - 1]
        off = off.cuda()
    mask = (torch.rand(T, generator=g) < 0.7).cuda() if masked else None
    dw = U.randn((T, k), seed=seed + 2) if weights else None
    lv = U.strided(l, stride) if stride else l
    b = balance_loss(lv, ids, score_func=func, d_seq_offsets=off, d_token_mask=mask)
    out = torch.full((T, E + stride), 7.0, device="cuda")[:, :E] if stride else None
    dl = router_backward(lv, ids, dw, score_func=func, renormalize=renorm, route_scale=scale, balance=b,
                         balance_grad=bg, z_grad=zg, d_dlogits=out)
    rc, rt, rb, rz, rdl, mag = reference(l, ids, func, off, mask, dw, renorm, scale, bg, zg)
    assert torch.equal(b.counts.cpu(), rc) and torch.equal(b.tokens.cpu(), rt)
    # the losses: each p and lse to 64 roundings, the sums in double
    assert abs(float(b.balance) - rb) <= 64 * 2.0 ** -24 * max(rb, 1e-30), (float(b.balance), rb)
    assert abs(float(b.z) - rz) <= 64 * 2.0 ** -24 * (rz + math.sqrt(rz)) + 1e-30, (float(b.z), rz)
    U.check(dl, rdl, 64 * 2.0 ** -24 * mag + 1e-37, f"dlogits {T} {E} {k} {S} {func} {renorm}")
    return b, dl


@pytest.mark.parametrize("func", [SOFTMAX, SIGMOID, SQRT_SOFTPLUS])
@pytest.mark.parametrize("E,k", [(1, 1), (3, 2), (8, 2), (31, 4), (33, 5), (64, 8), (100, 7), (127, 1), (128, 8),
                                 (255, 8), (256, 8), (257, 3), (512, 8), (700, 33), (1024, 16), (1025, 4), (3000, 8),
                                 (8192, 40)])
def test_expert_counts(cuda_device, func, E, k):
    run_case(37, E, k, 1, func, seed=E)
    run_case(37, E, k, 4, func, masked=True, dropped=True, renorm=False, scale=2.5, seed=E + 1)


@pytest.mark.parametrize("func", [SOFTMAX, SIGMOID, SQRT_SOFTPLUS])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 300, 4731, 20000])
def test_tokens(cuda_device, func, T):
    run_case(T, 64, 6, 1, func, seed=T)
    run_case(T, 256, 8, min(T, 9) + 1, func, masked=True, renorm=False, seed=T + 1)


@pytest.mark.parametrize("T,E,k,S", [(129, 64, 2, 1), (1000, 64, 8, 17), (4096, 33, 3, 30), (300, 500, 4, 4),
                                     (5, 256, 8, 2), (3, 3, 1, 40), (2048, 128, 8, 16), (2049, 128, 8, 16),
                                     (1025, 256, 8, 1), (9, 2000, 8, 1), (600, 1100, 3, 2), (1, 1024, 5, 1)])
def test_who_folds(cuda_device, T, E, k, S):
    """One block, a cluster of blocks or a launch of its own: sizes at the borders of each."""
    run_case(T, E, k, S, SOFTMAX, masked=True, seed=T)
    run_case(T, E, k, S, SIGMOID, renorm=False, dropped=True, seed=T + 1)


def test_many_short_sequences(cuda_device):
    run_case(3000, 16, 2, 2900, SOFTMAX, seed=3)
    run_case(40, 8, 2, 200, SIGMOID, masked=True, seed=4)


def test_strides(cuda_device):
    for E, stride in ((64, 8), (64, 3), (256, 4), (77, 5)):
        run_case(50, E, 4, 3, SOFTMAX, seed=E, stride=stride)
        run_case(50, E, 4, 3, SIGMOID, seed=E, stride=stride)


def test_parts_of_the_gradient(cuda_device):
    run_case(90, 40, 4, 3, SOFTMAX, weights=False, seed=1)
    run_case(90, 40, 4, 3, SIGMOID, weights=False, zg=0.0, seed=2)
    run_case(90, 40, 4, 3, SIGMOID, bg=0.0, seed=3)
    run_case(90, 40, 4, 3, SQRT_SOFTPLUS, bg=0.0, zg=0.0, seed=4)
    from objeta_b200.router import router_backward
    l = U.randn((50, 24), seed=1)
    ids = torch.topk(l, 3, dim=1).indices.to(torch.int32)
    dw = U.randn((50, 3), seed=2)
    mask = (torch.arange(50, device="cuda") % 3 > 0)
    for m in (None, mask):
        dl = router_backward(l, ids, dw, renormalize=True, d_token_mask=m)
        *_, rdl, mag = reference(l, ids, SOFTMAX, None, m, dw, True, 1.0, 0.0, 0.0)
        U.check(dl, rdl, 64 * 2.0 ** -24 * mag + 1e-37)
    inplace = l.clone()
    router_backward(inplace, ids, dw, renormalize=True, d_dlogits=inplace)
    assert torch.equal(inplace, router_backward(l, ids, dw, renormalize=True))


@pytest.mark.parametrize("func", [SOFTMAX, SIGMOID, SQRT_SOFTPLUS])
@pytest.mark.parametrize("E,k", [(8, 1), (64, 1), (200, 1), (64, 3), (1500, 1), (1500, 40), (64, 12)])
def test_equal_weight_gradients_cancel(cuda_device, func, E, k):
    """Renormalised weights sum to a constant: what their gradients have alike (with one slot, all) leaves
    nothing beside the losses' small gradients."""
    from objeta_b200.router import balance_loss, router_backward
    T = 50
    l = U.randn((T, E), scale=1.5, seed=E)
    ids = torch.topk(l, k, dim=1).indices.to(torch.int32)
    ids[3] = -1
    b = balance_loss(l, ids, score_func=func)
    args = dict(score_func=func, balance=b, balance_grad=0.01, z_grad=0.001)
    want = router_backward(l, ids, None, **args)
    dw = U.randn((T, 1), seed=1).expand(T, k).contiguous()
    dw[3] = math.nan  # of no expert: not looked at
    dl = router_backward(l, ids, dw, renormalize=True, **args)
    # w - mean is exact, mean wrong by 64 roundings; less the mean of that, 64 roundings of it: 2^-36 of w, which
    # reaches a logit through 1 / Q and the scores' derivatives, below 32 in all here; then the losses' own sums
    s = dw.nan_to_num().abs().max().double()
    U.check(dl, want.double(), 32 * 2.0 ** -36 * s + 64 * 2.0 ** -24 * want.double().abs().amax(1, keepdim=True)
            .expand(T, E), f"{func} {E} {k}")


def test_same_expert_twice(cuda_device):
    """A hash layer's table may name an expert twice: its gradients add up."""
    from objeta_b200.router import balance_loss, router_backward
    for E, k in ((8, 4), (100, 40), (2000, 70)):
        l = U.randn((20, E), seed=1)
        ids = torch.randint(0, max(2, E // 16), (20, k), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
        dw = U.randn((20, k), seed=2)
        for func in (SOFTMAX, SIGMOID):
            b = balance_loss(l, ids, score_func=func)
            dl = router_backward(l, ids, dw, score_func=func, renormalize=True, balance=b, balance_grad=0.1)
            rc, _, rb, _, rdl, mag = reference(l, ids, func, None, None, dw, True, 1.0, 0.1, 0.0)
            assert torch.equal(b.counts.cpu(), rc)
            U.check(dl, rdl, (64 + 2 * k) * 2.0 ** -24 * mag + 1e-37)  # k more roundings where all slots meet


def test_nothing_counts(cuda_device):
    from objeta_b200.router import balance_loss, router_backward
    l = U.randn((10, 16), seed=1)
    ids = torch.topk(l, 2, dim=1).indices.to(torch.int32)
    off = torch.tensor([4, 4, 4], dtype=torch.int32, device="cuda")
    none = torch.zeros(10, dtype=torch.bool, device="cuda")
    for kw in (dict(d_token_mask=none), dict(d_seq_offsets=off)):
        b = balance_loss(l, ids, **kw)
        assert not b.counts.any() and not b.tokens.any() and float(b.balance) == 0 and float(b.z) == 0
        assert not router_backward(l, ids, U.randn((10, 2)), balance=b, balance_grad=1.0, z_grad=1.0).any()
    b = balance_loss(l[:0], ids[:0])
    assert not b.counts.any() and float(b.balance) == 0 and float(b.z) == 0
    assert router_backward(l[:0], ids[:0], balance=b, balance_grad=1.0).shape == (0, 16)


def test_masked_experts(cuda_device):
    """Logits of -inf or the type's lowest value: no probability and no
    gradient there, and a row of only -inf adds nothing anywhere."""
    from objeta_b200.router import balance_loss, router_backward
    lowest = torch.finfo(torch.float32).min
    for func in (SOFTMAX, SIGMOID):
        for bad in (-math.inf, lowest):
            l = U.randn((12, 40), seed=5)
            ids = torch.topk(l[:, 20:], 3, dim=1).indices.to(torch.int32) + 20
            l[:, :20] = bad
            dw = U.randn((12, 3), seed=6)
            b = balance_loss(l, ids, score_func=func)
            dl = router_backward(l, ids, dw, score_func=func, renormalize=True, balance=b, balance_grad=0.5,
                                 z_grad=0.1)
            assert not dl[:, :20].any()
            sub = l[:, 20:].contiguous()
            # the same over the remaining experts: f has E = 40 in place of 20, so twice the balance
            _, _, rb, rz, rdl, mag = reference(sub, ids - 20, func, None, None, dw, True, 1.0, 1.0, 0.1)
            assert abs(float(b.balance) - 2 * rb) <= 64 * 2.0 ** -24 * 2 * rb
            assert abs(float(b.z) - rz) <= 64 * 2.0 ** -24 * (rz + math.sqrt(rz))
            U.check(dl[:, 20:].contiguous(), rdl, 64 * 2.0 ** -24 * mag + 1e-37)
        l = U.randn((5, 40), seed=5)
        l[2] = -math.inf
        ids = torch.topk(l, 3, dim=1).indices.to(torch.int32)
        b = balance_loss(l, ids, score_func=func)
        dl = router_backward(l, ids, U.randn((5, 3)), score_func=func, renormalize=True, balance=b, balance_grad=0.5,
                             z_grad=0.1)
        assert bool(torch.isfinite(dl).all()) and not dl[2].any() and math.isfinite(float(b.balance))
        assert math.isfinite(float(b.z)) and int(b.tokens[0]) == 5


def test_sqrt_softplus_branches(cuda_device):
    run_case(60, 32, 4, 1, SQRT_SOFTPLUS, spread=18.0, seed=2)


def test_scores_are_the_gates(cuda_device):
    """The routing weights that the gradient is of are those of deepseek_gate
    and router_topk_batched: differences of their own outputs."""
    from objeta_b200.ep import deepseek_gate, router_topk_batched
    from objeta_b200.router import router_backward
    T, E, k, h = 6, 12, 3, 0.01
    eye = torch.eye(E, device="cuda")
    l = U.randn((T, E), seed=3)
    dw = U.randn((T, k), seed=4)
    for func, renorm, scale in ((SOFTMAX, False, 1.0), (SOFTMAX, True, 1.0), (SIGMOID, True, 1.5),
                                (SQRT_SOFTPLUS, True, 2.0)):
        def route(v):
            if func == SOFTMAX:
                return router_topk_batched(v, k, renormalize=renorm)
            return deepseek_gate(eye, v, k, func, scale)
        ids, _ = route(l)
        dl = router_backward(l, ids, dw, score_func=func, renormalize=renorm, route_scale=scale)
        for e in range(E):
            step = torch.zeros(E, device="cuda")
            step[e] = h
            (ia, wa), (ib, wb) = route(l + step), route(l - step)
            same = (ia == ids).all(1) & (ib == ids).all(1)
            num = ((wa - wb).double() * dw.double()).sum(1) / (2 * h)
            # curvature h^2 |w'''| / 6 <= 2e-5 |dw|, f32 weights 2^-23 / h = 1.2e-5 |dw| per slot
            tol = 1e-4 * dw.double().abs().sum(1) * scale
            assert bool((((num - dl[:, e].double()).abs() <= tol) | ~same).all()), (func, e)
        assert int(same.sum()) >= 4


def test_gradient_against_differences(cuda_device):
    """The losses of the 64-bit definition, by central differences (step 1e-5:
    curvature 1e-10, rounding 1e-11)."""
    from objeta_b200.router import balance_loss, router_backward
    T, E, k = 7, 5, 2
    off = torch.tensor([1, 3, 3, 6], dtype=torch.int32, device="cuda")
    for func in (SOFTMAX, SIGMOID, SQRT_SOFTPLUS):
        l = U.randn((T, E), seed=8)
        ids = torch.topk(l, k, dim=1).indices.to(torch.int32)
        b = balance_loss(l, ids, score_func=func, d_seq_offsets=off)
        dl = router_backward(l, ids, score_func=func, balance=b, balance_grad=0.7, z_grad=0.2)

        def loss(v):
            s = scores64(v, func)
            p = s / s.sum(1, keepdim=True)
            tot = []
            for a, e in ((1, 3), (3, 6)):
                c = torch.bincount(ids[a:e].reshape(-1).long(), minlength=E).double()
                tot.append((p[a:e].mean(0) * c * E / (k * (e - a))).sum())
            return float(0.7 * (tot[0] + tot[1]) / 2 + 0.2 * torch.logsumexp(v[1:6], 1).square().mean())

        for t in range(T):
            for e in range(E):
                up, down = l.double().clone(), l.double().clone()
                up[t, e] += 1e-5
                down[t, e] -= 1e-5
                assert abs((loss(up) - loss(down)) / 2e-5 - float(dl[t, e])) <= 1e-6, (func, t, e)


@pytest.mark.parametrize("T,k,O", [(1, 1, 1), (1, 8, 4096), (5, 2, 33), (16, 2, 4096), (300, 8, 100), (700, 6, 260),
                                   (3, 1024, 8), (2500, 1, 2048)])
def test_combine_backward(cuda_device, T, k, O):
    from objeta_b200.router import moe_combine_backward
    V = T * k + 3
    dout, v = U.randn((T, O), seed=1), U.randn((V, O), seed=2)
    rows = torch.randint(0, V, (T, k), generator=torch.Generator().manual_seed(1)).to(torch.int32).cuda()
    dw = moe_combine_backward(dout, v, rows)
    prod = dout.double()[:, None] * v.double()[rows.long()]
    U.check(dw, prod.sum(-1), U.TOL * prod.abs().sum(-1))
    assert torch.equal(dw, moe_combine_backward(dout, v, rows))
    off = torch.empty(V * O + 1, device="cuda")[1:].view(V, O)  # 4-byte aligned rows
    off.copy_(v)
    dw = moe_combine_backward(dout, off, rows)
    U.check(dw, prod.sum(-1), U.TOL * prod.abs().sum(-1))


def test_combine_backward_flags_rows(cuda_device):
    from objeta_b200.quant import device_error_take
    from objeta_b200.router import moe_combine_backward
    device_error_take(cuda_device)
    dout, v = U.randn((2, 64), seed=1), U.randn((4, 64), seed=2)
    rows = torch.tensor([[0, 4], [-1, 3]], dtype=torch.int32, device="cuda")
    dw = moe_combine_backward(dout, v, rows)
    ref = (dout.double()[:, None] * v.double()[torch.tensor([[0, 0], [0, 3]], device="cuda")]).sum(-1)
    U.check(dw, ref, 1e-4 * torch.ones_like(ref))
    assert device_error_take(cuda_device) & 8


def test_repeat_streams_and_graphs(cuda_device):
    from objeta_b200.router import balance_loss, router_backward
    l = U.randn((5000, 128), seed=1)
    ids = torch.topk(l, 8, dim=1).indices.to(torch.int32)
    dw = U.randn((5000, 8), seed=2)

    def step(stream=None):
        b = balance_loss(l, ids, stream=stream)
        return b.counts, b.balance, b.z, router_backward(l, ids, dw, balance=b, balance_grad=0.1, z_grad=0.1,
                                                         stream=stream)

    want = step()
    assert all(torch.equal(a, b) for a, b in zip(want, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = step(side)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, _, s in graphs:
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for _, out, _ in graphs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_offsets_past_32_bits(cuda_device):
    """Logits, gradients and value rows beyond 2^31 elements."""
    from objeta_b200.router import balance_loss, moe_combine_backward, router_backward
    T, E, k = 300, 64, 4
    l = U.randn((T, E), seed=1)
    ids = torch.topk(l, k, dim=1).indices.to(torch.int32)
    dw = U.randn((T, k), seed=2)
    far = torch.empty(T, 1 << 23, device="cuda")
    far[:, :E] = l
    b, c = balance_loss(l, ids), balance_loss(far[:, :E], ids)
    assert torch.equal(b.counts, c.counts) and torch.equal(b.balance, c.balance) and torch.equal(b.z, c.z)
    args = dict(renormalize=True, balance=b, balance_grad=0.1, z_grad=0.1)
    want = router_backward(l, ids, dw, **args)
    router_backward(far[:, :E], ids, dw, d_dlogits=far[:, :E], **args)
    assert torch.equal(far[:, :E], want)
    del far
    V, O = (1 << 20) + 40, 2048
    v = torch.empty(V, O, device="cuda")
    rows = torch.tensor([[0, V - 1], [1 << 20, (1 << 20) - 1]], dtype=torch.int32, device="cuda")
    v[rows.long()] = U.randn((2, 2, O), seed=4)
    d = U.randn((2, O), seed=5)
    got = moe_combine_backward(d, v, rows)
    ref = (d.double()[:, None] * v[rows.long()].double()).sum(2)
    U.check(got, ref, U.TOL * (d.double()[:, None] * v[rows.long()].double()).abs().sum(2))


def test_argument_checks(cuda_device):
    from objeta_b200.router import balance_loss, moe_combine_backward, router_backward
    l = U.randn((6, 8))
    ids = torch.zeros(6, 2, dtype=torch.int32, device="cuda")
    for bad in (dict(d_ids=ids.long()), dict(d_ids=ids[:3]), dict(d_token_mask=torch.ones(5, dtype=torch.bool, device="cuda")),
                dict(d_seq_offsets=torch.zeros(1, dtype=torch.int32, device="cuda")),
                dict(d_seq_offsets=torch.zeros(2, dtype=torch.int64, device="cuda")), dict(d_logits=l.half()),
                dict(d_logits=l.t())):
        with pytest.raises(ValueError):
            balance_loss(**{**dict(d_logits=l, d_ids=ids), **bad})
    b = balance_loss(l, ids)
    with pytest.raises(ValueError):
        router_backward(l, ids, score_func=SIGMOID, balance=b)
    with pytest.raises(ValueError):
        router_backward(l, ids, balance=b, d_token_mask=torch.ones(6, dtype=torch.bool, device="cuda"))
    with pytest.raises(ValueError):
        router_backward(l, ids, d_dweights=torch.zeros(6, 3, device="cuda"))
    with pytest.raises(ValueError):
        moe_combine_backward(l, l, ids.long())


def test_router_training_step(cuda_device):
    """Routing, frozen Q4_0 experts, combine, and the gradient of the router's
    weight back through all of it, against the chain in 64 bits over the
    experts' own output rows."""
    from objeta_b200.dense import linear, linear_backward
    from objeta_b200.ep import ep_build_pairs, moe_combine, moe_pairs, router_topk_batched
    from objeta_b200.moe import MoeLayer
    from objeta_b200.quant import QGemvShape, QuantBackend, QuantFormat
    from objeta_b200.router import balance_loss, moe_combine_backward, router_backward
    T, H, I, E, k = 48, 256, 256, 16, 4
    qb = QuantBackend(0)
    pack = lambda r, c, s: qb.quantize_matrix_device(QuantFormat.Q4_0, U.randn((r, c), scale=0.05, seed=s),
                                                     QGemvShape.q4_0(r, c))
    layer = MoeLayer(QuantFormat.Q4_0, H, I, H, [pack(I, H, 3 * e) for e in range(E)],
                     [pack(I, H, 3 * e + 1) for e in range(E)], [pack(H, I, 3 * e + 2) for e in range(E)])
    x, wr, target = U.randn((T, H), seed=1), U.randn((E, H), scale=0.1, seed=2), U.randn((T, H), scale=0.1, seed=3)
    logits = linear(x, wr)
    ids, w = router_topk_batched(logits, k, renormalize=True)
    bal = balance_loss(logits, ids)
    pe, pt, po, cnt = ep_build_pairs(ids.view(1, T, k), 0, E)
    v = torch.empty(T * k, H, device="cuda")
    moe_pairs(layer, pe, pt, x, v, pair_out=po, d_count=cnt)
    slot = torch.arange(T * k, dtype=torch.int32, device="cuda").view(T, k)
    out = moe_combine(v, slot, w, torch.empty(T, H, device="cuda"))
    dout = out - target
    dw = moe_combine_backward(dout, v, slot)
    dl = router_backward(logits, ids, dw, renormalize=True, balance=bal, balance_grad=0.5, z_grad=0.05)
    _, dwr, _ = linear_backward(dl, x, wr, need_dx=False)
    W = wr.double().requires_grad_()
    L = x.double() @ W.t()
    s = torch.softmax(L, 1)
    q = torch.gather(s, 1, ids.long())
    q = q / q.sum(1, keepdim=True)
    o = (q[:, :, None] * v.double().view(T, k, H)).sum(1)
    counts = torch.bincount(ids.reshape(-1).long(), minlength=E).double()
    loss = 0.5 * (o - target.double()).square().sum() + 0.5 * (s.mean(0) * counts * E / (k * T)).sum() \
        + 0.05 * torch.logsumexp(L, 1).square().mean()
    ref = torch.autograd.grad(loss, W)[0]
    # every link is good to about 1e-5 of its terms; their sum over 48 tokens has no cancellation beyond 30x
    assert float((dwr.double() - ref).norm() / ref.norm()) <= 3e-4
