"""The dense products where accumulators are longest and values are not finite,
against 64-bit products."""
import math

import pytest

torch = pytest.importorskip("torch")

from tests import _dense_util as U  # noqa: E402

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt,K", [("f16", 16384), ("f16", 16448), ("f16", 65536), ("f16", 65600), ("bf16", 65536),
                                  ("bf16", 65600)])
def test_longest_accumulators_of_one_sign(cuda_device, dt, K):
    """Products of one sign over the longest k of an accumulator that is not promoted, and one k-block more, where
    the tiles fill the device: what truncation takes is a fraction of the result's rounding, and one-sided, so
    that the mean error shows it."""
    from objeta_b200.dense import linear
    T = N = 4096
    t = U.DT[dt]
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.rand(T, K, generator=g, device="cuda", dtype=t)
    w = torch.rand(N, K, generator=g, device="cuda", dtype=t) * 0.25
    y = linear(x, w)[::64, ::64]
    ref = x[::64].double() @ w[::64].double().t()
    half = torch.finfo(t).eps / 2
    loss = half / 4  # f16: a quarter of its half step (1.2e-4); bf16: of its largest (9.8e-4)
    U.check(y, ref, (half + loss) * ref, "y")
    # 4096 elements, each off by a rounding of at most half a step: their mean by half / sqrt(3) / 64 in a deviation,
    # six of which make half / 18
    mean = float(((y.double() - ref) / ref).mean())
    assert abs(mean) <= loss + half / 18, mean


def test_choice_of_tile_knows_the_type(cuda_device):
    """The same sizes in both 16-bit types, one after the other: each has its own longest accumulator."""
    from objeta_b200.dense import linear
    T = N = 2048
    K = 40000
    for dt in ("bf16", "f16", "bf16", "f16"):
        t = U.DT[dt]
        g = torch.Generator(device="cuda").manual_seed(7)
        x = torch.rand(T, K, generator=g, device="cuda", dtype=t)
        w = torch.rand(N, K, generator=g, device="cuda", dtype=t) * 0.25
        y = linear(x, w)[::32, ::32]
        ref = x[::32].double() @ w[::32].double().t()
        half = torch.finfo(t).eps / 2
        U.check(y, ref, 1.25 * half * ref, dt)
        assert abs(float(((y.double() - ref) / ref).mean())) <= half / 4 + half / 18, dt


@pytest.mark.parametrize("limit", [0.0, 1.0])
@pytest.mark.parametrize("T,H,I,O", [(2, 256, 128, 64), (16, 512, 300, 200), (17, 128, 64, 64), (300, 256, 192, 256),
                                     (700, 264, 800, 1000)])
def test_ffn_keeps_nan(cuda_device, T, H, I, O, limit):
    """NaN in a token makes its row NaN, also through the limited SwiGLU, and no other; in a weight all rows."""
    from objeta_b200.dense import ffn_bf16_tokens
    x = U.randn((T, H), seed=1)
    g, u = (U.randn((I, H), torch.bfloat16, 1 / math.sqrt(H), s) for s in (2, 3))
    d = U.randn((O, I), torch.bfloat16, 1 / math.sqrt(I), 4)
    want = ffn_bf16_tokens(g, u, d, x, swiglu_limit=limit)
    assert bool(torch.isfinite(want).all())
    bad = x.clone()
    bad[1, 5] = math.nan
    out = ffn_bf16_tokens(g, u, d, bad, swiglu_limit=limit)
    rest = torch.arange(T, device="cuda") != 1
    assert bool(torch.isnan(out[1]).all()) and torch.equal(out[rest], want[rest])
    for i in range(2):
        w = [g.clone(), u.clone()]
        w[i][I - 1, H - 1] = math.nan
        assert bool(torch.isnan(ffn_bf16_tokens(w[0], w[1], d, x, swiglu_limit=limit)).all()), i


def test_expert_parallel_shared_expert_of_every_batch(cuda_device):
    """Checks of the shared expert's weights, and the same tokens in batches of several sizes: within the bound of
    one another (the shared part's bits go with the batch)."""
    from objeta_b200.ep import ExpertParallelMoe, router_topk_batched
    from objeta_b200.moe import MoeLayer
    from objeta_b200.quant import QGemvShape, QuantBackend, QuantFormat
    from tests.test_dense_gpu import _ffn_ref
    T, H, I, E, k, Is = 40, 256, 256, 8, 2, 192
    qb = QuantBackend(0)
    pack = lambda r, c, s: qb.quantize_matrix_device(QuantFormat.Q4_0, U.randn((r, c), scale=0.05, seed=s),
                                                     QGemvShape.q4_0(r, c))
    layer = MoeLayer(QuantFormat.Q4_0, H, I, H, [pack(I, H, 3 * e) for e in range(E)],
                     [pack(I, H, 3 * e + 1) for e in range(E)], [pack(H, I, 3 * e + 2) for e in range(E)])
    g, u = U.randn((Is, H), torch.bfloat16, 1 / 16, 91), U.randn((Is, H), torch.bfloat16, 1 / 16, 92)
    d = U.randn((H, Is), torch.bfloat16, 1 / 14, 93)
    x = U.randn((T, H), seed=94)
    ids, w = router_topk_batched(U.randn((T, E), seed=95), k, renormalize=True)
    moe = ExpertParallelMoe(layer, E, k, shared=(g, u, d))
    routed = ExpertParallelMoe(layer, E, k).forward(x, ids, w)
    ref = _ffn_ref(g, u, d, x, routed, 0.0)
    at = 0
    for n in (1, 3, 16, 20):
        rows = slice(at, at + n)
        U.check(moe.forward(x[rows], ids[rows], w[rows]), ref[0][rows], ref[1][rows], f"{n} tokens")
        at += n
    for bad in ((g.half(), u.half(), d.half()), (g.float(), u.float(), d.float()), (g, u, d.t().contiguous().t()),
                (g.cpu(), u.cpu(), d.cpu()), (g[:, :128].contiguous(), u[:, :128].contiguous(), d)):
        with pytest.raises(ValueError, match="shared expert"):
            ExpertParallelMoe(layer, E, k, shared=bad)


@pytest.mark.parametrize("T,H", [(1, 200), (16, 256), (61, 33), (700, 264)])
def test_ffn_over_its_input(cuda_device, T, H):
    """x += ffn(x): x is read before the first result is written."""
    from objeta_b200.dense import ffn_bf16_tokens
    I = 136
    x = U.randn((T, H), seed=1)
    g, u = (U.randn((I, H), torch.bfloat16, 1 / math.sqrt(H), s) for s in (2, 3))
    d = U.randn((H, I), torch.bfloat16, 1 / math.sqrt(I), 4)
    want = ffn_bf16_tokens(g, u, d, x, d_residual=x)
    for _ in range(3):
        h = x.clone()
        assert ffn_bf16_tokens(g, u, d, h, d_residual=h, d_out=h) is h and torch.equal(h, want)


def test_results_over_operands_are_refused(cuda_device):
    from objeta_b200 import CudaError
    from objeta_b200.dense import linear, linear_backward
    from objeta_b200.router import router_backward
    x, w = U.randn((40, 64), torch.bfloat16, seed=1), U.randn((64, 64), torch.bfloat16, seed=2)
    for kw in (dict(d_y=x), dict(d_y=w[:40]), dict(d_z=x)):
        with pytest.raises(CudaError, match="overlaps"):
            linear(x, w, **kw)
    with pytest.raises(CudaError, match="overlaps"):
        linear_backward(x, U.randn((40, 64), torch.bfloat16), w, d_dx=x)
    l = U.randn((41, 8), seed=3)
    ids = torch.zeros(40, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(CudaError, match="overlaps"):
        router_backward(l[:40], ids, U.randn((40, 1)), d_dlogits=l[1:])
    # side by side in one buffer
    buf = torch.cat((x, torch.zeros_like(x)), 1)
    assert torch.equal(linear(buf[:, :64], w, d_y=buf[:, 64:]), linear(x, w))


@pytest.mark.parametrize("Is,shift", [(100, 0), (33, 0), (96, 1), (320, 3), (64, 0)])
def test_expert_parallel_shared_expert_of_any_width(cuda_device, Is, shift):
    """Widths and addresses that the one-token call does not take: a step of one token runs as one of more does."""
    from objeta_b200.ep import ExpertParallelMoe, router_topk_batched
    from objeta_b200.moe import MoeLayer
    from objeta_b200.quant import QGemvShape, QuantBackend, QuantFormat
    from tests.test_dense_gpu import _ffn_ref
    H, I, E, k = 256, 256, 4, 2
    qb = QuantBackend(0)
    pack = lambda r, c, s: qb.quantize_matrix_device(QuantFormat.Q4_0, U.randn((r, c), scale=0.05, seed=s),
                                                     QGemvShape.q4_0(r, c))
    layer = MoeLayer(QuantFormat.Q4_0, H, I, H, [pack(I, H, 3 * e) for e in range(E)],
                     [pack(I, H, 3 * e + 1) for e in range(E)], [pack(H, I, 3 * e + 2) for e in range(E)])

    def at(t):  # `shift` elements off 16-byte alignment
        buf = torch.empty(t.numel() + shift, dtype=t.dtype, device="cuda")[shift:].view(t.shape)
        return buf.copy_(t)

    g, u = (at(U.randn((Is, H), torch.bfloat16, 1 / 16, s)) for s in (91, 92))
    d = at(U.randn((H, Is), torch.bfloat16, 1 / 14, 93))
    x = U.randn((3, H), seed=94)
    ids, w = router_topk_batched(U.randn((3, E), seed=95), k, renormalize=True)
    moe, plain = ExpertParallelMoe(layer, E, k, shared=(g, u, d)), ExpertParallelMoe(layer, E, k)
    for n in (1, 3):
        ref, bound = _ffn_ref(g, u, d, x[:n], plain.forward(x[:n], ids[:n], w[:n]), 0.0)
        U.check(moe.forward(x[:n], ids[:n], w[:n]), ref, bound, f"{Is} {shift} {n}")
