"""The dense products of many tokens against 64-bit products: types, odd sizes,
strides, epilogues, gradients (also against differences), the shared expert of
a batch, streams and captured graphs."""
import math

import pytest

torch = pytest.importorskip("torch")

from tests import _dense_util as U  # noqa: E402

pytestmark = pytest.mark.gpu

PAIRS = [("bf16", "bf16", "bf16"), ("bf16", "bf16", "f32"), ("f16", "f16", "f16"), ("f16", "f16", "f32"),
         ("f32", "bf16", "f32"), ("f32", "f32", "f32")]
# tokens, in, out: one token, odd everything, a multiple of nothing, tiles and their borders
SIZES = [(1, 64, 64), (1, 4096, 256), (3, 7, 5), (17, 200, 129), (33, 1000, 257), (64, 64, 8), (128, 512, 384),
         (129, 520, 136), (250, 2048, 256), (300, 136, 1000), (513, 72, 264), (7, 5001, 33)]


def _case(T, K, N, xd, wd, seed=0):
    x = U.randn((T, K), U.DT[xd], seed=seed)
    w = U.randn((N, K), U.DT[wd], 1 / math.sqrt(K), seed=seed + 1)
    return x, w


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("xd,wd,yd", PAIRS)
def test_linear(cuda_device, xd, wd, yd, T, K, N):
    from objeta_b200.dense import linear
    x, w = _case(T, K, N, xd, wd)
    y = linear(x, w, out_dtype=U.DT[yd])
    _, _, ref, bound = U.linear_ref(x, w, None, "none", None, U.DT[yd])
    U.check(y, ref, bound, "y")


@pytest.mark.parametrize("act", U.ACTS)
@pytest.mark.parametrize("xd,wd,yd", PAIRS)
def test_linear_epilogue(cuda_device, xd, wd, yd, act):
    from objeta_b200.dense import linear
    for T, K, N in ((1, 256, 192), (45, 264, 133), (260, 384, 520)):
        x, w = _case(T, K, N, xd, wd, 3)
        yt = U.DT[yd]
        r = U.randn((T, N), yt, seed=9)
        z = torch.full((T, N), math.nan, dtype=yt, device="cuda")
        for bdt in {U.DT[wd], torch.float32}:
            b = U.randn((N,), bdt, 2.0, seed=8)
            y = linear(x, w, b, activation=act, d_residual=r, out_dtype=yt, d_z=z)
            rz, bz, ry, by = U.linear_ref(x, w, b, act, r, yt)
            U.check(z, rz, bz, "z")
            U.check(y, ry, by, "y")


def test_linear_activation_range(cuda_device):
    """Far arguments: no overflow inside an activation, and NaN stays NaN."""
    from objeta_b200.dense import linear
    v = torch.tensor([-3e38, -1e30, -1e4, -200.0, -90.0, -30.0, -5.0, -0.0, 0.0, 1e-30, 5.0, 30.0, 90.0, 1e4, 1e30],
                     device="cuda").view(-1, 1)
    one = torch.ones(1, 1, device="cuda")
    for act in U.ACTS:
        y = linear(v, one, activation=act)
        ref = U.act64(v.double(), act)
        # exp(-|v|) and its sums: 16 roundings of the terms, the arguments' rounding grows with |v|
        bound = 16 * 2.0 ** -24 * (ref.abs() + torch.clamp(v.double().abs(), max=200.0) * 1e-2 *
                                   (v.double().abs() < 200)) + 1e-38
        U.check(y, ref, bound, act)
        assert bool(torch.isnan(linear(torch.full((1, 1), math.nan, device="cuda"), one, activation=act)).all()), act


@pytest.mark.parametrize("xd,wd,yd", PAIRS)
@pytest.mark.parametrize("extra,offset", [(8, 0), (1, 0), (8, 1), (3, 5)])
def test_linear_strides(cuda_device, xd, wd, yd, extra, offset):
    """Padded rows and odd addresses, on every operand and result; what lies
    between the rows of y stays as it was."""
    from objeta_b200.dense import linear
    for T, K, N in ((1, 96, 40), (70, 130, 200)):
        x, w = _case(T, K, N, xd, wd, 5)
        yt = U.DT[yd]
        r = U.randn((T, N), yt, seed=6)
        buf = torch.full((T * (N + extra) + offset,), 7.0, dtype=yt, device="cuda")
        y = buf[offset:offset + T * (N + extra)].view(T, N + extra)[:, :N]
        zb = torch.full((T, N + extra), 7.0, dtype=yt, device="cuda")
        linear(U.strided(x, extra, offset), U.strided(w, extra, offset), d_residual=U.strided(r, extra, offset), d_y=y,
               d_z=zb[:, :N])
        rz, bz, ry, by = U.linear_ref(x, w, None, "none", r, yt)
        U.check(y, ry, by, "y")
        U.check(zb[:, :N], rz, bz, "z")
        rest = buf.clone()
        rest[offset:offset + T * (N + extra)].view(T, N + extra)[:, :N] = 7.0
        assert bool((rest == 7.0).all()) and bool((zb[:, N:] == 7.0).all())


def test_linear_residual_in_place(cuda_device):
    from objeta_b200.dense import linear
    for T, K, N in ((1, 2048, 512), (200, 256, 300)):
        x, w = _case(T, K, N, "bf16", "bf16", 7)
        r = U.randn((T, N), torch.bfloat16, seed=4)
        y = r.clone()
        linear(x, w, d_residual=y, d_y=y)
        _, _, ry, by = U.linear_ref(x, w, None, "none", r, torch.bfloat16)
        U.check(y, ry, by)


@pytest.mark.parametrize("wd", ["bf16", "f32"])
def test_linear_f32_keeps_f32(cuda_device, wd):
    """f32 operands of every magnitude: products as exact as f32 sums."""
    from objeta_b200.dense import linear
    T, K, N = 40, 300, 70
    g = torch.Generator(device="cuda").manual_seed(3)
    x = U.randn((T, K), seed=1) * torch.exp2(torch.randint(-60, 60, (T, 1), generator=g, device="cuda").float())
    w = (U.randn((N, K), seed=2) * torch.exp2(torch.randint(-40, 40, (N, 1), generator=g, device="cuda").float())
         ).to(U.DT[wd])
    y = linear(x, w)
    _, _, ref, bound = U.linear_ref(x, w, None, "none", None, torch.float32)
    U.check(y, ref, bound)
    # the average error is that of f32 sums: a few 2^-24, not a bf16 step
    rel = float((y.double() - ref).norm() / ref.norm())
    assert rel <= 1e-6, rel


@pytest.mark.parametrize("xd,wd,T,K,N", [("f32", "f32", 17, 136, 40000), ("f32", "f32", 32, 5000, 3000),
                                         ("f32", "f32", 1, 68, 20001), ("f32", "bf16", 1, 8200, 4000),
                                         ("f32", "bf16", 1000, 136, 65), ("f32", "f32", 100, 260, 600)])
def test_linear_few_f32_tokens(cuda_device, xd, wd, T, K, N):
    """f32 operands that the product splits itself: more tiles than the grid holds at once, many k-blocks, ragged
    ends; rows that the copy engine cannot read give the same."""
    from objeta_b200.dense import linear
    x, w = _case(T, K, N, xd, wd, 5)
    b, r = U.randn((N,), torch.float32, seed=8), U.randn((T, N), seed=9)
    y = linear(x, w, b, activation="silu", d_residual=r)
    _, _, ref, bound = U.linear_ref(x, w, b, "silu", r, torch.float32)
    U.check(y, ref, bound, "y")
    U.check(linear(U.strided(x, 3, 1), U.strided(w, 5, 1), b, activation="silu", d_residual=r), ref, bound, "strided")
    U.check(linear(U.strided(x, 4, 4), U.strided(w, 8, 8), b, activation="silu", d_residual=r), ref, bound, "aligned")


def test_linear_non_finite(cuda_device):
    """Inf and NaN reach their row (x) or column (w) of y and no other."""
    from objeta_b200.dense import linear
    for xd, wd, _ in PAIRS:
        for bad in (math.inf, -math.inf, math.nan):
            x, w = _case(40, 200, 150, xd, wd, 2)
            x[7, 11] = bad
            w[101, 5] = bad
            y = linear(x, w)
            fin = torch.isfinite(y)
            want = torch.ones_like(fin)
            want[7, :] = False
            want[:, 101] = False
            assert bool((fin == want).all()), (xd, wd, bad)


@pytest.mark.parametrize("T,K,N", [(300, 200, 400), (40, 203, 150), (700, 1000, 900)])
def test_non_finite_of_laid_out_operands(cuda_device, T, K, N):
    """The same for operands that become planes or images first, forwards and in both gradients."""
    from objeta_b200.dense import linear, linear_backward
    for xd, wd, _ in PAIRS:
        for bad in (math.inf, -math.inf, math.nan):
            x, w = _case(T, K, N, xd, wd, 2)
            dy = U.randn((T, N), U.DT[xd], seed=4)
            want = torch.ones(T, N, dtype=torch.bool, device="cuda")
            x[7, 11] = bad
            w[101, 5] = bad
            want[7, :] = False
            want[:, 101] = False
            assert bool((torch.isfinite(linear(x, w)) == want).all()), (xd, wd, bad)
            x, w = _case(T, K, N, xd, wd, 2)
            dy[9, 3] = bad  # its row of dx, its row of dw
            dx, dw, db = linear_backward(dy, x, w, need_dbias=True)
            rows = torch.isfinite(dx).all(1)
            assert not bool(torch.isfinite(dx[9]).any()) and int((~rows).sum()) == 1, (xd, wd, bad)
            rows = torch.isfinite(dw).all(1)
            assert not bool(torch.isfinite(dw[3]).any()) and int((~rows).sum()) == 1, (xd, wd, bad)
            assert int((~torch.isfinite(db)).sum()) == 1 and not bool(torch.isfinite(db[3]))


def test_linear_empty_and_repeat(cuda_device):
    from objeta_b200.dense import linear
    x, w = _case(0, 64, 32, "bf16", "bf16")
    assert linear(x, w).shape == (0, 32)
    for T in (1, 37, 700):
        x, w = _case(T, 1536, 640, "f32", "bf16", 2)
        a = linear(x, w, activation="silu")
        assert all(torch.equal(a, linear(x, w, activation="silu")) for _ in range(3))


BPAIRS = [("bf16", "bf16", "bf16", "bf16"), ("bf16", "bf16", "bf16", "f32"), ("bf16", "bf16", "f32", "f32"),
          ("bf16", "bf16", "f32", "bf16"), ("f16", "f16", "f16", "f16"), ("f16", "f16", "f16", "f32"),
          ("f16", "f16", "f32", "f16"), ("f32", "bf16", "f32", "f32"), ("f32", "bf16", "f32", "bf16"), ("f32", "f32", "f32", "f32")]


def _run_backward(T, K, N, xd, wd, yd, dwd, act, seed=0):
    from objeta_b200.dense import linear_backward
    x, w = _case(T, K, N, xd, wd, seed)
    dy = U.randn((T, N), U.DT[yd], seed=seed + 2)
    z = U.randn((T, N), U.DT[yd], seed=seed + 3) if act != "none" else None
    dx, dw, db = linear_backward(dy, x, w, z, activation=act, need_dbias=True, dw_dtype=U.DT[dwd])
    ref = U.backward_ref(dy, x, w, z, act, U.DT[dwd])
    for name, got in (("dx", dx), ("dw", dw), ("db", db)):
        U.check(got, *ref[name], f"{name} of {xd} {wd} {yd} {dwd} {act} {T} {K} {N}")


def test_backward_activation_range(cuda_device):
    """Far pre-activations: the powers of z overflow, the derivative is its limit; NaN stays NaN."""
    from objeta_b200.dense import linear_backward
    z = torch.tensor([-3e38, -1e30, -1e13, -1e4, -200.0, -129.0, -128.0, -90.0, -30.0, -5.0, -0.0, 0.0, 1e-30, 5.0,
                      30.0, 90.0, 129.0, 1e4, 1e13, 1e30, 3e38], device="cuda").view(-1, 1)
    far = torch.tensor([math.inf, -math.inf, math.nan], device="cuda").view(-1, 1)
    one = torch.ones(1, 1, device="cuda")
    for act in U.ACTS[1:]:
        dx = linear_backward(torch.ones_like(z), z, one, d_z=z, activation=act, need_dw=False)[0]
        ref = U.act_grad64(z, act)
        # 16 roundings; the exponent's argument, at most a few |z|, is rounded and its exponential off by as much;
        # below 1e-37 an exponential is flushed to 0
        bound = (16 + 8 * torch.clamp(z.double().abs(), max=200.0)) * 2.0 ** -24 * ref.abs() + 1e-36
        U.check(dx, ref, bound, act)
        dx = linear_backward(torch.ones_like(far), far, one, d_z=far, activation=act, need_dw=False)[0]
        assert dx[0] == 1 and dx[1] == 0 and (act == "relu" or bool(torch.isnan(dx[2]))), (act, dx)


def test_long_k_of_one_sign(cuda_device):
    """131072 products of one sign in f16: what the accumulators lose stays below the result's rounding."""
    from objeta_b200.dense import linear
    T = N = 4096
    K = 131072
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.rand(T, K, generator=g, device="cuda", dtype=torch.float16) * 0.5
    w = torch.rand(N, K, generator=g, device="cuda", dtype=torch.float16) * 0.5
    y = linear(x, w)[::64, ::64]
    ref = x[::64].double() @ w[::64].double().t()
    # an accumulator of 64 k-blocks takes 256 MMAs, each off by at most a step (2^-23); then f16's half step
    U.check(y, ref, (256 * 2.0 ** -23 + 32 * 2.0 ** -24 + 2.0 ** -11) * ref)


@pytest.mark.parametrize("xd,wd,yd,dwd", BPAIRS)
def test_backward_sizes(cuda_device, xd, wd, yd, dwd):
    for T, K, N in ((1, 64, 64), (3, 7, 5), (33, 1000, 257), (129, 520, 136), (400, 136, 256), (1025, 72, 48)):
        _run_backward(T, K, N, xd, wd, yd, dwd, "none")
        _run_backward(T, K, N, xd, wd, yd, dwd, "silu", 5)


@pytest.mark.parametrize("act", U.ACTS)
@pytest.mark.parametrize("xd,wd,yd,dwd", BPAIRS)
def test_backward_activations(cuda_device, xd, wd, yd, dwd, act):
    _run_backward(65, 200, 136, xd, wd, yd, dwd, act, 11)


@pytest.mark.parametrize("xd,wd,yd,dwd", BPAIRS)
def test_backward_strides_and_accumulate(cuda_device, xd, wd, yd, dwd):
    from objeta_b200.dense import linear_backward
    for (T, K, N), extra, offset in (((37, 96, 72), 8, 0), ((50, 61, 33), 3, 5)):
        x, w = _case(T, K, N, xd, wd, 1)
        dy = U.randn((T, N), U.DT[yd], seed=2)
        z = U.randn((T, N), U.DT[yd], seed=3)
        dw0, db0 = U.randn((N, K), U.DT[dwd], seed=4), U.randn((N,), seed=5)
        dxb = torch.full((T, K + extra), 7.0, dtype=x.dtype, device="cuda")
        dw, db = U.strided(dw0, extra, offset), db0.clone()
        linear_backward(U.strided(dy, extra, offset), U.strided(x, extra, offset), U.strided(w, extra, offset),
                        U.strided(z, extra, offset), activation="gelu", need_dbias=True, d_dx=dxb[:, :K], d_dw=dw,
                        d_dbias=db, accumulate=True)
        ref = U.backward_ref(dy, x, w, z, "gelu", U.DT[dwd], dw0, db0)
        for name, got in (("dx", dxb[:, :K]), ("dw", dw), ("db", db)):
            U.check(got, *ref[name], f"{name} {xd} {wd} {yd} {dwd} {extra}")
        assert bool((dxb[:, K:] == 7.0).all())


def test_backward_parts(cuda_device):
    """Each gradient alone, and the sums over no tokens."""
    from objeta_b200.dense import linear_backward
    x, w = _case(90, 128, 72, "bf16", "bf16", 1)
    dy = U.randn((90, 72), torch.bfloat16, seed=2)
    dx, dw, db = linear_backward(dy, x, w, need_dbias=True)
    assert torch.equal(linear_backward(dy, x, w, need_dw=False)[0], dx)
    assert torch.equal(linear_backward(dy, x, w, need_dx=False)[1], dw)
    assert torch.equal(linear_backward(dy, x, w, need_dx=False, need_dw=False, need_dbias=True)[2], db)
    e = linear_backward(dy[:0], x[:0], w, need_dbias=True)
    assert e[0].shape == (0, 128) and not e[1].any() and not e[2].any()
    one = torch.ones_like(dw)
    linear_backward(dy[:0], x[:0], w, need_dx=False, d_dw=one, accumulate=True)
    assert bool((one == 1).all())


@pytest.mark.parametrize("act", U.ACTS)
def test_backward_against_differences(cuda_device, act):
    """d/dp sum(dy act(x w^T + b)) by central differences in 64 bits, through
    the kept z.  Step 1e-6: rounding 1e-16 / 1e-6, curvature 1e-12."""
    from objeta_b200.dense import linear, linear_backward
    T, K, N = 5, 6, 4
    x, w, b = U.randn((T, K), seed=1), U.randn((N, K), seed=2), U.randn((N,), seed=3)
    dy = U.randn((T, N), seed=4)
    z = torch.empty(T, N, device="cuda")
    linear(x, w, b, activation=act, d_z=z)
    grads = dict(zip("xwb", linear_backward(dy, x, w, z, activation=act, need_dbias=True)))
    p = {"x": x.double(), "w": w.double(), "b": b.double()}

    def loss():
        return float((dy.double() * U.act64(p["x"] @ p["w"].t() + p["b"], act)).sum())

    for name, g in grads.items():
        flat = p[name].view(-1)
        for i in range(flat.numel()):
            keep = flat[i].item()
            flat[i] = keep + 1e-6
            up = loss()
            flat[i] = keep - 1e-6
            down = loss()
            flat[i] = keep
            # z was rounded to f32: its part of the gradient, and TOL of the sums (all below 30 here)
            assert abs((up - down) / 2e-6 - g.reshape(-1)[i].item()) <= 1e-4, (name, i)


def _ffn_ref(g, u, d, x, r, limit):
    G, Uu, X = g.double(), u.double(), x.double()
    gate, up = X @ G.t(), X @ Uu.t()
    gb, ub = U.product_bound(X, G), U.product_bound(X, Uu)
    if limit > 0:
        gate, up = torch.clamp(gate, max=limit), torch.clamp(up, -limit, limit)
    a = U.act64(gate, "silu") * up
    ab = 1.1 * gb * up.abs() + U.act64(gate, "silu").abs() * ub + 1.1 * gb * ub + 8 * 2.0 ** -24 * a.abs()
    D = d.double()
    out = a @ D.t()
    ob = U.product_bound(a, D) + ab @ D.abs().t()
    if r is not None:
        out = out + r.double()
        ob = ob + 2.0 ** -23 * (out.abs() + r.double().abs())
    return out, ob + U.half_step(torch.float32, out)


@pytest.mark.parametrize("T,H,I,O", [(1, 256, 128, 256), (5, 200, 72, 90), (16, 4096, 2048, 4096), (61, 33, 17, 41),
                                     (130, 512, 640, 384), (300, 256, 192, 256)])
@pytest.mark.parametrize("limit", [0.0, 0.4])
def test_ffn_tokens(cuda_device, T, H, I, O, limit):
    from objeta_b200.dense import ffn_bf16_tokens
    x = U.randn((T, H), seed=1)
    g, u = U.randn((I, H), torch.bfloat16, 1 / math.sqrt(H), 2), U.randn((I, H), torch.bfloat16, 1 / math.sqrt(H), 3)
    d = U.randn((O, I), torch.bfloat16, 1 / math.sqrt(I), 4)
    r = U.randn((T, O), seed=5)
    U.check(ffn_bf16_tokens(g, u, d, x, swiglu_limit=limit), *_ffn_ref(g, u, d, x, None, limit), "out")
    out = r.clone()
    ffn_bf16_tokens(g, u, d, x, d_residual=out, d_out=out, swiglu_limit=limit)
    U.check(out, *_ffn_ref(g, u, d, x, r, limit), "out, in place")


def test_ffn_tokens_matches_the_one_token_call(cuda_device):
    from objeta_b200.dense import ffn_bf16_tokens
    from objeta_b200.moe import ffn_bf16_device
    H, I = 2048, 512
    x = U.randn((9, H), seed=1)
    g, u = U.randn((I, H), torch.bfloat16, 0.02, 2), U.randn((I, H), torch.bfloat16, 0.02, 3)
    d = U.randn((H, I), torch.bfloat16, 0.02, 4)
    out = ffn_bf16_tokens(g, u, d, x)
    one = torch.empty(9, H, device="cuda")
    for t in range(9):
        ffn_bf16_device(g, u, d, H, I, H, x[t], one[t])
    ref, bound = _ffn_ref(g, u, d, x, None, 0.0)
    U.check(out, ref, bound)
    U.check(one, ref, bound)


def test_streams_and_graphs(cuda_device):
    """A side stream, and two graphs captured from it and replayed at once:
    each call has its own scratch."""
    from objeta_b200.dense import linear, linear_backward
    x, w = _case(96, 1000, 136, "f32", "f32", 1)
    dy = U.randn((96, 136), seed=2)
    want = (linear(x, w), *linear_backward(dy, x, w)[:2])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = (linear(x, w, stream=side), *linear_backward(dy, x, w, stream=side)[:2])
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((linear(x, w), *linear_backward(dy, x, w)[:2]))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, o))


def test_many_streams_at_once(cuda_device):
    """Products of every kind of tile side by side on the device: the same bits as one after another."""
    from objeta_b200.dense import ffn_bf16_tokens, linear, linear_backward
    cases = []
    for xd, wd, T, K, N in (("f32", "f32", 250, 2048, 256), ("bf16", "bf16", 1, 4096, 4096), ("f32", "bf16", 30, 2048, 512),
                            ("bf16", "bf16", 1500, 512, 2048), ("f32", "f32", 700, 512, 1024), ("f16", "f16", 60, 1000, 3000)):
        x, w = _case(T, K, N, xd, wd, T)
        dy = U.randn((T, N), U.DT[xd], seed=3)
        cases.append(lambda x=x, w=w: (linear(x, w),))
        cases.append(lambda x=x, w=w, dy=dy: linear_backward(dy, x, w, need_dbias=True))
    g, u = (U.randn((512, 1024), torch.bfloat16, 0.03, i) for i in (1, 2))
    d = U.randn((1024, 512), torch.bfloat16, 0.04, 3)
    for T in (16, 300):
        cases.append(lambda x=U.randn((T, 1024), seed=T): (ffn_bf16_tokens(g, u, d, x),))
    want = [f() for f in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for turn in range(6):
        for i, f in enumerate(cases):
            with torch.cuda.stream(streams[(i + turn) % 4]):
                got.append((i, f()))
    torch.cuda.synchronize()
    for i, r in got:
        assert all(torch.equal(a, b) for a, b in zip(want[i], r)), i


def test_offsets_past_32_bits(cuda_device):
    """Outputs, dz images and strided rows beyond 2^31 elements."""
    from objeta_b200.dense import linear, linear_backward
    T, K, N = 70000, 64, 32768
    x, w = _case(T, K, N, "bf16", "bf16", 1)
    y = linear(x, w)
    rows = torch.tensor([0, 65535, 65536, 65537, T - 1], device="cuda")
    _, _, ref, bound = U.linear_ref(x[rows], w, None, "none", None, torch.bfloat16)
    U.check(y[rows], ref, bound, "y")
    dx, _, db = linear_backward(y, x, w, y, activation="relu", need_dw=False, need_dbias=True)
    r = U.backward_ref(y[rows], x[rows], w, y[rows], "relu", torch.bfloat16)
    U.check(dx[rows], *r["dx"], "dx")
    pos = torch.zeros(N, dtype=torch.double, device="cuda")
    for i in range(0, T, 7000):
        pos += torch.relu(y[i:i + 7000].double()).sum(0)
    U.check(db, pos, U.TOL * pos + 1e-30, "db")
    del y, dx
    buf = torch.empty(300, 1 << 23, device="cuda", dtype=torch.bfloat16)[:, :K]  # rows 2^23 elements apart
    buf.copy_(x[:300])
    assert torch.equal(linear(buf, w[:100]), linear(x[:300].contiguous(), w[:100]))


def test_c_entry_with_the_streams_workspace(cuda_device):
    """NULL scratch: the per-stream workspace, as the other device entries."""
    import ctypes
    from objeta_b200 import _lib
    from objeta_b200.dense import _LinearDesc, linear
    x, w = _case(20, 300, 50, "f32", "bf16", 1)
    y = torch.empty(20, 50, device="cuda")
    d = _LinearDesc(tokens=20, in_features=300, out_features=50, x_dtype=0, w_dtype=2, y_dtype=0)
    _lib.call("objb_linear_device", ctypes.byref(d), x.data_ptr(), w.data_ptr(), None, None, y.data_ptr(), None, None,
              0, torch.cuda.current_stream().cuda_stream)
    assert torch.equal(y, linear(x, w))


@pytest.mark.parametrize("xd,wd,yd", PAIRS)
def test_large_tiles(cuda_device, xd, wd, yd):
    """Results that fill the SMs with the largest tiles, ragged on both sides,
    more tiles than the grid holds at once, one k-block and many."""
    from objeta_b200.dense import linear
    for T, K, N, act in ((1500, 200, 1800, "none"), (2049, 40, 1537, "silu"), (2600, 1000, 5000, "gelu_tanh"),
                         (8000, 64, 1000, "relu"), (4100, 72, 4100, "none")):
        x, w = _case(T, K, N, xd, wd, 4)
        yt = U.DT[yd]
        b, r = U.randn((N,), U.DT[wd], seed=8), U.randn((T, N), yt, seed=9)
        z = torch.empty(T, N, dtype=yt, device="cuda")
        y = linear(x, w, b, activation=act, d_residual=r, d_z=z, out_dtype=yt)
        rz, bz, ry, by = U.linear_ref(x, w, b, act, r, yt)
        U.check(z, rz, bz, "z")
        U.check(y, ry, by, "y")
        assert torch.equal(y, linear(x, w, b, activation=act, d_residual=r, out_dtype=yt))


@pytest.mark.parametrize("xd,wd", [("f32", "bf16"), ("f32", "f32")])
def test_long_k_f32(cuda_device, xd, wd):
    """Hundreds of k-blocks and more tiles than the grid holds at once, forwards and for both gradients."""
    from objeta_b200.dense import linear
    x, w = _case(1500, 20000, 2600, xd, wd, 6)
    _, _, ref, bound = U.linear_ref(x, w, None, "none", None, torch.float32)
    y = linear(x, w)
    U.check(y, ref, bound)
    assert float((y.double() - ref).norm() / ref.norm()) <= 1e-6  # f32 sums, not bf16 steps
    _run_backward(20000, 2600, 1500, xd, wd, "f32", "f32", "none", 7)
    _run_backward(1500, 2600, 20000, xd, wd, "f32", "f32", "none", 8)


@pytest.mark.parametrize("xd,wd,yd,dwd", BPAIRS)
def test_large_tiles_backward(cuda_device, xd, wd, yd, dwd):
    _run_backward(1600, 1704, 1601, xd, wd, yd, dwd, "none", 3)
    _run_backward(2603, 1801, 4056, xd, wd, yd, dwd, "silu", 4)
    _run_backward(130, 2700, 2600, xd, wd, yd, dwd, "none", 5)


def test_large_tiles_ffn(cuda_device):
    from objeta_b200.dense import ffn_bf16_tokens
    for T, H, I, O in ((700, 264, 800, 1000), (1001, 72, 1500, 136)):
        x, r = U.randn((T, H), seed=1), U.randn((T, O), seed=5)
        g, u = U.randn((I, H), torch.bfloat16, 1 / math.sqrt(H), 2), U.randn((I, H), torch.bfloat16, 1 / math.sqrt(H), 3)
        d = U.randn((O, I), torch.bfloat16, 1 / math.sqrt(I), 4)
        U.check(ffn_bf16_tokens(g, u, d, x, d_residual=r), *_ffn_ref(g, u, d, x, r, 0.0), "out")


@pytest.mark.parametrize("T", [1, 5, 40])
def test_expert_parallel_layer_with_a_shared_expert(cuda_device, T):
    """ExpertParallelMoe(shared=...): the routed output plus the shared expert."""
    from objeta_b200.ep import ExpertParallelMoe, router_topk_batched
    from objeta_b200.moe import MoeLayer
    from objeta_b200.quant import QGemvShape, QuantBackend, QuantFormat
    H, I, E, k, Is = 256, 256, 8, 2, 192
    qb = QuantBackend(0)
    pack = lambda r, c, s: qb.quantize_matrix_device(QuantFormat.Q4_0, U.randn((r, c), scale=0.05, seed=s),
                                                     QGemvShape.q4_0(r, c))
    layer = MoeLayer(QuantFormat.Q4_0, H, I, H, [pack(I, H, 3 * e) for e in range(E)],
                     [pack(I, H, 3 * e + 1) for e in range(E)], [pack(H, I, 3 * e + 2) for e in range(E)])
    g, u = U.randn((Is, H), torch.bfloat16, 1 / 16, 91), U.randn((Is, H), torch.bfloat16, 1 / 16, 92)
    d = U.randn((H, Is), torch.bfloat16, 1 / 14, 93)
    x = U.randn((T, H), seed=94)
    ids, w = router_topk_batched(U.randn((T, E), seed=95), k, renormalize=True)
    routed = ExpertParallelMoe(layer, E, k).forward(x, ids, w)
    both = ExpertParallelMoe(layer, E, k, shared=(g, u, d)).forward(x, ids, w)
    U.check(both, *_ffn_ref(g, u, d, x, routed, 0.0))
    with pytest.raises(ValueError):
        ExpertParallelMoe(layer, E, k, shared=(g, u, d.t().contiguous()))
