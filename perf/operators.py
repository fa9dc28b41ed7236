"""What the dense and router-training operators are measured on: their cases,
their plain forms and the framework's calls.

Operators (``case["op"]``):

* ``linear``: y = act(x W^T + b) + r, optionally with z = x W^T + b kept;
* ``linear_backward``: dx, dW, db of act(x W^T + b) from dy and the kept z;
* ``ffn``: the bf16 SwiGLU FFN (shared expert) of T tokens, added to the routed
  experts' sum;
* ``router``: per-expert counts, balance and z losses of packed sequences, then
  the gradient of the logits through the routing weights and both losses;
* ``combine_backward``: the routing weights' gradient of the top-k combine.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
ACTS = ("none", "relu", "silu", "gelu", "gelu_tanh")
SCORES = ("softmax", "sigmoid", "sqrt_softplus")
SQRT_2_OVER_PI = math.sqrt(2.0 / math.pi)
# the largest drawn product (2 T K N), below that of the largest listed case
MAX_FLOPS = 4.0e11


def _linear(name, T, K, N, x, w, y, act="none", bias=False, residual=False, z=False):
    c = {"op": "linear", "T": T, "K": K, "N": N, "x": x, "w": w, "y": y, "act": act, "bias": bias,
         "residual": residual, "z": z}
    return dict(c, name=name) if name else c


def _backward(name, T, K, N, x, w, y, act="none", dw="w", bias=True):
    c = {"op": "linear_backward", "T": T, "K": K, "N": N, "x": x, "w": w, "y": y, "act": act, "dw": dw, "bias": bias}
    return dict(c, name=name) if name else c


def _ffn(name, T, H, I, limit=0.0):
    c = {"op": "ffn", "T": T, "H": H, "I": I, "limit": limit}
    return dict(c, name=name) if name else c


def _router(name, T, E, k, S, score, renorm, masked):
    c = {"op": "router", "T": T, "E": E, "k": k, "S": S, "score": score, "renorm": renorm, "masked": masked}
    return dict(c, name=name) if name else c


def _combine(name, T, k, O):
    c = {"op": "combine_backward", "T": T, "k": k, "O": O}
    return dict(c, name=name) if name else c


def listed():
    return [
        # one decoded token through a projection with a skip connection: latency
        _linear("projection_1_token", 1, 4096, 4096, "bf16", "bf16", "bf16", bias=True, residual=True),
        # a ragged decode batch through the vocabulary head, f32 logits: the weight's bytes
        _linear("vocabulary_37_tokens", 37, 2048, 151936, "bf16", "bf16", "f32"),
        # routing logits of a decode batch at an expert-parallel layer, f32 throughout
        _linear("router_logits_250", 250, 2048, 256, "f32", "f32", "f32", bias=True),
        # a training or prompt pass through a wide hidden layer: the matrix units
        _linear("hidden_4096_tokens", 4096, 4096, 14336, "bf16", "bf16", "bf16", act="silu", bias=True, z=True),
        # the router projection's gradients over a training batch, f32
        _backward("router_backward_4000", 4000, 2048, 256, "f32", "f32", "f32"),
        # a dense layer's gradients over a training batch, fp16
        _backward("hidden_backward_2048", 2048, 4096, 4096, "f16", "f16", "f16", act="gelu_tanh"),
        # the shared expert of a decode batch, added to the routed experts' sum
        _ffn("shared_expert_16", 16, 4096, 2048),
        # the shared expert of a prompt
        _ffn("shared_expert_1000", 1000, 4096, 2048, limit=10.0),
        # a small router's step: latency
        _router("router_8_experts", 64, 8, 2, 1, "softmax", True, False),
        # a training batch of packed, padded sequences over a wide router
        _router("router_256_packed", 32768, 256, 8, 23, "sigmoid", True, True),
        # routing weights' gradients of a few tokens
        _combine("combine_16_tokens", 16, 2, 4096),
        # and of a training batch
        _combine("combine_4096_tokens", 4096, 8, 2048),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of lo..hi: whole multiples of 64 and 8 mostly, odd ones among them."""
    n = _log(rng, lo, hi)
    step = rng.choice((64, 64, 8, 1))
    return max(lo, n // step * step)


def draw(rng):
    op = rng.choice(("linear", "linear", "linear_backward", "linear_backward", "ffn", "router", "router",
                     "combine_backward"))
    if op in ("linear", "linear_backward"):
        while True:
            T, K, N = _log(rng, 1, 8192), _size(rng, 64, 8192), _size(rng, 8, 16384)
            if 2.0 * T * K * N * (2 if op == "linear_backward" else 1) <= MAX_FLOPS / 2:
                break
        x, w = rng.choice((("bf16", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("f32", "bf16"), ("f32", "f32")))
        act = rng.choice(ACTS)
        if op == "linear":
            y = "f32" if x == "f32" else rng.choice((x, x, "f32"))
            return _linear(None, T, K, N, x, w, y, act, rng.random() < 0.5, rng.random() < 0.5, rng.random() < 0.3)
        return _backward(None, T, K, N, x, w, x, act, "w" if w == x else "f32", rng.random() < 0.7)
    if op == "ffn":
        return _ffn(None, _log(rng, 1, 2048), 64 * rng.randint(4, 72), 64 * rng.randint(4, 40),
                    rng.choice((0.0, 0.0, 10.0, 1.5)))
    if op == "router":
        E = rng.choice((rng.randint(4, 64), rng.randint(64, 512), 64, 128, 256))
        T = _log(rng, 1, 32768)
        return _router(None, T, E, rng.randint(1, min(8, E)), min(T, rng.choice((1, 1, rng.randint(2, 40)))),
                       rng.choice(SCORES), rng.random() < 0.6, rng.random() < 0.5)
    return _combine(None, _log(rng, 1, 4096), rng.randint(1, 8), _size(rng, 64, 4096))


# ------------------------------------------------------------------ inputs
def _randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32) * scale).to(dtype)


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    op = case["op"]
    s = {"case": case}
    if op in ("linear", "linear_backward"):
        T, K, N = case["T"], case["K"], case["N"]
        xt, wt, yt = DTYPES[case["x"]], DTYPES[case["w"]], DTYPES[case["y"]]
        s["x"] = _randn(g, T, K, dtype=xt)
        s["w"] = _randn(g, N, K, dtype=wt, scale=1.0 / math.sqrt(K))
        if op == "linear":
            s["bias"] = _randn(g, N, dtype=wt, scale=0.1) if case["bias"] else None
            s["residual"] = _randn(g, T, N, dtype=yt) if case["residual"] else None
        else:
            # the incoming gradient, and the z that the forward pass kept (none without an activation)
            s["dy"] = _randn(g, T, N, dtype=yt)
            s["z"] = _randn(g, T, N, dtype=yt) if case["act"] != "none" else None
    elif op == "ffn":
        T, H, I = case["T"], case["H"], case["I"]
        s["x"] = _randn(g, T, H)
        s["gate"] = _randn(g, I, H, dtype=torch.bfloat16, scale=0.02)
        s["up"] = _randn(g, I, H, dtype=torch.bfloat16, scale=0.02)
        s["down"] = _randn(g, H, I, dtype=torch.bfloat16, scale=0.02)
        s["routed"] = _randn(g, T, H)
    elif op == "router":
        T, E, k, S = case["T"], case["E"], case["k"], case["S"]
        popular = _randn(g, E)  # some experts are wanted more than others
        s["logits"] = _randn(g, T, E, scale=1.5) + popular
        s["ids"] = torch.topk(s["logits"], k, dim=1).indices.to(torch.int32)
        s["dw"] = _randn(g, T, k)
        # S sequences of different lengths, one of them empty where there are several, and rows behind the last
        cuts = torch.sort(torch.randint(0, T + 1, (S,), generator=g, device="cuda"))[0].to(torch.int32)
        first = torch.zeros(1, dtype=torch.int32, device="cuda")
        s["offsets"] = torch.cat((first, cuts)) if S > 1 else None
        if S > 2:
            s["offsets"][2] = s["offsets"][1]
        s["mask"] = torch.rand(T, generator=g, device="cuda") < 0.9 if case["masked"] else None
    else:
        T, k, O = case["T"], case["k"], case["O"]
        s["dout"] = _randn(g, T, O)
        s["v"] = _randn(g, T * k, O)
        s["slot_row"] = torch.randperm(T * k, generator=g, device="cuda").to(torch.int32).view(T, k)
    return s


# ------------------------------------------------------------- plain forms
def _act(z, act):
    if act == "relu":
        return torch.clamp(z, min=0.0)
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z / math.sqrt(2.0)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(SQRT_2_OVER_PI * (z + 0.044715 * z * z * z)))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-z))
        return sg * (1.0 + z * (1.0 - sg))
    if act == "gelu":
        return 0.5 * (1.0 + torch.erf(z / math.sqrt(2.0))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi)
    if act == "gelu_tanh":
        t = torch.tanh(SQRT_2_OVER_PI * (z + 0.044715 * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * SQRT_2_OVER_PI * (1.0 + 3 * 0.044715 * z * z)
    return torch.ones_like(z)


def _plain_linear(s):
    c = s["case"]
    yt = DTYPES[c["y"]]
    z = s["x"].float() @ s["w"].float().t()
    if s["bias"] is not None:
        z = z + s["bias"].float()
    y = _act(z, c["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return {"y": y.to(yt), "z": z.to(yt)} if c["z"] else {"y": y.to(yt)}


def _plain_linear_backward(s):
    c = s["case"]
    x, w = s["x"].float(), s["w"].float()
    dz = s["dy"].float()
    if s["z"] is not None:
        dz = dz * _act_grad(s["z"].float(), c["act"])
    out = {"dx": (dz @ w).to(s["x"].dtype),
           "dw": (dz.t() @ x).to(torch.float32 if c["dw"] == "f32" else s["w"].dtype)}
    if c["bias"]:
        out["db"] = dz.sum(0)
    return out


def _plain_ffn(s):
    limit = s["case"]["limit"]
    g = s["x"] @ s["gate"].float().t()
    u = s["x"] @ s["up"].float().t()
    if limit > 0:
        g = torch.clamp(g, max=limit)
        u = torch.clamp(u, min=-limit, max=limit)
    a = g / (1.0 + torch.exp(-g)) * u
    return {"out": s["routed"] + a @ s["down"].float().t()}


def _plain_router(s):
    """In 64 bits: a mean over all tokens, whose differences from each token's
    own value the gradient consists of."""
    c = s["case"]
    T, E, k, S = c["T"], c["E"], c["k"], c["S"]
    l = s["logits"].double()
    ids = s["ids"].long()
    t = torch.arange(T, device=l.device)
    if s["offsets"] is None:
        seq = torch.zeros(T, dtype=torch.long, device=l.device)
    else:
        seq = torch.searchsorted(s["offsets"].long(), t, right=True) - 1  # S: behind the last sequence
    valid = seq < S
    if s["mask"] is not None:
        valid = valid & s["mask"]
    seq = torch.where(valid, seq, torch.full_like(seq, S))
    member = (seq[:, None] == torch.arange(S, device=l.device)).double()  # [T, S]
    top = l.max(1, keepdim=True).values
    ex = torch.exp(l - top)
    lse = torch.log(ex.sum(1)) + top[:, 0]
    soft = ex / ex.sum(1, keepdim=True)
    if c["score"] == "softmax":
        sc, dsc = soft, None
    elif c["score"] == "sigmoid":
        sc = 1.0 / (1.0 + torch.exp(-l))
        dsc = sc * (1.0 - sc)
    else:
        sp = torch.where(l > 20.0, l, torch.log1p(torch.exp(torch.clamp(l, max=20.0))))
        sc = torch.sqrt(sp)
        dsc = torch.where(l > 20.0, torch.ones_like(l), 1.0 / (1.0 + torch.exp(-l))) / (2.0 * sc)
    total = sc.sum(1, keepdim=True)
    p = sc / total
    hot = torch.zeros(T, E, dtype=torch.double, device=l.device)
    hot.scatter_add_(1, ids, torch.ones_like(ids, dtype=torch.double))
    counts = member.t() @ hot  # [S, E]
    n = member.sum(0)
    some = (n > 0).sum()
    n1 = torch.clamp(n, min=1.0)[:, None]
    f = counts * E / (k * n1)
    P = (member.t() @ p) / n1
    balance = (f * P).sum() / torch.clamp(some, min=1)
    N = torch.clamp(n.sum(), min=1.0)
    z = (lse * lse * valid).sum() / N
    # gradients
    q = torch.gather(sc, 1, ids)
    gq = s["dw"].double()
    if c["renorm"]:
        Q = q.sum(1, keepdim=True)
        gq = (gq - (gq * q).sum(1, keepdim=True) / Q) / Q
    gp = 0.01 * (member @ (f / n1)) / torch.clamp(some, min=1)
    gs = torch.zeros_like(sc).scatter_add_(1, ids, gq)
    if dsc is None:
        gs = gs + gp
        dl = sc * (gs - (gs * sc).sum(1, keepdim=True))
    else:
        gs = gs + (gp - (gp * p).sum(1, keepdim=True)) / total
        dl = gs * dsc
    dl = dl + 0.001 * 2.0 * lse[:, None] * soft / N
    dl = torch.where(valid[:, None], dl, torch.zeros_like(dl))
    return {"counts": counts.to(torch.int32), "balance": balance.float(), "z": z.float(), "dlogits": dl.float()}


def _plain_combine(s):
    return {"dw": (s["dout"][:, None, :] * s["v"][s["slot_row"].long()]).sum(-1)}


PLAIN = {"linear": _plain_linear, "linear_backward": _plain_linear_backward, "ffn": _plain_ffn,
         "router": _plain_router, "combine_backward": _plain_combine}


# ------------------------------------------------------ the framework's calls
def _own(s):
    from objeta_b200 import dense, router
    c = s["case"]
    op = c["op"]
    if op == "linear":
        z = torch.empty(c["T"], c["N"], dtype=DTYPES[c["y"]], device="cuda") if c["z"] else None
        y = dense.linear(s["x"], s["w"], s["bias"], activation=c["act"], d_residual=s["residual"],
                         out_dtype=DTYPES[c["y"]], d_z=z)
        return {"y": y, "z": z} if c["z"] else {"y": y}
    if op == "linear_backward":
        dx, dw, db = dense.linear_backward(s["dy"], s["x"], s["w"], s["z"], activation=c["act"],
                                           need_dbias=c["bias"],
                                           dw_dtype=torch.float32 if c["dw"] == "f32" else s["w"].dtype)
        return {"dx": dx, "dw": dw, "db": db} if c["bias"] else {"dx": dx, "dw": dw}
    if op == "ffn":
        return {"out": dense.ffn_bf16_tokens(s["gate"], s["up"], s["down"], s["x"], d_residual=s["routed"],
                                             swiglu_limit=c["limit"])}
    if op == "router":
        b = router.balance_loss(s["logits"], s["ids"], score_func=SCORES.index(c["score"]),
                                d_seq_offsets=s["offsets"], d_token_mask=s["mask"])
        dl = router.router_backward(s["logits"], s["ids"], s["dw"], score_func=SCORES.index(c["score"]),
                                    renormalize=c["renorm"], balance=b, balance_grad=0.01, z_grad=0.001)
        return {"counts": b.counts, "balance": b.balance, "z": b.z, "dlogits": dl}
    return {"dw": router.moe_combine_backward(s["dout"], s["v"], s["slot_row"])}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    size = {"f32": 4, "bf16": 2, "f16": 2}
    if op == "linear":
        T, K, N = case["T"], case["K"], case["N"]
        y = T * N * size[case["y"]]
        return {"bytes": T * K * size[case["x"]] + N * K * size[case["w"]] + y * (1 + case["z"] + case["residual"])
                + (N * size[case["w"]] if case["bias"] else 0), "flops": 2.0 * T * K * N}
    if op == "linear_backward":
        T, K, N = case["T"], case["K"], case["N"]
        wb = size[case["w"]]
        return {"bytes": T * N * size[case["y"]] * (1 + (case["act"] != "none")) + 2 * T * K * size[case["x"]]
                + N * K * (wb + (4 if case["dw"] == "f32" else wb)) + (4 * N if case["bias"] else 0),
                "flops": 4.0 * T * K * N}
    if op == "ffn":
        T, H, I = case["T"], case["H"], case["I"]
        return {"bytes": 3 * H * I * 2 + 3 * T * H * 4, "flops": 6.0 * T * H * I}
    if op == "router":
        T, E, k, S = case["T"], case["E"], case["k"], case["S"]
        return {"bytes": 8 * T * E + 8 * T * k + 4 * S * E + (4 * S + 4 if S > 1 else 0) + (T if case["masked"] else 0),
                "flops": 20.0 * T * E}
    T, k, O = case["T"], case["k"], case["O"]
    return {"bytes": 4 * (T * k * O + T * O + 2 * T * k), "flops": 2.0 * T * k * O}


# --------------------------------------------------------- 64-bit references
def _exact_act(z, act):
    F = torch.nn.functional
    return {"none": lambda v: v * 1.0, "relu": F.relu, "silu": F.silu, "gelu": F.gelu,
            "gelu_tanh": lambda v: F.gelu(v, approximate="tanh")}[act](z)


def _exact_scores(l, score):
    if score == "softmax":
        return torch.softmax(l, 1)
    if score == "sigmoid":
        return torch.sigmoid(l)
    return torch.sqrt(torch.nn.functional.softplus(l, threshold=20.0))


def exact(case, seed):
    """From the definitions in 64 bits; the gradients by differentiating them."""
    s = prepare(case, seed)
    op = case["op"]
    d = {k: v.double() if isinstance(v, torch.Tensor) and v.is_floating_point() else v for k, v in s.items()}
    if op == "linear":
        z = torch.nn.functional.linear(d["x"], d["w"], d["bias"])
        y = _exact_act(z, case["act"])
        y = y if d["residual"] is None else y + d["residual"]
        return {"y": y, "z": z} if case["z"] else {"y": y}
    if op == "linear_backward":
        dz = d["dy"]
        if d["z"] is not None:
            z = d["z"].requires_grad_()
            dz = torch.autograd.grad(_exact_act(z, case["act"]), z, d["dy"])[0]
        out = {"dx": torch.einsum("tn,nk->tk", dz, d["w"]), "dw": torch.einsum("tn,tk->nk", dz, d["x"])}
        if case["bias"]:
            out["db"] = torch.einsum("tn->n", dz)
        return out
    if op == "ffn":
        L = torch.nn.functional.linear
        g, u = L(d["x"], d["gate"]), L(d["x"], d["up"])
        if case["limit"] > 0:
            g, u = torch.minimum(g, torch.full_like(g, case["limit"])), u.clip(-case["limit"], case["limit"])
        return {"out": d["routed"] + L(torch.nn.functional.silu(g) * u, d["down"])}
    if op == "router":
        T, E, k, S = case["T"], case["E"], case["k"], case["S"]
        l = d["logits"].requires_grad_()
        off = [0, T] if s["offsets"] is None else s["offsets"].tolist()
        keep = torch.ones(T, dtype=torch.bool, device=l.device) if s["mask"] is None else s["mask"]
        sc = _exact_scores(l, case["score"])
        p = sc / sc.sum(1, keepdim=True)
        counts = torch.zeros(S, E, dtype=torch.int32, device=l.device)
        terms, rows = [], []
        for i in range(S):
            r = torch.arange(off[i], off[i + 1], device=l.device)
            r = r[keep[r]]
            if r.numel():
                counts[i] = torch.bincount(s["ids"][r].reshape(-1).long(), minlength=E).to(torch.int32)
                terms.append((p[r].mean(0) * counts[i].double() * E / (k * r.numel())).sum())
                rows.append(r)
        if not rows:
            zero = torch.zeros((), dtype=torch.double, device=l.device)
            return {"counts": counts, "balance": zero, "z": zero, "dlogits": torch.zeros_like(l.detach())}
        balance = torch.stack(terms).mean()
        r = torch.cat(rows)
        z = torch.logsumexp(l[r], 1).square().mean()
        w = torch.gather(sc, 1, s["ids"].long())[r]
        if case["renorm"]:
            w = w / w.sum(1, keepdim=True)
        dl = torch.autograd.grad((w * d["dw"][r]).sum() + 0.01 * balance + 0.001 * z, l)[0]
        return {"counts": counts, "balance": balance.detach(), "z": z.detach(), "dlogits": dl}
    return {"dw": torch.einsum("to,tko->tk", d["dout"], d["v"][s["slot_row"].long()])}
