"""Training a router on frozen experts: load counts, balance and z losses, and
the gradients of the router's logits and of the routing weights.

A step over T tokens, beside ``router_topk_batched`` / ``deepseek_gate``,
``ExpertParallelMoe`` or ``moe_pairs`` and ``moe_combine``::

    logits = linear(x, w_router)                       # dense.py
    ids, w = router_topk_batched(logits, k, renormalize=True)
    bal = balance_loss(logits, ids)
    ... v = moe_pairs(...); out = moe_combine(v, slot_row, w, out) ...
    dw = moe_combine_backward(dout, v, slot_row)
    dlogits = router_backward(logits, ids, dw, renormalize=True, balance=bal,
                              balance_grad=1e-2, z_grad=1e-3)
    _, dw_router, _ = linear_backward(dlogits, x, w_router, need_dx=False)

Results carry no autograd graph; the gradients are these calls' own.

The reference has no training; the scores are those of its router and gate
(crates/objeta-cuda/src/bin/deepseek_single_layer_moe.rs:720-740, 768-881).
"""
from __future__ import annotations

import ctypes
from dataclasses import dataclass

import torch

from . import _lib
from ._launch import matrix, on_device, run
from .ep import SOFTMAX

c_size = ctypes.c_size_t
c_int = ctypes.c_int
c_float = ctypes.c_float
c_void_p = ctypes.c_void_p

_lib.register_signatures({
    "objb_balance_loss_scratch_bytes": (c_int, [c_size, c_size, c_size, ctypes.POINTER(c_size)]),
    "objb_balance_loss_device": (c_int, [c_void_p, c_size, c_void_p, c_void_p, c_void_p, c_size, c_size, c_size,
                                         c_size, c_int, c_void_p, c_void_p, c_void_p, c_void_p, c_void_p, c_size,
                                         c_void_p]),
    "objb_router_backward_device": (c_int, [c_void_p, c_size, c_void_p, c_void_p, c_void_p, c_void_p, c_size,
                                            c_void_p, c_void_p, c_size, c_size, c_size, c_int, c_int, c_float,
                                            c_float, c_float, c_void_p, c_size, c_void_p]),
    "objb_moe_combine_backward_device": (c_int, [c_void_p, c_void_p, c_size, c_void_p, c_size, c_size, c_size,
                                                 c_void_p, c_void_p]),
})


_F32, _I32, _MASK = (torch.float32,), (torch.int32,), (torch.bool, torch.uint8)


@dataclass
class BalanceLoss:
    """What ``balance_loss`` returns; ``router_backward`` takes it back."""
    counts: object       # int32 [S, E]: selections of each expert
    sums: object         # f32 [at + 2 S + 3]: from `at` on balance, z, scales [S + 1], the bits of tokens [S]
    at: int
    score_func: int
    seq_offsets: object
    token_mask: object

    @property
    def balance(self):
        """f32 scalar tensor."""
        return self.sums[self.at]

    @property
    def z(self):
        """f32 scalar tensor."""
        return self.sums[self.at + 1]

    @property
    def scales(self):
        """f32 [S + 1]: the gradients' factors, E / (k n^2 S') and then 2 / N."""
        return self.sums[self.at + 2:self.at + self.counts.shape[0] + 3]

    @property
    def tokens(self):
        """int32 [S]: counted tokens."""
        return self.sums[self.at + self.counts.shape[0] + 3:].view(torch.int32)


def _routing(d_logits, d_ids, d_seq_offsets, d_token_mask):
    T, E, ld = matrix("d_logits", d_logits, None, _F32)
    dev = d_logits.device
    on_device("d_ids", d_ids, dev, _I32)
    size = d_ids.shape
    if len(size) != 2 or size[0] != T:
        raise ValueError(f"d_ids has shape {tuple(size)}, expected ({T}, top_k)")
    mask = off = None
    S = 1
    if d_token_mask is not None:
        on_device("d_token_mask", d_token_mask, dev, _MASK, (T,))
        mask = d_token_mask.data_ptr()
    if d_seq_offsets is not None:
        on_device("d_seq_offsets", d_seq_offsets, dev, _I32)
        S = d_seq_offsets.numel() - 1
        if d_seq_offsets.dim() != 1 or S < 1:
            raise ValueError("d_seq_offsets: expected [num_seqs + 1] offsets")
        off = d_seq_offsets.data_ptr()
    return dev, ld, T, E, size[1], S, mask, off


def balance_loss(d_logits, d_ids, score_func: int = SOFTMAX, d_seq_offsets=None, d_token_mask=None,
                 stream=None) -> BalanceLoss:
    """Per-expert counts and the balance and z losses of a routed batch.

    d_logits f32 [T, E] (rows may be strided), d_ids int32 [T, k] the selected
    experts (entries outside 0..E-1, such as the gate's -1, count nowhere).
    ``d_seq_offsets`` int32 [S + 1], ascending: sequence q holds tokens
    [off[q], off[q+1]); tokens before the first and behind the last belong to
    none.  Without it all tokens are one sequence.  ``d_token_mask`` bool [T]:
    tokens to count.  With p the scores shared out to 1 per token, n_q the
    counted tokens of q, S' the sequences that have any and N all of them:

    * balance = 1/S' sum_q sum_e (E counts[q, e] / (k n_q)) (1/n_q sum_t p[t, e])
    * z = 1/N sum_t logsumexp(l_t)^2

    (both 0 where no token counts).  Masked experts' logits, -inf or the lowest
    f32 beside larger ones (under sqrt-softplus all below about -88.7, where
    the gate's log1p(exp(-l)) overflows), have score 0.  A token whose logits
    are all -inf counts but adds nothing to either loss.  Sums over tokens are
    folded in a fixed order:
    the same call gives the same bits.
    """
    dev, ld, T, E, k, S, mask, off = _routing(d_logits, d_ids, d_seq_offsets, d_token_mask)
    counts, sums, at = run(dev, stream, _balance_loss, d_logits, ld, d_ids, mask, off, S, T, E, k, int(score_func),
                           dev)
    return BalanceLoss(counts, sums, at, int(score_func), d_seq_offsets, d_token_mask)


def _balance_loss(st, d_logits, ld, d_ids, mask, off, S, T, E, k, func, dev):
    n = c_size()
    _lib.call("objb_balance_loss_scratch_bytes", T, E, S, ctypes.byref(n))
    n = n.value
    at = n // 4 if n <= 65536 else 0  # a small scratch is in front of the sums: one allocation less
    counts = torch.empty(S, E, dtype=torch.int32, device=dev)
    sums = torch.empty(at + 2 * S + 3, dtype=torch.float32, device=dev)
    base = sums.data_ptr()
    scratch = base if at else torch.empty(n, dtype=torch.uint8, device=dev)
    base += 4 * at
    _lib.call("objb_balance_loss_device", d_logits.data_ptr(), ld, d_ids.data_ptr(), mask, off, S, T, E, k, func,
              counts.data_ptr(), base + 4 * (S + 3), base, base + 8, scratch if at else scratch.data_ptr(), n, st)
    return counts, sums, at


def router_backward(d_logits, d_ids, d_dweights=None, score_func: int = SOFTMAX, renormalize: bool = False,
                    route_scale: float = 1.0, balance: BalanceLoss | None = None, balance_grad: float = 0.0,
                    z_grad: float = 0.0, d_token_mask=None, d_dlogits=None, stream=None):
    """The gradient of the router's logits, f32 [T, E], in one pass.

    ``d_dweights`` f32 [T, k] (or None): the gradient of the routing weights
    w_j = route_scale * s[ids_j], divided by sum_j s[ids_j] with
    ``renormalize`` (``router_topk_batched``: softmax, scale 1;
    ``deepseek_gate``: its score function and scale, renormalised unless
    softmax).  ``balance``: the ``balance_loss`` result of the same logits and
    ids, whose two losses enter with the factors ``balance_grad`` and
    ``z_grad``; its offsets and mask then say which tokens count (else
    ``d_token_mask``).  Rows of tokens that do not count are zero.
    ``d_dlogits`` may be ``d_logits`` itself.
    """
    d_off = None
    if balance is not None:
        if int(score_func) != balance.score_func:
            raise ValueError(f"score_func {score_func} differs from the balance loss's {balance.score_func}")
        if d_token_mask is not None:
            raise ValueError("the token mask of a call with a balance loss is the balance loss's")
        d_off, d_token_mask = balance.seq_offsets, balance.token_mask
    dev, ld, T, E, k, S, mask, off = _routing(d_logits, d_ids, d_off, d_token_mask)
    counts = scales = dw = None
    if balance is not None:
        on_device("balance.counts", balance.counts, dev, _I32, (S, E))
        counts, scales = balance.counts.data_ptr(), balance.sums.data_ptr() + 4 * balance.at + 8
    if d_dweights is not None:
        on_device("d_dweights", d_dweights, dev, _F32, (T, k))
        dw = d_dweights.data_ptr()
    ldo = E
    if d_dlogits is not None:
        ldo = matrix("d_dlogits", d_dlogits, dev, _F32, (T, E))[2]
    return run(dev, stream, _router_backward, d_logits, ld, d_ids, dw, mask, off, S, counts, scales, T, E, k,
               int(score_func), int(bool(renormalize)), float(route_scale), float(balance_grad), float(z_grad),
               d_dlogits, ldo, dev)


def _router_backward(st, d_logits, ld, d_ids, dw, mask, off, S, counts, scales, T, E, k, func, renorm, scale, bg, zg,
                     d_dlogits, ldo, dev):
    if d_dlogits is None:
        d_dlogits = torch.empty(T, E, dtype=torch.float32, device=dev)
    _lib.call("objb_router_backward_device", d_logits.data_ptr(), ld, d_ids.data_ptr(), dw, mask, off, S, counts,
              scales, T, E, k, func, renorm, scale, bg, zg, d_dlogits.data_ptr(), ldo, st)
    return d_dlogits


def moe_combine_backward(d_dout, d_v, slot_row, d_dw=None, stream=None):
    """The routing weights' gradient of ``moe_combine``: dw[t, j] = sum_o
    d_dout[t, o] * d_v[slot_row[t, j], o], f32 [T, k].  A row outside d_v is
    read as row 0 and flagged (device error word bit 8), as the combine does."""
    dev = on_device("d_dout", d_dout, None, _F32)
    on_device("d_v", d_v, dev, _F32)
    on_device("slot_row", slot_row, dev, _I32)
    if d_v.dim() != 2 or slot_row.dim() != 2:
        raise ValueError("expected d_dout [T, O], d_v [V, O] and slot_row [T, k]")
    T, k = slot_row.shape
    V, O = d_v.shape
    if d_dout.shape != (T, O):
        raise ValueError(f"d_dout has shape {tuple(d_dout.shape)}, expected ({T}, {O})")
    if d_dw is not None:
        on_device("d_dw", d_dw, dev, _F32, (T, k))
    return run(dev, stream, _combine_backward, d_dout, d_v, V, slot_row, T, k, O, d_dw, dev)


def _combine_backward(st, d_dout, d_v, V, slot_row, T, k, O, d_dw, dev):
    if d_dw is None:
        d_dw = torch.empty(T, k, dtype=torch.float32, device=dev)
    _lib.call("objb_moe_combine_backward_device", d_dout.data_ptr(), d_v.data_ptr(), V, slot_row.data_ptr(), T, k, O,
              d_dw.data_ptr(), st)
    return d_dw
