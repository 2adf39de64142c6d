"""Log-probabilities of given tokens, row entropies and the best alternatives, with their gradient.

``token_logprobs`` starts from logits; ``linear_logprobs`` from hidden states and the output weight, in row chunks, so that
neither the logits nor their gradient exist as a whole.  The reference project has no counterpart.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from maester_b200.ops import reference as ref
from maester_b200.ops.functional import _C, _acc_or_return, use_native

MAX_TOP = 64                        # alternatives of one row
CHUNK_BYTES = 1 << 30               # fp32 logits that ``linear_logprobs`` holds at a time
_NATIVE = (torch.bfloat16, torch.float16, torch.float32)


class TokenLogprobs(NamedTuple):
    logprobs: torch.Tensor | None       # fp32 [...]: log p(token); 0 where the token is -100
    entropy: torch.Tensor | None        # fp32 [...]: -sum p log p
    top_logprobs: torch.Tensor | None   # fp32 [..., top]: the best alternatives, best first
    top_tokens: torch.Tensor | None     # int64 [..., top]: their ids; equal logits in the order of their ids


def _check(tokens, lead, device, V, scale, entropy, top) -> None:
    if not (isinstance(scale, (int, float)) and 1e-8 <= scale <= 1e8):   # (logits up to 1e30 times it are fp32 numbers)
        raise ValueError(f"the logit scale has to be a number in [1e-8, 1e8], got {scale!r}")
    if not (isinstance(top, int) and 0 <= top <= min(MAX_TOP, V)):
        raise ValueError(f"top has to be a whole number in [0, {min(MAX_TOP, V)}], got {top!r}")
    if tokens is None:
        if not (entropy or top):
            raise ValueError("nothing to compute: give tokens, or ask for the entropy or for alternatives")
        return
    if tokens.dtype not in (torch.int64, torch.int32):
        raise TypeError(f"tokens have to be int64 or int32, got {tokens.dtype}")
    if tokens.shape != lead:
        raise ValueError(f"tokens {tuple(tokens.shape)} do not fit rows of shape {tuple(lead)}")
    if tokens.device != device:
        raise ValueError(f"tokens are on {tokens.device}, the rows on {device}")


def _dense_f32(g: torch.Tensor | None) -> torch.Tensor | None:
    return g if g is None or (g.dtype is torch.float32 and g.is_contiguous()) else g.to(torch.float32).contiguous()


class _TokenLogprobs(Function):
    @staticmethod
    def forward(ctx, x, tokens, scale, entropy, top):
        lp, ent, top_lp, top_id, stats = _C().logprobs_fwd(x, tokens, scale, entropy, top, True)
        ctx.save_for_backward(x, tokens, stats, top_id)
        ctx.scale = scale
        if top_id is not None:
            ctx.mark_non_differentiable(top_id)
        ctx.set_materialize_grads(False)
        return lp, ent, top_lp, top_id

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, g_top, _):
        x, tokens, stats, top_id = ctx.saved_tensors
        if g_lp is None and g_ent is None and g_top is None:
            return None, None, None, None, None
        g = [_dense_f32(t) for t in (g_lp, g_ent, g_top)]
        return _C().logprobs_bwd(x, tokens, ctx.scale, stats, g[0], g[1], top_id, g[2]), None, None, None, None


def _shaped(out, lead, top) -> TokenLogprobs:
    if len(lead) == 1:
        return TokenLogprobs(*out)
    return TokenLogprobs(*(None if t is None else t.view((*lead, *((top,) if i >= 2 else ()))) for i, t in enumerate(out)))


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, scale: float = 1.0, entropy: bool = False,
                   top: int = 0) -> TokenLogprobs:
    """Per row of ``scale * logits`` [..., V]: the log-probability of ``tokens`` [...], the entropy, and the ``top`` best
    tokens with their log-probabilities; what was not asked for is None.

    All results are fp32 whatever the type of the logits (bf16, fp16, fp32; rows may have any pitch).  A row whose token is
    -100 is skipped: log-probability and entropy 0, alternatives -inf with id -1, no gradient.  A -inf logit (or one whose
    distance from the row's maximum is beyond fp32) has probability 0; a row without a finite logit, or with NaN or +inf, has
    no distribution: its numbers are NaN, its alternatives are still in order (NaN above +inf).  A token id outside [0, V)
    gives NaN and a device status error (``ops.cuda.check_status``); on the CPU it raises.  ``scale`` is a number in
    [1e-8, 1e8].  Gradients flow to the logits from log-probabilities, entropies and the alternatives' log-probabilities.
    The first call on a device has to run outside a stream capture."""
    if logits.dim() < 1 or not logits.is_floating_point():
        raise TypeError("logits have to be a floating-point tensor with a vocabulary dimension")
    V, lead = logits.shape[-1], logits.shape[:-1]
    if V == 0:
        raise ValueError("the vocabulary is empty")
    _check(tokens, lead, logits.device, V, scale, entropy, top)
    x = logits if logits.dim() == 2 else logits.reshape(math.prod(lead), V)
    t = None
    if tokens is not None:
        t = tokens if len(lead) == 1 else tokens.reshape(-1)
        if t.dtype != torch.int64:
            t = t.to(torch.int64)
        if not t.is_contiguous():
            t = t.contiguous()
    if not (x.is_cuda and x.dtype in _NATIVE):
        return _shaped(ref.token_logprobs(x, t, scale, entropy, top), lead, top)
    if x.stride(1) != 1 and V > 1:
        x = x.contiguous()
    if torch.is_grad_enabled() and x.requires_grad:
        out = _TokenLogprobs.apply(x, t, scale, entropy, top)
    else:
        out = _C().logprobs_fwd(x, t, scale, entropy, top, False)[:4]
    return _shaped(out, lead, top)


class _LinearLogprobs(Function):
    """Forward: a chunk of fp32 logits at a time, reduced to a few numbers per row.  Backward: the chunk's logits again
    (the same product gives the same bits), their gradient in bf16, and the two products that consume it."""

    @staticmethod
    def forward(ctx, h, w, tokens, scale, entropy, top):
        C = _C()
        need = ctx.needs_input_grad[0] or ctx.needs_input_grad[1]
        parts = []
        for r0, r1 in _chunks(h.shape[0], w.shape[0]):
            logits = C.gemm(h[r0:r1], w, epi=C.EPI_F32)
            parts.append(C.logprobs_fwd(logits, None if tokens is None else tokens[r0:r1], scale, entropy, top, need))
        lp, ent, top_lp, top_id, stats = (None if c[0] is None else c[0] if len(c) == 1 else torch.cat(c)
                                          for c in zip(*parts))
        ctx.save_for_backward(h, w, tokens, stats, top_id)
        ctx.scale = scale
        if top_id is not None:
            ctx.mark_non_differentiable(top_id)
        ctx.set_materialize_grads(False)
        return lp, ent, top_lp, top_id

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, g_top, _):
        C = _C()
        h, w, tokens, stats, top_id = ctx.saved_tensors
        if g_lp is None and g_ent is None and g_top is None:
            return (None,) * 6
        M, D = h.shape
        V = w.shape[0]
        g = [_dense_f32(t) for t in (g_lp, g_ent, g_top)]
        # a row of dh is one product (fp32 sum over the whole vocabulary, rounded once, the same bits every time); dw adds
        # the chunks up in fp32
        dh = torch.empty(M, D, device=h.device, dtype=h.dtype) if ctx.needs_input_grad[0] else None
        dw = None
        chunks = _chunks(M, V)
        dl_buf = torch.empty(max(r1 - r0 for r0, r1 in chunks), (V + 7) // 8 * 8, device=h.device, dtype=torch.bfloat16)

        def products(buf, _acc):
            for r0, r1 in chunks:
                at = lambda t: None if t is None else t[r0:r1]
                logits = C.gemm(h[r0:r1], w, epi=C.EPI_F32)
                dl = C.logprobs_bwd(logits, at(tokens), ctx.scale, stats[r0:r1], at(g[0]), at(g[1]), at(top_id), at(g[2]),
                                    out=dl_buf[:r1 - r0, :V])
                del logits
                if dh is not None:
                    C.gemm(dl, w, b_mn=True, out=dh[r0:r1])
                if buf is not None:
                    C.gemm(dl, h[r0:r1], a_mn=True, b_mn=True, out=buf, epi=C.EPI_F32_ACC)

        if ctx.needs_input_grad[1]:
            dw = _acc_or_return(w, products)
        else:
            products(None, True)
        return dh, dw, None, None, None, None


class _PlainLinearLogprobs(Function):
    """The same off the native products' path (other types than bf16, odd widths, the CPU): logits are a plain product in 32
    bits (64 where either operand has them), a chunk of rows at a time, formed again in the backward pass."""

    @staticmethod
    def forward(ctx, h, w, tokens, scale, entropy, top):
        ctx.wide = torch.float64 if torch.float64 in (h.dtype, w.dtype) else torch.float32
        ctx.args = scale, entropy, top
        ctx.save_for_backward(h, w, tokens)
        wt = w.to(ctx.wide).T
        parts = []
        for r0, r1 in _chunks(h.shape[0], w.shape[0]):
            t = None if tokens is None else tokens[r0:r1]
            parts.append(_of_logits(_product(h[r0:r1].to(ctx.wide), wt), t, scale, entropy, top))
        out = tuple(None if c[0] is None else c[0] if len(c) == 1 else torch.cat(c) for c in zip(*parts))
        if out[3] is not None:
            ctx.mark_non_differentiable(out[3])
        ctx.set_materialize_grads(False)
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, *grads):
        h, w, tokens = ctx.saved_tensors
        grads = grads[:3]
        if all(g is None for g in grads):
            return (None,) * 6
        ww = w.to(ctx.wide)
        dh = torch.empty(h.shape, device=h.device, dtype=h.dtype) if ctx.needs_input_grad[0] else None
        mg = getattr(w, "main_grad", None)
        dw = None
        if ctx.needs_input_grad[1]:
            dw = mg if mg is not None else torch.zeros(w.shape, device=w.device, dtype=ctx.wide)
        for r0, r1 in _chunks(h.shape[0], w.shape[0]):
            hh = h[r0:r1].to(ctx.wide)
            logits = _product(hh, ww.T).detach().requires_grad_(True)
            with torch.enable_grad():
                out = _of_logits(logits, None if tokens is None else tokens[r0:r1], *ctx.args)
            some = [(o, g[r0:r1]) for o, g in zip(out[:3], grads) if g is not None]
            dl, = torch.autograd.grad([o for o, _ in some], [logits], [g for _, g in some])
            if dh is not None:
                dh[r0:r1] = _product(dl, ww)
            if dw is not None:
                dw.add_(_product(dl.T, hh))
        return dh, None if dw is None or mg is not None else dw.to(w.dtype), None, None, None, None


def _product(a: torch.Tensor, b: torch.Tensor) -> torch.Tensor:
    with torch.autocast(a.device.type, enabled=False):      # (in the operands' own type)
        return a @ b


def _of_logits(logits, tokens, scale, entropy, top):
    """(log-probabilities, entropies, alternatives', their ids) of a matrix of logits, by kernel where there is one."""
    if logits.is_cuda and logits.dtype in _NATIVE:
        return tuple(token_logprobs(logits, tokens, scale=scale, entropy=entropy, top=top))
    return ref.token_logprobs(logits, tokens, scale, entropy, top)


def _chunks(rows: int, V: int) -> list[tuple[int, int]]:
    step = max(128, CHUNK_BYTES // (4 * V) // 128 * 128)
    return [(r0, min(rows, r0 + step)) for r0 in range(0, rows, step)] or [(0, 0)]


def linear_logprobs(h: torch.Tensor, w: torch.Tensor, tokens: torch.Tensor | None = None, *, logit_scale: float = 1.0,
                    entropy: bool = False, top: int = 0) -> TokenLogprobs:
    """``token_logprobs`` of the logits ``h @ w.T * logit_scale`` for hidden states ``h`` [..., D] and an output weight
    ``w`` [V, D], with gradients to both (into ``w.main_grad`` where there is one).  Logits are fp32 and live one chunk of
    rows at a time, whatever the types of ``h`` and ``w``; bf16 with a width that 8 divides runs in the framework's own
    products, the rest in plain ones (and 64-bit operands in 64 bits)."""
    if not (h.is_floating_point() and w.is_floating_point()):
        raise TypeError(f"hidden states and weight have to be floating-point tensors, got {h.dtype} and {w.dtype}")
    if h.dim() < 1 or w.dim() != 2 or h.shape[-1] != w.shape[1]:
        raise ValueError(f"hidden states {tuple(h.shape)} do not fit the weight {tuple(w.shape)}")
    if w.device != h.device:
        raise ValueError(f"the weight is on {w.device}, the hidden states on {h.device}")
    V, lead = w.shape[0], h.shape[:-1]
    if V == 0:
        raise ValueError("the vocabulary is empty")
    _check(tokens, lead, h.device, V, logit_scale, entropy, top)
    rows = math.prod(lead)
    h2 = h.reshape(rows, h.shape[-1])
    t = None if tokens is None else tokens.reshape(-1).to(torch.int64).contiguous()
    if use_native(h2, w) and w.dtype == torch.bfloat16 and h2.shape[1] % 8 == 0 and rows > 0:
        h2, w2 = h2.contiguous(), w if w.is_contiguous() else w.contiguous()
        with _C().on_device(h2):
            out = _LinearLogprobs.apply(h2, w2, t, logit_scale, entropy, top)
    else:
        out = _PlainLinearLogprobs.apply(h2, w, t, logit_scale, entropy, top)
    return _shaped(out, lead, top)
