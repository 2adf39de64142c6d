"""Plain-PyTorch definitions of every hot op: the CPU execution path and the numerics oracle.

Every function here is differentiable through ordinary autograd and computes in fp32 internally.
The CUDA kernels in ``maester_b200/csrc`` are tested against these.  Semantics follow the
reference models: Gemma RMSNorm ``x̂·(1+w)`` in fp32 (maester/models/gemma/model.py:155-175),
half-split and interleaved RoPE (gemma/model.py:97-106, llama/model.py:133-168), inclusive sliding
window ``0 <= q-kv <= W`` AND same-document (gemma/model.py:203-256), tanh-GELU GeGLU
(gemma/model.py:189-195), SwiGLU (llama/model.py:308-309), mean cross-entropy with
``ignore_index=-100``.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F

IGNORE_INDEX = -100


def rmsnorm(x: torch.Tensor, w: torch.Tensor | None, eps: float, unit_offset: bool = False,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """``residual + x * rsqrt(mean(x², -1) + eps) * (w or 1+w)``; fp32 math, result in x.dtype."""
    xf = x.float()
    y = xf * torch.rsqrt(xf.pow(2).mean(-1, keepdim=True) + eps)
    if w is not None:
        y = y * ((1.0 + w.float()) if unit_offset else w.float())
    y = y.to(x.dtype)
    if residual is not None:
        y = residual + y
    return y


def layernorm(x, w, b, eps):
    return F.layer_norm(x.float(), (x.shape[-1],), None if w is None else w.float(),
                        None if b is None else b.float(), eps).to(x.dtype)


def rope_inv_freq(rot_dim: int, theta: float, scaling_factor: float = 1.0, device=None) -> torch.Tensor:
    """``theta^(-2i/rot_dim) / scaling_factor`` for i in [0, rot_dim/2), fp32."""
    idx = torch.arange(0, rot_dim, 2, device=device)[: rot_dim // 2].float()
    return (1.0 / (theta ** (idx / rot_dim))) / scaling_factor


def apply_rope(x: torch.Tensor, pos: torch.Tensor, inv_freq: torch.Tensor, layout: str,
               attn_factor: float = 1.0) -> torch.Tensor:
    """Rotate the first ``2*len(inv_freq)`` channels of every head.

    x: [B, S, H, hd]; pos: [B, S] integer positions; layout "half" pairs channel i with i+rot/2,
    "interleaved" pairs 2i with 2i+1.  Channels beyond the rotary width pass through.
    """
    rot = inv_freq.numel() * 2
    ang = pos.to(torch.float32)[..., None] * inv_freq.to(torch.float32)  # [B,S,rot/2]
    cos = (ang.cos() * attn_factor)[:, :, None, :]
    sin = (ang.sin() * attn_factor)[:, :, None, :]
    xr = x[..., :rot].float()
    if layout == "half":
        a, b = xr[..., : rot // 2], xr[..., rot // 2:]
        out = torch.cat([a * cos - b * sin, a * sin + b * cos], dim=-1)
    elif layout == "interleaved":
        a, b = xr[..., 0::2], xr[..., 1::2]
        out = torch.stack([a * cos - b * sin, a * sin + b * cos], dim=-1).flatten(-2)
    else:
        raise ValueError(f"unknown rope layout {layout}")
    out = out.to(x.dtype)
    if rot < x.shape[-1]:
        out = torch.cat([out, x[..., rot:]], dim=-1)
    return out


def qk_norm_rope(q, k, q_w, k_w, pos, inv_freq, layout, eps, unit_offset):
    """Optional per-head RMSNorm of q and k (weights of size head_dim) followed by RoPE."""
    if q_w is not None:
        q = rmsnorm(q, q_w, eps, unit_offset)
    if k_w is not None:
        k = rmsnorm(k, k_w, eps, unit_offset)
    if inv_freq is not None:
        q = apply_rope(q, pos, inv_freq, layout)
        k = apply_rope(k, pos, inv_freq, layout)
    return q, k


def attention_mask(seq_q: int, seq_kv: int, causal: bool, window: int | None,
                   doc_ids: torch.Tensor | None, device=None, q_offset: int = 0) -> torch.Tensor:
    """Dense boolean mask [B or 1, 1, Sq, Skv]; True = attend."""
    q = torch.arange(seq_q, device=device)[:, None] + q_offset
    kv = torch.arange(seq_kv, device=device)[None, :]
    m = torch.ones(seq_q, seq_kv, dtype=torch.bool, device=device)
    if causal:
        m = m & (q >= kv)
    if window is not None and window > 0:
        m = m & (q - kv <= window)
    m = m[None, None]
    if doc_ids is not None:
        d = doc_ids.to(device)
        same = d[:, q_offset:q_offset + seq_q, None] == d[:, None, :seq_kv]
        m = m & same[:, None]
    return m


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, causal: bool = True,
              window: int | None = None, doc_ids: torch.Tensor | None = None,
              return_lse: bool = False):
    """Masked softmax attention with GQA.  q: [B,S,H,hd], k/v: [B,S,KV,hd(v)] → [B,S,H,hd_v]."""
    B, S, H, _ = q.shape
    KV = k.shape[2]
    g = H // KV
    qf = q.float().permute(0, 2, 1, 3)  # B,H,S,hd
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(g, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(g, dim=1)
    scores = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    mask = attention_mask(S, k.shape[1], causal, window, doc_ids, device=q.device)
    scores = scores.masked_fill(~mask, float("-inf"))
    lse = torch.logsumexp(scores, dim=-1)
    p = torch.exp(scores - lse[..., None])
    p = torch.where(mask, p, torch.zeros_like(p))
    out = torch.matmul(p, vf).permute(0, 2, 1, 3).to(q.dtype)
    if return_lse:
        return out, lse
    return out


def geglu(gate_up: torch.Tensor) -> torch.Tensor:
    """``gelu_tanh(gate) * up`` for gate_up = [gate | up] concatenated on the last dim."""
    g, u = gate_up.float().chunk(2, dim=-1)
    return (F.gelu(g, approximate="tanh") * u).to(gate_up.dtype)


def swiglu(gate_up: torch.Tensor) -> torch.Tensor:
    g, u = gate_up.float().chunk(2, dim=-1)
    return (F.silu(g) * u).to(gate_up.dtype)


def linear(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    return F.linear(x, w)


def embedding(tokens: torch.Tensor, w: torch.Tensor, scale: float | None = None) -> torch.Tensor:
    h = F.embedding(tokens, w)
    if scale is not None:
        h = h * torch.tensor(scale, dtype=h.dtype, device=h.device)
    return h


def linear_cross_entropy(h: torch.Tensor, w: torch.Tensor, labels: torch.Tensor,
                         logit_scale: float = 1.0, reduction: str = "mean") -> torch.Tensor:
    """CE(h·Wᵀ·logit_scale, labels) with ignore_index=-100; softmax in fp32."""
    logits = F.linear(h, w).float() * logit_scale
    return F.cross_entropy(logits, labels, ignore_index=IGNORE_INDEX, reduction=reduction)


def cross_entropy(logits: torch.Tensor, labels: torch.Tensor) -> torch.Tensor:
    return F.cross_entropy(logits.float().flatten(0, -2), labels.flatten(), ignore_index=IGNORE_INDEX)


def adamw_step(p32, g32, m, v, step: int, lr: float, beta1: float, beta2: float, eps: float,
               wd: float, grad_scale: float = 1.0, out_lp: torch.Tensor | None = None) -> None:
    """Decoupled AdamW on fp32 tensors in place; optionally emits a low-precision copy of p."""
    g = g32 * grad_scale
    m.mul_(beta1).add_(g, alpha=1 - beta1)
    v.mul_(beta2).addcmul_(g, g, value=1 - beta2)
    bc1 = 1 - beta1 ** step
    bc2 = 1 - beta2 ** step
    denom = (v.sqrt() / math.sqrt(bc2)).add_(eps)
    p32.mul_(1 - lr * wd).addcdiv_(m, denom, value=-lr / bc1)
    if out_lp is not None:
        out_lp.copy_(p32)


def newton_schulz(g: torch.Tensor, steps: int = 5, eps: float = 1e-7) -> torch.Tensor:
    """Quintic Newton–Schulz orthogonalisation in bf16 (maester/optimizers/muon.py:22-49)."""
    a, b, c = 3.4445, -4.7750, 2.0315
    x = g.to(torch.bfloat16)
    transposed = x.shape[-2] > x.shape[-1]
    if transposed:
        x = x.mT
    x = x / (x.norm(dim=(-2, -1), keepdim=True) + eps)
    for _ in range(steps):
        A = x @ x.mT
        Bm = b * A + (c * A) @ A   # the scaled matrix is the left factor, as in the reference: same bf16 roundings
        x = a * x + Bm @ x
    if transposed:
        x = x.mT
    return x


# --------------------------------------------------------------------------- token log-probabilities
def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor | None, scale: float = 1.0, entropy: bool = False,
                   top: int = 0):
    """``(logprobs, entropy, top_logprobs, top_tokens)`` of the rows of ``logits`` [R, V] (see ``ops.token_logprobs``)."""
    V = logits.shape[-1]
    x = logits if logits.dtype == torch.float64 else logits.float()
    scored = torch.ones(x.shape[0], dtype=torch.bool, device=x.device) if tokens is None else tokens != IGNORE_INDEX
    if tokens is not None and bool((scored & ((tokens < 0) | (tokens >= V))).any()):
        raise ValueError(f"token ids have to be in [0, {V}) or {IGNORE_INDEX}")
    if tokens is not None:     # (a row that is not scored may have no distribution: its gradient is 0 all the same)
        x = torch.where(scored[:, None], x, torch.zeros_like(x))
    m = x.detach().amax(dim=-1, keepdim=True)      # taken off before the scale: logits of the lowest value do not overflow
    logp = torch.log_softmax((x - torch.where(m.isfinite(), m, torch.zeros_like(m))) * scale, dim=-1)
    lp = ent = top_lp = top_id = None
    if tokens is not None:
        at = torch.where(scored, tokens, torch.zeros_like(tokens))
        lp = torch.where(scored, logp.gather(1, at[:, None])[:, 0], torch.zeros_like(logp[:, 0]))
    if entropy:
        p = logp.exp()
        plogp = torch.where(p == 0, torch.zeros_like(p), p * torch.where(p == 0, torch.zeros_like(logp), logp))
        ent = torch.where(scored, -plogp.sum(-1), torch.zeros_like(plogp[:, 0]))
    if top:
        # a stable descending sort keeps the lowest index of equal values first; NaN sorts above +inf
        top_id = torch.sort(x.detach() + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
        top_lp = torch.where(scored[:, None], logp.gather(1, top_id), torch.full_like(logp[:, :top], -math.inf))
        top_id = torch.where(scored[:, None], top_id, torch.full_like(top_id, -1))
    return lp, ent, top_lp, top_id


# --------------------------------------------------------------------------- e4m3 with power-of-two block scales
E4M3_MAX = 448.0
E4M3_TINY = 2.0 ** -9    # smallest positive code
FP8_BLOCK = 128          # values of a contraction that share a scale
FP8_MIN_EXP, FP8_MAX_EXP = -117, 120


def pow2(k: torch.Tensor) -> torch.Tensor:
    """``2^k`` in fp32 for whole ``k`` in [-126, 127] (exact: the exponent field itself)."""
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def fp8_block_exponents(amax: torch.Tensor, k_min: int) -> torch.Tensor:
    """Smallest whole ``k`` in [k_min, 120] with ``amax <= 448 * 2^k``."""
    mant, e = torch.frexp(amax)                       # amax = mant * 2^e with 0.5 <= mant < 1, and 448 = 0.875 * 2^9
    k = torch.where(mant <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, k, torch.full_like(k, k_min)).clamp(k_min, FP8_MAX_EXP)


def _finite_abs(x: torch.Tensor) -> torch.Tensor:
    """|x|, and 0 where x is not finite: infinities and NaN become the NaN code and leave their block's scale alone."""
    a = x.abs()
    return torch.where(a <= torch.finfo(torch.float32).max, a, torch.zeros_like(a))


def fp8_quantize(x: torch.Tensor, square: bool = False) -> tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes [R, C rounded up to 128] and biased exponents uint8 [R, C blocks] of a matrix: one scale for every 128
    values of a row, or (``square``) for every 128 x 128 tile."""
    rows, cols = x.shape
    nb = -(-cols // FP8_BLOCK)
    f = F.pad(x.float(), (0, nb * FP8_BLOCK - cols)).view(rows, nb, FP8_BLOCK)
    amax = _finite_abs(f).amax(dim=2)
    if square:
        rb = -(-rows // FP8_BLOCK)
        amax = F.pad(amax, (0, 0, 0, rb * FP8_BLOCK - rows)).view(rb, FP8_BLOCK, nb).amax(dim=1, keepdim=True)
        amax = amax.expand(rb, FP8_BLOCK, nb).reshape(-1, nb)[:rows]
    k = fp8_block_exponents(amax, FP8_MIN_EXP)
    codes = (f * pow2(-k)[:, :, None]).to(torch.float8_e4m3fn).view(rows, nb * FP8_BLOCK)
    return codes, (k + 127).to(torch.uint8)


def fp8_pack_exponents(exps: torch.Tensor) -> torch.Tensor:
    """[R, blocks] exponent bytes in the order of the block-scaled matrix unit: [R/128, blocks/4, 32, 4, 4] with row
    ``32 i + j`` of 128 at [j, i] and zeros past the end."""
    rows, nb = exps.shape
    rt, kt = -(-rows // 128), -(-nb // 4)
    full = F.pad(exps, (0, kt * 4 - nb, 0, rt * 128 - rows))
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous()


def fp8_unpack_exponents(scales: torch.Tensor, rows: int, blocks: int) -> torch.Tensor:
    rt, kt = scales.shape[:2]
    return scales.permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :blocks]


def fp8_dequantize(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    """fp32 values of codes [R, 128 blocks] with exponents [R, blocks]."""
    rows, nb = exps.shape
    return (codes.float().view(rows, nb, FP8_BLOCK) * pow2(exps.to(torch.int32) - 127)[:, :, None]).view(rows, -1)


# --------------------------------------------------------------------------- AdamW with 8-bit or 32-bit moments
STATE_BLOCK = 256        # values of an optimizer state that share a scale
STATE_MIN_EXP, ROOT_MIN_EXP = -117, -54   # (the square of the smallest root code is still a normal number)


def _mix32(x: int) -> int:
    for shift, factor in ((16, 0x9E3779B9), (15, 0xB7E15163), (16, 1)):    # (digits of the golden ratio and of e)
        x = (x ^ (x >> shift)) * factor & 0xFFFFFFFF
    return x


def state_noise_key(step: int) -> int:
    """32 bits that stand for a step number."""
    return _mix32(_mix32(step & 0xFFFFFFFF) + 0x6A09E667 & 0xFFFFFFFF)


def state_noise(step: int, first: int, n: int, device=None) -> torch.Tensor:
    """32 random bits (int64) for values ``first`` .. ``first + n - 1`` of the flat states in a step: a hash of the step and
    of the value's group of 8, and a linear congruence along the group."""
    m32 = 0xFFFFFFFF
    i = torch.arange(first, first + n, dtype=torch.int64, device=device)
    x = (i >> 3) * 0x9E3779B9 + state_noise_key(step) & m32
    for shift, factor in ((16, 0xB7E15163), (15, 0x6A09E667), (16, 1)):
        x = (x ^ (x >> shift)) * factor & m32
    out = x
    for j in range(1, 8):
        x = x * 0x6A09E667 + 0xBB67AE85 & m32
        out = torch.where(i & 7 == j, x, out)
    return out


def _code_below(a: torch.Tensor, add) -> tuple[torch.Tensor, torch.Tensor]:
    """(the largest code that is at most ``a`` in [0, 448], the distance to the next one); with ``add`` in [0, 2^20) the bits
    below a code's last place are added up first, in units of 2^-20 of that distance."""
    low = torch.where(a < 2.0 ** -6, torch.full_like(a, 2.0 ** -6), torch.zeros_like(a))     # below it codes keep one distance
    z = ((a + low).view(torch.int32) + add) & -(1 << 20)
    z, gap = z.view(torch.float32), (z & 0x7F800000).view(torch.float32) * 0.125
    return z - low, gap


def state_round(y: torch.Tensor, noise: torch.Tensor) -> torch.Tensor:
    """Values in [-448, 448] rounded to one of their two neighbouring codes, so that the expectation is the value."""
    a, _ = _code_below(y.abs(), (noise >> 12).to(torch.int32))
    return torch.where(y.isnan(), y, torch.copysign(a, y))


def state_round_root(y: torch.Tensor, noise: torch.Tensor) -> torch.Tensor:
    """Values in [0, 448] rounded to one of their two neighbouring codes, so that the expectation of the SQUARE is the value's;
    what is not zero does not become zero."""
    lo, gap = _code_below(y, 0)
    u1 = ((noise & 0x7FFFFF).to(torch.int32) | 0x3F800000).view(torch.float32)  # 1 + u
    q = gap * (2 * lo + gap)                                                      # hi^2 - lo^2
    at = (u1.double() * q.double() + (lo * lo - q).double()).float()              # lo^2 + u q, rounded once
    out = torch.where(y * y > at, lo + gap, lo)
    out = torch.where(y > 0, out.clamp_min(E4M3_TINY), out)
    return torch.where(y.isnan(), y, out)


def state_encode(x: torch.Tensor, root: bool = False,
                 noise: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and biased block exponents of a flat state whose length is a multiple of 256; ``root``: a value that is not
    zero does not become zero.  Rounded to nearest, or with ``noise`` (``state_noise``) to a neighbour whose expectation is
    the value, for a root in the squares.  What is a code already stays one."""
    b = x.view(-1, STATE_BLOCK)
    k = fp8_block_exponents(_finite_abs(b).amax(dim=1), ROOT_MIN_EXP if root else STATE_MIN_EXP)
    y = b * pow2(-k)[:, None]
    if noise is not None:
        y = torch.where(y.isinf(), torch.full_like(y, math.nan), y)
        n = noise.view(-1, STATE_BLOCK)
        y = state_round_root(y, n) if root else state_round(y, n)
    elif root:
        y = torch.where(y > 0, y.clamp_min(E4M3_TINY), y)
    return y.to(torch.float8_e4m3fn).view(-1), (k + 127).to(torch.uint8)


def state_decode(codes: torch.Tensor, exps: torch.Tensor) -> torch.Tensor:
    return (codes.float().view(-1, STATE_BLOCK) * pow2(exps.to(torch.int32) - 127)[:, None]).view(-1)


def adamw_multi_step(p: torch.Tensor, g: torch.Tensor, m: torch.Tensor, v: torch.Tensor, *, b1: float, b2: float,
                     decay: float, step_size: float, inv_root: float, eps: float):
    """One AdamW step on flat fp32 values, every operation rounded on its own; returns new (p, m, sqrt(v), v).
    ``decay`` = 1 - lr wd, ``step_size`` = lr / (1 - b1^t), ``inv_root`` = 1 / sqrt(1 - b2^t)."""
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    root = v.sqrt()
    return p * decay - m / (root * inv_root + eps) * step_size, m, root, v
