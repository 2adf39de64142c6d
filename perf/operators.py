"""Measured cases of three operators of a training step that scores tokens, multiplies in 8 bits and keeps its optimizer's
state in 8 bits.

``logprobs``  log-probabilities of given tokens, the entropy of every row and the best alternatives, from logits, with the
              gradient of log-probability and entropy (``ops.token_logprobs``);
``linear``    ``x @ w.T`` with both operands in e4m3 and a power-of-two scale for every block of 128 values of the
              contraction (128 x 128 for the weight), with its gradients (``ops.linear_fp8``);
``adamw``     one AdamW step over many tensors, its two moments held in 8 bits with a power-of-two scale for every 256
              values, or in 32 bits (``optimizers.AdamWMulti``).

``run`` computes the plain form with elementary torch operations where ``own`` is false and calls the framework where it is
true.  ``exact`` says what the outputs are in 64 bits.
"""
import math
import random

import torch

own = False

IGNORE = -100      # token of a row that is not scored
BLOCK = 128        # values of the contraction that share a scale
STATE_BLOCK = 256  # values of an optimizer state that share a scale
E4M3_MAX = 448.0


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decoding step of 16 sequences over the largest vocabulary here: the 20 best alternatives beside each token
        dict(name="logprobs token", op="logprobs", rows=16, vocab=262144, dtype="bf16", top=20, grad=False, scale=1.0, pad=0),
        # scoring the tokens of a packed prompt, five alternatives each
        dict(name="logprobs prompt", op="logprobs", rows=4099, vocab=128256, dtype="bf16", top=5, grad=False, scale=1.0, pad=0),
        # a policy's training step: log-probabilities and entropy with their gradient, at a temperature
        dict(name="logprobs train", op="logprobs", rows=4096, vocab=102400, dtype="bf16", top=0, grad=True, scale=1.25, pad=0),
        # 32-bit logits of an odd vocabulary, rows cut out of a padded matrix
        dict(name="logprobs odd", op="logprobs", rows=1001, vocab=32003, dtype="f32", top=3, grad=True, scale=0.5, pad=61),
        # a few tokens through a feed-forward projection whose weight was laid out once
        dict(name="linear token", op="linear", tokens=4, inner=4096, outer=14336, train=False),
        # a whole prompt of odd length through a gate-and-up projection
        dict(name="linear prompt", op="linear", tokens=5003, inner=2560, outer=20480, train=False),
        # a projection in a training step: output, input gradient and weight gradient, everything quantised on the way
        dict(name="linear train", op="linear", tokens=16384, inner=4096, outer=4096, train=True),
        # sizes that no tile divides
        dict(name="linear odd", op="linear", tokens=333, inner=1100, outer=777, train=True),
        # the tensors of a two-layer debug model
        dict(name="adamw small", op="adamw", tensors=20, total=2_000_000, bits=8, dtype="f32", copy=True),
        # a block-wise list of weights and norms, 32-bit masters with the 16-bit copy that the next step computes with
        dict(name="adamw large", op="adamw", tensors=170, total=400_000_000, bits=8, dtype="f32", copy=True),
        # 16-bit parameters without masters
        dict(name="adamw bf16", op="adamw", tensors=60, total=100_000_000, bits=8, dtype="bf16", copy=False),
        # the same step with 32-bit states
        dict(name="adamw 32", op="adamw", tensors=90, total=120_000_000, bits=32, dtype="f32", copy=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["logprobs", "linear", "adamw"])
    if op == "logprobs":
        vocab = _log(rng, 1000, 262208)
        rows = _log(rng, 1, max(1, min(8192, 400_000_000 // vocab)))
        dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
        grad = rng.random() < 0.5
        return dict(op=op, rows=rows, vocab=vocab, dtype=dtype, top=rng.choice([0, 1, 5, 20, 64]), grad=grad,
                    scale=round(rng.uniform(0.3, 2.0), 3), pad=rng.choice([0, 0, 8, rng.randrange(1, 100)]))
    if op == "linear":
        train = rng.random() < 0.5
        inner, outer = _log(rng, 64, 16384), _log(rng, 64, 20480)
        tokens = _log(rng, 1, max(1, min(16384, 250_000_000_000 // (inner * outer))))
        return dict(op=op, tokens=tokens, inner=inner, outer=outer, train=train)
    bits = rng.choice([8, 8, 32])
    total = _log(rng, 10_000, 200_000_000)
    dtype = rng.choice(["f32", "f32", "bf16"])  # a 16-bit parameter has no 16-bit copy beside it
    return dict(op=op, tensors=_log(rng, 1, 300), total=total, bits=bits, dtype=dtype,
                copy=dtype == "f32" and rng.random() < 0.7)


_DTYPE = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def _sizes(case):
    """Element counts of the tensors of an optimizer case: a few large matrices among many vectors, odd ones with them."""
    r = random.Random(case["tensors"] * 1_000_003 + case["total"])
    weight = [math.exp(r.uniform(0.0, 7.0)) for _ in range(case["tensors"])]
    share = case["total"] / sum(weight)
    return [max(1, int(w * share)) for w in weight]


def _offsets(sizes):
    """Where every tensor and its states begin in the flat buffers: each starts on a block of its own."""
    at, offs = 0, []
    for n in sizes:
        offs.append(at)
        at += (n + STATE_BLOCK - 1) // STATE_BLOCK * STATE_BLOCK
    return offs, at


def work(case):
    if case["op"] == "logprobs":
        size = 4 if case["dtype"] == "f32" else 2
        n, rows = case["rows"] * case["vocab"], case["rows"]
        small = rows * (8 + 8 + case["top"] * 12 + (8 if case["grad"] else 0))
        # with the gradient the logits are read once for the values, and again once those are known
        return {"bytes": n * size * (3 if case["grad"] else 1) + small, "flops": n * (10 if case["grad"] else 5)}
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["inner"], case["outer"]
        if case["train"]:
            return {"bytes": 2 * (2 * t * k + 2 * n * k + 2 * t * n), "flops": 6 * t * k * n}
        return {"bytes": 2 * t * k + n * k + n * k // BLOCK + 2 * t * n, "flops": 2 * t * k * n}
    n = sum(_sizes(case))
    p = 4 if case["dtype"] == "f32" else 2
    state = 2 * (1 + 1 / STATE_BLOCK) if case["bits"] == 8 else 8
    return {"bytes": n * (2 * p + p + 2 * state + (2 if case["copy"] else 0)), "flops": 20 * n}


# ------------------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(int(seed))
    if case["op"] == "logprobs":
        rows, vocab, dt = case["rows"], case["vocab"], _DTYPE[case["dtype"]]
        wide = torch.empty(rows, vocab + case["pad"], device=dev, dtype=dt)
        # a language model's logits: a broad bulk and a few candidates that stand out
        for r0 in range(0, rows, 512):
            part = torch.randn(min(512, rows - r0), vocab + case["pad"], device=dev, generator=g) * 2.0
            hot = torch.randint(0, vocab, (part.shape[0], 24), device=dev, generator=g)
            part.scatter_add_(1, hot, torch.rand(hot.shape, device=dev, generator=g) * 16.0)
            wide[r0:r0 + part.shape[0]] = part.to(dt)
        logits = wide[:, :vocab]
        best = logits.argmax(dim=1)
        other = torch.randint(0, vocab, (rows,), device=dev, generator=g)
        pick = torch.rand(rows, device=dev, generator=g)
        tokens = torch.where(pick < 0.6, best, other)
        if case["grad"]:  # the prompt's own tokens are not trained on
            tokens = torch.where(torch.rand(rows, device=dev, generator=g) < 0.1, torch.full_like(tokens, IGNORE), tokens)
        s = dict(case=case, logits=logits, tokens=tokens)
        if case["grad"]:
            s["g_logprob"] = torch.randn(rows, device=dev, generator=g) / rows
            s["g_entropy"] = torch.randn(rows, device=dev, generator=g) * (0.01 / rows)
            s["logits"] = logits.detach().requires_grad_(True)
        return s
    if case["op"] == "linear":
        t, k, n = case["tokens"], case["inner"], case["outer"]
        # activations with channels of very different size, as they come out of a norm; weights of the usual spread
        chan = torch.exp(torch.randn(k, device=dev, generator=g) * 0.7)
        x = (torch.randn(t, k, device=dev, generator=g) * chan).to(torch.bfloat16)
        w = (torch.randn(n, k, device=dev, generator=g) * (k ** -0.5)).to(torch.bfloat16)
        s = dict(case=case, x=x)
        if case["train"]:
            s["w"], s["x"] = w.requires_grad_(True), x.requires_grad_(True)
            s["dy"] = (torch.randn(t, n, device=dev, generator=g) * 1e-3).to(torch.bfloat16)
        else:  # a program that serves keeps the weight's codes and scales
            codes, exps = _quantize(w, square=True)
            s["codes"], s["scales"] = codes, _pack(exps, n)
        return s
    sizes = _sizes(case)
    offs, total = _offsets(sizes)
    dt = _DTYPE[case["dtype"]]
    # gradients whose size differs from tensor to tensor; zeros between the tensors
    size = torch.zeros(total, device=dev)
    for n, o, e in zip(sizes, offs, torch.randn(len(sizes), generator=torch.Generator().manual_seed(int(seed))).tolist()):
        size[o:o + n] = math.exp(1.5 * e) * 1e-3
    inside = (size > 0).float()
    p = (torch.randn(total, device=dev, generator=g) * inside * 0.02).to(dt)
    grad = (torch.randn(total, device=dev, generator=g) * size).to(dt)
    s = dict(case=case, sizes=sizes, offs=offs, p=p, grad=grad, step=0,
             copy=torch.zeros(total, device=dev, dtype=torch.bfloat16) if case["copy"] else None,
             hyper=dict(lr=3e-4, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1))
    # states as they are some way into a run
    m1 = torch.randn(total, device=dev, generator=g) * size * 0.3
    v1 = (torch.rand(total, device=dev, generator=g) + 0.05) * size ** 2
    if case["bits"] == 8:
        s["m"], s["m_exp"] = _state_codes(m1, -117, False)
        s["r"], s["r_exp"] = _state_codes(v1.sqrt(), -54, True)
    else:
        s["m"], s["v"] = m1, v1
    if own:  # the optimizer that a program builds once, over the same tensors and with the same states
        from maester_b200.optimizers import AdamWMulti
        params, copies = [], {}
        for n, o in zip(sizes, offs):
            q = torch.nn.Parameter(s["p"][o:o + n])
            q.grad = s["grad"][o:o + n]
            if s["copy"] is not None:
                copies[q] = s["copy"][o:o + n]
            params.append(q)
        opt = AdamWMulti(params, state_bits=case["bits"], **s["hyper"])
        if copies:
            opt.attach_copies(copies)
        flat = opt.state_buffers()
        for mine, theirs in (("m", "exp_avg"), ("m_exp", "exp_avg_exp"), ("r", "exp_avg_root"),
                             ("r_exp", "exp_avg_root_exp"), ("v", "exp_avg_sq")):
            if mine in s:
                flat[theirs].copy_(s[mine])
                s[mine] = flat[theirs]
        s["opt"] = opt
    return s


# ------------------------------------------------------------------------------------------------ plain forms
def _pow2(k):
    """2^k in 32 bits for whole k in [-126, 127]."""
    return ((k.to(torch.int32) + 127) << 23).view(torch.float32)


def _block_exponents(amax):
    """Smallest whole k with amax <= 448 * 2^k (far below every limit for a block of zeros)."""
    mant, e = torch.frexp(amax)  # amax = mant * 2^e, 0.5 <= mant < 1; 448 = 0.875 * 2^9
    k = torch.where(mant <= 0.875, e - 9, e - 8)
    return torch.where(amax > 0, k, torch.full_like(k, -200))


def _finite_abs(x):
    a = x.abs()
    return torch.where(a <= torch.finfo(torch.float32).max, a, torch.zeros_like(a))


def _quantize(x, square):
    """e4m3 codes [rows, columns padded to 128] and biased block exponents [rows, column blocks] of a matrix."""
    rows, cols = x.shape
    nb = (cols + BLOCK - 1) // BLOCK
    f = torch.zeros(rows, nb * BLOCK, device=x.device)
    f[:, :cols] = x.float()
    amax = _finite_abs(f).view(rows, nb, BLOCK).amax(dim=2)
    if square:
        rb = (rows + BLOCK - 1) // BLOCK
        full = torch.zeros(rb * BLOCK, nb, device=x.device)
        full[:rows] = amax
        amax = full.view(rb, BLOCK, nb).amax(dim=1, keepdim=True).expand(rb, BLOCK, nb).reshape(rb * BLOCK, nb)[:rows]
    k = _block_exponents(amax).clamp(-117, 120)
    y = f.view(rows, nb, BLOCK) * _pow2(-k)[:, :, None]
    return y.to(torch.float8_e4m3fn).view(rows, nb * BLOCK), (k + 127).to(torch.uint8)


def _pack(exps, rows):
    """Exponents in the order in which the matrix unit takes them: for 128 rows and 4 blocks, row r of the 128 at
    16 (r mod 32) + 4 (r div 32)."""
    nb = exps.shape[1]
    rt, kt = (rows + 127) // 128, (nb + 3) // 4
    full = torch.zeros(rt * 128, kt * 4, device=exps.device, dtype=torch.uint8)
    full[:rows, :nb] = exps
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous()


def _unpack(scales, rows, nb):
    rt, kt = scales.shape[:2]
    return scales.permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)[:rows, :nb]


def _dequantize(codes, exps):
    rows, nb = exps.shape
    return (codes.float().view(rows, nb, BLOCK) * _pow2(exps.to(torch.int32) - 127)[:, :, None]).view(rows, nb * BLOCK)


def _state_codes(x, k_min, keep):
    """Codes and biased exponents of a flat state; ``keep``: what is not zero does not become zero."""
    b = x.view(-1, STATE_BLOCK)
    k = _block_exponents(_finite_abs(b).amax(dim=1)).clamp(k_min, 120)
    y = b * _pow2(-k)[:, None]
    if keep:
        y = torch.where(y > 0, y.clamp_min(2.0 ** -9), y)
    return y.to(torch.float8_e4m3fn).view(-1), (k + 127).to(torch.uint8)


def _plain_logprobs(s):
    case, raw, tokens = s["case"], s["logits"].detach(), s["tokens"]
    rows, vocab = raw.shape
    scored = tokens != IGNORE
    at = torch.where(scored, tokens, torch.zeros_like(tokens))[:, None]
    x = raw.float()
    d = (x - x.amax(dim=1, keepdim=True)) * case["scale"]
    e = d.exp()
    total = e.sum(dim=1, keepdim=True)
    log_total = total.log()
    zero = torch.zeros(rows, device=x.device)
    logprob = torch.where(scored, (d.gather(1, at) - log_total)[:, 0], zero)
    entropy = (log_total - (d * e).sum(dim=1, keepdim=True) / total)
    out = {"logprob": logprob, "entropy": torch.where(scored, entropy[:, 0], zero)}
    if case["top"]:
        # order by value, ties by the lowest index: one whole key of both
        bits = (x + 0.0).view(torch.int32).to(torch.int64)
        order = torch.where(bits >= 0, bits, -2 ** 31 - 1 - bits)
        key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(vocab, device=x.device))
        best = torch.topk(key, case["top"], dim=1).values
        token = (1 << 20) - 1 - (best & ((1 << 20) - 1))
        value = d.gather(1, token) - log_total
        out["top_tokens"] = torch.where(scored[:, None], token, torch.full_like(token, -1))
        out["top_logprobs"] = torch.where(scored[:, None], value, torch.full_like(value, -math.inf))
    if case["grad"]:
        prob = e / total
        logp = d - log_total
        gl = torch.where(scored, s["g_logprob"], zero)[:, None]
        ge = torch.where(scored, s["g_entropy"], zero)[:, None]
        grad = prob * -(gl + ge * (logp + entropy))
        grad.scatter_add_(1, at, gl)
        out["grad"] = (grad * case["scale"]).to(raw.dtype)
    return out


def _plain_linear(s):
    case = s["case"]
    x = s["x"].detach()
    k, n = case["inner"], case["outer"]
    if not case["train"]:
        nb = (k + BLOCK - 1) // BLOCK
        w = _dequantize(s["codes"], _unpack(s["scales"], n, nb))
        return (_dequantize(*_quantize(x, False)) @ w.T).to(torch.bfloat16)
    w, dy = s["w"].detach(), s["dy"]
    wq = _dequantize(*_quantize(w, True))
    y = _dequantize(*_quantize(x, False)) @ wq.T
    dx = _dequantize(*_quantize(dy, False))[:, :n] @ wq[:, :k]
    dw = _dequantize(*_quantize(dy.T, False)) @ _dequantize(*_quantize(x.T, False)).T
    return {"y": y.to(torch.bfloat16), "dx": dx.to(torch.bfloat16), "dw": dw.to(torch.bfloat16)}


def _plain_adamw(s):
    case, h = s["case"], s["hyper"]
    s["step"] += 1
    b1, b2 = h["betas"]
    bc1, root2 = 1 - b1 ** s["step"], math.sqrt(1 - b2 ** s["step"])
    g, p = s["grad"].float(), s["p"].float()
    if case["bits"] == 8:
        m = (s["m"].float().view(-1, STATE_BLOCK) * _pow2(s["m_exp"].to(torch.int32) - 127)[:, None]).view(-1)
        r = (s["r"].float().view(-1, STATE_BLOCK) * _pow2(s["r_exp"].to(torch.int32) - 127)[:, None]).view(-1)
        v = r * r
    else:
        m, v = s["m"], s["v"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * g * (1 - b2)
    root = v.sqrt()
    p = p * (1 - h["lr"] * h["weight_decay"]) - m / (root * (1 / root2) + h["eps"]) * (h["lr"] / bc1)
    s["p"].copy_(p)
    if s["copy"] is not None:
        s["copy"].copy_(s["p"])
    if case["bits"] == 8:
        for key, value, k_min, keep in (("m", m, -117, False), ("r", root, -54, True)):
            codes, exps = _state_codes(value, k_min, keep)
            s[key].copy_(codes)
            s[key + "_exp"].copy_(exps)
    else:
        s["m"].copy_(m)
        s["v"].copy_(v)
    return _adamw_outputs(s)


def _adamw_outputs(s):
    return {k: s[k] for k in ("p", "copy", "m", "m_exp", "r", "r_exp", "v") if s.get(k) is not None}


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    case = state["case"]
    if case["op"] == "logprobs":
        if not own:
            return _plain_logprobs(state)
        from maester_b200 import ops
        got = ops.token_logprobs(state["logits"], state["tokens"], scale=case["scale"], entropy=True, top=case["top"])
        out = {"logprob": got.logprobs.detach(), "entropy": got.entropy.detach()}
        if case["top"]:
            out["top_tokens"], out["top_logprobs"] = got.top_tokens, got.top_logprobs.detach()
        if case["grad"]:
            out["grad"], = torch.autograd.grad([got.logprobs, got.entropy], [state["logits"]],
                                               [state["g_logprob"], state["g_entropy"]])
        return out
    if case["op"] == "linear":
        if not own:
            return _plain_linear(state)
        from maester_b200 import ops
        if not case["train"]:
            w = ops.Fp8Blocks(state["codes"], state["scales"], case["inner"])
            return ops.linear_fp8(state["x"], w)
        y = ops.linear_fp8(state["x"], state["w"])
        dx, dw = torch.autograd.grad([y], [state["x"], state["w"]], [state["dy"]])
        return {"y": y.detach(), "dx": dx, "dw": dw}
    if not own:
        return _plain_adamw(state)
    state["opt"].step()
    return _adamw_outputs(state)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_e4m3(y):
    """Nearest e4m3 value, ties to even, by arithmetic on doubles: steps of 2^(e-3) inside [2^e, 2^(e+1)), of 2^-9 below 2^-6."""
    _, e = torch.frexp(y)
    step = torch.exp2((e - 1).clamp_min(-6).double() - 3)
    return torch.round(y / step) * step


def _exact_blocks(x, square):
    """The values that a quantised matrix stands for."""
    rows, cols = x.shape
    rb, nb = -(-rows // BLOCK), -(-cols // BLOCK)
    f = torch.zeros(rb * BLOCK, nb * BLOCK, device=x.device, dtype=torch.float64)
    f[:rows, :cols] = x.double()
    f = f.view(rb, BLOCK, nb, BLOCK)
    top = f.abs().amax(dim=(1, 3) if square else 3, keepdim=True) / E4M3_MAX
    mant, e = torch.frexp(top)
    unit = torch.exp2(torch.where(mant == 0.5, e - 1, e).clamp(-117, 120).double())
    return (_exact_e4m3(f / unit) * unit).view(rb * BLOCK, nb * BLOCK)[:rows, :cols]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "logprobs":
        n, tokens = case["vocab"], s["tokens"]
        parts = {"logprob": [], "entropy": [], "top_logprobs": [], "grad": []}
        for r0 in range(0, case["rows"], 256):
            z = s["logits"].detach()[r0:r0 + 256].double() * case["scale"]
            t = tokens[r0:r0 + 256]
            live = (t != IGNORE)
            logp = z - torch.logsumexp(z, dim=1, keepdim=True)
            p = logp.exp()
            one = (torch.arange(n, device=z.device)[None] == t[:, None]).double()
            h = -(p * logp).sum(dim=1)
            parts["logprob"].append((logp * one).sum(dim=1))
            parts["entropy"].append(h * live)
            if case["top"]:
                best = logp.sort(dim=1, descending=True).values[:, :case["top"]]
                parts["top_logprobs"].append(torch.where(live[:, None], best, torch.full_like(best, -math.inf)))
            if case["grad"]:
                gl = (s["g_logprob"][r0:r0 + 256].double() * live)[:, None]
                ge = (s["g_entropy"][r0:r0 + 256].double() * live)[:, None]
                parts["grad"].append(case["scale"] * (gl * (one - p) - ge * p * (logp + h[:, None])))
        out = {k: torch.cat(v) for k, v in parts.items() if v}
        if case["top"]:
            out["top_tokens"] = None
        return out
    if case["op"] == "linear":
        x = _exact_blocks(s["x"].detach(), False)
        if not case["train"]:
            k, n = case["inner"], case["outer"]
            nb = s["codes"].shape[1] // BLOCK
            unit = torch.exp2(_unpack(s["scales"], n, nb).double() - 127)
            w = s["codes"].double() * unit.repeat_interleave(BLOCK, dim=1)
            return x @ w[:, :k].T
        w = _exact_blocks(s["w"].detach(), True)
        y = x @ w.T
        dx = _exact_blocks(s["dy"], False) @ w
        dw = _exact_blocks(s["dy"].T, False) @ _exact_blocks(s["x"].detach().T, False).T
        return {"y": y, "dx": dx, "dw": dw}
    h = s["hyper"]
    b1, b2 = h["betas"]
    g, p = s["grad"].double(), s["p"].double()
    if case["bits"] == 8:
        m = s["m"].double() * torch.exp2(s["m_exp"].double() - 127).repeat_interleave(STATE_BLOCK)
        v = (s["r"].double() * torch.exp2(s["r_exp"].double() - 127).repeat_interleave(STATE_BLOCK)) ** 2
    else:
        m, v = s["m"].double(), s["v"].double()
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g ** 2
    p = p - h["lr"] * (h["weight_decay"] * p + (m / (1 - b1)) / ((v / (1 - b2)).sqrt() + h["eps"]))
    out = {"p": p}
    if case["copy"]:
        out["copy"] = p
    if case["bits"] == 32:
        out["m"], out["v"] = m, v
    else:  # what the next step finds is a rounding of these to 8 bits: no value in 64 bits of its own
        out |= {"m": None, "m_exp": None, "r": None, "r_exp": None}
    return out
