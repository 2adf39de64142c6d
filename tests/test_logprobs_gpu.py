"""``ops.token_logprobs`` and ``ops.linear_logprobs`` against the formulas in 64 bits.

Tolerances (u = 2^-24, half a step of fp32): an exponent's argument has at most three roundings (3 |z| u relative to
exp), the exponential 2^-22; the weighted mean of |z| over a row is at most log V < 13; a sum of V values takes at most
V / 256 + 32 additions one after the other.  So log s is within E = (80 + V / 256) u of its value, a log-probability within
E + 4 |lp| u, an entropy within E (2 + log V), a probability within (E + 3 |lp| u) p, and a gradient adds half a step of its
own type.
"""
import math

import pytest
import torch

from maester_b200 import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: U}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -25, torch.float32: 1e-38}


@pytest.fixture(autouse=True)
def _status():
    from maester_b200.ops import cuda as C
    yield
    C.check_status()


def _logits(rows, V, dtype, pad=0, spread=3.0):
    x = torch.randn(rows, V + pad, device="cuda") * spread
    x[:, : max(1, V // 50)] += 6.0
    return x.to(dtype)[:, :V]


def _exact(x, tokens, scale):
    """(logprob of every token, entropy) in 64 bits."""
    z = x.double() * scale
    z = z - z.amax(1, keepdim=True).clamp_min(-1e300)     # (a row of -3.4e38 has no room for log V beside it, in 64 bits either)
    logp = z - torch.logsumexp(z, 1, keepdim=True)
    p = logp.exp()
    return logp, -(torch.where(p > 0, p * logp, torch.zeros_like(p))).sum(1)


def _order(x, top):
    """ids by value, ties by the lowest id"""
    return torch.sort(x.float() + 0.0, dim=1, descending=True, stable=True).indices[:, :top]


def _err(V):
    return (80 + V / 256) * U


def _check_fwd(got, x, tokens, scale, top):
    V = x.shape[1]
    logp, h = _exact(x, tokens, scale)
    live = tokens != -100
    at = torch.where(live, tokens, 0)
    want = torch.where(live, logp.gather(1, at[:, None])[:, 0], 0.0)
    assert got.logprobs.dtype == got.entropy.dtype == torch.float32
    masked = want == -math.inf
    assert torch.equal(got.logprobs.double()[masked], want[masked])
    assert ((got.logprobs.double() - want).abs()[~masked] <= _err(V) + 4 * want.abs()[~masked] * U).all()
    assert ((got.entropy.double() - torch.where(live, h, 0.0)).abs() <= _err(V) * (2 + math.log(V))).all()
    if top:
        ids = _order(x, top)
        assert torch.equal(got.top_tokens, torch.where(live[:, None], ids, -1))
        want = torch.where(live[:, None], logp.gather(1, ids), -math.inf)
        fin = want > -math.inf
        assert torch.equal(got.top_logprobs == -math.inf, ~fin)
        assert ((got.top_logprobs.double() - want).abs()[fin] <= _err(V) + 4 * want.abs()[fin] * U).all()
    else:
        assert got.top_tokens is None and got.top_logprobs is None


SHAPES = [(1, 1), (1, 2), (3, 7), (5, 64), (2, 255), (2, 257), (9, 1000), (33, 4099), (4, 32003), (1, 65537), (7, 128256),
          (2, 262144), (1, 262144), (300, 5001), (1500, 129)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V", SHAPES)
def test_values(rows, V, dtype):
    for pad, scale, top in ((0, 1.0, min(5, V)), (3, 0.7, 0), (8, 1.9, min(64, V))):
        x = _logits(rows, V, dtype, pad)
        tokens = torch.randint(0, V, (rows,), device="cuda")
        if rows > 2:
            tokens[1] = -100
        _check_fwd(ops.token_logprobs(x, tokens, scale=scale, entropy=True, top=top), x, tokens, scale, top)


@pytest.mark.parametrize("kind", ["constant", "ascending", "descending", "zeros", "steps", "masked", "one", "lowest", "all lowest"])
@pytest.mark.parametrize("rows,V", [(3, 50), (2, 5000), (1, 200001), (260, 3001)])
def test_orders_and_masks(kind, rows, V):
    """Rows that a threshold or a tie-break could get wrong: equal values, sorted values, signed zeros, masks."""
    base = torch.arange(V, device="cuda", dtype=torch.float32)
    x = {"constant": torch.full((V,), -3.25, device="cuda"), "ascending": base / V * 8, "descending": -base / V * 8,
         "zeros": torch.where(base % 2 == 0, 0.0, -0.0), "steps": (base % 7), "masked": torch.where(base % 11 == 5, base % 13, -math.inf),
         "one": torch.where(base == V - 1, 1.0, -math.inf), "lowest": torch.where(base % 5 == 2, base / V, -math.inf),
         "all lowest": torch.full((V,), -math.inf, device="cuda")}[kind]
    scale = 1.0
    for dtype in (torch.float32, torch.bfloat16):
        xs = x.to(dtype)[None].repeat(rows, 1)
        if "lowest" in kind:
            xs = xs.clamp_min(torch.finfo(dtype).min)
        tokens = torch.full((rows,), V - 1, device="cuda")
        _check_fwd(ops.token_logprobs(xs, tokens, scale=scale, entropy=True, top=min(40, V)), xs, tokens, scale, min(40, V))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V", [(700, 6), (700, 100), (800, 4099), (1200, 16003), (601, 32000)])
def test_rows_that_share_an_sm(rows, V, dtype):
    """More rows than blocks of 256 threads fit on the GPU at once: blocks are smaller then.  Random rows, and one whose
    best values lie next to each other, one that ascends, one that is constant, one without a finite value but the last."""
    x = _logits(rows, V, dtype, 1)
    x[3, V // 2:V // 2 + 70] = 50.0
    x[4] = torch.arange(V, device="cuda") / V
    x[5] = -2.5
    x[6, :-1] = -math.inf
    tokens = torch.randint(0, V, (rows,), device="cuda")
    tokens[1], tokens[6] = -100, V - 1
    for top in sorted({0, 1, min(20, V), min(33, V), min(64, V)}):
        _check_fwd(ops.token_logprobs(x, tokens, scale=0.9, entropy=True, top=top), x, tokens, 0.9, top)


@pytest.mark.parametrize("scale,size", [(1e8, 1e-7), (1e8, 9e29), (1e-8, 1e9), (1.0, 9e29), (1.0, 3e38)])
def test_scales_and_sizes_at_the_ends(scale, size):
    """The largest logits times the largest scale, up to the ends of fp32: small distances, or one value that has it all."""
    x = torch.linspace(-1, 1, 2000, device="cuda")[None].repeat(2, 1) * size
    x[1] = x[1].flip(0)
    tokens = torch.tensor([1999, 3], device="cuda")
    got = ops.token_logprobs(x, tokens, scale=scale, entropy=True, top=4)
    z = x.double() * scale
    logp = torch.log_softmax(z - z.amax(1, keepdim=True), 1)
    want = logp.gather(1, tokens[:, None])[:, 0]
    far = want < -3e38      # beyond fp32
    assert (got.logprobs[far] == -math.inf).all()
    assert ((got.logprobs.double() - want).abs() <= _err(2000) + 4 * want.abs() * U)[~far].all()
    ent = -(logp.exp() * logp).nan_to_num(0.0).sum(1)
    assert ((got.entropy.double() - ent).abs() <= _err(2000) * (2 + math.log(2000))).all()
    assert torch.equal(got.top_tokens, _order(x, 4))


@pytest.mark.parametrize("scale,size", [(0.1, 2.0 ** 27), (0.1, 2.0 ** 29), (0.1, 2.0 ** 30), (0.05, -2.0 ** 30), (1e-3, 2.0 ** 36),
                                        (1.0, 2.0 ** 25), (1.0, -2.0 ** 26), (1.0, 2.0 ** 40)])
def test_close_logits_far_from_zero(scale, size):
    """Neighbouring fp32 numbers around `size`, the largest ones last or first: what a product with the scale rounds away is
    larger than their distances.  The gradient's tolerance is that of ``test_gradient``'s probabilities."""
    V = 4000
    step = abs(size) * 2.0 ** -23
    x = (size + (torch.arange(V, device="cuda", dtype=torch.float64) // 571) * step).float()[None].repeat(2, 1)
    x[:, 100:2000] = size / 4 if size > 0 else size * 4
    x[1] = x[1].flip(0)
    x.requires_grad_()
    tokens = torch.tensor([V - 1, 1], device="cuda")
    got = ops.token_logprobs(x, tokens, scale=scale, entropy=True, top=10)
    with torch.no_grad():
        _check_fwd(got, x, tokens, scale, 10)
        logp, h = _exact(x, tokens, scale)
    dx, = torch.autograd.grad(got.logprobs.sum() + got.entropy.sum(), x)
    p = logp.exp()
    one = (torch.arange(V, device="cuda")[None] == tokens[:, None]).double()
    lp = torch.where(p > 0, logp, 0.0)
    want = scale * (one - p - p * (lp + h[:, None]))
    # (a probability below 2^-126, e^-87, is no normal fp32 number and may be taken for 0: here they go down to e^-91)
    room = p * (2 + lp.abs() + h[:, None]) + one
    assert ((dx.double() - want).abs() <= 4 * scale * (_err(V) + 3 * lp.abs() * U) * room + scale * room * (p < 2.0 ** -126)).all()


def test_rows_without_a_distribution():
    x = torch.zeros(5, 3000, device="cuda")
    x[0] = -math.inf
    x[1, 2900] = math.nan
    x[2, 7] = math.inf
    x[3, 0] = -math.inf
    got = ops.token_logprobs(x, torch.zeros(5, dtype=torch.int64, device="cuda"), entropy=True, top=2)
    assert got.logprobs[:3].isnan().all() and got.entropy[:3].isnan().all() and got.top_logprobs[:3].isnan().all()
    assert got.top_tokens[:3].tolist() == [[0, 1], [2900, 0], [7, 0]]
    assert got.logprobs[3].item() == -math.inf and got.top_tokens[3].tolist() == [1, 2]
    assert abs(got.logprobs[4].item() + math.log(3000)) < 1e-5 and abs(got.entropy[3].item() - math.log(2999)) < 1e-5


def _grad_want(x, tokens, scale, gl, ge, gt, ids):
    logp, h = _exact(x, tokens, scale)
    p, live = logp.exp(), (tokens != -100).double()[:, None]
    one = (torch.arange(x.shape[1], device="cuda")[None] == tokens[:, None]).double()
    all_ = gl.double()[:, None]
    hot = all_ * one
    if gt is not None:
        all_ = all_ + gt.double().sum(1, keepdim=True)
        hot = hot.scatter_add(1, ids, gt.double())
    lp = torch.where(p > 0, logp, 0.0)
    want = live * scale * (hot - p * (all_ + ge.double()[:, None] * (lp + h[:, None])))
    size = gl.double().abs()[:, None] + (0 if gt is None else gt.double().abs().sum(1, keepdim=True))
    size = size + ge.double().abs()[:, None] * (lp.abs() + h[:, None] + 1)
    slack = scale * (size * p * (2 * _err(x.shape[1]) + 6 * lp.abs() * U) + 8 * U * hot.abs())
    return want, slack


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,V", [(1, 1), (3, 7), (2, 257), (33, 4099), (7, 128256), (1, 262144), (300, 5001)])
def test_gradient(rows, V, dtype):
    for pad, scale, top in ((0, 1.0, 0), (5, 0.6, min(6, V)), (8, 1.3, 0)):
        x = _logits(rows, V, dtype, pad)
        tokens = torch.randint(0, V, (rows,), device="cuda")
        if rows > 2:
            tokens[1] = -100
        tokens[0] = _order(x, 1)[0, 0]                       # a token that is also an alternative
        x.requires_grad_(True)
        out = ops.token_logprobs(x, tokens, scale=scale, entropy=True, top=top)
        gl, ge = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda")
        gt = torch.randn(rows, top, device="cuda") if top else None
        outs, gs = [out.logprobs, out.entropy], [gl, ge]
        if top:
            live = (tokens != -100)[:, None]
            outs, gs = outs + [out.top_logprobs], gs + [gt]
        dx, = torch.autograd.grad(outs, [x], gs)
        assert dx.dtype == dtype and dx.shape == x.shape
        ids = _order(x.detach(), top) if top else None
        want, slack = _grad_want(x.detach(), tokens, scale, gl, ge, gt, ids)
        assert ((dx.double() - want).abs() <= slack + want.abs() * HALF[dtype] * 1.01 + TINY[dtype]).all()
        if rows > 2:
            assert not dx[1].any()


def test_gradient_of_parts_and_masks():
    """Only some outputs used, broadcast gradients, -inf logits: zero gradient there, none turned into NaN."""
    x = _logits(4, 777, torch.float32)
    x[:, 100:300] = -math.inf
    x.requires_grad_(True)
    tokens = torch.tensor([5, 6, 300, 776], device="cuda")
    ones, zeros = torch.ones(4, device="cuda"), torch.zeros(4, device="cuda")
    for use, gl, ge in ((lambda o: o.logprobs.sum(), ones, zeros), (lambda o: o.entropy.sum(), zeros, ones)):
        dx, = torch.autograd.grad(use(ops.token_logprobs(x, tokens, entropy=True, top=3)), [x])
        want, slack = _grad_want(x.detach(), tokens, 1.0, gl, ge, None, None)
        assert not dx[:, 100:300].any() and ((dx.double() - want).abs() <= slack + want.abs() * U * 1.01 + 1e-38).all()
    only, = torch.autograd.grad(ops.token_logprobs(x, entropy=True).entropy.sum(), [x])
    assert torch.equal(only, dx)


def test_gradient_against_differences():
    """Central differences of the fp32 outputs in direction d: their rounding, E / h, and the third derivative, h^2."""
    x = (torch.randn(3, 40, device="cuda")).requires_grad_(True)
    tokens = torch.tensor([1, 0, 39], device="cuda")
    f = lambda v: (lambda o: (o.logprobs * 0.7 + o.entropy * 0.3).double().sum() + o.top_logprobs.double().sum() * 0.2)(
        ops.token_logprobs(v, tokens, scale=0.9, entropy=True, top=2))
    dx, = torch.autograd.grad(f(x), [x])
    d = torch.randn_like(x)
    h = 2.0 ** -6
    with torch.no_grad():
        num = (f(x + h * d) - f(x - h * d)) / (2 * h)
    assert abs(num.item() - (dx * d).sum().item()) < 3 * 10 * _err(40) * 5 / h + 10 * h * h


def test_layouts_streams_and_capture():
    x3 = torch.randn(2, 5, 1003, device="cuda", dtype=torch.bfloat16)
    tokens = torch.randint(0, 1003, (2, 5), device="cuda", dtype=torch.int32)
    want = ops.token_logprobs(x3.reshape(10, 1003), tokens.reshape(10).long(), entropy=True, top=4)
    for x in (x3, x3.transpose(0, 1).contiguous().transpose(0, 1), x3.permute(2, 0, 1).contiguous().permute(1, 2, 0)):
        got = ops.token_logprobs(x, tokens, entropy=True, top=4)
        assert got.top_tokens.shape == (2, 5, 4) and got.logprobs.shape == (2, 5)
        for a, b in zip(got, want):
            assert torch.equal(a.reshape(-1), b.reshape(-1))
    one = ops.token_logprobs(x3[0, 0], tokens[0, 0], entropy=True, top=4)
    assert one.logprobs.shape == () and torch.equal(one.top_tokens, want.top_tokens[0])
    row = x3[0, :1].expand(5, 1003)                              # rows that share their memory
    assert torch.equal(ops.token_logprobs(row, tokens[0]).logprobs[:1], want.logprobs[:1])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.token_logprobs(x3, tokens, entropy=True, top=4)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(other.logprobs.view(-1), want.logprobs)
    buf = x3.clone()
    graphs = []
    for _ in range(2):                                           # two graphs of the same call
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = ops.token_logprobs(buf, tokens, entropy=True, top=4)
        graphs.append((g, out))
    buf.copy_(torch.randn_like(buf))
    fresh = ops.token_logprobs(buf, tokens, entropy=True, top=4)
    for g, out in graphs:
        g.replay()
        for a, b in zip(out, fresh):
            assert torch.equal(a, b)
    empty = ops.token_logprobs(buf[:0], tokens[:0], entropy=True, top=2)
    assert empty.logprobs.shape == (0, 5) and empty.top_tokens.shape == (0, 5, 2)


def test_same_bits_every_time():
    x = _logits(40, 70001, torch.bfloat16).requires_grad_(True)
    tokens = torch.randint(0, 70001, (40,), device="cuda")
    runs = []
    for _ in range(3):
        o = ops.token_logprobs(x, tokens, entropy=True, top=20)
        runs.append([*o, *torch.autograd.grad((o.logprobs + o.entropy).sum(), [x])])
    for r in runs[1:]:
        assert all(torch.equal(a, b) for a, b in zip(r, runs[0]))


def test_a_token_outside_the_vocabulary_is_reported():
    from maester_b200.ops import cuda as C
    x = torch.randn(3, 100, device="cuda", requires_grad=True)
    got = ops.token_logprobs(x, torch.tensor([5, 100, -1], device="cuda"), entropy=True, top=1)
    assert got.logprobs.isnan().tolist() == [False, True, True]
    dx, = torch.autograd.grad(got.logprobs.sum(), [x])
    assert dx.isnan().all(1).tolist() == [False, True, True] and dx[0].isfinite().all()
    with pytest.raises(RuntimeError, match="status 8"):
        C.check_status()


@pytest.mark.parametrize("rows,V,D", [(1, 1000, 64), (130, 4099, 256), (700, 32003, 128)])
def test_linear_logprobs(rows, V, D, monkeypatch):
    """Chunks of 128 rows against the whole product: logits in fp32 within D half steps of sum |h||w|."""
    from maester_b200.ops import logprobs
    monkeypatch.setattr(logprobs, "CHUNK_BYTES", 4 * V * 256)
    h = torch.randn(rows, D, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    w = (torch.randn(V, D, device="cuda") * D ** -0.5).to(torch.bfloat16).requires_grad_(True)
    tokens = torch.randint(0, V, (rows,), device="cuda")
    tokens[rows // 2:rows // 2 + (rows > 1)] = -100
    gl, ge = torch.randn(rows, device="cuda"), torch.randn(rows, device="cuda") * 0.1
    got = ops.linear_logprobs(h, w, tokens, logit_scale=1.5, entropy=True, top=3)
    dh, dw = torch.autograd.grad([got.logprobs, got.entropy], [h, w], [gl, ge], retain_graph=True)
    logits = h.detach().double() @ w.detach().double().T
    off = 2 * D * U * (h.detach().double().abs() @ w.detach().double().abs().T).max().item() * 1.5
    logp, ent = _exact(logits, tokens, 1.5)
    live = tokens != -100
    want = torch.where(live, logp.gather(1, tokens.clamp_min(0)[:, None])[:, 0], 0.0)
    assert ((got.logprobs.double() - want).abs() <= 2 * off + _err(V) + 4 * want.abs() * U).all()
    assert ((got.entropy.double() - torch.where(live, ent, 0.0)).abs() <= (2 * off + _err(V)) * (2 + math.log(V))).all()
    # gradients: every dlogit is rounded to bf16 (half a step 2^-8), the result once more; sums of independent roundings
    g, slack = _grad_want(logits, tokens, 1.5, gl, ge, None, None)
    g_err = g.abs() * 2.0 ** -8 + slack + 4 * off * g.abs()
    for a, b, e in ((dh, g @ w.detach().double(), g_err @ w.detach().double().abs()),
                    (dw, g.T @ h.detach().double(), g_err.T @ h.detach().double().abs())):
        assert ((a.double() - b).abs() <= e + b.abs() * 2.0 ** -8 + 1e-30).all()
    w.main_grad = torch.ones(V, D, device="cuda")
    dh2, = torch.autograd.grad([got.logprobs, got.entropy], [h], [gl, ge], retain_graph=True)
    assert torch.equal(dh, dh2)
    w.main_grad.fill_(1.0)      # (every pass through the node adds to the buffer)
    torch.autograd.backward([got.logprobs, got.entropy], [gl, ge])
    assert w.grad is None and ((w.main_grad.double() - 1 - g.T @ h.detach().double()).abs()
                               <= g_err.T @ h.detach().double().abs() + 2.0 ** -22 * (1 + w.main_grad.abs())).all()
    with torch.no_grad():
        again = ops.linear_logprobs(h, w, tokens, logit_scale=1.5, entropy=True, top=3)
    assert torch.equal(again.logprobs, got.logprobs) and torch.equal(again.top_tokens, got.top_tokens)
