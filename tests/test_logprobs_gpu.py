"""Token log probabilities on the GPU against a plain 64-bit implementation.

Tolerances. A sum of V exponentials in fp32 is off, relatively, by the exponential (2^-22), its
argument's rounding (|d| 2^-24 for a term exp(d); weighted by the terms themselves at most log V + 1)
and at most V / 256 + 64 additions: ts = 2^-22 + (log V + 1) 2^-23 + (V / 256 + 64) 2^-24. A log
probability (z - m) - log s adds one rounding of each part; the entropy log s - u / s carries ts on a
value of at most log V + 1 twice. The gradient is a product with p (ts, and |log p| 2^-22 for its
exponent), rounded once to the logits' type; the given tokens' own terms add 2^-22 of their sum.
"""

import math

import pytest
import torch

from nuvla_forge_b200 import _native as nat
from nuvla_forge_b200.ops import logprobs as lp
from nuvla_forge_b200.ops import token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _gen(seed):
    return torch.Generator(DEV).manual_seed(seed)


def _plain64(x, t, k, ignore, g_lp, g_h, g_top):
    z = x.double()
    dead = (z == -math.inf).all(-1)
    m = torch.where(dead, torch.zeros_like(z[:, 0]), z.amax(-1))
    e = (z - m[:, None]).exp()
    s = e.sum(-1)
    logp = (z - m[:, None]) - s.log()[:, None]
    p = e / s[:, None]
    plogp = torch.where(p > 0, p * logp, torch.zeros_like(p))
    H = -plogp.sum(-1)
    keep = t != ignore
    given = logp[torch.arange(len(t), device=t.device), torch.where(keep, t, torch.zeros_like(t))]
    given = torch.where(keep, given, torch.zeros_like(given))
    ids = torch.sort(x.float(), dim=-1, descending=True, stable=True)[1][:, :k]
    top = logp.gather(1, ids)
    whole = g_lp.double() * keep + g_top.double().sum(-1)
    dx = -(p * whole[:, None]) - g_h.double()[:, None] * (plogp + p * H[:, None])
    hot = torch.zeros_like(dx)
    at = torch.where(keep, t, torch.zeros_like(t))[:, None]
    hot.scatter_add_(1, at, (g_lp.double() * keep)[:, None])
    hot.scatter_add_(1, ids, g_top.double())
    big = torch.zeros_like(dx)
    big.scatter_add_(1, at, (g_lp.double().abs() * keep)[:, None])
    big.scatter_add_(1, ids, g_top.double().abs())
    V = x.shape[1]
    ts = 2.0 ** -22 + (math.log(V) + 1) * 2.0 ** -23 + (V / 256 + 64) * 2.0 ** -24
    mag = whole.abs()[:, None] + g_h.double().abs()[:, None] * (torch.where(p > 0, logp.abs(), torch.zeros_like(p)) + H[:, None] + 1)
    # the gradient's factor (g + e (log p + H)): its own rounding, and the error of log p + H (3 ts (log V + 1))
    rel = 2 * ts + (torch.where(p > 0, logp.abs(), torch.zeros_like(p)) + 4) * 2.0 ** -22
    tol_dx = p * (mag * rel + g_h.double().abs()[:, None] * 3 * ts * (math.log(V) + 1)) + big * 2.0 ** -22
    out = dict(given=given, H=H, top=top, ids=ids, dx=dx + hot, tol_dx=tol_dx, ts=ts)
    dead2 = dead[:, None]
    out["H"] = torch.where(dead, torch.zeros_like(H), H)
    out["given"] = torch.where(dead & keep, torch.full_like(given, -math.inf), torch.where(keep, given, torch.zeros_like(given)))
    out["top"] = torch.where(dead2, torch.full_like(top, -math.inf), top)
    for n in ("dx", "tol_dx"):
        out[n] = torch.where(dead2, torch.zeros_like(out[n]), out[n])
    return out


def _close(a, b, tol):
    inf = torch.isinf(b)
    assert torch.equal(a.double()[inf], b[inf])
    d = (a.double() - b)[~inf].abs()
    tol = (tol if torch.is_tensor(tol) else torch.full_like(b, tol))[~inf]
    assert (d <= tol).all(), float((d / tol).max())


def _check(x, t, k, seed=0, ignore=-100):
    g = _gen(seed + 100)
    M, V = x.shape
    g_lp, g_h, g_top = (torch.randn(s, generator=g, device=DEV) for s in ((M,), (M,), (M, k)))
    ref = _plain64(x, t, k, ignore, g_lp, g_h, g_top)
    leaf = x.detach().requires_grad_(True)
    r = token_logprobs(leaf, t, top_k=k, ignore_index=ignore)
    ts, logV = ref["ts"], math.log(V)
    _close(r.logprobs, ref["given"], ts + 2.0 ** -22 * (ref["given"].abs() + logV + 1))
    _close(r.entropy, ref["H"], 3 * ts * (logV + 1) + 2.0 ** -23)
    outs, grads = [r.logprobs, r.entropy], [g_lp, g_h]
    if k:
        assert r.top_tokens.dtype == torch.int64 and torch.equal(r.top_tokens, ref["ids"])
        _close(r.top_logprobs, ref["top"], ts + 2.0 ** -22 * (ref["top"].abs() + logV + 1))
        outs.append(r.top_logprobs)
        grads.append(g_top)
    else:
        assert r.top_tokens is None and r.top_logprobs is None
    (dx,) = torch.autograd.grad(outs, leaf, grads)
    assert dx.dtype == x.dtype and dx.shape == x.shape
    tiny = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -126, torch.float32: 2.0 ** -126}[x.dtype]
    _close(dx, ref["dx"], torch.finfo(x.dtype).eps / 2 * ref["dx"].abs() + ref["tol_dx"] * (1 + 2 ** -7) + tiny)
    lp.check_status()
    return r, dx


def _logits(M, V, dtype, seed, spread=2.0):
    g = _gen(seed)
    x = torch.randn(M, V, generator=g, device=DEV) * spread
    t = torch.randint(0, V, (M,), generator=g, device=DEV)
    x[torch.arange(M, device=DEV), t] += torch.rand(M, generator=g, device=DEV) * 12
    return x.to(dtype), t


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,V,k", [(1, 1, 1), (3, 2, 2), (1, 31, 31), (5, 32, 32), (4, 33, 5), (2, 1000, 0), (7, 4099, 20),
                                   (1, 32000, 5), (130, 32000, 5), (3, 32003, 32), (2, 65537, 7), (1, 151936, 32),
                                   (600, 2049, 1), (2, 300007, 10)])
def test_values_and_gradient(dtype, M, V, k):
    x, t = _logits(M, V, dtype, seed=M + V)
    if M > 2:
        t[1] = -100
    _check(x, t, k)


@pytest.mark.parametrize("dtype", TYPES)
def test_ties_take_the_lowest_index(dtype):
    """Rows of few distinct values, of one value, and of zeros of both signs."""
    g = _gen(1)
    for V in (40, 3000, 40000, 100001):
        x = torch.randint(-3, 4, (6, V), generator=g, device=DEV).to(dtype)
        x[0] = 1.5
        x[1] = 0.0
        x[1, ::2] = -0.0
        x[2] = torch.arange(V, device=DEV).float().clamp(max=60000).to(dtype) * 1e-3      # rising
        x[3] = -x[2]                                                                    # falling
        x[4] = -float("inf")
        x[4, V - 3:] = 2.0                                                              # fewer live ones than k
        t = torch.randint(0, V, (6,), generator=g, device=DEV)
        _check(x, t, 32)
        _check(x, t, 3)


@pytest.mark.parametrize("dtype", TYPES)
def test_masked_logits(dtype):
    """-inf and the type's lowest value in masked places, rows with nothing left, targets that are masked."""
    for V in (50, 32003):
        x, t = _logits(8, V, dtype, seed=V)
        low = torch.finfo(dtype).min
        x[0, ::2] = -float("inf")
        x[1, 1::3] = low
        x[2] = -float("inf")
        x[3] = low
        x[4] = -float("inf")
        x[4, 17] = 3.0
        t[4] = 17
        x[5, t[5]] = -float("inf")
        t[6] = -100
        x[6] = -float("inf")
        _check(x, t, 6)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [3, 40, 2001, 32003, 150001])
def test_rows_with_their_mass_on_one_token_keep_their_digits(dtype, V):
    """log p = -log(1 + r) for a small r: the relative error is that of r (ts), not 2^-24 / r; so is that of the
    gradient at the token, g r / (1 + r), and of the entropy (both parts positive)."""
    g = _gen(V)
    for M in (1, 5, 300):
        x = (torch.randn(M, V, generator=g, device=DEV) * 2).to(dtype)
        t = torch.randint(0, V, (M,), generator=g, device=DEV)
        x[torch.arange(M, device=DEV), t] = (14 + 8 * torch.rand(M, generator=g, device=DEV)).to(dtype)
        one, none = torch.ones(M, device=DEV), torch.zeros(M, device=DEV)
        ref = _plain64(x, t, 0, -100, one, none, torch.zeros(M, 0, device=DEV))
        lp64 = torch.log_softmax(x.double(), -1)
        r64 = torch.where(torch.nn.functional.one_hot(t, V).bool(), torch.zeros_like(lp64), (x.double() - x.double().gather(1, t[:, None])).exp()).sum(-1)
        leaf = x.clone().requires_grad_(True)
        r = token_logprobs(leaf, t, top_k=1)
        rel = ref["ts"] + 2.0 ** -21
        want = -torch.log1p(r64)
        assert ((r.logprobs.double() - want).abs() <= rel * want.abs()).all()
        assert torch.equal(r.top_logprobs[:, 0], r.logprobs) and torch.equal(r.top_tokens[:, 0], t)
        H = torch.log1p(r64) - ((lp64 - lp64.gather(1, t[:, None])).exp() * (x.double() - x.double().gather(1, t[:, None]))).sum(-1) / (1 + r64)
        assert ((r.entropy.double() - H).abs() <= 2 * rel * H + 2.0 ** -120).all()
        (dx,) = torch.autograd.grad(r.logprobs.sum(), leaf)
        at = dx.gather(1, t[:, None])[:, 0].double()
        tiny = {torch.float16: 2.0 ** -25}.get(dtype, 2.0 ** -126)
        assert ((at - r64 / (1 + r64)).abs() <= (rel + torch.finfo(dtype).eps / 2) * r64 + tiny).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_nan_and_infinite_logits_stay_in_their_rows(dtype):
    for V in (64, 40000):
        x, t = _logits(5, V, dtype, seed=3)
        x[1, 7] = float("nan")
        x[2, 9] = float("inf")
        x[3] = float("nan")
        leaf = x.clone().requires_grad_(True)
        r = token_logprobs(leaf, t, top_k=4)
        (dx,) = torch.autograd.grad(r.logprobs.sum() + r.entropy.sum() + r.top_logprobs.sum(), leaf)
        for i in (1, 2, 3):
            assert r.logprobs[i].isnan() and r.entropy[i].isnan() and dx[i].isnan().any()
        for i in (0, 4):
            assert r.logprobs[i].isfinite() and r.entropy[i].isfinite() and dx[i].isfinite().all()
        assert ((r.top_tokens >= 0) & (r.top_tokens < V)).all()


def test_strides_shapes_and_missing_targets():
    g = _gen(4)
    for dtype in TYPES:
        base = torch.randn(6, 5, 1003, generator=g, device=DEV).to(dtype)
        t = torch.randint(0, 1001, (6, 5), generator=g, device=DEV)
        whole = token_logprobs(base[..., 1:1002].contiguous(), t, top_k=3)
        cut = token_logprobs(base[..., 1:1002], t, top_k=3)                # rows that start anywhere
        for a, b in zip(whole, cut):
            assert a.shape == b.shape and torch.allclose(a.float(), b.float(), rtol=1e-5, atol=1e-5)
        col = token_logprobs(base[..., 1:1002].transpose(0, 1).contiguous().transpose(0, 1), t, top_k=3)
        assert torch.equal(col.top_tokens, whole.top_tokens)
        turned = base[0, :, 1:1002].T.contiguous().T                        # columns contiguous
        assert torch.equal(token_logprobs(turned, top_k=3).top_tokens, whole.top_tokens[0])
        same = token_logprobs(base[0, 0, :1000].expand(4, 1000), torch.arange(4, device=DEV))   # one row, four targets
        _check(base[0, 0, :1000].expand(4, 1000), torch.arange(4, device=DEV), 2)
        assert same.logprobs.shape == (4,)
        none = token_logprobs(base[0], top_k=2)
        assert none.logprobs is None and none.top_tokens.shape == (5, 2)
    empty = token_logprobs(torch.zeros(0, 10, device=DEV), torch.zeros(0, dtype=torch.int64, device=DEV), top_k=2)
    assert empty.logprobs.shape == (0,) and empty.top_tokens.shape == (0, 2)


def test_gradient_of_each_output_alone_and_of_an_empty_batch():
    x, t = _logits(5, 777, torch.float32, seed=5)
    t[2] = -100
    z = x.double()
    P = torch.softmax(z, -1)
    hot = torch.zeros_like(P)
    hot[torch.arange(5, device=DEV), t.clamp(min=0)] = 1
    hot[2] = 0
    H = -(P * P.log()).sum(-1, keepdim=True)
    want = {"logprobs": hot - P * (t != -100)[:, None], "entropy": -P * (P.log() + H)}
    for name, ref in want.items():
        leaf = x.clone().requires_grad_(True)
        r = token_logprobs(leaf, t, top_k=4)
        getattr(r, name).sum().backward()
        # 777 terms: ts is below 3e-5, factors below log V + 2
        assert (leaf.grad.double() - ref).abs().max() < 3e-5
    leaf = torch.zeros(0, 10, device=DEV, requires_grad=True)
    token_logprobs(leaf, torch.zeros(0, dtype=torch.int64, device=DEV)).logprobs.sum().backward()
    assert leaf.grad.shape == (0, 10)


def test_second_derivatives_are_refused():
    x, t = _logits(3, 100, torch.float32, seed=12)
    leaf, w = x.requires_grad_(True), torch.ones(3, device=DEV, requires_grad=True)
    (dx,) = torch.autograd.grad((token_logprobs(leaf, t).logprobs * w).sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        dx.square().sum().backward()


def test_gradient_against_differences():
    """Directional central differences of the 64-bit function; the gradient is computed in fp32."""
    x, t = _logits(3, 501, torch.float32, seed=6)
    g = _gen(60)
    g1, g2, g3 = (torch.randn(s, generator=g, device=DEV) for s in ((3,), (3,), (3, 5)))
    ids = torch.sort(x, dim=-1, descending=True, stable=True)[1][:, :5]

    def f(z):
        logp = torch.log_softmax(z, -1)
        return (logp.gather(1, t[:, None])[:, 0] * g1).sum() - ((logp.exp() * logp).sum(-1) * g2).sum() + \
            (logp.gather(1, ids) * g3).sum()

    leaf = x.clone().requires_grad_(True)
    r = token_logprobs(leaf, t, top_k=5)
    (dx,) = torch.autograd.grad([r.logprobs, r.entropy, r.top_logprobs], leaf, [g1, g2, g3])
    for _ in range(5):
        d = torch.randn(3, 501, generator=g, device=DEV, dtype=torch.float64)
        h = 1e-5
        num = float(f(x.double() + h * d) - f(x.double() - h * d)) / (2 * h)
        # |dx|_1 is below 60 here: its fp32 errors (ts < 3e-5 relative) and those of the differences (1e-8)
        assert abs(num - float((dx.double() * d).sum())) < 3e-5 * float((dx.double() * d).abs().sum()) + 1e-6


def test_bad_targets_are_reported_and_not_read():
    x, t = _logits(4, 1000, torch.bfloat16, seed=7)
    good = token_logprobs(x, t)
    for bad in (1000, -1, 2 ** 62, -2 ** 63):
        t2 = t.clone()
        t2[1] = bad
        leaf = x.clone().requires_grad_(True)
        r = token_logprobs(leaf, t2)
        assert r.logprobs[1].isnan() and torch.equal(r.logprobs[[0, 2, 3]], good.logprobs[[0, 2, 3]])
        r.entropy.sum().backward()
        assert leaf.grad.isfinite().all()
        with pytest.raises(RuntimeError, match="outside the vocabulary"):
            lp.check_status()
    own = token_logprobs(x, torch.where(t > 500, torch.full_like(t, -1), t), ignore_index=-1)
    assert torch.equal(own.logprobs == 0, t > 500)
    lp.check_status()


def test_captured_forward_and_backward_follow_new_inputs():
    x, t = _logits(64, 3001, torch.bfloat16, seed=8)
    static = x.clone().requires_grad_(True)
    gr = torch.cuda.CUDAGraph()
    g = torch.ones(64, device=DEV)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.autograd.grad(token_logprobs(static, t, top_k=3).logprobs, static, g)
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        r = token_logprobs(static, t, top_k=3)
        (dx,) = torch.autograd.grad(r.logprobs, static, g)
    y, t2 = _logits(64, 3001, torch.bfloat16, seed=9)
    with torch.no_grad():
        static.copy_(y)
    t.copy_(t2)
    gr.replay()
    torch.cuda.synchronize()
    leaf = y.clone().requires_grad_(True)
    e = token_logprobs(leaf, t2, top_k=3)
    (de,) = torch.autograd.grad(e.logprobs, leaf, g)
    assert torch.equal(r.logprobs, e.logprobs) and torch.equal(r.top_tokens, e.top_tokens) and torch.equal(dx, de)


def test_rows_past_32_bits():
    """Row offsets beyond 2^31 values: the last rows are read and their gradient written there."""
    V = 32000
    M = 2 ** 31 // V + 3
    x = torch.zeros(M, V, device=DEV, dtype=torch.bfloat16)
    y, t3 = _logits(3, V, torch.bfloat16, seed=10)
    x[-3:] = y
    t = torch.full((M,), -100, device=DEV)
    t[-3:] = t3
    leaf = x.requires_grad_(True)
    r = token_logprobs(leaf, t, top_k=2)
    one, none = torch.ones(3, device=DEV), torch.zeros(3, device=DEV)
    ref = _plain64(y, t3, 2, -100, one, none, torch.zeros(3, 2, device=DEV))
    # against the definition, not against a call of three rows: that one divides each row over several
    # blocks, so its sums are added in another order and either is within the tolerance of the exact value
    _close(r.logprobs[-3:].detach(), ref["given"], ref["ts"] + 2.0 ** -22 * (ref["given"].abs() + math.log(V) + 1))
    assert torch.equal(r.top_tokens[-3:], ref["ids"])
    (dx,) = torch.autograd.grad(r.logprobs.sum(), leaf)
    _close(dx[-3:], ref["dx"], torch.finfo(torch.bfloat16).eps / 2 * ref["dx"].abs() + ref["tol_dx"] * (1 + 2 ** -7) + 2.0 ** -126)
    assert not dx[:-3].any()


def test_repeats_are_bit_identical_and_native():
    x, t = _logits(700, 32003, torch.bfloat16, seed=11)
    nat.reset_launch_count()
    a = token_logprobs(x, t, top_k=8)
    assert nat.launch_count() == 1
    for _ in range(3):
        b = token_logprobs(x, t, top_k=8)
        assert all(torch.equal(p, q) for p, q in zip(a, b))
