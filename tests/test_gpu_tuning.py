"""-m gpu: the operators that tune a caption model on its samples (losses from logits, embedding with its sorted gradient, gradient norm and
clipping) against plain implementations in 64 bits on the same inputs.

Tolerances, in units u = 2^-24 (half a step of fp32):
  * one exponential: exp(t), t = x - max, is off by (3 |t| + 2) u relatively (the difference, its product with log2 e, that constant, and the
    instruction); under the softmax t averages below ln V, so a sum is off by less than (3 * 16 + 2) u from it, and by V / threads more where a
    thread adds its V / threads terms in fp32.  log-probability: (64 + V / 64) u absolutely, + u |logp| for the stored value.
  * a gradient w (1[c = id] - p): |w| times twice that (p and w both hang on it), p <= 1 and p |t| < 1: (256 + V / 32) u max|w| absolutely; a type of
    fewer bits adds half a step of the value, and fp16 half of its smallest step 2^-24."""
import math

import pytest
import torch

from tests.gpu_util import report

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
PAD = 1


@pytest.fixture(scope="module")
def ops():
    from bmt_amd import ops as o
    return o


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def within(got, want, tol, name):
    g, w = got.detach().double(), want.detach().double()
    assert g.shape == w.shape, (name, g.shape, w.shape)
    bad = ~(((g - w).abs() <= tol) | (torch.isnan(g) & torch.isnan(w)) | (g == w))
    assert not bool(bad.any()), report(got, want, name) + f"\n  {int(bad.sum())} of {bad.numel()} outside {tol if isinstance(tol, float) else float(tol.max()):.3e}"


def make_logits(kind, B, T, V, dtype, g, scale=2.5):
    def randn(*s):
        return (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)
    if kind == "plain":
        return randn(B, T, V)
    if kind == "shifted":
        return randn(B, T + 1, V)[:, :-1]
    if kind == "later":                # every row starts at an odd element
        return randn(B * T * V + 3)[3:].view(B, T, V)
    if kind == "padded":               # a vocabulary that was rounded up
        return randn(B, T, V + 13)[:, :, 5:V + 5]
    if kind == "transposed":
        return randn(T, B, V).transpose(0, 1)
    if kind == "columns":              # the vocabulary is not the last dimension
        return randn(B, V, T).transpose(1, 2)
    if kind == "sparse":               # much room between the rows
        return randn(B, 5 * T, V)[:, ::5]
    return randn(1, T, V).expand(B, T, V)


def logp64(x, ids):
    x = x.double()
    V = x.shape[-1]
    lp = torch.log_softmax(x, -1).gather(-1, ids.clamp(0, V - 1)[..., None])[..., 0]
    return torch.where((ids >= 0) & (ids < V), lp, torch.full_like(lp, float("nan")))


SHAPES = [(1, 1, 1), (3, 5, 7), (1, 1, 10000), (2, 3, 1000), (5, 7, 4099), (4, 150, 2051), (2, 2, 33001), (3, 1, 131075), (2, 1, 300001)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,V", SHAPES)
def test_token_logp_and_its_gradient(ops, dtype, B, T, V):
    g = gen(V + B)
    for kind in ("plain", "shifted"):
        x = make_logits(kind, B, T, V, dtype, g).requires_grad_(True)
        ids = torch.randint(0, V, (B, T), device="cuda", generator=g)
        mask = torch.rand(B, T, device="cuda", generator=g) > 0.3
        up = torch.randn(B, T, device="cuda", generator=g)
        got = ops.token_logp(x, ids, mask)
        (dx,) = torch.autograd.grad(got, x, up)
        lp = torch.where(mask, logp64(x.detach(), ids), torch.zeros(B, T, device="cuda", dtype=torch.float64))
        within(got, lp, (64 + V / 64) * U + U * lp.abs(), f"logp {kind}")
        w = torch.where(mask, up, torch.zeros_like(up)).double()
        want = -torch.softmax(x.detach().double(), -1) * w[..., None]
        want.scatter_add_(-1, ids[..., None], w[..., None])
        within(dx, want, (256 + V / 32) * U * w.abs().amax() + HALF[dtype] * want.abs() + TINY[dtype], f"dlogits {kind}")
        assert dx.dtype == dtype and bool((dx[~mask] == 0).all())


@pytest.mark.parametrize("kind", ["later", "padded", "transposed", "columns", "sparse", "expanded"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts_of_logits_ids_and_masks(ops, kind, dtype):
    B, T, V = 3, 6, 1237
    g = gen(7)
    x = make_logits(kind, B, T, V, dtype, g).requires_grad_(True)
    ids = torch.randint(0, V, (B, T + 1), device="cuda", generator=g)[:, 1:]
    mask = (torch.rand(T, B, device="cuda", generator=g) > 0.2).t()
    old = (logp64(x.detach(), ids) + 0.1).float().t().contiguous().t()
    adv = torch.randn(B, 1, device="cuda", generator=g)
    loss, stats = ops.policy_loss(x, ids, old, adv, mask=mask)
    (dx,) = torch.autograd.grad(loss, x)
    x64 = x.detach().double().requires_grad_(True)
    lp = logp64(x64, ids)
    want = policy64(lp, old, adv, None, mask)[0]
    (d64,) = torch.autograd.grad(want, x64)
    n = float(mask.sum())
    w = adv.abs().max() * 2 / n
    within(loss, want, (64 + V / 64) * U * 2 * float(adv.abs().max()) + U * abs(float(want.detach())), "loss")
    within(stats.logp, torch.where(mask, lp, torch.zeros_like(lp)), (64 + V / 64) * U + U * lp.abs(), "logp")
    within(dx, d64, (256 + V / 32) * U * w + HALF[dtype] * d64.abs(), "dlogits")


def policy64(lp, old, adv, ref, mask, lo=0.2, hi=0.2, beta=0.0, reduction="token"):
    adv = adv.double()
    adv = adv[:, None] if adv.dim() == 1 else adv
    rho = torch.exp(lp - old.double()) if old is not None else torch.exp(lp - lp.detach())
    u, c = rho * adv, rho.clamp(1 - lo, 1 + hi) * adv
    each = -torch.minimum(u, c)
    kl = torch.zeros_like(lp)
    if ref is not None:
        d = ref.double() - lp
        kl = torch.exp(d) - d - 1
        each = each + beta * kl
    m = mask.double()
    each = torch.where(mask, each, torch.zeros_like(each))
    n = m.sum().clamp(min=1)
    if reduction == "sum":
        loss = each.sum()
    elif reduction == "token":
        loss = each.sum() / n
    else:
        loss = (each.sum(1) / m.sum(1).clamp(min=1)).mean()
    return loss, (torch.where(mask, kl, torch.zeros_like(kl)).sum() / n).detach(), (((u > c) & mask).double().sum() / n).detach()


def policy_inputs(B, T, V, dtype, g, kl=True, per_token=False):
    x = make_logits("plain", B, T, V, dtype, g)
    ids = torch.randint(0, V, (B, T), device="cuda", generator=g)
    length = torch.randint(0, T + 1, (B, 1), device="cuda", generator=g)
    length[0] = T
    if B > 2:
        length[1] = 0
    mask = torch.arange(T, device="cuda")[None] < length
    lp = logp64(x, ids)
    off = 0.25 * torch.randn(B, T, device="cuda", generator=g).double()
    for border in (0.8, 1.3):          # (the gradient jumps there: no ratio within 1e-3 of a border)
        off = torch.where(((-off).exp() - border).abs() < 1e-3, off + 0.01, off)
    old = (lp + off).float()
    ref = (lp + 0.2 * torch.randn(B, T, device="cuda", generator=g)).float() if kl else None
    adv = torch.randn(*((B, T) if per_token else (B,)), device="cuda", generator=g)
    return x, ids, mask, old, ref, adv


@pytest.mark.parametrize("reduction", ["token", "sequence", "sum"])
@pytest.mark.parametrize("B,T,V,dtype", [(8, 1, 10000, torch.float32), (4, 29, 1000, torch.float32), (150, 130, 17, torch.float32), (3000, 1, 5, torch.bfloat16), (2, 900, 260, torch.float16),
                                         (1, 20, 32001, torch.bfloat16), (1, 600, 16385, torch.float32), (40, 29, 1501, torch.bfloat16), (3, 300, 777, torch.float16),
                                         (2, 2, 131075, torch.bfloat16), (1, 2, 300001, torch.float32), (700, 1, 4101, torch.float32)])
def test_policy_loss_and_its_gradient(ops, reduction, B, T, V, dtype):
    g = gen(B * T + V)
    for kl, beta in ((True, 0.1), (False, 0.0)):
        x, ids, mask, old, ref, adv = policy_inputs(B, T, V, dtype, g, kl, per_token=kl)
        x.requires_grad_(True)
        loss, stats = ops.policy_loss(x, ids, old, adv, ref, mask, None, 0.2, 0.3, beta, reduction)
        (dx,) = torch.autograd.grad(loss, x)
        lp = logp64(x.detach(), ids).requires_grad_(True)
        want, klm, clipped = policy64(lp, old, adv, ref, mask, 0.2, 0.3, beta, reduction)
        (w,) = torch.autograd.grad(want, lp)
        # every row's loss moves by |d loss / d lp| times the error of lp; ratios below 4 * 0.25 sigma: e
        e_lp = (64 + V / 64) * U
        rows = float((policy64(lp.detach(), old, adv, ref, mask, 0.2, 0.3, beta, "sum")[0]).abs()) if reduction == "sum" else 1.0
        within(loss, want, 4 * e_lp * float(adv.abs().max()) * (float(mask.sum()) if reduction == "sum" else 1.0) + U * rows + U * abs(float(want)), "loss")
        within(stats.kl, klm, 4 * e_lp + U * float(klm), "kl")
        within(stats.clip_fraction, clipped, U, "clip fraction")
        d = -torch.softmax(x.detach().double(), -1) * w[..., None]
        d.scatter_add_(-1, ids[..., None], w[..., None])
        within(dx, d, (256 + V / 32) * U * float(w.abs().max()) * 2 + HALF[dtype] * d.abs() + TINY[dtype], "dlogits")
        assert bool((dx[~mask] == 0).all())
        with torch.no_grad():          # the form without a gradient reads the rows another way
            loss2, stats2 = ops.policy_loss(x, ids, old, adv, ref, mask, None, 0.2, 0.3, beta, reduction)
        within(stats2.logp, stats.logp, 2 * e_lp + 2 * U * stats.logp.abs().double(), "logp of the two forms")
        assert not loss2.requires_grad and not stats.logp.requires_grad


def test_policy_loss_against_differences(ops):
    """d loss along a direction, from the 64-bit loss at two near points: off by (step^2 / 6) times the third derivative, far below the tolerance"""
    g = gen(3)
    x, ids, mask, old, ref, adv = policy_inputs(4, 9, 501, torch.float32, g)
    x.requires_grad_(True)
    loss, _ = ops.policy_loss(x, ids, old, adv, ref, mask, None, 0.2, 0.3, 0.1, "token")
    (dx,) = torch.autograd.grad(loss, x)
    for _ in range(3):
        way = torch.randn(*x.shape, device="cuda", generator=g).double()
        at = lambda h: policy64(logp64(x.detach().double() + h * way, ids), old, adv, ref, mask, 0.2, 0.3, 0.1, "token")[0]      # noqa: E731
        want = (at(1e-5) - at(-1e-5)) / 2e-5
        tol = (256 + 501 / 32) * U * 2 * float(adv.abs().max()) * float(way.abs().sum()) / float(mask.sum()) + 1e-8
        within((dx.double() * way).sum(), want, tol, "directional derivative")


def test_policy_loss_upstream_gradient_and_kept_graphs(ops):
    g = gen(11)
    x, ids, mask, old, ref, adv = policy_inputs(5, 17, 1234, torch.bfloat16, g)
    x.requires_grad_(True)

    def loss():
        return ops.policy_loss(x, ids, old, adv, ref, mask, None, 0.2, 0.2, 0.05, "token")[0]
    (one,) = torch.autograd.grad(loss(), x)
    kept = loss()
    (a,) = torch.autograd.grad(kept * 0.5, x, retain_graph=True)
    (b,) = torch.autograd.grad(kept, x, retain_graph=True)
    (c,) = torch.autograd.grad(kept, x)
    # halving is exact in bf16 (no value of these is subnormal); the recomputed gradient takes the same steps as the fused one
    assert torch.equal(a, (one * 0.5)) and torch.equal(b, one) and torch.equal(c, one)
    (kept2 := loss()).backward()
    x2 = x.grad.clone()
    loss().backward()                  # accumulates
    assert torch.equal(x2, one) and torch.equal(x.grad, one + one)
    x.grad = None
    kept3 = loss()
    with torch.no_grad():
        x.add_(1.0)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        kept3.backward()


def test_rows_that_do_not_count_leak_nothing(ops):
    """NaN and infinities behind the mask, a batch whose mask leaves nothing, ids that only masked rows may hold"""
    B, T, V = 4, 5, 999
    g = gen(5)
    for dtype in (torch.float32, torch.float16):
        x, ids, _, old, ref, adv = policy_inputs(B, T, V, dtype, g)
        ids = ids.clamp(min=2)
        ids[1] = PAD
        ids[2, 3:] = PAD
        x[1, 0], x[1, 1], x[1, 2, ::2], x[1, 3] = float("nan"), float("inf"), -float("inf"), -float("inf")
        old[1], ref[1] = float("nan"), float("inf")
        x.requires_grad_(True)
        for reduction in ("token", "sequence", "sum"):
            loss, stats = ops.policy_loss(x, ids, old, adv, ref, None, PAD, 0.2, 0.2, 0.1, reduction)
            (dx,) = torch.autograd.grad(loss, x)
            assert bool(torch.isfinite(loss)) and bool(torch.isfinite(dx).all()) and bool((dx[1] == 0).all()) and bool((dx[2, 3:] == 0).all())
            assert bool((stats.logp[1] == 0).all()) and bool(torch.isfinite(stats.kl))
        none = torch.zeros(B, T, dtype=torch.bool, device="cuda")
        ids[0, 0] = V + 7
        loss, stats = ops.policy_loss(x, ids, old, adv, ref, none)
        (dx,) = torch.autograd.grad(loss, x)
        assert float(loss) == 0.0 and float(stats.kl) == 0.0 and float(stats.clip_fraction) == 0.0 and bool((dx == 0).all())
        lp = ops.token_logp(x, ids, none)
        assert bool((lp == 0).all()) and bool((torch.autograd.grad(lp.sum(), x)[0] == 0).all())
        # an id outside the vocabulary in a row that counts is loud
        assert bool(torch.isnan(ops.token_logp(x.detach(), ids)[0, 0])) and bool(torch.isnan(ops.policy_loss(x, ids, old, adv, ref, None, PAD)[0]))


def test_nothing_is_held_where_no_graph_is_recorded(ops):
    x = torch.randn(4, 64, 4096, device="cuda", requires_grad=True)
    ids = torch.randint(0, 4096, (4, 64), device="cuda")
    row, seq = torch.zeros(4, 64, device="cuda"), torch.zeros(4, device="cuda")
    for call in (lambda: ops.policy_loss(x, ids, row, seq), lambda: ops.preference_loss(x, ids, seq), lambda: ops.token_logp(x, ids)):
        torch.cuda.reset_peak_memory_stats()
        held = torch.cuda.memory_allocated()
        with torch.no_grad():
            call()
        assert torch.cuda.max_memory_allocated() - held < x.numel() * 4 // 8


def test_vocabularies_with_forbidden_tokens(ops):
    """-inf and the type's lowest value among the logits: probability 0 and gradient 0 there, and a row of nothing but the lowest value is uniform"""
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        V = 1003
        x = make_logits("plain", 1, 4, V, dtype, gen(2))
        ids = torch.tensor([[5, 6, 7, 8]], device="cuda")
        x[0, 0, 100:] = -float("inf")
        x[0, 1, 100:] = torch.finfo(dtype).min
        x[0, 2] = torch.finfo(dtype).min
        x[0, 3, ::2] = -float("inf")
        x[0, 3, 8] = 1.0
        x.requires_grad_(True)
        lp = ops.token_logp(x, ids)
        (dx,) = torch.autograd.grad(lp.sum(), x)
        want = logp64(x.detach(), ids)
        within(lp, want, (64 + V / 64) * U + U * want.abs(), "logp")
        assert bool((dx[0, 0, 100:] == 0).all()) and bool((dx[0, 1, 100:] == 0).all()) and bool(torch.isfinite(dx).all())
        assert abs(float(lp[0, 2]) + math.log(V)) <= (64 + V / 64) * U + U * math.log(V)
        y = x.detach().clone()
        y[0, 0], y[0, 1, 3] = -float("inf"), float("nan")
        y[0, 2, 9] = float("inf")
        lp = ops.token_logp(y, ids)          # a row without any probability, a NaN, an infinity: NaN, and only there
        assert bool(torch.isnan(lp[0, :3]).all()) and bool(torch.isfinite(lp[0, 3]))


def test_policies_that_lie_far_apart(ops):
    """ratios from 0 to beyond fp32's exponential: the clipped side where the advantage asks for it, the ratio itself elsewhere"""
    V, B = 40, 6
    x = torch.zeros(B, 1, V, device="cuda")
    x[5, 0, 3] = -float("inf")                      # the sampled token has no probability any more
    x.requires_grad_(True)
    ids = torch.full((B, 1), 3, device="cuda")
    lp = -math.log(V)
    old = torch.tensor([lp - 3.0, lp + 3.0, lp - 0.4999, lp + 0.5001, lp - 60.0, lp], device="cuda")[:, None]
    for sign in (1.0, -1.0):
        adv = torch.full((B,), sign, device="cuda")
        loss, stats = ops.policy_loss(x, ids, old, adv, reduction="sum")
        (dx,) = torch.autograd.grad(loss, x)
        rho = torch.tensor([math.exp(lp - o) for o in old[:5, 0].double().tolist()] + [0.0], dtype=torch.float64, device="cuda")
        u, c = rho * sign, rho.clamp(0.8, 1.2) * sign
        want = -torch.minimum(u, c).sum()
        # lp to (64 + V / 64) u, old to u |old|: the ratios to their sum relatively
        tol = (66 + abs(lp) + 60) * U
        within(loss, want, tol * float(rho.sum() if sign < 0 else 8.0), "loss")
        w = -torch.where(u <= c, u, torch.zeros_like(u))
        within(dx[:5, 0, 3], w[:5] * (1 - 1 / V), 2 * tol * w[:5].abs(), "dlogits at the tokens")
        assert float(dx[5].abs().max()) == 0.0


def test_on_policy_samples(ops):
    g = gen(9)
    x, ids, mask, _, ref, adv = policy_inputs(3, 8, 300, torch.float32, g)
    x.requires_grad_(True)
    loss, stats = ops.policy_loss(x, ids, None, adv, ref, mask, kl_coef=0.1)
    (dx,) = torch.autograd.grad(loss, x)
    x64 = x.detach().double().requires_grad_(True)
    want = policy64(logp64(x64, ids), None, adv, ref, mask, beta=0.1)[0]
    (d64,) = torch.autograd.grad(want, x64)
    within(loss, want, 4 * (64 + 300 / 64) * U + U, "loss")
    within(dx, d64, (256 + 300 / 32) * U * 2 * float(adv.abs().max()) / float(mask.sum()), "dlogits")
    assert float(stats.clip_fraction) == 0.0


def preference64(lp, ref, mask, beta, ls, mean):
    m = mask.double()
    S = torch.where(mask, lp, torch.zeros_like(lp)).sum(1)
    if mean:
        S = S / m.sum(1).clamp(min=1)
    r = beta * (S - ref.double())
    P = lp.shape[0] // 2
    z = r[:P] - r[P:]
    return -((1 - ls) * torch.nn.functional.logsigmoid(z) + ls * torch.nn.functional.logsigmoid(-z)).mean(), r


@pytest.mark.parametrize("B,T,V,dtype", [(2, 1, 10000, torch.float32), (6, 29, 1000, torch.float32), (8, 70, 1501, torch.bfloat16), (2, 300, 2777, torch.float16),
                                         (4, 2, 300001, torch.float32), (600, 3, 65, torch.float32)])
@pytest.mark.parametrize("ls,mean", [(0.0, False), (0.1, True)])
def test_preference_loss_and_its_gradient(ops, B, T, V, dtype, ls, mean):
    g = gen(B + T + V)
    x = make_logits("shifted", B, T, V, dtype, g).requires_grad_(True)
    ids = torch.randint(2, max(V, 3), (B, T), device="cuda", generator=g)
    mask = torch.rand(B, T, device="cuda", generator=g) > 0.2
    if B > 2:
        mask[B - 1] = False          # a rejected caption that holds nothing
    ref = (preference64(logp64(x.detach(), ids), torch.zeros(B, device="cuda"), mask, 1.0, 0.0, mean)[1] + torch.randn(B, device="cuda", generator=g)).float()
    loss, rewards = ops.preference_loss(x, ids, ref, mask, beta=0.3, label_smoothing=ls, mean_logp=mean)
    (dx,) = torch.autograd.grad(loss * 2.0, x)
    lp = logp64(x.detach(), ids).requires_grad_(True)
    want, r = preference64(lp, ref, mask, 0.3, ls, mean)
    (w,) = torch.autograd.grad(want * 2.0, lp)
    # a sequence's sum is off by T times a log-probability's error and the rounding of its T stored values
    e = 0.3 * (T if not mean else 1) * ((64 + V / 64) * U + U * float(lp.detach().abs().max()))
    within(rewards, r, e + U * r.abs(), "rewards")
    within(loss, want, 2 * e + U * abs(float(want)), "loss")
    d = -torch.softmax(x.detach().double(), -1) * w[..., None]
    d.scatter_add_(-1, ids[..., None], w[..., None])
    # w moves by 0.3 * e (the sigmoid's slope is below 1) beside its own rounding
    wmax = float(w.abs().max())
    within(dx, d, (256 + V / 32) * U * wmax + 2 * e * wmax + HALF[dtype] * d.abs() + TINY[dtype], "dlogits")
    assert bool((dx[~mask] == 0).all())
    with torch.no_grad():
        assert torch.equal(ops.preference_loss(x, ids, ref, mask, beta=0.3, label_smoothing=ls, mean_logp=mean)[0], loss)


def test_preference_of_impossible_tokens(ops):
    """a rejected caption of probability 0 is as bad as can be: z = inf, loss 0, no gradient; the preferred one: loss inf"""
    V = 50
    x = torch.zeros(2, 1, V, device="cuda")
    x[1, 0, 7] = -float("inf")
    ids = torch.full((2, 1), 7, device="cuda")
    loss, r = ops.preference_loss(x, ids, torch.zeros(2, device="cuda"))
    assert float(loss) == 0.0 and float(r[1]) == -float("inf")
    assert float(ops.preference_loss(x.flip(0).contiguous(), ids, torch.zeros(2, device="cuda"))[0]) == float("inf")


# ----------------------------------------------------------------------------- embedding
def embedding64(ids, W, scale, dout, pad):
    V, D = W.shape
    i = ids.clamp(0, V - 1)
    s = float(torch.tensor(scale, dtype=torch.float32))
    out = W.double()[i] * s
    dW, absum, most = torch.zeros(V, D, device="cuda", dtype=torch.float64), torch.zeros(V, D, device="cuda", dtype=torch.float64), 0
    if dout is not None and ids.numel():
        keep = ids.reshape(-1) != (-1 << 62 if pad is None else pad)
        flat = i.reshape(-1)[keep]
        d = dout.reshape(-1, D)[keep].double() * s
        dW.index_put_((flat,), d, accumulate=True)
        absum.index_put_((flat,), d.abs(), accumulate=True)
        most = int(torch.bincount(flat, minlength=1).max()) if flat.numel() else 0
    return out, dW, absum, most


def check_embedding(ops, ids, W, scale, dout, pad, name):
    W = W.detach().requires_grad_(True)
    out = ops.embedding(ids, W, scale, pad)
    (dW,) = torch.autograd.grad(out, W, dout)
    want, d64, absum, most = embedding64(ids, W.detach(), scale, dout, pad)
    half, tiny = HALF[W.dtype], TINY[W.dtype]
    within(out, want, (half + U) * want.abs() + tiny, f"{name} out")          # the product in fp32, then the type
    # additions a value passes through: up to 2048 positions at most 32 of one wave, or a quarter of a token's positions and the 3 sums of the
    # quarters; beyond, 32 positions and then a quarter of their sums, and 3.  + the scale (and the type)
    within(dW, d64, (36 + most / (4 if ids.numel() <= 2048 else 32)) * U * absum + half * d64.abs() + tiny, f"{name} dW")
    assert torch.equal(dW, torch.autograd.grad(ops.embedding(ids, W, scale, pad), W, dout)[0]), name      # the same bits
    with torch.no_grad():
        assert torch.equal(ops.embedding(ids, W, scale, pad), out)
    return dW


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("N,V,D", [((1,), 1, 1), ((3, 1), 7, 3), ((31,), 10, 64), ((33,), 3, 300), ((32, 29), 10000, 300), ((5, 1000), 997, 66), ((40, 500), 50000, 36),
                                   ((66, 1000), 2000, 20), ((2, 3, 4), 300007, 1024), ((4096,), 1, 130), ((2, 6000), 300007, 12), ((300, 1000), 70000, 8), ((9000,), 2, 16),
                                   ((9001,), 600000, 4)])
def test_embedding_and_its_gradient(ops, dtype, N, V, D):
    g = gen(V + D)
    W = (0.4 * torch.randn(V, D, device="cuda", generator=g)).to(dtype)
    ids = (torch.rand(*N, device="cuda", generator=g) ** 6 * V).long().clamp(max=V - 1)          # few tokens hold most positions
    dout = torch.randn(*N, D, device="cuda", generator=g).to(dtype)
    dW = check_embedding(ops, ids, W, math.sqrt(D), dout, None, "zipf")
    seen = torch.zeros(V, dtype=torch.bool, device="cuda")
    seen[ids.reshape(-1)] = True
    assert bool((dW[~seen] == 0).all())


@pytest.mark.parametrize("what", ["all_one", "all_pad", "two", "runs", "outside", "none"])
def test_embedding_of_uncommon_batches(ops, what):
    V, D, n, g = 500, 48, 3000, gen(1)
    ids = torch.randint(0, V, (n,), device="cuda", generator=g)
    if what == "all_one":
        ids[:] = 17
    elif what == "all_pad":
        ids[:] = PAD
    elif what == "two":                  # two long runs that meet inside a run of 32, and short ones around them
        ids[:40], ids[40:1111], ids[1111:2500] = 3, 8, 9
    elif what == "runs":                 # runs of 31, 32, 33, 64 positions of the sorted order
        ids = torch.cat([torch.full((k,), v, device="cuda") for v, k in enumerate((31, 32, 33, 64, 1, 0, 65, 32, 96, 33))]).long()
        ids = ids[torch.randperm(len(ids), device="cuda", generator=g)]
    elif what == "outside":              # clamped to the table, as the framework's other lookups do
        ids[::3], ids[1::3] = -5, V + 1000
    else:
        ids = ids[:0]
    W = torch.randn(V, D, device="cuda", generator=g)
    dout = torch.randn(ids.numel(), D, device="cuda", generator=g)
    dW = check_embedding(ops, ids, W, 2.0, dout, PAD, what)
    assert bool((dW[PAD] == 0).all())


def test_embedding_layouts(ops):
    """a table inside a wider buffer, ids and gradients with strides, one gradient for all positions, rows at odd addresses"""
    g = gen(4)
    for dtype in (torch.float32, torch.bfloat16):
        wide = torch.randn(200, 80, device="cuda", generator=g).to(dtype)
        odd = torch.randn(200 * 33 + 1, device="cuda", generator=g).to(dtype)[1:].view(200, 33)
        ids = torch.randint(0, 200, (11, 14), device="cuda", generator=g).t()[:, ::2]
        for name, W in (("columns", wide[:, 3:67]), ("transposed", wide.t()[:, :64]), ("odd", odd), ("expanded", wide[:, :1].expand(200, 40))):
            W = W[:80] if name == "transposed" else W
            i = ids.clamp(max=W.shape[0] - 1)
            D = W.shape[1]
            dout = torch.randn(*i.shape, 2 * D, device="cuda", generator=g).to(dtype)
            check_embedding(ops, i, W, 1.5, dout[..., :D], None, name)
            check_embedding(ops, i, W, 1.5, dout[:1, :1, :D].expand(*i.shape, D), None, name + " one gradient")


@pytest.mark.parametrize("D,N", [(40, 60), (37, 60), (3, 900), (1, 10), (301, 900)])
def test_embedding_into_a_static_gradient_buffer(ops, D, N):
    from bmt_amd.parallel import GradientReducer
    g = gen(6)
    other = torch.nn.Parameter(torch.zeros(3, device="cuda"))          # (the table's buffer starts behind it, at an odd element)
    W = torch.nn.Parameter(torch.randn(300, D, device="cuda", generator=g))
    red = GradientReducer([other, W], overlap=False)
    ids = torch.randint(0, 50, (4, N), device="cuda", generator=g)
    dout = torch.randn(4, N, D, device="cuda", generator=g)
    red.zero_grad()
    W.grad[7] += 3.0
    ops.embedding(ids, W, 2.0, PAD).backward(dout)
    ops.embedding(ids, W, 2.0, PAD).backward(dout)
    _, d64, absum, most = embedding64(ids, W.detach(), 2.0, dout, PAD)
    d64 *= 2
    d64[7] += 3.0
    within(W.grad, d64, (36 + most / (4 if ids.numel() <= 2048 else 32)) * U * 2 * absum + 4 * U * d64.abs(), "static gradient")
    red.remove()


# ----------------------------------------------------------------------------- gradient norm and clipping
def gradients(g, odd=True):
    shapes = [(1000, 300), (7,), (0, 5), (8192,), (8193,), (1,), (), (64, 33), (3, 5, 7), (40000,), (2, 0)]
    kinds = [torch.float32, torch.bfloat16, torch.float16]
    ts = []
    for k, s in enumerate(shapes):
        n = math.prod(s)
        base = torch.randn(n + 3, device="cuda", generator=g).to(kinds[k % 3])
        ts.append(base[(k % 4 if odd else 0):][:n].view(s))
    ts.append(torch.randn(50, 60, device="cuda", generator=g).t())          # dense in another order
    return ts


def norm64(ts, inf):
    flat = torch.cat([t.double().reshape(-1) for t in ts])
    return flat.abs().max() if inf else flat.norm()


@pytest.mark.parametrize("norm_type", [2.0, float("inf")])
@pytest.mark.parametrize("where", ["in_place", "fp32", "bf16_odd"])
@pytest.mark.parametrize("max_norm", [0.5, 1e9])
def test_gradient_norm_and_clipping(norm_type, where, max_norm):
    from bmt_amd.optim import GradClipper
    ts = gradients(gen(8))
    before = [t.clone() for t in ts]
    if where == "in_place":
        outs = None
    else:
        dt = torch.float32 if where == "fp32" else torch.bfloat16
        outs = [torch.full((t.numel() + 1,), 7.0, device="cuda", dtype=dt)[where != "fp32":][:t.numel()].view(t.shape) if t.is_contiguous()
                else torch.empty_like(t, dtype=dt) for t in ts]
    scale = torch.tensor([0.25], device="cuda")
    for s in (None, scale):
        for t, b in zip(ts, before):
            t.copy_(b)
        clip = GradClipper(ts, max_norm, outs, norm_type)
        want = norm64(before, norm_type != 2.0) * (1.0 if s is None else 0.25)
        only = clip(s, apply=False)
        assert all(torch.equal(t, b) for t, b in zip(ts, before))
        got = clip(s)
        assert torch.equal(got, only)
        within(got, want, U * float(want), "norm")          # 64-bit sums: the stored value's rounding
        coef = min(1.0, max_norm / (float(want) + 1e-6)) * (1.0 if s is None else 0.25)
        within(clip.coef, torch.tensor(coef), 4 * U * coef, "coef")
        for t, b in zip(outs or ts, before):
            w = b.double() * coef
            # the factor's and the product's rounding, then the type's
            within(t, w, 6 * U * w.abs() + HALF[t.dtype] * w.abs() + TINY[t.dtype], "clipped")
        if outs is not None:
            assert all(torch.equal(t, b) for t, b in zip(ts, before))


def test_gradient_norm_of_extreme_values():
    from bmt_amd.optim import GradClipper
    big = torch.full((5000,), 1e30, device="cuda")          # squares beyond fp32
    assert abs(float(GradClipper([big], 1.0)(apply=False)) / (1e30 * math.sqrt(5000)) - 1) < 1e-6
    small = torch.full((5000,), 1e-30, device="cuda")
    assert abs(float(GradClipper([small], 1.0)(apply=False)) / (1e-30 * math.sqrt(5000)) - 1) < 1e-6
    for norm_type in (2.0, float("inf")):
        a, b = torch.ones(10, device="cuda"), torch.ones(9000, device="cuda")
        b[8999] = float("inf")
        assert float(GradClipper([a, b], 1.0, norm_type=norm_type)()) == float("inf")
        assert bool((a == 0).all()) and bool(torch.isnan(b[8999])) and bool((b[:8999] == 0).all())          # as torch does: inf * 0
        a, b = torch.ones(10, device="cuda"), torch.ones(9000, device="cuda")
        a[3], b[5] = float("nan"), float("inf")
        assert bool(torch.isnan(GradClipper([a, b], 1.0, norm_type=norm_type)())) and bool(torch.isnan(a).all()) and bool(torch.isnan(b).all())
        zero = [torch.zeros(3, device="cuda"), torch.zeros(0, device="cuda")]
        assert float(GradClipper(zero, 1.0, norm_type=norm_type)()) == 0.0
        assert float(GradClipper([zero[1]], 1.0, norm_type=norm_type)()) == 0.0
    neg = [torch.tensor([3.0, -4.0], device="cuda")]
    assert float(GradClipper(neg, 1.0)(torch.tensor(-1.0, device="cuda"))) == 5.0 and float(neg[0][0]) < 0


def test_clipper_refuses_what_it_cannot_do():
    from bmt_amd.optim import GradClipper
    a = torch.randn(100, device="cuda")
    for bad in ([a, a], [a[:50], a[40:]], [a[::2]], [a.double()], [a.long()], []):
        with pytest.raises(ValueError):
            GradClipper(bad, 1.0)
    for out in ([a[1:]], [torch.empty(99, device="cuda")], [], [torch.empty(10, 10, device="cuda")]):
        with pytest.raises(ValueError):
            GradClipper([a], 1.0, out)
    with pytest.raises(ValueError):
        GradClipper([torch.randn(4, 5, device="cuda")], 1.0, [torch.empty(5, 4, device="cuda").t()])
    for kw in (dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(max_norm=1.0, norm_type=1.0), dict(max_norm=1.0, eps=-1.0)):
        with pytest.raises(ValueError):
            GradClipper([a], **kw)
    clip = GradClipper([a], 1.0)
    with pytest.raises(ValueError):
        clip(scale=torch.ones(2, device="cuda"))
    a.set_(torch.randn(100, device="cuda"))
    with pytest.raises(RuntimeError, match="moved"):
        clip()


def test_losses_refuse_device_tensors_of_the_wrong_kind(ops):
    x, ids = torch.zeros(2, 3, 5, device="cuda"), torch.zeros(2, 3, device="cuda", dtype=torch.int64)
    row = torch.zeros(2, 3, device="cuda")
    for kw in (dict(advantages=None), dict(advantages=torch.zeros(3, device="cuda")), dict(advantages=row.double()), dict(old_logp=row[:, :1]), dict(ref_logp=row[0]),
               dict(reduction="mean"), dict(kl_coef=0.1), dict(clip_low=-0.1), dict(clip_high=float("nan"))):
        with pytest.raises(ValueError):
            ops.policy_loss(x, ids, **{"old_logp": row, "advantages": row, **kw})
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.policy_loss(x, ids, row, row.cpu())
    with pytest.raises(ValueError):
        ops.policy_loss(x[:0], ids[:0], row[:0], row[:0])
    for bad in ((x[:1], ids[:1], row[0, :1]), (x, ids, row), (x, ids, row[:, 0].double()), (x[:, :0], ids[:, :0], row[:, 0])):
        with pytest.raises(ValueError):
            ops.preference_loss(*bad)
    with pytest.raises(ValueError):
        ops.preference_loss(x, ids, row[:, 0], label_smoothing=1.1)
    for bad in ((ids.int(), row), (ids, row[0]), (ids, row.double()), (ids, row[:, :0])):
        with pytest.raises(ValueError):
            ops.embedding(*bad)
    assert ops.token_logp(x[:0], ids[:0]).shape == (0, 3) and ops.token_logp(x[:, :0], ids[:, :0]).shape == (2, 0)


# ----------------------------------------------------------------------------- together, on streams, in graphs
def tuning_step(ops, W, head, ids, old, ref, adv, clipper):
    """embed -> a linear head -> policy loss -> gradients -> clipping, over static gradient buffers"""
    e = ops.embedding(ids, W, math.sqrt(W.shape[1]), PAD)
    loss, stats = ops.policy_loss(e @ head, ids.roll(-1, 1), old, adv, ref, None, PAD, kl_coef=0.1)
    dW, dh = torch.autograd.grad(loss, (W, head))
    clipper.grads[0].copy_(dW)
    clipper.grads[1].copy_(dh)
    return loss.detach(), stats.kl, clipper(), clipper.grads[0], clipper.grads[1]


def step_inputs(seed, V=600, D=32, B=6, T=20):
    g = gen(seed)
    ids = torch.randint(2, V, (B, T), device="cuda", generator=g)
    ids[0, 10:] = PAD
    old = -6.0 + 0.3 * torch.randn(B, T, device="cuda", generator=g)
    return ids, old, old + 0.1, torch.randn(B, device="cuda", generator=g)


def test_a_step_on_a_side_stream_and_in_a_graph(ops):
    from bmt_amd.optim import GradClipper
    g = gen(21)
    W = (0.1 * torch.randn(600, 32, device="cuda", generator=g)).requires_grad_(True)
    head = (0.1 * torch.randn(32, 600, device="cuda", generator=g)).requires_grad_(True)
    bufs = [torch.zeros_like(W), torch.zeros_like(head)]
    clipper = GradClipper([b.detach() for b in bufs], 0.01)
    batches = [step_inputs(s) for s in (1, 2, 3)]
    want = [[t.clone() for t in tuning_step(ops, W, head, *b, clipper)] for b in batches]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for b, w in zip(batches, want):
            got = [t.clone() for t in tuning_step(ops, W, head, *b, clipper)]
            side.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(got, w))
    static = [t.clone() for t in batches[0]]
    side = torch.cuda.Stream()
    alone = torch.cuda.CUDAGraph()
    lonely = [torch.full((5000,), 3.0, device="cuda")]
    plans = [GradClipper(lonely, 1.0)]
    with torch.cuda.graph(alone):          # a graph that outlives its plan
        norm = plans.pop()()
    junk = [torch.full((4096,), float("nan"), device="cuda") for _ in range(64)]
    for _ in range(2):
        lonely[0].fill_(3.0)
        alone.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - 3.0 * math.sqrt(5000)) < 1e-3 and abs(float(lonely[0].norm()) - 1.0) < 1e-5
    del junk
    clippers = [GradClipper([torch.zeros_like(W).detach(), torch.zeros_like(head).detach()], 0.01) for _ in range(2)]
    graphs, outs = [], []
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for c in clippers:
            tuning_step(ops, W, head, *static, c)
    torch.cuda.current_stream().wait_stream(side)
    for c in clippers:          # two graphs of the same step: neither shares a workspace with the other
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(tuning_step(ops, W, head, *static, c))
        graphs.append(graph)
    for turn in range(2):
        for b, w in zip(batches, want):
            for s, t in zip(static, b):
                s.copy_(t)
            for graph in graphs:
                graph.replay()
            torch.cuda.synchronize()
            for o in outs:
                assert all(torch.equal(x, y) for x, y in zip(o, w)), turn
            eager = tuning_step(ops, W, head, *b, clipper)
            assert all(torch.equal(x, y) for x, y in zip(eager, w))


def test_caption_model_tuned_on_samples(ops):
    """the caption model's own decoder states and generator under PolicyLoss and PreferenceLoss: the parameters' gradients are those of the plain
    losses on the same log-probabilities; then clipped and stepped"""
    from bmt_amd import synthetic as syn
    from bmt_amd.loss.policy import PolicyLoss, PreferenceLoss
    from bmt_amd.model.captioning_module import BiModalTransformer
    from bmt_amd.optim import FusedAdam, GradClipper
    from bmt_amd.train import make_masks
    cfg = syn.cfg_config0(dout_p=0.0)
    cfg.device = "cuda:0"
    torch.manual_seed(0)
    V, B, T = 60, 4, 9
    model = BiModalTransformer(cfg, syn.FakeTrainDataset(V, syn.make_glove(V, cfg.d_model_caps))).to("cuda:0")
    batch = syn.make_cap_batch(cfg, B, 12, 40, T, V, seed=5)
    fs = {k: v.cuda() for k, v in batch["feature_stacks"].items()}
    caps = batch["captions"].cuda()
    x, y = caps[:, :-1].contiguous(), caps[:, 1:]
    masks = make_masks(fs, x, "audio_video", syn.PAD_IDX)
    params = [p for p in model.parameters() if p.requires_grad]
    valid = y != syn.PAD_IDX
    g = gen(31)
    with torch.no_grad():
        base = ops.token_logp(model(fs, x, masks), y, pad_idx=syn.PAD_IDX)
    old, ref = base + 0.05 * torch.randn(*y.shape, device="cuda", generator=g), base + 0.05 * torch.randn(*y.shape, device="cuda", generator=g)
    adv = torch.randn(B, device="cuda", generator=g)

    def plain_policy(pred):
        lp = pred.gather(-1, y[..., None])[..., 0].double()
        return policy64(lp, old, adv, ref, valid, 0.2, 0.2, 0.1, "token")[0].float()

    def plain_preference(pred):
        lp = pred.gather(-1, y[..., None])[..., 0].double()
        return preference64(lp, (ref * valid).sum(1), valid, 0.1, 0.0, False)[0].float()

    policy, preference = PolicyLoss(pad_idx=syn.PAD_IDX, kl_coef=0.1), PreferenceLoss(pad_idx=syn.PAD_IDX)
    for own, plain in ((lambda p: policy(p, y, old, adv, ref)[0], plain_policy), (lambda p: preference(p, y, (ref * valid).sum(1))[0], plain_preference)):
        got = torch.autograd.grad(own(model(fs, x, masks)), params)
        want = torch.autograd.grad(plain(model(fs, x, masks)), params)
        num = math.sqrt(sum(float((a.double() - b.double()).square().sum()) for a, b in zip(got, want)))
        den = math.sqrt(sum(float(b.double().square().sum()) for b in want))
        # the two gradients of the logits differ by fp32 roundings; every later operand of the backward pass is a bf16 plane, where such a
        # difference moves a value by at most one step, 2^-7 of it -- all of them at once would move the whole by that
        assert den > 0 and num <= 2.0 ** -7 * den, (num, den)
    opt = FusedAdam(params, lr=1e-3)
    loss, stats = policy(model(fs, x, masks), y, old, adv, ref)
    loss.backward()
    clipper = GradClipper([p.grad for p in params], max_norm=0.1)
    before = [p.detach().clone() for p in params]
    norm = float(norm64([p.grad for p in params], False))
    assert abs(float(clipper()) - norm) <= U * norm
    after = float(norm64([p.grad for p in params], False))
    assert abs(after - min(norm, 0.1 * norm / (norm + 1e-6))) <= 8 * U * norm + 1e-9
    opt.step()
    assert any(not torch.equal(a, b) for a, b in zip(before, params)) and all(bool(torch.isfinite(p).all()) for p in params)


def caption_step(grad_clip, V=60, B=4, T=9):
    from bmt_amd import synthetic as syn
    from bmt_amd.model.captioning_module import BiModalTransformer
    from bmt_amd.train import CaptioningTrainStep
    cfg = syn.cfg_config0(dout_p=0.0)
    cfg.device, cfg.grad_clip, cfg.lr = "cuda:0", grad_clip, 1e-4
    torch.manual_seed(0)
    model = BiModalTransformer(cfg, syn.FakeTrainDataset(V, syn.make_glove(V, cfg.d_model_caps))).to("cuda:0")
    batch = syn.make_cap_batch(cfg, B, 12, 40, T, V, seed=5)
    fs = {k: v.cuda() for k, v in batch["feature_stacks"].items()}
    return CaptioningTrainStep(model, cfg, syn.PAD_IDX, static_grads=True), fs, batch["captions"].cuda()


@pytest.mark.parametrize("grad_clip", [0.05, 1e6])
def test_train_step_clips_its_arena(grad_clip):
    """cfg.grad_clip with static gradient buffers: p.grad holds what normalising and torch's clip_grad_norm_ give, eagerly and in replayed graphs"""
    step, fs, caps = caption_step(grad_clip)
    kl, n = step._forward_backward(fs, caps)
    step._reduce(kl, n)
    raw = [p.grad.detach().double().clone() for p in step.params]
    scale = float(step.grad_scale)
    before = [p.detach().clone() for p in step.params]
    step._optimize()
    norm = math.sqrt(sum(float((r * scale).square().sum()) for r in raw))
    coef = min(1.0, grad_clip / (norm + 1e-6)) * scale
    for p, r in zip(step.params, raw):
        within(p.grad, r * coef, 8 * U * (r * coef).abs(), "clipped")          # the factor's roundings and the product's
    assert step.optimizer.grad_scale is step.grad_scale and any(not torch.equal(a, b) for a, b in zip(before, step.params))
    step.capture(fs, caps)
    for _ in range(3):
        step.replay(fs, caps)
        torch.cuda.synchronize()
        total = math.sqrt(sum(float(p.grad.double().square().sum()) for p in step.params))
        assert 0 < total <= grad_clip * (1 + 1e-5)
        assert abs(float(step._clipper.coef)) > 0 and all(bool(torch.isfinite(p).all()) for p in step.params)
        assert grad_clip > 1 or abs(total - grad_clip) <= 1e-4 * grad_clip
        float(sum(p.sum() for p in step.params))          # (the program's own work between the replays)
    step.uncapture()


def test_vocabulary_embedder_without_positions_uses_the_sorted_gradient(ops):
    from bmt_amd.model.blocks import VocabularyEmbedder
    torch.manual_seed(0)
    emb = VocabularyEmbedder(300, 40).cuda()
    ids = torch.randint(0, 60, (5, 33), device="cuda", generator=gen(2))
    up = torch.randn(5, 33, 40, device="cuda", generator=gen(3))
    W = emb.embedder.weight
    out = emb(ids)
    assert torch.equal(out, W.detach()[ids] * torch.tensor(math.sqrt(40), dtype=torch.float32))
    (dW,) = torch.autograd.grad(out, W, up)
    _, d64, absum, most = embedding64(ids, W.detach(), math.sqrt(40), up, None)
    within(dW, d64, (36 + most / 4) * U * absum, "dW")


def test_losses_behind_a_generator_skip_its_softmax(ops, monkeypatch):
    """applied to a Generator's untouched output the losses' gradient goes straight to the generator's products: what the way through its
    log-softmax gives, alone, beside another consumer of the same output, and not at all where the output was written to"""
    from bmt_amd.model.generators import Generator
    torch.manual_seed(0)
    generator = Generator(48, 203).cuda()
    g = gen(12)
    x = torch.randn(3, 7, 48, device="cuda", generator=g).requires_grad_(True)
    ids = torch.randint(2, 203, (3, 7), device="cuda", generator=g)
    old, adv = torch.full((3, 7), -5.3, device="cuda"), torch.randn(3, device="cuda", generator=g)
    other = torch.randn(3, 7, 203, device="cuda", generator=g) * 1e-3
    seq = torch.zeros(2, device="cuda")
    leaves = [x, generator.linear.weight, generator.linear.bias]
    losses = {"policy": lambda p: ops.policy_loss(p, ids, old, adv)[0], "logp": lambda p: ops.token_logp(p, ids).square().mean(),
              "preference": lambda p: ops.preference_loss(p.narrow(0, 0, 2), ids[:2], seq)[0]}
    for name, loss in losses.items():
        for extra in (False, True):
            got = {}
            for fused in (True, False):
                monkeypatch.setattr(ops, "FUSE_GEN_LOSS", fused)
                pred = generator(x)
                total = loss(pred) + ((pred * other).sum() if extra else 0.0)
                got[fused] = torch.autograd.grad(total, leaves)
            for a, b in zip(got[True], got[False]):
                # the same values up to fp32 roundings before the bf16 operand plane, where one of them moves a value by at most a step: 2^-7 of it
                assert float((a - b).double().norm()) <= 2.0 ** -7 * float(b.double().norm()), (name, extra)
    monkeypatch.setattr(ops, "FUSE_GEN_LOSS", True)
    pred = generator(x)
    calls = []
    monkeypatch.setattr(ops.GenLogitsFn, "apply", lambda *a, f=ops.GenLogitsFn.apply: (calls.append(1), f(*a))[1])
    ops.token_logp(pred, ids)
    ops.token_logp(pred * 1.0, ids)
    assert len(calls) == 1
    ops.policy_loss(pred, ids, old, adv)
    assert len(calls) == 2
    with torch.no_grad():
        assert ops.token_logp(generator(x), ids).shape == (3, 7)
    first = torch.autograd.grad(ops.policy_loss(pred, ids, old, adv)[0] * 2.0, leaves, retain_graph=True)
    assert all(torch.isfinite(t).all() for t in first)


# ----------------------------------------------------------------------------- beyond 32 bits, and two calls at once
def test_logits_beyond_32_bit_offsets(ops):
    """2.2e9 logits: the last rows against 64 bits"""
    R, V = 66001, 33001
    x = torch.empty(1, R, V, device="cuda", dtype=torch.bfloat16)
    g = gen(1)
    for part in x[0].split(8192):
        part.copy_(torch.randn(part.shape, device="cuda", generator=g, dtype=torch.bfloat16))
    x.requires_grad_(True)
    ids = torch.randint(0, V, (1, R), device="cuda", generator=g)
    mask = torch.zeros(1, R, dtype=torch.bool, device="cuda")
    mask[0, -3:], mask[0, 100] = True, True
    adv = torch.ones(1, device="cuda")
    lp = logp64(x.detach()[:, -3:], ids[:, -3:])
    loss, stats = ops.policy_loss(x, ids, None, adv, mask=mask, reduction="sum")
    (dx,) = torch.autograd.grad(loss, x)
    within(stats.logp[:, -3:], lp, (64 + V / 64) * U + U * lp.abs(), "logp")
    want = torch.softmax(x.detach()[:, -3:].double(), -1)
    want.scatter_add_(-1, ids[:, -3:, None], torch.full((1, 3, 1), -1.0, device="cuda", dtype=torch.float64))
    tol = (256 + V / 32) * U + HALF[torch.bfloat16] * want.abs()
    within(dx[:, -3:], want, tol, "dlogits")
    assert int((dx[0, 101:-3].amax(1) != 0).sum()) == 0
    d2 = torch.autograd.grad(ops.token_logp(x, ids, mask).sum(), x)[0]
    within(d2[:, -3:], -want, tol, "token_logp's dlogits")


def test_embedding_beyond_32_bit_offsets(ops):
    """2.3e9 values of output and gradient"""
    N, V, D = 280001, 40, 8200
    g = gen(2)
    W = torch.randn(V, D, device="cuda", generator=g).bfloat16().requires_grad_(True)
    ids = torch.randint(0, V - 1, (N,), device="cuda", generator=g)
    ids[-1] = V - 1          # a token that only the last position holds
    out = ops.embedding(ids, W, 2.0)
    assert torch.equal(out[-5:], W.detach()[ids[-5:]] * 2.0)
    dout = torch.zeros(N, D, device="cuda", dtype=torch.bfloat16)
    dout[-1], dout[0] = 1.0, 0.5
    (dW,) = torch.autograd.grad(out, W, dout)
    want = torch.zeros(V, D, device="cuda")
    want[V - 1] += 2.0
    want[ids[0]] += 1.0
    assert torch.equal(dW.float(), want)


def test_a_gradient_beyond_32_bit_offsets():
    from bmt_amd.optim import GradClipper
    n = 2 ** 31 + 12345
    t = torch.zeros(n, device="cuda", dtype=torch.bfloat16)
    t[-1], t[0], t[n // 2] = 4.0, 2.0, 4.0
    assert float(GradClipper([t], 3.0)()) == 6.0
    assert [float(t[i]) for i in (0, n // 2, n - 1)] == [1.0, 2.0, 2.0] and float(t[1:5].abs().sum()) == 0.0


def test_many_rows_of_few_tokens(ops):
    """a million rows: several adding and counting workgroups"""
    B, T, V = 1000, 1003, 6
    g = gen(3)
    x = torch.randn(B, T, V, device="cuda", generator=g).requires_grad_(True)
    ids = torch.randint(0, V, (B, T), device="cuda", generator=g)
    mask = torch.rand(B, T, device="cuda", generator=g) > 0.5
    old, adv = torch.full((B, T), -2.0, device="cuda"), torch.randn(B, device="cuda", generator=g)
    for reduction in ("token", "sequence"):
        loss, stats = ops.policy_loss(x, ids, old, adv, old - 0.1, mask, kl_coef=0.1, reduction=reduction)
        (dx,) = torch.autograd.grad(loss, x)
        x64 = x.detach().double().requires_grad_(True)
        want, kl, clipped = policy64(logp64(x64, ids), old, adv, old - 0.1, mask, beta=0.1, reduction=reduction)
        (d64,) = torch.autograd.grad(want, x64)
        # (ratios up to e^2 here; rows whose ratio is at a border to rounding: none may differ by more than its own size, and few do)
        near = (dx.double() - d64).abs() > (256 + V / 32) * U * 16 * float(d64.abs().max())
        assert int(near.any(-1).sum()) <= 20
        within(loss, want, 1e-6 * float(adv.abs().max()), "loss")
        within(stats.kl, kl, 16 * 64 * U, "kl")
        within(stats.clip_fraction, clipped, 20 / float(mask.sum()) + U, "clip fraction")


def test_calls_at_once_on_two_streams(ops):
    """independent calls issued alternately on two streams, and from two threads: each has the result it has alone"""
    import threading
    from bmt_amd.optim import GradClipper
    g = gen(8)
    V, B, T = 5003, 6, 40
    xs = [torch.randn(B, T, V, device="cuda", generator=g).requires_grad_(True) for _ in range(2)]
    ids = [torch.randint(0, V, (B, T), device="cuda", generator=g) for _ in range(2)]
    rows = [torch.full((B, T), -9.0, device="cuda") + torch.randn(B, T, device="cuda", generator=g) for _ in range(2)]
    Ws = [torch.randn(V, 64, device="cuda", generator=g).requires_grad_(True) for _ in range(2)]
    ups = [torch.randn(B, T, 64, device="cuda", generator=g) for _ in range(2)]
    grads = [[torch.randn(100000, device="cuda", generator=g) for _ in range(5)] for _ in range(2)]
    outs = [[torch.empty_like(t) for t in ts] for ts in grads]
    clips = [GradClipper(a, 0.5, b) for a, b in zip(grads, outs)]

    def work(k):
        loss, _ = ops.policy_loss(xs[k], ids[k], rows[k], rows[k][:, 0], rows[k], kl_coef=0.1)
        (dx,) = torch.autograd.grad(loss, xs[k])
        pl, r = ops.preference_loss(xs[k], ids[k], rows[k][:, 1])
        (dp,) = torch.autograd.grad(pl, xs[k])
        (dW,) = torch.autograd.grad(ops.embedding(ids[k], Ws[k], 3.0), Ws[k], ups[k])
        return [loss.detach(), dx, pl.detach(), r, dp, dW, clips[k](), outs[k][4].clone()]

    alone = [work(k) for k in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(5):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(work(k))
    torch.cuda.synchronize()

    def loop(k):
        with torch.cuda.stream(streams[k]):
            for _ in range(5):
                got[k].append(work(k))
            streams[k].synchronize()
    threads = [threading.Thread(target=loop, args=(k,)) for k in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for k in range(2):
        assert len(got[k]) == 10
        for r in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(r, alone[k]))


# ----------------------------------------------------------------------------- calls at the edges of what the documentation allows
def test_a_kl_term_that_is_only_watched_may_be_infinite(ops):
    """kl_coef 0 with a reference: its KL term is a number to look at, and tokens that the reference rules out leave loss and gradient alone"""
    g = gen(21)
    x = torch.randn(2, 3, 40, device="cuda", generator=g).requires_grad_(True)
    ids = torch.randint(0, 40, (2, 3), device="cuda", generator=g)
    adv = torch.randn(2, device="cuda", generator=g)
    ref = torch.full((2, 3), -2.0, device="cuda")
    ref[1, 1] = -float("inf")
    old = logp64(x.detach(), ids).float()
    loss, stats = ops.policy_loss(x, ids, old, adv, ref)
    (dx,) = torch.autograd.grad(loss, x)
    alone = ops.policy_loss(x, ids, old, adv)[0]
    assert torch.equal(loss, alone) and torch.equal(dx, torch.autograd.grad(alone, x)[0]) and bool(torch.isfinite(dx).all())
    assert float(stats.kl) == float("inf")


def test_preference_labels_that_are_all_wrong(ops):
    """label_smoothing 1: only -log sigmoid(-z) counts, which is 0 where the first caption is impossible"""
    x = torch.zeros(2, 1, 50, device="cuda")
    x[0, 0, 7] = -float("inf")
    ids = torch.full((2, 1), 7, device="cuda")
    x.requires_grad_(True)
    loss, _ = ops.preference_loss(x, ids, torch.zeros(2, device="cuda"), label_smoothing=1.0)
    (dx,) = torch.autograd.grad(loss, x)
    assert float(loss) == 0.0 and bool((dx == 0).all())


@pytest.mark.parametrize("n", [40, 5000, 20000])      # (ids in registers, ids split by owner first)
def test_ids_that_are_clamped_to_the_padding_row_add_nothing_to_it(ops, n):
    V, D, g = 30, 8, gen(n)
    ids = torch.randint(-9, V + 9, (n,), device="cuda", generator=g)
    W = torch.randn(V, D, device="cuda", generator=g).requires_grad_(True)
    dout = torch.randint(-3, 4, (n, D), device="cuda", generator=g).float()      # (sums of small integers: exact)
    for pad in (0, V - 1, -4):
        (dW,) = torch.autograd.grad(ops.embedding(ids, W, 1.0, pad), W, dout)
        at = ids.clamp(0, V - 1)
        keep = (ids != pad) & (at != pad)
        want = torch.zeros(V, D, device="cuda").index_add_(0, at[keep], dout[keep])
        assert torch.equal(dW, want), pad


def test_a_table_of_one_row_in_any_layout(ops):
    W = torch.randn(6, 1, device="cuda").t()          # (1, 6), strides (1, 1)
    W.requires_grad_(True)
    ids = torch.zeros(3, dtype=torch.int64, device="cuda")
    out = ops.embedding(ids, W)
    (dW,) = torch.autograd.grad(out, W, torch.ones_like(out))
    assert torch.equal(out, W.detach().expand(3, 6)) and bool((dW == 3).all())


def test_embedding_of_more_ids_than_short_chunks_hold(ops):
    """over 16 M positions the chunks of the split grow"""
    g = gen(3)
    V, D, n = 1000, 4, (1 << 24) + 100001
    ids = torch.randint(0, V, (n,), device="cuda", generator=g)
    dout = torch.randint(-1, 2, (n, D), device="cuda", generator=g).float()      # (a token's sum stays far below 2^24: exact)
    W = torch.randn(V, D, device="cuda", generator=g).requires_grad_(True)
    (dW,) = torch.autograd.grad(ops.embedding(ids, W, 1.0, PAD), W, dout)
    want = torch.zeros(V, D, device="cuda", dtype=torch.float64).index_add_(0, ids, dout.double())
    want[PAD] = 0
    assert torch.equal(dW.double(), want)


def test_inputs_that_get_no_gradient_may_ask_for_one(ops):
    g = gen(22)
    x = torch.randn(2, 3, 20, device="cuda", generator=g)
    ids = torch.randint(0, 20, (2, 3), device="cuda", generator=g)
    old, adv, ref = (torch.randn(2, 3, device="cuda", generator=g).requires_grad_(True) for _ in range(3))
    loss, _ = ops.policy_loss(x, ids, old, adv, ref, kl_coef=0.1)
    assert not loss.requires_grad
    pair, _ = ops.preference_loss(x, ids, torch.zeros(2, device="cuda", requires_grad=True))
    assert not pair.requires_grad
    x.requires_grad_(True)
    again, _ = ops.policy_loss(x, ids, old, adv, ref, kl_coef=0.1)
    dx, dold = torch.autograd.grad(again, (x, old), allow_unused=True)
    assert torch.equal(again, loss) and dold is None and bool((dx != 0).any())


def test_a_gradient_of_a_gradient_is_refused(ops):
    x = torch.randn(2, 3, 20, device="cuda").requires_grad_(True)
    W = torch.randn(20, 4, device="cuda").requires_grad_(True)
    ids = torch.zeros(2, 3, dtype=torch.int64, device="cuda")
    row = torch.ones(2, 3, device="cuda")
    for leaf, call in ((x, lambda: ops.policy_loss(x, ids, row, row)[0]), (x, lambda: ops.preference_loss(x, ids, torch.zeros(2, device="cuda"))[0]),
                       (x, lambda: ops.token_logp(x, ids).sum()), (W, lambda: ops.embedding(ids, W).sum())):
        (d,) = torch.autograd.grad(call(), leaf)
        (same,) = torch.autograd.grad(call(), leaf, create_graph=True)
        assert torch.equal(d, same)
        with pytest.raises(RuntimeError):
            same.sum().backward()


def test_a_clipping_plan_is_not_made_inside_a_capture():
    from bmt_amd.optim import GradClipper
    t = torch.ones(100, device="cuda")
    plan = GradClipper([t], 1.0)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="before the capture"):
            GradClipper([t], 1.0)
        norm = plan()
    for _ in range(2):
        t.fill_(1.0)
        graph.replay()
        torch.cuda.synchronize()
        assert abs(float(norm) - 10.0) < 1e-5 and abs(float(t.norm()) - 1.0) < 1e-5
