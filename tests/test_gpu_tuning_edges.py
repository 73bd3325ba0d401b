"""-m gpu: the operators that tune a caption model at values, layouts and lifetimes beyond those of test_gpu_tuning.py, against 64 bits.  u = 2^-24, half
a step of fp32; every test derives its own tolerance."""
import pytest
import torch

from tests.gpu_util import report

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF = {torch.float32: 0.0, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


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
    assert not bool(bad.any()), report(got, want, name) + f"\n  {int(bad.sum())} of {bad.numel()} outside"


# ----------------------------------------------------------------------------- policy loss
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V", [40, 140001])          # (a row in registers, a row that is read twice)
def test_gradient_of_the_kl_term_for_any_reference(ops, dtype, V):
    """d / d logp of beta (e^d - d - 1) is beta (1 - e^d): finite, and beta itself, where the reference rules the token out (d = -inf) or holds its
    type's lowest value.  The loss is infinite, or as large as the reference says, in such a row; every gradient is finite"""
    refs = [-float("inf"), torch.finfo(torch.float32).min, torch.finfo(torch.bfloat16).min, -1e16, -1e7, -60.0, -12.0, 0.0, 3.0]
    B, beta, g = len(refs), 0.25, gen(V)
    x = torch.randn(B, 1, V, device="cuda", generator=g).to(dtype)
    ids = torch.randint(0, V, (B, 1), device="cuda", generator=g)
    x.requires_grad_(True)
    lp = torch.log_softmax(x.detach().double(), -1).gather(-1, ids[..., None])[..., 0]
    old, adv = lp.float(), torch.randn(B, device="cuda", generator=g)
    ref = torch.tensor(refs, device="cuda")[:, None]
    loss, stats = ops.policy_loss(x, ids, old, adv, ref, kl_coef=beta, reduction="sum")
    (dx,) = torch.autograd.grad(loss, x)
    d = ref.double() - lp
    w = -adv.double()[:, None] * torch.exp(lp - old.double()) - beta * torch.expm1(d)
    assert bool(torch.isfinite(w).all())
    p = torch.softmax(x.detach().double(), -1)
    want = w[..., None] * (torch.zeros_like(p).scatter_(-1, ids[..., None], 1.0) - p)
    # logp is off by less than (3 * 16 + 2) u (one exponential, t = x - max below 16) and a few more of the sum: 64 u; w moves by (|A| + beta e^d) times
    # that and is rounded; p and its product with w: 64 u of |w|; a type of fewer bits adds half a step
    each = (adv.abs().double()[:, None] + beta * torch.exp(d) + w.abs()) * 64 * U
    within(dx, want, each[..., None] + HALF[dtype] * want.abs(), "dlogits")
    assert float(loss) == float("inf") and float(stats.kl) == float("inf")
    rest, _ = ops.policy_loss(x[3:], ids[3:], old[3:], adv[3:], ref[3:], kl_coef=beta, reduction="sum")
    total = (-adv.double()[3:, None] * torch.exp(lp - old.double())[3:] + beta * (torch.expm1(d) - d)[3:]).sum()
    within(rest, total, 2 * U * abs(float(total)), "loss")          # (1e16 of it: the loss's own rounding, and beta is exact)
