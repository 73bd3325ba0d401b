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


def softmax64(x):
    """(torch.softmax of float64 rows of more than 1024 elements takes fp32 exponentials on this GPU: up to 1.8e-6 off)"""
    x = x.detach().double()
    e = torch.exp(x - x.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


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
    p = softmax64(x)
    want = w[..., None] * (torch.zeros_like(p).scatter_(-1, ids[..., None], 1.0) - p)
    # logp is off by less than (3 * 16 + 2) u (one exponential, t = x - max below 16) and a few more of the sum: 64 u; w moves by (|A| + beta e^d) times
    # that and is rounded; p and its product with w: 64 u of |w|; a type of fewer bits adds half a step
    each = (adv.abs().double()[:, None] + beta * torch.exp(d) + w.abs()) * 64 * U
    within(dx, want, each[..., None] + HALF[dtype] * want.abs(), "dlogits")
    assert float(loss) == float("inf") and float(stats.kl) == float("inf")
    rest, _ = ops.policy_loss(x[3:], ids[3:], old[3:], adv[3:], ref[3:], kl_coef=beta, reduction="sum")
    total = (-adv.double()[3:, None] * torch.exp(lp - old.double())[3:] + beta * (torch.expm1(d) - d)[3:]).sum()
    within(rest, total, 2 * U * abs(float(total)), "loss")          # (1e16 of it: the loss's own rounding, and beta is exact)


# ----------------------------------------------------------------------------- losses on a Generator's own output
def behind_a_generator(V=203, D=48, B=4, T=7):
    from bmt_amd.model.generators import Generator
    torch.manual_seed(0)
    generator, g = Generator(D, V).cuda(), gen(12)
    x = torch.randn(B, T, D, device="cuda", generator=g).requires_grad_(True)
    ids = torch.randint(2, V, (B, T), device="cuda", generator=g)
    old, adv = torch.full((B, T), -5.3, device="cuda"), torch.randn(B, device="cuda", generator=g)
    seq = torch.zeros(B, device="cuda")
    from bmt_amd import ops
    losses = {"policy": lambda p: ops.policy_loss(p, ids, old, adv)[0], "policy_times_3": lambda p: ops.policy_loss(p, ids, old, adv)[0] * 3.0,
              "logp": lambda p: ops.token_logp(p, ids).square().mean(), "preference": lambda p: ops.preference_loss(p, ids, seq)[0]}
    return generator, x, losses


LOSSES = ["policy", "policy_times_3", "logp", "preference"]


@pytest.mark.parametrize("name", LOSSES)
def test_a_generator_s_output_sees_its_gradient(ops, monkeypatch, name):
    """hooks, retain_grad and torch.autograd.grad on the output itself get what the loss gives logits that are leaves, and the way behind the output
    runs without the log-softmax's backward"""
    generator, x, losses = behind_a_generator()
    calls = []
    monkeypatch.setattr(ops.lib, "bmt_log_softmax_bwd", lambda *a, f=ops.lib.bmt_log_softmax_bwd: (calls.append(1), f(*a))[1])
    pred = generator(x)
    leaf = pred.detach().clone().requires_grad_(True)
    (want,) = torch.autograd.grad(losses[name](leaf), leaf)
    (got,) = torch.autograd.grad(losses[name](pred), pred, retain_graph=True)
    assert torch.equal(got, want)
    seen = []
    pred.retain_grad()
    pred.register_hook(lambda g: seen.append(g.clone()))
    losses[name](pred).backward()
    assert len(seen) == 1 and torch.equal(seen[0], want) and torch.equal(pred.grad, want)
    assert not calls
    (losses[name](generator(x)) + losses[name](generator(x)) * 0.0).backward()
    assert not calls
    pred = generator(x)
    (losses[name](pred) + pred.mean()).backward()          # another consumer: the sum of the gradients goes the whole way
    assert len(calls) == 1


@pytest.mark.parametrize("name", LOSSES)
def test_the_way_past_a_generator_s_log_softmax(ops, monkeypatch, name):
    """the same gradients as through it: fp32 roundings of the logits' gradient, after which every operand is a bf16 plane, where one of them moves a
    value by at most a step, 2^-7 of it"""
    generator, x, losses = behind_a_generator()
    leaves, got = [x, generator.linear.weight, generator.linear.bias], {}
    for fused in (True, False):
        monkeypatch.setattr(ops, "FUSE_GEN_LOSS", fused)
        got[fused] = torch.autograd.grad(losses[name](generator(x)), leaves)
    for a, b in zip(got[True], got[False]):
        assert float((a - b).double().norm()) <= 2.0 ** -7 * float(b.double().norm())


@pytest.mark.parametrize("what", ["weight", "output"])
def test_a_generator_written_to_before_the_backward_pass_is_noticed(ops, what):
    generator, x, losses = behind_a_generator()
    for name in LOSSES:
        pred = generator(x)
        loss = losses[name](pred)
        with torch.no_grad():
            (generator.linear.weight if what == "weight" else pred).mul_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


class Watched(torch.autograd.Function):
    """a node in front of the generator that holds an object: alive as long as the pass is"""

    @staticmethod
    def forward(ctx, x, held):
        ctx.held = held
        return x * 1.0

    @staticmethod
    def backward(ctx, d):
        return d, None


class Held:
    pass


@pytest.mark.parametrize("backward", [True, False])
@pytest.mark.parametrize("name", LOSSES)
def test_a_pass_ends_with_its_loss(ops, name, backward):
    """once loss and output are dropped nothing of a pass lives on: neither the log-probabilities nor the graph in front of the generator"""
    import gc
    import weakref
    generator, x, losses = behind_a_generator()
    ops.context().gen_handles.clear()
    sizes, held = [], []
    for _ in range(4):
        h = Held()
        held.append(weakref.ref(h))
        pred = generator(Watched.apply(x, h))
        loss = losses[name](pred)
        if backward:
            loss.backward()
        del pred, loss, h
        gc.collect()
        sizes.append(torch.cuda.memory_allocated())
        assert held[-1]() is None
    assert sizes[1] == sizes[2] == sizes[3] and not ops.context().gen_handles


@pytest.mark.parametrize("name", LOSSES)
def test_a_generator_with_static_gradient_buffers(ops, name):
    """GradientReducer, a loss on the generator's output, GradClipper: the buffers hold the gradients, and every use of a parameter that the forward
    pass counted is settled by the backward pass alone, step after step"""
    from bmt_amd.optim import GradClipper
    from bmt_amd.parallel import GradientReducer
    generator, x, losses = behind_a_generator()
    params = [generator.linear.weight, generator.linear.bias]
    want = torch.autograd.grad(losses[name](generator(x)), params)
    reducer = GradientReducer(params)
    try:
        clipper = GradClipper([p.grad for p in params], max_norm=1e9)
        for _ in range(3):
            reducer.zero_grad()
            losses[name](generator(x)).backward()
            assert all(p._bmt_uses == 0 for p in params) and not ops.context().gen_handles
            reducer.finish()
            norm = clipper()
            for p, w in zip(params, want):
                # (sums over 28 rows of the same operands, in another order: 28 u of their absolute sum, which stays below 28 times the largest)
                assert float((p.grad - w).abs().max()) <= 28 * 28 * U * float(w.abs().max())
            total = sum(float(p.grad.double().square().sum()) for p in params) ** 0.5
            assert abs(float(norm) - total) <= 2 * U * total
    finally:
        reducer.remove()


# ----------------------------------------------------------------------------- ids outside the vocabulary
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
@pytest.mark.parametrize("V", [7, 1000, 140001])
def test_ids_outside_the_vocabulary_give_nan_rows(ops, dtype, V):
    """value and gradient of such a row are NaN throughout, whichever loss asks and however far outside the id is; other rows are as without it"""
    g = gen(V)
    outside = [-1, V, V + 13, -(1 << 40), (1 << 35) + 3, (1 << 62)]
    B, T = len(outside) + 2, 2
    x = torch.randn(B, T, V, device="cuda", generator=g).to(dtype).requires_grad_(True)
    good = torch.randint(0, V, (B, T), device="cuda", generator=g)
    ids = good.clone()
    ids[:len(outside), 0] = torch.tensor(outside, device="cuda")
    bad = ids != good
    up = torch.randn(B, T, device="cuda", generator=g)
    lp, lp_good = ops.token_logp(x, ids), ops.token_logp(x, good)
    assert bool(torch.isnan(lp[bad]).all()) and torch.equal(lp[~bad], lp_good[~bad])
    (dx,), (want,) = torch.autograd.grad(lp, x, up), torch.autograd.grad(lp_good, x, up)
    assert bool(torch.isnan(dx[bad]).all()) and torch.equal(dx[~bad], want[~bad])
    loss, _ = ops.policy_loss(x, ids, None, up, reduction="sum")
    (dx,) = torch.autograd.grad(loss, x, retain_graph=True)
    (dx2,) = torch.autograd.grad(loss * 2.0, x)
    assert torch.isnan(loss) and all(bool(torch.isnan(d[bad]).all()) and bool(torch.isfinite(d[~bad]).all()) for d in (dx, dx2))
    loss, rewards = ops.preference_loss(x, ids, torch.zeros(B, device="cuda"))
    (dx,) = torch.autograd.grad(loss, x)
    hit = bad.any(1)
    pair = hit[:B // 2] | hit[B // 2:]
    assert torch.isnan(loss) and torch.equal(torch.isnan(rewards), hit)
    assert torch.equal(torch.isnan(dx).all(2).all(1), pair.repeat(2)) and bool(torch.isfinite(dx[~pair.repeat(2)]).all())
    masked = ids.clone()
    mask = ~bad
    assert bool(torch.isfinite(torch.autograd.grad(ops.policy_loss(x, masked, None, up, mask=mask)[0], x)[0]).all())


# ----------------------------------------------------------------------------- clipping plans
def test_a_clipping_plan_dropped_behind_a_call_on_another_stream(ops):
    """its tile table belongs to the stream it was made on; while a call on another stream may still read it, that memory goes to nobody else"""
    from bmt_amd.optim import GradClipper
    work = torch.randn(4096, 4096, device="cuda")
    grads = [torch.full((100003,), 0.5, device="cuda"), torch.full((33,), 0.25, device="cuda")]
    plan = GradClipper(grads, max_norm=1.0)
    table = (plan._tiles.data_ptr(), plan._tiles.numel())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(50):          # (tens of milliseconds in front of the call)
            work = work @ work
            work = work / work.norm()
        norm = plan()
        behind = side.record_event()
    del plan
    taken = [torch.empty(table[1], dtype=torch.uint8, device="cuda") for _ in range(64)]
    where = [t.data_ptr() for t in taken]
    still_running = not behind.query()
    side.synchronize()
    assert still_running and table[0] not in where
    want = (100003 * 0.25 + 33 * 0.0625) ** 0.5
    assert abs(float(norm) - want) <= 2 * U * want
    for t, v in zip(grads, (0.5, 0.25)):
        assert float((t - v / (want + 1e-6)).abs().max()) <= 4 * U * v / want


def test_another_clipping_bound_in_front_of_a_capture_without_warm_up(ops):
    """cfg.grad_clip may change between eager steps and a capture that runs none of its own"""
    from tests.test_gpu_tuning import caption_step
    step, fs, caps = caption_step(1e6)
    for _ in range(2):
        step(fs, caps)
    step.cfg.grad_clip = 0.05
    step.capture(fs, caps, warmup=0)
    for _ in range(3):
        step.replay(fs, caps)
        torch.cuda.synchronize()
        total = sum(float(p.grad.double().square().sum()) for p in step.params) ** 0.5
        # (clipped: the norm is at least 0.05, so eps = 1e-6 takes at most 2e-5 of the total; the factor and every product are rounded)
        assert abs(total - 0.05) <= 0.05 * (2e-5 + 8 * U)
        float(sum(p.sum() for p in step.params))          # (the program's own work between the replays)
    step.uncapture()
    step.cfg.grad_clip = 0.025
    step(fs, caps)
    total = sum(float(p.grad.double().square().sum()) for p in step.params) ** 0.5
    assert abs(total - 0.025) <= 0.025 * (4e-5 + 8 * U)
    for bound in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            step._clipper.max_norm = bound


# ----------------------------------------------------------------------------- embedding
@pytest.mark.parametrize("static", [False, True])
@pytest.mark.parametrize("n", [4097, 1 << 22])
def test_gradient_of_very_frequent_tokens(ops, n, static):
    """an element's value passes through at most 7 additions of a wave, the 3 that join its four waves, 64 bits from there and one rounding (and one
    more where it is added to a buffer): 12 u of the absolute sum, however frequent the token is"""
    V, D, g = 5, 16, gen(n)
    ids = torch.tensor([0, 3, 4], device="cuda")[torch.randint(0, 3, (n,), device="cuda", generator=g)]
    ids[7] = 2
    dout = torch.rand(n, D, device="cuda", generator=g)
    W = torch.nn.Parameter(torch.randn(V, D, device="cuda", generator=g))
    want = torch.stack([dout[ids == v].double().sum(0) * 1.5 for v in range(V)])
    if static:
        from bmt_amd.parallel import GradientReducer
        reducer = GradientReducer([W])
        try:
            ops.embedding(ids, W, 1.5).backward(dout)
            got = W.grad.clone()
        finally:
            reducer.remove()
    else:
        (got,) = torch.autograd.grad(ops.embedding(ids, W, 1.5), W, dout)
        assert torch.equal(got, torch.autograd.grad(ops.embedding(ids, W, 1.5), W, dout)[0])
    within(got, want, 12 * U * want, "dW")


# ----------------------------------------------------------------------------- every element of a gradient, relative to itself
def test_exponentials_of_an_fp32_gradient_have_no_bias(ops):
    """exp(t) in a gradient errs by roundings, which average out, and not with t: the mean relative errors of elements near t = -60 and near t = -3
    differ by less than 2 u.  (The roundings of t log2 e are at most 2.6e-6 there; the mean over 50 000 of them is off by less than six of its own
    deviations, 6 * 2.6e-6 / 3^1/2 / 50000^1/2 = 4e-8, and 2 u = 1.2e-7.)"""
    n, g = 50000, gen(5)
    far, near = -62.0 + 4.0 * torch.rand(n, device="cuda", generator=g), -4.0 + 2.0 * torch.rand(n, device="cuda", generator=g)
    x = torch.cat([torch.zeros(1, device="cuda"), far, near])[None, None].requires_grad_(True)
    ids = torch.zeros(1, 1, dtype=torch.int64, device="cuda")
    want = -softmax64(x)[0, 0, 1:]
    for loss in (ops.token_logp(x, ids).sum(), ops.policy_loss(x, ids, None, -torch.ones(1, device="cuda"))[0]):
        (dx,) = torch.autograd.grad(loss, x)
        rel = (dx[0, 0, 1:].double() / want - 1.0).view(2, n).mean(1)
        assert abs(float(rel[0] - rel[1])) < 2 * U, rel


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,T,V", [(3, 2, 7), (2, 3, 1000), (5, 7, 4099), (2, 2, 33001), (4, 1, 131075), (2, 1, 300001), (700, 1, 4101), (600, 1, 16385)])
def test_every_element_of_a_gradient(ops, dtype, B, T, V):
    """Off the target the gradient is -w p, one product after another, so its error is bounded relative to itself: exp by its argument (t = x - max and
    t log2 e rounded: 2 |t| u) and the instruction (2 u), 1 / sum (the sum's terms err by (2 |t| + 2) u each, under p |t| averages below ln V + 1 < 14:
    30 u, and its rounding), two products: (2 |t| + 36) u; the type adds half a step, fp16 half of its smallest one.  At the target w - w p: that of p,
    and 2 u |w|.  w is exact but for the preference loss, where it is a sigmoid of rewards: beta = 0.1 times 64 u, and its rounding: 8 u more"""
    g = gen(V + B)
    x = (torch.randn(B, T, V, device="cuda", generator=g) * 2.5).to(dtype).requires_grad_(True)
    ids = torch.randint(0, V, (B, T), device="cuda", generator=g)
    up = torch.randn(B, T, device="cuda", generator=g)
    x64 = x.detach().double()
    t = (x64 - x64.amax(-1, keepdim=True)).abs()
    p = softmax64(x)
    at = torch.zeros_like(p).scatter_(-1, ids[..., None], 1.0)
    cases = [("logp", up.double(), 0.0, lambda: (ops.token_logp(x, ids) * up).sum()),
             ("policy", -up.double(), 0.0, lambda: ops.policy_loss(x, ids, None, up, reduction="sum")[0])]
    cases.append(("policy times 0.5", -0.5 * up.double(), 0.0, lambda: ops.policy_loss(x, ids, None, up, reduction="sum")[0] * 0.5))
    if B % 2 == 0 and T == 1:
        S = torch.log_softmax(x64, -1).gather(-1, ids[..., None])[..., 0].sum(1)
        z = 0.1 * (S[:B // 2] - S[B // 2:])
        d = -0.1 / (B // 2) * torch.sigmoid(-z)
        cases.append(("preference", torch.cat([d, -d])[:, None], 8.0, lambda: ops.preference_loss(x, ids, torch.zeros(B, device="cuda"))[0]))
    tiny = 2.0 ** -25 if dtype == torch.float16 else 0.0
    for name, w, more, loss in cases:
        (dx,) = torch.autograd.grad(loss(), x)
        w = w[..., None]
        want = w * (at - p)
        tol = (2 * t + 36 + more) * U * (w * p).abs() + at * (2 + more) * U * w.abs() + HALF[dtype] * want.abs() * (1 + 2.0 ** -8) + tiny
        within(dx, want, tol, name)


# ----------------------------------------------------------------------------- gradient buckets
@pytest.mark.parametrize("name", LOSSES)
def test_buckets_behind_a_loss_on_a_generator_s_output(ops, name):
    """every bucket is handed to its collective once, with the gradients that the pass ends with"""
    from bmt_amd.parallel import GradientReducer
    generator, x, losses = behind_a_generator()
    reducer = GradientReducer([generator.linear.weight, generator.linear.bias], bucket_bytes=1)
    reducer.world, handed = 2, []          # (as one of two ranks; the collective is this list)
    reducer._reduce_bucket = lambda b: handed.append((b["flat"], b["flat"].clone()))
    try:
        for _ in range(2):
            handed.clear()
            reducer.zero_grad()
            losses[name](generator(x)).backward()
            assert len(handed) == len(reducer.buckets) == 2
            reducer.finish()
            assert len(handed) == 2 and all(torch.equal(flat, at) and bool((at != 0).any()) for flat, at in handed)
    finally:
        reducer.remove()


def test_buckets_of_an_overlapped_step_are_reduced_once_and_complete(ops):
    from tests.test_gpu_tuning import caption_step
    single, fs, caps = caption_step(None)
    from bmt_amd.train import CaptioningTrainStep
    step = CaptioningTrainStep(single.model, single.cfg, single.pad_idx, data_parallel=True, bucket_bytes=1 << 14)
    reducer, handed = step.reducer, []
    reducer.world = 2
    reducer._reduce_bucket = lambda b: handed.append((b["flat"], b["flat"].clone()))
    assert len(reducer.buckets) > 4
    for _ in range(2):
        handed.clear()
        kl, n = step._forward_backward(fs, caps)
        inside = len(handed)
        step._reduce(kl, n)
        assert inside > 0 and len(handed) == len(reducer.buckets)
        assert sorted(f.data_ptr() for f, _ in handed) == sorted(b["flat"].data_ptr() for b in reducer.buckets)
        assert all(torch.equal(flat, at) for flat, at in handed)
        step._optimize()
    reducer.remove()


def test_buckets_of_an_overlapped_proposal_step_are_reduced_once_and_complete(ops, golden):
    """the same where products run as autograd reaches them, weights are read through views, and the reduction ends inside the step"""
    from bmt_amd.model.proposal_generator import MultimodalProposalGenerator
    from bmt_amd.train import ProposalTrainStep
    from tests.test_gpu_proposal import _prop_cfg
    g, cfg = golden("tiny_prop.npz"), _prop_cfg()
    cfg.lr, cfg.grad_clip = 1e-3, None
    model = MultimodalProposalGenerator(cfg, {"audio": [float(a) for a in g.np("anchors_audio")], "video": [float(a) for a in g.np("anchors_video")]})
    model.load_state_dict(g.sub("sd/"))
    step = ProposalTrainStep(model.cuda(), cfg, pad_idx=1, data_parallel=True, bucket_bytes=1 << 12)
    reducer, handed, checks = step.reducer, [], []
    reducer.world = 2
    reducer._reduce_bucket = lambda b: handed.append((b["flat"], b["flat"].clone()))

    def finish(inner=reducer.finish):
        inside = len(handed)
        inner()
        checks.append((inside, len(handed), all(torch.equal(flat, at) for flat, at in handed)))
    reducer.finish = finish
    fs, targets = {k: g[k].cuda() for k in ("rgb", "flow", "audio")}, g["targets"].cuda()
    for _ in range(2):
        handed.clear()
        step(fs, targets)
    n = len(reducer.buckets)
    assert n > 4 and checks == [(n, n, True)] * 2
    reducer.remove()
