"""The operators of a caption model's tuning step, as cases that can be timed: the clipped policy loss and the paired preference loss from
logits (with their gradients), the scaled embedding lookup with its gradient, and the global gradient norm with clipping.

``run`` computes a case in its plain form (elementary torch operations, 32 bits, rows' scalars in 64) or, where ``own`` is true, through the
framework's entry points; ``exact`` computes the definition in 64 bits."""
import math

import torch

own = False

PAD = 1                    # the framework's padding token
DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
LARGEST = 2.2e9            # bytes of the largest listed case: no drawn case is larger


def listed():
    return [
        # one decoding step of eight sampled captions scored at once: T = 1, latency counts
        {"name": "policy_step_fp32", "op": "policy", "dtype": "fp32", "B": 8, "T": 1, "V": 10000, "view": False, "masked": "pad", "kl": 0.05, "adv": "seq", "reduction": "token"},
        # the framework's caption batch (B = 32, 29 predicted tokens, V = 10 000, ragged), tuned on sampled captions
        {"name": "policy_captions_fp32", "op": "policy", "dtype": "fp32", "B": 32, "T": 29, "V": 10000, "view": False, "masked": "pad", "kl": 0.05, "adv": "seq", "reduction": "token"},
        # long sampled sequences over a larger vocabulary, 16-bit logits, mean over each sequence first
        {"name": "policy_long_bf16", "op": "policy", "dtype": "bf16", "B": 16, "T": 512, "V": 32000, "view": False, "masked": "mask", "kl": 0.02, "adv": "token", "reduction": "sequence"},
        # logits[:, :-1] of an odd vocabulary: rows that start at every alignment, strides that do not collapse; no KL term
        {"name": "policy_odd_view_bf16", "op": "policy", "dtype": "bf16", "B": 9, "T": 130, "V": 20011, "view": True, "masked": "mask", "kl": 0.0, "adv": "seq", "reduction": "token"},
        # 32 pairs of preferred / rejected captions through the caption model
        {"name": "preference_captions_fp32", "op": "preference", "dtype": "fp32", "B": 64, "T": 29, "V": 10000, "view": False, "masked": "pad", "smooth": 0.0, "mean": False},
        # eight pairs of long sequences, 16-bit logits
        {"name": "preference_long_bf16", "op": "preference", "dtype": "bf16", "B": 16, "T": 1024, "V": 32000, "view": False, "masked": "mask", "smooth": 0.1, "mean": False},
        # a few short pairs, odd vocabulary, shifted view, length-normalised
        {"name": "preference_odd_fp16", "op": "preference", "dtype": "fp16", "B": 6, "T": 37, "V": 12345, "view": True, "masked": "mask", "smooth": 0.0, "mean": True},
        # the embedding of one decoding step (no gradient): 32 tokens
        {"name": "embedding_step_fp32", "op": "embedding", "dtype": "fp32", "B": 32, "T": 1, "V": 10000, "D": 300, "grad": False},
        # the framework's caption batch through a trained table: 32 x 29 tokens, 10 000 x 300
        {"name": "embedding_captions_fp32", "op": "embedding", "dtype": "fp32", "B": 32, "T": 29, "V": 10000, "D": 300, "grad": True},
        # a training batch of long sequences, 16-bit table, a few very frequent tokens
        {"name": "embedding_long_bf16", "op": "embedding", "dtype": "bf16", "B": 32, "T": 2048, "V": 32000, "D": 1024, "grad": True},
        # the gradients of a model of the caption model's size (50 M fp32 values in one arena), clipped into the optimizer's buffers
        {"name": "clip_captions_fp32", "op": "clip", "dtype": "fp32", "layers": 4, "width": 1024, "V": 300, "norm": "l2", "inplace": False},
        # 16-bit gradients of a larger model into fp32 buffers
        {"name": "clip_large_bf16", "op": "clip", "dtype": "bf16", "layers": 24, "width": 1024, "V": 10001, "norm": "l2", "inplace": False},
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    while True:
        op = rng.choice(["policy", "preference", "embedding", "clip"])
        case = {"op": op, "dtype": rng.choice(["fp32", "bf16", "fp16"])}
        if op in ("policy", "preference"):
            case.update(B=log(1, 64) if op == "policy" else 2 * log(1, 32), T=log(1, 1024), V=log(500, 130000), view=rng.random() < 0.3, masked=rng.choice(["pad", "mask"]))
            if op == "policy":
                case.update(kl=rng.choice([0.0, 0.02, 0.1]), adv=rng.choice(["seq", "token"]), reduction=rng.choice(["token", "sequence"]))
            else:
                case.update(smooth=rng.choice([0.0, 0.1]), mean=rng.random() < 0.5)
        elif op == "embedding":
            case.update(B=log(1, 64), T=log(1, 2048), V=log(500, 130000), D=log(64, 4096), grad=rng.random() < 0.8)
        else:
            case.update(layers=log(1, 24), width=log(64, 1024), V=log(100, 32000), norm=rng.choice(["l2", "l2", "inf"]), inplace=rng.random() < 0.3)
        if work(case)["bytes"] <= LARGEST:
            return case


def _shapes(case):
    d = case["width"]
    layer = [(d, d), (d,)] * 4 + [(4 * d, d), (4 * d,), (d, 4 * d), (d,)] + [(d,)] * 4
    return layer * case["layers"] + [(case["V"], d), (case["V"],), (2 * d + 1,), (3,), (1,)]


def work(case):
    e = DTYPES[case["dtype"]].itemsize
    if case["op"] in ("policy", "preference"):
        rows = case["B"] * case["T"]
        return {"bytes": 2 * rows * case["V"] * e + rows * 32, "flops": 8 * rows * case["V"]}
    if case["op"] == "embedding":
        n, d, v = case["B"] * case["T"], case["D"], case["V"]
        fwd = n * 8 + (min(n, v) + n) * d * e
        return {"bytes": fwd + ((n + v) * d * e + n * 8 if case["grad"] else 0), "flops": (2 if case["grad"] else 1) * n * d}
    n = sum(math.prod(s) for s in _shapes(case))
    return {"bytes": n * e + (0 if case["inplace"] else n * 4), "flops": 3 * n}


def _frequent(n, v, g):
    """token ids as text has them: the k-th most frequent one with a share of about 1 / k"""
    p = 1.0 / (torch.arange(v, device="cuda", dtype=torch.float64) + 2.7)
    cdf = torch.cumsum(p / p.sum(), 0)
    return torch.searchsorted(cdf, torch.rand(n, device="cuda", dtype=torch.float64, generator=g)).clamp_(max=v - 1)


def _logp64(logits, ids):
    """log-probabilities of the ids in 64 bits, a few rows at a time"""
    out = []
    for x, t in zip(logits.reshape(-1, logits.shape[-1]).split(512), ids.reshape(-1).split(512)):
        out.append(torch.log_softmax(x.double(), -1).gather(1, t[:, None])[:, 0])
    return torch.cat(out).view(ids.shape)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, device="cuda", generator=g)

    st = {"case": case}
    if case["op"] in ("policy", "preference"):
        B, T, V = case["B"], case["T"], case["V"]
        full = torch.empty(B, T + 1 if case["view"] else T, V, device="cuda", dtype=dt)
        for b in range(B):
            full[b] = randn(*full[b].shape) * 2.5
        ids = 2 + _frequent(B * T, V - 2, g).view(B, T)
        length = torch.randint(1, T + 1, (B, 1), device="cuda", generator=g)
        length[torch.arange(B, device="cuda") % 3 == 0] = T          # (a third of the sequences run to the end)
        if B > 4:
            length[B - 1] = 0 if case["masked"] == "mask" else 1     # (one that holds nothing)
        inside = torch.arange(T, device="cuda")[None] < length
        if case["masked"] == "pad":
            ids = torch.where(inside, ids, torch.full_like(ids, PAD))
        else:
            inside &= torch.rand(B, T, device="cuda", generator=g) > 0.05      # (tokens of a prompt or a tool in the middle are not trained on)
            st["mask"] = inside
        logits = full[:, :-1] if case["view"] else full
        # the sampled tokens stand out of the distribution, as sampled ones do
        logits.scatter_add_(2, ids[..., None], (4.0 + randn(B, T, 1)).to(dt))
        st.update(logits=logits.detach().requires_grad_(True), ids=ids)
        lp = _logp64(logits.detach(), ids)
        if case["op"] == "policy":
            # an earlier policy's log-probabilities; the gradient jumps at the borders of the clip range, where either side is right: none lies there
            old = 0.2 * randn(B, T).double()
            for border in (0.8, 1.2):
                near = ((-old).exp() - border).abs() < 1e-3
                old = torch.where(near, old + 0.01, old)
            st["old"] = (lp + old).float()
            st["ref"] = (lp + 0.15 * randn(B, T)).float() if case["kl"] else None
            st["adv"] = randn(B) if case["adv"] == "seq" else randn(B, T)
        else:
            w = inside.double()
            ref = (w * (lp + 0.1 * randn(B, T))).sum(1)
            st["ref"] = (ref / w.sum(1).clamp(min=1) if case["mean"] else ref).float()
    elif case["op"] == "embedding":
        B, T, V, D = case["B"], case["T"], case["V"], case["D"]
        ids = 2 + _frequent(B * T, V - 2, g).view(B, T)
        length = torch.randint(1, T + 1, (B, 1), device="cuda", generator=g)
        length[::2] = T
        st["ids"] = torch.where(torch.arange(T, device="cuda")[None] < length, ids, torch.full_like(ids, PAD))
        st["W"] = (0.4 * randn(V, D)).to(dt).requires_grad_(case["grad"])
        st["dout"] = randn(B, T, D).to(dt) if case["grad"] else None
    else:
        shapes = _shapes(case)
        sizes = [math.prod(s) for s in shapes]
        arena = randn(sum(sizes)).mul_(1e-3).to(dt)
        st["grads"] = [t.view(s).mul_(1 + i % 7) for i, (t, s) in enumerate(zip(arena.split(sizes), shapes))]
        if case["inplace"]:          # a settled run: the norm stays below the bound, step after step
            st["out"], st["max_norm"] = arena, 1e4
            views = None
        else:
            st["out"] = torch.empty(arena.numel(), device="cuda")
            st["max_norm"] = 0.5 if case["norm"] == "l2" else 1e-3
            views = st["views"] = [t.view(s) for t, s in zip(st["out"].split(sizes), shapes)]
        if own:
            from bmt_amd.optim import GradClipper
            st["clipper"] = GradClipper(st["grads"], st["max_norm"], norm_type=2.0 if case["norm"] == "l2" else math.inf, out=views)
    return st


def _valid(st):
    return st["mask"] if "mask" in st else st["ids"] != PAD


def _statistics(x, ids):
    """exp(x - max), its sums (64 bits) and the log-probabilities of the ids (64 bits)"""
    m = x.amax(-1, keepdim=True)
    at = x.gather(-1, ids[..., None])
    e = x.sub_(m).exp_()
    s = e.sum(-1, keepdim=True, dtype=torch.float64)
    return e, s, ((at.double() - m.double()) - s.log())[..., 0]


def _logit_grad(e, s, w, ids, dt):
    """w (1[c = id] - softmax)"""
    d = e.mul_((-w[..., None] / s).float())
    return d.scatter_add_(-1, ids[..., None], w.float()[..., None]).to(dt)


def _policy_rows(st, lp, c):
    valid, adv = _valid(st), st["adv"].double()
    adv = adv[:, None] if adv.dim() == 1 else adv
    rho = (lp - st["old"].double()).exp()
    u, cl = rho * adv, rho.clamp(0.8, 1.2) * adv
    loss, w = -torch.minimum(u, cl), -torch.where(u <= cl, u, torch.zeros_like(u))
    kl = torch.zeros_like(lp)
    if c["kl"]:
        d = st["ref"].double() - lp
        kl = d.expm1() - d
        loss, w = loss + c["kl"] * kl, w - c["kl"] * d.expm1()
    n = valid.sum().clamp(min=1).double()
    norm = 1.0 / n if c["reduction"] == "token" else 1.0 / (c["B"] * valid.sum(1, keepdim=True).clamp(min=1).double())
    zero = torch.zeros_like(lp)
    return {"loss": torch.where(valid, loss * norm, zero).sum(), "kl": torch.where(valid, kl, zero).sum() / n,
            "clipped": torch.where(valid, (u > cl).double(), zero).sum() / n, "logp": torch.where(valid, lp, zero),
            "w": torch.where(valid, w * norm, zero)}


def _preference_rows(st, lp, c):
    valid = _valid(st)
    inv = 1.0 / valid.sum(1).clamp(min=1).double() if c["mean"] else torch.ones(c["B"], device=lp.device, dtype=torch.float64)
    r = 0.1 * (torch.where(valid, lp, torch.zeros_like(lp)).sum(1) * inv - st["ref"].double())
    P = c["B"] // 2
    z, ls = r[:P] - r[P:], c["smooth"]
    loss = ((1 - ls) * torch.log1p((-z.abs()).exp()) + (1 - ls) * (-z).clamp(min=0) + ls * torch.log1p((-z.abs()).exp()) + ls * z.clamp(min=0)).mean()
    d = -(0.1 / P) * ((1 - ls) * torch.sigmoid(-z) - ls * torch.sigmoid(z))
    w = torch.cat([d, -d]) * inv
    return {"loss": loss, "rewards": r, "w": torch.where(valid, w[:, None], torch.zeros_like(lp))}


def _rounded(rows, dt):
    return {k: v.to(dt) for k, v in rows.items() if k != "w"}


def run(state):
    c = state["case"]
    if own:
        return _run_own(state, c)
    if c["op"] in ("policy", "preference"):
        e, s, lp = _statistics(state["logits"].detach().to(torch.float32, copy=True), state["ids"])
        rows = (_policy_rows if c["op"] == "policy" else _preference_rows)(state, lp, c)
        return {**_rounded(rows, torch.float32), "dlogits": _logit_grad(e, s, rows["w"], state["ids"], state["logits"].dtype)}
    if c["op"] == "embedding":
        W, scale = state["W"].detach(), math.sqrt(c["D"])
        out = (W[state["ids"]].float() * scale).to(W.dtype)
        if not c["grad"]:
            return {"out": out}
        dW = torch.zeros(c["V"], c["D"], device=W.device)
        dW.index_add_(0, state["ids"].reshape(-1), state["dout"].reshape(-1, c["D"]).float())
        dW[PAD] = 0
        return {"out": out, "dW": dW.mul_(scale).to(W.dtype)}
    if c["norm"] == "l2":
        norm = torch.stack([g.float().square().sum(dtype=torch.float64) for g in state["grads"]]).sum().sqrt()
    else:
        norm = torch.stack([g.abs().amax().double() for g in state["grads"]]).amax()
    coef = (state["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    for g, o in zip(state["grads"], state["grads"] if c["inplace"] else state["views"]):
        o.copy_(g.float() * coef)
    return {"norm": norm.float(), "out": state["out"]}


def _run_own(state, c):
    from bmt_amd import ops
    if c["op"] == "policy":
        loss, stats = ops.policy_loss(state["logits"], state["ids"], state["old"], state["adv"], ref_logp=state["ref"], mask=state.get("mask"),
                                      pad_idx=None if "mask" in state else PAD, kl_coef=c["kl"], reduction=c["reduction"])
        (dlogits,) = torch.autograd.grad(loss, state["logits"])
        return {"loss": loss, "kl": stats.kl, "clipped": stats.clip_fraction, "logp": stats.logp, "dlogits": dlogits}
    if c["op"] == "preference":
        loss, rewards = ops.preference_loss(state["logits"], state["ids"], state["ref"], mask=state.get("mask"), pad_idx=None if "mask" in state else PAD,
                                            beta=0.1, label_smoothing=c["smooth"], mean_logp=c["mean"])
        (dlogits,) = torch.autograd.grad(loss, state["logits"])
        return {"loss": loss, "rewards": rewards, "dlogits": dlogits}
    if c["op"] == "embedding":
        out = ops.embedding(state["ids"], state["W"], scale=math.sqrt(c["D"]), pad_idx=PAD)
        if not c["grad"]:
            return {"out": out}
        (dW,) = torch.autograd.grad(out, state["W"], state["dout"])
        return {"out": out, "dW": dW}
    return {"norm": state["clipper"](), "out": state["out"]}


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("policy", "preference"):
        logits, ids = st["logits"].detach(), st["ids"]
        B, T, V = logits.shape
        lp = _logp64(logits, ids).requires_grad_(True)
        valid = (st["mask"] if "mask" in st else ids != PAD).double()
        if case["op"] == "policy":
            adv = st["adv"].double()
            adv = adv.unsqueeze(1).expand(B, T) if adv.dim() == 1 else adv
            rho = torch.exp(lp - st["old"].double())
            inside = torch.clamp(rho, 1 - 0.2, 1 + 0.2)
            each = -torch.minimum(rho * adv, inside * adv)
            kl = torch.zeros_like(lp)
            if case["kl"]:
                diff = st["ref"].double() - lp
                kl = torch.exp(diff) - diff - 1
                each = each + case["kl"] * kl
            n = max(1.0, float(valid.sum()))
            per = (each * valid).sum(1) / valid.sum(1).clamp(min=1)
            loss = (each * valid).sum() / n if case["reduction"] == "token" else per.mean()
            more = {"kl": ((kl * valid).sum() / n).detach(), "clipped": ((rho * adv > inside * adv).double() * valid).sum() / n, "logp": (lp * valid).detach()}
        else:
            P = B // 2
            total = (lp * valid).sum(1)
            if case["mean"]:
                total = total / valid.sum(1).clamp(min=1)
            r = 0.1 * (total - st["ref"].double())
            z = r[:P] - r[P:]
            loss = -((1 - case["smooth"]) * torch.nn.functional.logsigmoid(z) + case["smooth"] * torch.nn.functional.logsigmoid(-z)).mean()
            more = {"rewards": r.detach()}
        (dlp,) = torch.autograd.grad(loss, lp)
        dlogits = torch.empty(B, T, V, device="cuda", dtype=torch.float64)
        for b in range(B):
            d = torch.softmax(logits[b].double(), -1).neg_()
            d[torch.arange(T, device="cuda"), ids[b]] += 1
            torch.mul(d, dlp[b][:, None], out=dlogits[b])
        return {"loss": loss.detach(), **more, "dlogits": dlogits}
    if case["op"] == "embedding":
        D, V = case["D"], case["V"]
        out = st["W"].detach().double()[st["ids"]] * math.sqrt(D)
        if not case["grad"]:
            return {"out": out}
        flat = st["ids"].reshape(-1)
        dW = torch.zeros(V, D, device="cuda", dtype=torch.float64)
        keep = flat != PAD
        dW.index_put_((flat[keep],), st["dout"].reshape(-1, D)[keep].double() * math.sqrt(D), accumulate=True)
        return {"out": out, "dW": dW}
    flat = torch.cat([g.reshape(-1) for g in st["grads"]]).double()
    norm = flat.norm() if case["norm"] == "l2" else flat.abs().max()
    return {"norm": norm, "out": flat * min(1.0, st["max_norm"] / (float(norm) + 1e-6))}
