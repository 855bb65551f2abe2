"""What is measured of the fine-tuning operators: log-probabilities of given labels, the preference loss and the clipped
policy loss with their gradients, gradient clipping over many tensors, and the Adam step that clips as it reads.

`own` chooses what run() calls: False computes the operators in plain torch, True calls spice_amd.ops."""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}


def listed():
    return [
        # a sampled token is scored while an answer is being written: one row, forward only
        dict(name="logprobs one token", kind="logprobs", layout="tokens", n=1, l=1, c=32000, dtype="bf16", shift=False, pad=0,
             temperature=0.7, grad=False),
        # scoring answers for a loss of the user's own: next-token shift as a view, vocabulary padded in memory, odd size
        dict(name="logprobs shifted padded", kind="logprobs", layout="tokens", n=4, l=1023, c=50001, dtype="bf16", shift=True,
             pad=47, temperature=1.0, grad=True),
        # the shortest pair: two odd answers of one prompt
        dict(name="preference one odd pair", kind="preference", layout="tokens", n=2, l=37, c=50001, dtype="fp16", shift=False,
             pad=0, loss="ipo", average=True, beta=0.1, smoothing=0.0, scale=128.0),
        # a batch of four answer pairs
        dict(name="preference token pairs", kind="preference", layout="tokens", n=8, l=1024, c=32000, dtype="bf16", shift=False,
             pad=0, loss="sigmoid", average=False, beta=0.1, smoothing=0.1, scale=1.0),
        # four pictures with a better and a worse label map each, at the segmentation benchmark's size
        dict(name="preference mask pairs", kind="preference", layout="pixels", n=8, l=512 * 512, c=21, dtype="fp32", shift=False,
             pad=0, loss="sigmoid", average=True, beta=2.0, smoothing=0.0, scale=1.0),
        # one short answer
        dict(name="policy short answer", kind="policy", layout="tokens", n=1, l=7, c=32000, dtype="fp16", shift=False, pad=0,
             reduction="token", kl=0.05, temperature=1.0, scale=1.0),
        # a group of eight answers to one prompt, large vocabulary
        dict(name="policy answer group", kind="policy", layout="tokens", n=8, l=512, c=131072, dtype="bf16", shift=False, pad=0,
             reduction="sequence", kl=0.05, temperature=1.0, scale=1.0),
        # sampled label maps with a reward each, at the segmentation benchmark's size
        dict(name="policy sampled masks", kind="policy", layout="pixels", n=8, l=512 * 512, c=21, dtype="fp32", shift=False, pad=0,
             reduction="token", kl=0.1, temperature=1.0, scale=1.0),
        # a toy network: a dozen small tensors, launches count
        dict(name="clip toy network", kind="clip", tensors=12, least=5, most=2304, dtype="fp32", out="fp32"),
        # about the tensors of a ResNet-50 segmentation model, half-precision gradients clipped into fp32 ones
        dict(name="clip bf16 into fp32", kind="clip", tensors=190, least=21, most=2359296, dtype="bf16", out="fp32"),
        # the same model's update
        dict(name="adam segmentation model", kind="adam", tensors=190, least=21, most=2359296, dtype="fp32", decoupled=False),
        # a network of some 800 million parameters
        dict(name="adam large network", kind="adam", tensors=200, least=5, most=1 << 26, dtype="fp32", decoupled=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["logprobs", "preference", "policy", "clip", "adam"])
    if kind in ("clip", "adam"):
        tensors = rng.choice([1, 2, 7, 33, 97, 161, 257])
        most = _log(rng, 64, 1 << 24)
        case = dict(kind=kind, tensors=tensors, least=min(most, _log(rng, 1, 64)), most=most, dtype=rng.choice(["fp32", "bf16", "fp16"]))
        if kind == "clip":
            return dict(case, out=rng.choice([case["dtype"], "fp32"]))
        return dict(case, decoupled=rng.random() < 0.5)
    layout = rng.choice(["tokens", "tokens", "pixels"])
    n = rng.choice([2, 4, 6, 8, 16]) if kind == "preference" else _log(rng, 1, 16)
    if layout == "tokens":
        c = _log(rng, 1000, 131072)
        l = _log(rng, 1, max(2, min(4096, (1 << 28) // (n * c))))
    else:
        c = rng.choice([2, 5, 19, 21, 64, 150])
        l = _log(rng, 1, max(2, min(512 * 512, (1 << 25) // (n * c))))
    case = dict(kind=kind, layout=layout, n=n, l=l, c=c, dtype=rng.choice(["bf16", "fp16", "fp32"]),
                shift=layout == "tokens" and rng.random() < 0.3, pad=rng.choice([0, 0, 3, 64]) if layout == "tokens" else 0)
    # half-precision gradients of a mean over many positions need the loss scale that training in fp16 uses
    scale = 2.0 ** round(math.log2(n * l)) if case["dtype"] == "fp16" else 1.0
    if kind == "preference":
        average = layout == "pixels" or rng.random() < 0.5
        return dict(case, scale=scale if average else 1.0, average=average, loss=rng.choice(["sigmoid", "ipo"]),
                    beta=rng.choice([0.1, 0.5, 2.0] if average else [0.05, 0.1]), smoothing=rng.choice([0.0, 0.1]))
    if kind == "policy":
        return dict(case, scale=scale, reduction=rng.choice(["token", "sequence"]), kl=rng.choice([0.0, 0.05]), temperature=rng.choice([1.0, 0.7]))
    return dict(case, temperature=rng.choice([1.0, 0.7, 2.0]), grad=rng.random() < 0.7)


# ---- inputs


def _sizes(case):
    """Element counts of the tensors: spread over their logarithm, every third one odd."""
    k, lo, hi = case["tensors"], case["least"], case["most"]
    got = [int(round(lo * (hi / lo) ** (i / (k - 1)))) if k > 1 else hi for i in range(k)]
    return [s | 1 if i % 3 == 1 else s for i, s in enumerate(got)]


def _views(flat, sizes):
    """Tensors laid out in one buffer, each on a 64-element boundary, as the trainer's gradient buckets lay them."""
    at, got = 0, []
    for s in sizes:
        got.append(flat[at:at + s])
        at += -(-s // 64) * 64
    return got


def _flat(sizes, dtype, gen, scale):
    """Normal values in the tensors, zeros between them."""
    total = sum(-(-s // 64) * 64 for s in sizes)
    flat = torch.zeros(total, device="cuda", dtype=dtype)
    for v in _views(flat, sizes):
        v.normal_(0.0, scale, generator=gen)
    return flat


def _prepare_tensors(case, gen):
    sizes = _sizes(case)
    if case["kind"] == "clip":
        grads = _flat(sizes, _TYPES[case["dtype"]], gen, 0.02)
        out = torch.zeros(grads.numel(), device="cuda", dtype=_TYPES[case["out"]])
        limit = 0.25 * 0.02 * math.sqrt(sum(sizes))
        return dict(case=case, grads=grads, out=out, grad_list=_views(grads, sizes), out_list=_views(out, sizes), limit=limit)
    kind = _TYPES[case["dtype"]]
    params, grads = _flat(sizes, kind, gen, 0.05), _flat(sizes, kind, gen, 0.02)
    m, v = _flat(sizes, torch.float32, gen, 0.003), _flat(sizes, torch.float32, gen, 0.01).square_()
    state = dict(case=case, params=params, grads=grads, m=m, v=v, step=torch.full((1,), 10, dtype=torch.int64, device="cuda"),
                 limit=0.25 * 0.02 * math.sqrt(sum(sizes)))
    for k in ("params", "grads", "m", "v"):
        state[k + "_list"] = _views(state[k], sizes)
    return state


def _ignore(case):
    return 255 if case["layout"] == "pixels" else -100


def _class_dim(case):
    return 1 if case["layout"] == "pixels" else 2


def _prepare_logits(case, gen):
    n, l, c, dev, kind = case["n"], case["l"], case["c"], "cuda", _TYPES[case["dtype"]]
    pixels = case["layout"] == "pixels"
    rows = l + 1 if case["shift"] else l
    labels = torch.randint(0, c, (n, rows), device=dev, generator=gen)
    shape = (n, c, rows) if pixels else (n, rows, c + case["pad"])
    logits = torch.empty(shape, device=dev, dtype=kind).normal_(0.0, 1.5, generator=gen)
    if case["shift"]:
        logits, labels = logits[:, :-1], labels[:, 1:]
    if case["pad"]:
        logits = logits[..., :c]
    # the label stands out, as a trained model's does
    at = labels.unsqueeze(_class_dim(case))
    logits.scatter_(_class_dim(case), at, logits.gather(_class_dim(case), at) + 5.0)
    # a prompt in front and padding behind each answer; a few ignored pixels; the last of many sequences is empty
    if pixels:
        out = torch.rand(n, l, device=dev, generator=gen) < 0.05
    else:
        begin = (torch.rand(n, 1, device=dev, generator=gen) * 0.4 * l).long()
        end = l - (torch.rand(n, 1, device=dev, generator=gen) * 0.3 * l).long()
        at = torch.arange(l, device=dev)
        out = (at < begin) | (at >= end)
    if n >= 8:
        out[n - 1] = True
    return logits, labels.masked_fill(out, _ignore(case)), out


def _true_logprobs(case, logits, labels, out):
    t = case.get("temperature", 1.0)
    z = logits.double() / t
    d = _class_dim(case)
    return (z.gather(d, labels.masked_fill(out, 0).unsqueeze(d)) - torch.logsumexp(z, d, keepdim=True)).squeeze(d)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    if case["kind"] in ("clip", "adam"):
        return _prepare_tensors(case, gen)
    n, l, dev = case["n"], case["l"], "cuda"
    logits, labels, out = _prepare_logits(case, gen)
    state = dict(case=case, logits=logits, labels=labels)
    if case["kind"] == "logprobs":
        state["weight"] = torch.randn(n, l, device=dev, generator=gen)
        return state
    logp = _true_logprobs(case, logits, labels, out)
    state["ref"] = (logp + 0.2 * torch.randn(n, l, device=dev, generator=gen).double()).float()
    if case["kind"] == "preference":
        # training has moved the better half's log-probabilities up and the other half's down
        up = 0.02 if case["average"] else 10.0 / l
        state["ref"][: n // 2] -= up
        state["ref"][n // 2:] += up
    if case["kind"] == "policy":
        state["advantages"] = torch.randn(n, device=dev, generator=gen)
        # how far the policy has moved since it sampled; no ratio lies on a border of the clipping, where both
        # branches are right
        moved = 0.15 * torch.randn(n, l, device=dev, generator=gen).double()
        for border in (math.log(0.8), math.log(1.25)):
            moved = torch.where((moved - border).abs() < 1e-3, moved + 3e-3, moved)
        state["old"] = (logp - moved).float()
    return state


# ---- the operators in plain torch


def _plain_softmax(state, total=torch.float32):
    """(log-probability of the label, softmax, mask of the counted positions, the label to gather): in 32 bits, the
    sum of the exponentials and its logarithm in `total`."""
    case, d = state["case"], _class_dim(state["case"])
    keep = state["labels"] != _ignore(case)
    at = torch.where(keep, state["labels"], 0).unsqueeze(d)
    z = state["logits"].float()
    if case.get("temperature", 1.0) != 1.0:
        z = z / case["temperature"]
    z = z - z.amax(d, keepdim=True)
    e = torch.exp(z)
    s = e.sum(d, keepdim=True, dtype=total)
    logp = (z.gather(d, at).to(total) - torch.log(s)).squeeze(d)
    return torch.where(keep, logp, 0.0), e / s.float(), keep, at


def _plain_grad(state, p, at, weight):
    """d sum(weight * logp) / d logits."""
    case, d = state["case"], _class_dim(state["case"])
    w = (weight / case.get("temperature", 1.0)).unsqueeze(d)
    return (p * -w).scatter_add(d, at, w).to(state["logits"].dtype)


def _plain_logprobs(state):
    logp, p, keep, at = _plain_softmax(state)
    if not state["case"]["grad"]:
        return [logp]
    return [logp, _plain_grad(state, p, at, torch.where(keep, state["weight"], 0.0))]


def _plain_preference(state):
    case = state["case"]
    # a sequence's log ratio is a small difference of many log-probabilities: they are taken in 64 bits
    logp, p, keep, at = _plain_softmax(state, torch.float64)
    count = keep.sum(1).clamp(min=1).double() if case["average"] else torch.ones((), dtype=torch.float64, device=logp.device)
    total = (torch.where(keep, logp - state["ref"].double(), 0.0)).sum(1) / count
    half, beta, eps = case["n"] // 2, case["beta"], case["smoothing"]
    h = total[:half] - total[half:]
    if case["loss"] == "sigmoid":
        up, down = torch.sigmoid(beta * h), torch.sigmoid(-beta * h)
        loss = -(1 - eps) * torch.log(up) - eps * torch.log(down)
        dh = -beta * ((1 - eps) * down - eps * up)
    else:
        loss = (h - 0.5 / beta) ** 2
        dh = 2 * (h - 0.5 / beta)
    w = torch.cat([dh, -dh]) * (case["scale"] / half) / count
    grad = _plain_grad(state, p, at, torch.where(keep, w.float().unsqueeze(1), 0.0))
    return [loss.mean().float(), (beta * total).float(), grad]


def _plain_policy(state):
    case = state["case"]
    logp, p, keep, at = _plain_softmax(state)
    adv = state["advantages"].unsqueeze(1)
    ratio = torch.exp(logp - state["old"])
    free, clipped = ratio * adv, ratio.clamp(0.8, 1.25) * adv
    over = free > clipped
    back = torch.exp(state["ref"] - logp)
    kl = back - (state["ref"] - logp) - 1.0
    valid = keep.sum(1)
    if case["reduction"] == "token":
        share = (1.0 / valid.sum().clamp(min=1).double()).expand(case["n"], 1)
    else:
        share = (1.0 / (valid.clamp(min=1).double() * case["n"])).unsqueeze(1)
    mean = lambda x: (torch.where(keep, x, 0.0).double() * share).sum()  # noqa: E731
    surrogate, far = mean(-torch.minimum(free, clipped)), mean(kl)
    part = (over & keep).sum().double() / valid.sum().clamp(min=1)
    if case["kl"] == 0.0:
        far = torch.zeros_like(far)
    out = torch.stack([surrogate + case["kl"] * far, surrogate, far, part]).float()
    dl = torch.where(over, 0.0, -free) + case["kl"] * (1.0 - back)
    return [out, logp, _plain_grad(state, p, at, torch.where(keep, dl * (case["scale"] * share).float(), 0.0))]


def _plain_norm(state):
    norm = state["grads"].double().square().sum().sqrt()
    return norm.float(), (state["limit"] / (norm + 1e-6)).clamp(max=1.0).float()


def _plain_clip(state):
    norm, scale = _plain_norm(state)
    state["out"].copy_(state["grads"].float() * scale)
    return [norm, state["out"]]


_ADAM = dict(lr=1e-3, beta1=0.9, beta2=0.999, eps=1e-8, weight_decay=1e-2)


def _plain_adam(state):
    lr, b1, b2, eps, wd = _ADAM["lr"], _ADAM["beta1"], _ADAM["beta2"], _ADAM["eps"], _ADAM["weight_decay"]
    norm, scale = _plain_norm(state)
    state["step"] += 1
    t = state["step"].double()
    p, g = state["params"].float(), state["grads"].float() * scale
    if state["case"]["decoupled"]:
        p = p * (1.0 - lr * wd)
    else:
        g = g + wd * p
    state["m"].mul_(b1).add_(g, alpha=1.0 - b1)
    state["v"].mul_(b2).add_(g * g, alpha=1.0 - b2)
    denom = state["v"].sqrt() * (1.0 / torch.sqrt(1.0 - b2 ** t)).float() + eps
    state["params"].copy_(p - (lr / (1.0 - b1 ** t)).float() * state["m"] / denom)
    return [norm, state["params"], state["m"], state["v"], state["step"]]


# ---- the framework's calls


def _own(state):
    from spice_amd import ops
    case = state["case"]
    if case["kind"] == "clip":
        return [ops.clip_grad_norm(state["grad_list"], state["limit"], out=state["out_list"]), state["out"]]
    if case["kind"] == "adam":
        norm = ops.adam_step(state["params_list"], state["grads_list"], state["m_list"], state["v_list"], state["step"],
                             lr=_ADAM["lr"], betas=(_ADAM["beta1"], _ADAM["beta2"]), eps=_ADAM["eps"],
                             weight_decay=_ADAM["weight_decay"], decoupled=case["decoupled"], max_norm=state["limit"])
        return [norm, state["params"], state["m"], state["v"], state["step"]]
    logits, labels = state["logits"], state["labels"]
    how = dict(class_dim=_class_dim(case), ignore_index=_ignore(case))
    if case["kind"] == "logprobs":
        logp, lse = ops.token_logprobs(logits, labels, temperature=case["temperature"], **how)
        if not case["grad"]:
            return [logp]
        return [logp, ops.token_logprobs_grad(logits, labels, lse, state["weight"], temperature=case["temperature"], **how)]
    if case["kind"] == "preference":
        return list(ops.preference_loss(logits, labels, state["ref"], beta=case["beta"],
                                        label_smoothing=case["smoothing"] if case["loss"] == "sigmoid" else 0.0,
                                        loss_type=case["loss"], average=case["average"], want_grad=True,
                                        grad_scale=case["scale"], **how))
    return list(ops.policy_loss(logits, labels, state["old"], state["advantages"],
                                ref_logprobs=state["ref"] if case["kl"] else None, clip_low=0.2, clip_high=0.25,
                                kl_weight=case["kl"], reduction=case["reduction"], temperature=case["temperature"],
                                want_grad=True, grad_scale=case["scale"], **how))


_PLAIN = {"logprobs": _plain_logprobs, "preference": _plain_preference, "policy": _plain_policy, "clip": _plain_clip,
          "adam": _plain_adam}


def run(state):
    return _own(state) if own else _PLAIN[state["case"]["kind"]](state)


def work(case):
    size = {"fp32": 4, "fp16": 2, "bf16": 2}
    if case["kind"] in ("clip", "adam"):
        e, g = sum(_sizes(case)), size[case["dtype"]]
        if case["kind"] == "clip":
            return {"bytes": e * (g + size[case["out"]]), "flops": 3 * e}
        return {"bytes": e * (3 * g + 16), "flops": 14 * e}
    p, e = case["n"] * case["l"], size[case["dtype"]]
    x = p * case["c"]
    if case["kind"] == "logprobs":
        return {"bytes": x * e + 12 * p + (x * e + 4 * p if case["grad"] else 0), "flops": (7 if case["grad"] else 4) * x}
    if case["kind"] == "preference":
        return {"bytes": 2 * x * e + 12 * p, "flops": 7 * x}
    return {"bytes": 2 * x * e + (20 if case["kl"] else 16) * p, "flops": 7 * x}


# ---- the definitions in 64 bits


def _exact_tensors(state):
    case = state["case"]
    flat = torch.cat([g.double() for g in state["grads_list" if case["kind"] == "adam" else "grad_list"]])
    norm = torch.linalg.vector_norm(flat)
    scale = min(1.0, state["limit"] / (norm.item() + 1e-6))
    del flat
    if case["kind"] == "clip":
        return [norm, state["grads"].double() * scale]
    lr, b1, b2, t = _ADAM["lr"], _ADAM["beta1"], _ADAM["beta2"], int(state["step"].item()) + 1
    p, g = state["params"].double(), state["grads"].double() * scale
    if case["decoupled"]:
        p = p - lr * _ADAM["weight_decay"] * p
    else:
        g = g + _ADAM["weight_decay"] * p
    m = state["m"].double() + (1.0 - b1) * (g - state["m"].double())
    v = state["v"].double() + (1.0 - b2) * (g.square() - state["v"].double())
    p = p - lr * (m / (1.0 - b1 ** t)) / ((v / (1.0 - b2 ** t)).sqrt() + _ADAM["eps"])
    return [norm, p, m, v, None]


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] in ("clip", "adam"):
        return _exact_tensors(state)
    d, n = _class_dim(case), case["n"]
    keep = state["labels"] != _ignore(case)
    x = state["logits"].double().requires_grad_(True)
    chosen = torch.where(keep, state["labels"], 0).unsqueeze(d)
    logp = torch.log_softmax(x / case.get("temperature", 1.0), d).gather(d, chosen).squeeze(d) * keep
    if case["kind"] == "logprobs":
        if not case["grad"]:
            return [logp.detach()]
        return [logp.detach(), torch.autograd.grad((logp * state["weight"].double()).sum(), x)[0]]
    tokens = keep.sum(1).clamp(min=1).double()
    ref = state["ref"].double()
    if case["kind"] == "preference":
        s = ((logp - ref) * keep).sum(1)
        if case["average"]:
            s = s / tokens
        h = s[: n // 2] - s[n // 2:]
        if case["loss"] == "sigmoid":
            loss = -(1 - case["smoothing"]) * torch.nn.functional.logsigmoid(case["beta"] * h) \
                - case["smoothing"] * torch.nn.functional.logsigmoid(-case["beta"] * h)
        else:
            loss = (h - 1.0 / (2.0 * case["beta"])).square()
        loss = loss.mean()
        return [loss.detach(), (case["beta"] * s).detach(), torch.autograd.grad(case["scale"] * loss, x)[0]]
    adv = state["advantages"].double().unsqueeze(1)
    r = torch.exp(logp - state["old"].double())
    inside = r.clamp(1.0 - 0.2, 1.0 + 0.25)
    surrogate = -torch.min(r * adv, inside * adv) * keep
    far = (torch.exp(ref - logp) + (logp - ref) - 1.0) * keep
    if case["reduction"] == "token":
        surrogate, far = surrogate.sum() / keep.sum().clamp(min=1), far.sum() / keep.sum().clamp(min=1)
    else:
        surrogate, far = (surrogate.sum(1) / tokens).mean(), (far.sum(1) / tokens).mean()
    if not case["kl"]:
        far = 0.0 * far
    total = surrogate + case["kl"] * far
    part = (((r * adv) > (inside * adv)) & keep).sum() / keep.sum().clamp(min=1).double()
    return [torch.stack([total, surrogate, far, part]).detach(), logp.detach(), torch.autograd.grad(case["scale"] * total, x)[0]]
