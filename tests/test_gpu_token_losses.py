"""Label log-probabilities, preference loss and clipped policy loss on the GPU against the 64-bit oracle.

Tolerances, with u = 2^-24 (half a step of fp32) and D the spread of a position's finite logits over T:
 * exp((x - m) / T): x - m rounds once, its product with log2(e) / T twice, each by u relative, so the exponent is off by at
   most 2 u D and the exponential by that plus the instruction's 2 u; a sum of C of them adds at most one u a step on the
   longest chain, min(C, 256 + C / 64) steps: s is off by R = u (2 D + 4 + steps) relative;
 * logp = d / T - log s: R, plus 2 u of each term and of the result;
 * a gradient w (1[label] - p) / T: w (p (2 R) + 4 u), plus half a step of the logits' type, plus half its least value.
What sums or multiplies these (a sequence's log ratio, a ratio's exponential) carries the bound through its derivative."""
import math

import pytest
import torch

from oracle import tokenloss as ot
from spice_amd import ops
from spice_amd.pruning.losses import ClippedPolicyLoss, PreferenceLoss, token_logprobs

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
LEAST = {torch.float32: 2.0 ** -126, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}

# (layout, n, positions, c, dtype): single positions and classes, odd sizes, vocabularies over every kernel's row length
SHAPES = [
    ("last", 1, (1,), 1, torch.float32), ("last", 1, (1,), 7, torch.bfloat16), ("last", 3, (), 257, torch.float32),
    ("last", 2, (5,), 33, torch.float16), ("last", 2, (3,), 1000, torch.float32), ("last", 2, (4,), 4097, torch.bfloat16),
    ("last", 2, (2, 3), 8192, torch.float16), ("last", 2, (3,), 32000, torch.bfloat16), ("last", 2, (2,), 50001, torch.float16),
    ("last", 1, (3,), 65537, torch.float32), ("last", 2, (1,), 131072, torch.bfloat16), ("last", 1, (2,), 200003, torch.bfloat16),
    ("last", 1, (2,), 150001, torch.float32), ("last", 2, (700,), 5, torch.float32), ("last", 1, (130,), 64, torch.bfloat16),
    ("planes", 1, (1,), 1, torch.float32), ("planes", 2, (7, 9), 5, torch.float32), ("planes", 2, (16, 16), 21, torch.float32),
    ("planes", 3, (33,), 19, torch.bfloat16), ("planes", 2, (64, 36), 21, torch.float16), ("planes", 2, (5, 3), 150, torch.float32),
    ("planes", 2, (12, 40), 200, torch.float32), ("planes", 1, (700,), 300, torch.bfloat16), ("planes", 2, (301,), 60, torch.float16),
    ("planes", 1, (601,), 100, torch.float32), ("planes", 1, (129,), 33, torch.float32), ("planes", 2, (260,), 128, torch.float16),
    ("last", 3, (50,), 31, torch.float32), ("last", 3, (50,), 127, torch.float32), ("last", 2, (33,), 255, torch.float16),
    ("last", 2, (9,), 767, torch.float32), ("last", 2, (9,), 20479, torch.float32), ("last", 1, (2,), 86015, torch.float32),
    ("planes", 1, (9000,), 2, torch.float16), ("planes", 1, (40, 41), 64, torch.bfloat16), ("planes", 2, (6,), 3001, torch.float32),
]
IDS = ["%s-%d-%s-%d-%s" % (s[0], s[1], "x".join(map(str, s[2])), s[3], str(s[4])[6:]) for s in SHAPES]


@pytest.fixture(scope="module")
def dev():
    assert torch.cuda.is_available()
    return torch.device("cuda:0")


def _inputs(layout, n, positions, c, dtype, seed=0, ignore=None):
    """(logits, labels, class_dim, ignore_index): about a sixth of the positions ignored, the label's logit raised."""
    g = torch.Generator().manual_seed(seed)
    ignore = (255 if c <= 255 else -100) if ignore is None else ignore
    x = 2.0 * torch.randn(n, *positions, c, generator=g)
    y = torch.randint(0, c, (n, *positions), generator=g)
    x.scatter_add_(-1, y.unsqueeze(-1), torch.full((n, *positions, 1), 4.0))
    y = torch.where(torch.rand(n, *positions, generator=g) < 1 / 6, ignore, y)
    if layout != "last":
        x = x.movedim(-1, 1)
    if layout == "planes":
        x = x.contiguous()
    return x.to(dtype), y, -1 if layout == "last" else 1, ignore


def _last(t, class_dim):
    return t.movedim(class_dim, -1)


def _bounds(x, class_dim, t):
    """(R, bound of logp without its own rounding): of the logits' positions, 64 bits."""
    z = _last(x.double(), class_dim)
    c = z.shape[-1]
    fine = torch.isfinite(z)
    top = torch.where(fine, z, -math.inf).amax(-1)
    low = torch.where(fine, z, math.inf).amin(-1)
    spread = torch.nan_to_num((top - low) / t, 0.0, 0.0, 0.0)
    r = U * (2 * spread + 4 + min(c, 256 + c / 64))
    return r, r + U * (2 * spread + 2 * math.log(c + 1) + 2)


def _grad_tol(x, g64, w, class_dim, t):
    """Bound of each gradient value; w: |weight| of each position (with whatever error it carries already in `extra`)."""
    r, _ = _bounds(x, class_dim, t)
    p = torch.softmax(torch.nan_to_num(_last(x.double(), class_dim), -math.inf, math.inf, -math.inf) / t, -1).nan_to_num(0.0)
    tol = (w / t).unsqueeze(-1) * (p * 2 * r.unsqueeze(-1) + 4 * U)
    tol = tol.movedim(-1, class_dim if class_dim == 1 else -1)
    return tol + HALF_STEP[x.dtype] * (g64.abs() + tol) + LEAST[x.dtype] / 2


def _close(got, want, tol, what=""):
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape, what
    off = (got - want).abs()
    bad = ~(off <= tol) & ~(torch.isnan(got) & torch.isnan(want)) & ~(got == want)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:5], want[bad][:5], float((off / tol).nan_to_num(0.0).max()))


@pytest.mark.parametrize("shape", SHAPES, ids=IDS)
@pytest.mark.parametrize("t", [1.0, 0.7])
def test_token_logprobs_and_gradient(dev, shape, t):
    x, y, d, ignore = _inputs(*shape)
    how = dict(class_dim=d, temperature=t, ignore_index=ignore)
    v = x.double().requires_grad_(True)
    want, keep = ot.token_logprobs(v, y, **how)
    weight = torch.randn(y.shape, generator=torch.Generator().manual_seed(1))
    g64, = torch.autograd.grad((want * weight.double()).sum(), v)
    xd, yd = x.to(dev), y.to(dev)
    logp, stats = ops.token_logprobs(xd, yd, **how)
    assert logp.dtype == torch.float32 and stats.shape == (*y.shape, 2)
    _close(logp, want.detach(), _bounds(x, d, t)[1] + 2 * U * want.detach().abs(), "logp")
    assert (logp.cpu()[~keep] == 0).all()
    grad = ops.token_logprobs_grad(xd, yd, stats, weight.to(dev), scale=4.0, **how)
    assert grad.dtype == x.dtype and grad.shape == x.shape
    _close(grad, 4 * g64, _grad_tol(x, 4 * g64, 4 * weight.abs().double(), d, t), "grad")
    # one weight a sequence, a factor on the device, and what a second call gives
    ws = weight.reshape(y.shape[0], -1)[:, 0].contiguous()
    wide = ws.view(-1, *([1] * (y.dim() - 1))).expand(y.shape)
    s64, = torch.autograd.grad((ot.token_logprobs(v, y, **how)[0] * wide.double()).sum(), v)
    half = torch.full((1,), 0.5, device=dev)
    seq = ops.token_logprobs_grad(xd, yd, stats, ws.to(dev), device_scale=half, **how)
    _close(seq, 0.5 * s64, _grad_tol(x, 0.5 * s64, 0.5 * wide.abs().double(), d, t), "grad a sequence")
    assert torch.equal(seq, ops.token_logprobs_grad(xd, yd, stats, ws.to(dev), device_scale=half, **how))
    assert torch.equal(logp, ops.token_logprobs(xd, yd, **how)[0])


@pytest.mark.parametrize("layout, positions, c", [("last", (6,), 5000), ("last", (40,), 9), ("planes", (8, 12), 21), ("planes", (5, 7), 70)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("t", [1.0, 0.7, 1.44269502, 3.0])
def test_excluded_classes_and_rubbish_in_ignored_positions(dev, layout, positions, c, dtype, t):
    """-inf and the type's lowest value as masks of classes, a row with nothing left, +inf, NaN; an ignored position may
    hold anything and gives zeros."""
    x, y, d, ignore = _inputs(layout, 2, positions, c, dtype, seed=5)
    rows = _last(x, d).reshape(-1, c).clone()
    lab = y.reshape(-1)
    lab[0], lab[1], lab[2], lab[3], lab[4], lab[5] = 1, 2, 3, 4, ignore, ignore
    rows[0, c // 2:] = -math.inf
    rows[1, 4:] = torch.finfo(dtype).min
    rows[2, :] = -math.inf
    rows[3, 0] = math.inf
    rows[4, :] = math.nan
    rows[5, ::2] = math.inf
    lab[6], lab[7] = 0, c - 1
    rows[6, 0] = -math.inf                     # the label itself is excluded
    rows[7, :] = torch.finfo(dtype).min       # a plain row at the lowest value
    x = rows.reshape(2, *positions, c).movedim(-1, d).contiguous()
    how = dict(class_dim=d, ignore_index=ignore, temperature=t)
    v = x.double().requires_grad_(True)
    want, keep = ot.token_logprobs(v, y, **how)
    weight = torch.rand(y.shape, generator=torch.Generator().manual_seed(2)) + 0.5
    logp, stats = ops.token_logprobs(x.to(dev), y.to(dev), **how)
    tol = _bounds(x, d, t)[1] + 2 * U * want.detach().abs().nan_to_num(0.0, 0.0, 0.0)
    got, ref = logp.cpu().double().reshape(-1), want.detach().reshape(-1)
    assert torch.isnan(got[2]) and torch.isnan(ref[2]) and torch.isnan(got[3]) and got[6] == -math.inf
    assert got[4] == 0 and got[5] == 0
    rest = torch.ones(len(got), dtype=torch.bool)
    rest[[2, 3, 6]] = False
    _close(got[rest], ref[rest], tol.reshape(-1)[rest])
    grad = ops.token_logprobs_grad(x.to(dev), y.to(dev), stats, weight.to(dev), **how)
    g = _last(grad, d).reshape(-1, c).cpu().double()
    assert (g[4] == 0).all() and (g[5] == 0).all() and torch.isnan(g[2]).all()
    assert (g[0, c // 2:] == 0).all() and (g[1, 4:] == 0).all()
    g64, = torch.autograd.grad((want * weight.double()).sum(), v)
    g64 = torch.where(torch.isfinite(g64), g64, torch.zeros((), dtype=g64.dtype))
    gt = _last(_grad_tol(x, g64, weight.double(), d, t), d).reshape(-1, c)
    rest[6] = True                             # p of the label is 0 there: w (1 - 0) at the label, -w p elsewhere
    p6 = torch.softmax(rows[6].double() / t, -1) / t
    expect = _last(g64, d).reshape(-1, c).clone()
    expect[6] = -weight.reshape(-1)[6].double() * p6
    expect[6, 0] += weight.reshape(-1)[6].double() / t
    rest[3] = rest[2] = False
    gt[6] = gt[6] + HALF_STEP[dtype] * expect[6].abs()
    _close(g[rest], expect[rest], gt[rest])


@pytest.mark.parametrize("layout, c", [("last", 3000), ("last", 6), ("planes", 21), ("planes", 100)])
def test_labels_that_are_no_class_give_nan(dev, layout, c):
    x, y, d, ignore = _inputs(layout, 2, (12,), c, torch.float32, seed=6)
    y[:] = 1
    y[0, 3], y[1, 0], y[1, 1], y[0, 0] = c, -7, ignore, c + (1 << 33)
    how = dict(class_dim=d, ignore_index=ignore)
    logp, stats = ops.token_logprobs(x.to(dev), y.to(dev), **how)
    bad = torch.zeros(2, 12, dtype=torch.bool)
    bad[0, 3] = bad[1, 0] = bad[0, 0] = True
    assert torch.equal(torch.isnan(logp.cpu()), bad)
    grad = ops.token_logprobs_grad(x.to(dev), y.to(dev), stats, torch.ones(2, device=dev), **how)
    nan = torch.isnan(_last(grad.cpu(), d))
    assert torch.equal(nan.all(-1), bad) and torch.equal(nan.any(-1), bad)
    total, rewards, _ = ops.preference_loss(x.to(dev), y.to(dev), torch.zeros(2, 12, device=dev), **how)
    assert torch.isnan(total) and torch.isnan(rewards).all()
    out, _, grad = ops.policy_loss(x.to(dev), y.to(dev), torch.zeros(2, 12, device=dev), torch.ones(2, device=dev),
                                   want_grad=True, **how)
    assert torch.isnan(out[0]) and torch.equal(torch.isnan(_last(grad.cpu(), d)).all(-1), bad)


def _views(dev, c):
    """Views with strides of their own, and the dense tensor each stands for."""
    g = torch.Generator().manual_seed(8)
    big = torch.randn(2, 9, c + 13, generator=g).to(dev)
    yield "next-token shift", big[:, :-1, :c], -1
    yield "odd offset", big[:, 1:, 3:c + 3], -1
    yield "every second position", big[:, ::2, :c], -1
    yield "every second class", torch.randn(2, 8, 2 * c, generator=g).to(dev)[:, :, ::2], -1
    yield "transposed", torch.randn(2, c, 7, generator=g).to(dev).transpose(1, 2), -1
    yield "sequences apart", torch.randn(4, 5, c, generator=g).to(dev)[::2], -1
    yield "one sequence for all", torch.randn(1, 6, c, generator=g).to(dev).expand(3, 6, c), -1
    yield "channel slice", torch.randn(2, c + 6, 4, 6, generator=g).to(dev)[:, 2:c + 2], 1
    yield "channels last", torch.randn(2, c, 4, 6, generator=g).to(dev).contiguous(memory_format=torch.channels_last), 1
    yield "pixels from an odd place", torch.randn(2 * c * 24 + 1, generator=g).to(dev)[1:].view(2, c, 4, 6), 1


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("c", [21, 6001])
def test_views_are_read_as_they_are(dev, dtype, c):
    for name, view, d in _views(dev, c):
        view = view.to(dtype) if dtype == view.dtype else torch.empty_strided(
            view.shape, view.stride(), dtype=dtype, device=dev).copy_(view) if 0 not in view.stride() else view[:1].to(dtype).expand(view.shape)
        shape = _last(view, d).shape[:-1]
        y = torch.randint(0, c, shape, generator=torch.Generator().manual_seed(9)).to(dev)
        y.reshape(-1)[1] = -100
        how = dict(class_dim=d, ignore_index=-100)
        logp, stats = ops.token_logprobs(view, y, **how)
        dense = view.contiguous()
        want, st = ops.token_logprobs(dense, y, **how)
        tol = _bounds(dense.cpu(), d, 1.0)[1] + 2 * U * want.cpu().double().abs()
        v64 = dense.cpu().double()
        _close(logp, ot.token_logprobs(v64, y.cpu(), **how)[0], tol, name)
        w = torch.ones(shape, device=dev)
        grad = ops.token_logprobs_grad(view, y, stats, w, **how)
        assert grad.is_contiguous()
        x64 = v64.requires_grad_(True)
        g64, = torch.autograd.grad(ot.token_logprobs(x64, y.cpu(), **how)[0].sum(), x64)
        _close(grad, g64, _grad_tol(dense.cpu(), g64, torch.ones(shape, dtype=torch.float64), d, 1.0), name)
    with pytest.raises(ValueError, match="one stride"):
        ops.token_logprobs(torch.zeros(2, 4, 6, 3, device=dev).transpose(1, 2), torch.zeros(2, 6, 4, dtype=torch.int64, device=dev),
                           class_dim=-1)


def test_views_of_labels_and_long_offsets(dev):
    """Labels as a shifted view; logits whose offsets pass 2^31 elements."""
    x = torch.randn(2, 8, 100, generator=torch.Generator().manual_seed(1)).to(dev)
    y = torch.randint(0, 100, (2, 9), generator=torch.Generator().manual_seed(2)).to(dev)
    got, _ = ops.token_logprobs(x, y[:, 1:], class_dim=-1, ignore_index=-100)
    want, _ = ops.token_logprobs(x, y[:, 1:].contiguous(), class_dim=-1, ignore_index=-100)
    assert torch.equal(got, want)
    far = torch.zeros((1 << 31) + 50000, dtype=torch.bfloat16, device=dev)
    view = far.as_strided((2, 1, 40001), ((1 << 31) + 7, 40001, 1))
    view[1].copy_(torch.randn(1, 40001, generator=torch.Generator().manual_seed(3)))
    lab = torch.tensor([[5], [40000]], device=dev)
    logp, stats = ops.token_logprobs(view, lab, class_dim=-1, ignore_index=-100)
    dense = view.cpu()
    want = ot.token_logprobs(dense.double(), lab.cpu(), class_dim=-1, ignore_index=-100)[0]
    _close(logp, want, _bounds(dense, -1, 1.0)[1] + 2 * U * want.abs())


def _ratio_tol(x, want, keep, d, t, average):
    """Bound of each sequence's log ratio: the positions' bounds added up (their mean)."""
    tol = _bounds(x, d, t)[1] + 3 * U * want.abs()
    n = x.shape[0]
    tol = torch.where(keep, tol, torch.zeros((), dtype=tol.dtype)).reshape(n, -1).sum(1)
    return tol / keep.reshape(n, -1).sum(1).clamp(min=1) if average else tol


PAIRS = [("last", 2, (1,), 11, torch.float32), ("last", 4, (37,), 1031, torch.bfloat16), ("last", 2, (9,), 50001, torch.float16),
         ("last", 6, (5000,), 7, torch.float32), ("last", 2, (), 300, torch.float32), ("planes", 4, (24, 20), 21, torch.float32),
         ("planes", 2, (70, 70), 5, torch.float16), ("planes", 64, (3,), 19, torch.bfloat16), ("planes", 2, (30, 22), 150, torch.float32),
         ("planes", 4, (700,), 300, torch.float16), ("last", 2, (3000,), 90, torch.float32)]


@pytest.mark.parametrize("shape", PAIRS, ids=lambda s: "%s-%d-%s-%d" % (s[0], s[1], "x".join(map(str, s[2])), s[3]))
@pytest.mark.parametrize("loss_type, smoothing, average", [("sigmoid", 0.0, False), ("sigmoid", 0.1, True), ("ipo", 0.0, True)])
def test_preference_loss(dev, shape, loss_type, smoothing, average):
    x, y, d, ignore = _inputs(*shape, seed=11)
    y[-1] = ignore     # the last sequence holds nothing
    beta, t, scale = 0.3, 1.0, 8.0
    how = dict(class_dim=d, ignore_index=ignore, temperature=t)
    lp, keep = ot.token_logprobs(x.double(), y, **how)
    g = torch.Generator().manual_seed(12)
    ref = (lp + 0.3 * torch.randn(y.shape, generator=g, dtype=torch.float64)).float()
    ref = torch.where(keep, ref, math.nan)    # not read there
    v = x.double().requires_grad_(True)
    total, rewards = ot.preference(v, y, ref.nan_to_num(0.0), beta=beta, label_smoothing=smoothing, loss_type=loss_type,
                                   average=average, **how)
    g64, = torch.autograd.grad(scale * total, v)
    opts = dict(beta=beta, label_smoothing=smoothing, loss_type=loss_type, average=average, **how)
    got, rew, grad = ops.preference_loss(x.to(dev), y.to(dev), ref.to(dev), want_grad=True, grad_scale=scale, **opts)
    tr = _ratio_tol(x, lp, keep, d, t, average)
    _close(rew, rewards.detach(), beta * tr + 2 * U * rewards.detach().abs(), "rewards")
    n = x.shape[0]
    th = tr[: n // 2] + tr[n // 2:]
    r = (rewards.detach() / beta)
    h = r[: n // 2] - r[n // 2:]
    steep = (2 * (h - 1 / (2 * beta)).abs() + th) if loss_type == "ipo" else torch.full_like(h, beta)
    _close(got, total.detach(), (steep * th).mean() + 2 * U * total.detach().abs(), "total")
    # d total / d logp of a sequence and its error
    counts = keep.reshape(n, -1).sum(1).clamp(min=1).double() if average else torch.ones(n, dtype=torch.float64)
    dh = (2 * (h - 1 / (2 * beta)) if loss_type == "ipo" else
          -beta * ((1 - smoothing) * torch.sigmoid(-beta * h) - smoothing * torch.sigmoid(beta * h)))
    ddh = (2 * th if loss_type == "ipo" else beta * beta / 4 * th) + 4 * U * dh.abs()
    w = torch.cat([dh, dh]).abs() / (n // 2) / counts * scale
    dw = torch.cat([ddh, ddh]) / (n // 2) / counts * scale
    wide = lambda s: s.view(-1, *([1] * (y.dim() - 1))).expand(y.shape)  # noqa: E731
    extra = (wide(dw) / t).unsqueeze(d if d == 1 else -1)
    _close(grad, g64, _grad_tol(x, g64, wide(w), d, t) + extra, "grad")
    again = ops.preference_loss(x.to(dev), y.to(dev), ref.to(dev), want_grad=True, grad_scale=scale, **opts)
    assert torch.equal(again[0], got) and torch.equal(again[1], rew) and torch.equal(again[2], grad)
    # the module: same values; an upstream factor reaches the gradient
    loss = PreferenceLoss(beta=beta, label_smoothing=smoothing, loss_type=loss_type, average=average, **how)
    leaf = x.to(dev).requires_grad_(True)
    res = loss(leaf, y.to(dev), ref.to(dev))
    assert torch.equal(res["total"].detach(), got) and torch.equal(res["rewards"], rew) and not res["rewards"].requires_grad
    (scale * res["total"]).backward()
    assert torch.equal(leaf.grad, grad)
    with torch.no_grad():
        assert torch.equal(loss(leaf, y.to(dev), ref.to(dev))["total"], got)


def test_preference_sides_and_extremes(dev):
    """The preferred half is the first; log ratios of thousands saturate without overflow."""
    x = torch.zeros(2, 4, 3, device=dev)
    y = torch.zeros(2, 4, dtype=torch.int64, device=dev)
    base = ops.token_logprobs(x, y, class_dim=-1)[0]
    up = base.clone()
    up[0] -= 1e4      # the reference finds the preferred answer far less likely: the policy moved the right way
    total, rewards, grad = ops.preference_loss(x, y, up, beta=1.0, class_dim=-1, want_grad=True)
    # the second answer's ratio: four log-probabilities in fp64 less their fp32 roundings, each within half a step (2^-24
    # between 1 and 2) of log(1/3) = -1.0986
    assert total == 0 and rewards[0] == 4e4 and abs(rewards[1].item()) <= 4 * U and (grad == 0).all()
    up[0] += 2e4
    total, _, grad = ops.preference_loss(x, y, up, beta=1.0, class_dim=-1, want_grad=True)
    assert abs(total.item() - 4e4) <= 4e4 * 2.0 ** -23 * 4
    # factor -1 on every position of the first sequence: the gradient lifts the label, 1 - 1/3, and lowers the rest
    want = torch.tensor([-2 / 3, 1 / 3, 1 / 3], device=dev).expand(4, 3)
    assert ((grad[0] - want).abs() <= 8 * U).all() and ((grad[1] + want).abs() <= 8 * U).all()


ROWS = [("last", 1, (1,), 9, torch.float32), ("last", 3, (41,), 1025, torch.bfloat16), ("last", 2, (7,), 50001, torch.float16),
        ("last", 2, (3,), 140001, torch.bfloat16), ("last", 5, (4500,), 6, torch.float32), ("last", 4, (), 700, torch.float32),
        ("planes", 3, (24, 20), 21, torch.float32), ("planes", 2, (70, 70), 5, torch.float16), ("planes", 40, (3,), 19, torch.bfloat16),
        ("planes", 1, (30, 5), 100, torch.float32), ("planes", 2, (30, 22), 150, torch.float32), ("planes", 4, (700,), 300, torch.float16),
        ("last", 3, (20,), 21, torch.float32), ("last", 3, (20,), 100, torch.bfloat16), ("last", 2, (600,), 300, torch.float32),
        ("planes", 3, (5, 7), 1000, torch.float32)]


@pytest.mark.parametrize("shape", ROWS, ids=lambda s: "%s-%d-%s-%d" % (s[0], s[1], "x".join(map(str, s[2])), s[3]))
@pytest.mark.parametrize("reduction, kl, t, each", [("token", 0.0, 1.0, False), ("sequence", 0.2, 0.7, True)])
def test_policy_loss(dev, shape, reduction, kl, t, each):
    x, y, d, ignore = _inputs(*shape, seed=21)
    if x.shape[0] > 2:
        y[1] = ignore
    how = dict(class_dim=d, ignore_index=ignore, temperature=t)
    lp, keep = ot.token_logprobs(x.double(), y, **how)
    g = torch.Generator().manual_seed(22)
    moved = 0.3 * torch.randn(y.shape, generator=g, dtype=torch.float64)
    for border in (math.log(0.8), math.log(1.3)):    # at the border either branch is right
        moved = torch.where((moved - border).abs() < 1e-2, moved + 3e-2, moved)
    old = torch.where(keep, (lp - moved).float(), math.nan)
    ref = torch.where(keep, (lp + 0.3 * torch.randn(y.shape, generator=g, dtype=torch.float64)).float(), math.nan)
    adv = torch.randn(y.shape if each else (x.shape[0],), generator=g)
    wide = adv.double() if each else adv.double().view(-1, *([1] * (y.dim() - 1))).expand(y.shape)
    scale, opts = 4.0, dict(clip_low=0.2, clip_high=0.3, kl_weight=kl, reduction=reduction, **how)
    v = x.double().requires_grad_(True)
    want = ot.policy(v, y, old.nan_to_num(0.0), wide.float(), ref=ref.nan_to_num(0.0) if kl else None, **opts)
    g64, = torch.autograd.grad(scale * want[0], v)
    args = (x.to(dev), y.to(dev), old.to(dev), adv.to(dev))
    refd = ref.to(dev) if kl else None
    out, logp, grad = ops.policy_loss(*args, ref_logprobs=refd, want_grad=True, grad_scale=scale, **opts)
    tl = _bounds(x, d, t)[1] + 2 * U * lp.abs()
    _close(logp, lp, tl, "logp")
    n = x.shape[0]
    # a ratio is off by the error of its logarithm and the exponential's 3 u; a mean averages the bounds
    ratio = torch.exp(torch.where(keep, moved, 0.0)) + 1e-3
    t_r = wide.abs() * ratio * (tl + U * (4 + moved.abs()))
    q = torch.where(keep, (ref.double() - lp), 0.0)
    t_k = (torch.exp(q) + 1) * (tl + U * (6 + q.abs())) + 4 * U
    zero = torch.zeros((), dtype=torch.float64)
    share = keep.sum().clamp(min=1).double().reciprocal().expand(y.shape) if reduction == "token" else (
        1.0 / (keep.reshape(n, -1).sum(1).clamp(min=1).double() * n)).view(-1, *([1] * (y.dim() - 1))).expand(y.shape)
    mean = lambda e: (torch.where(keep, e, zero) * share).sum()  # noqa: E731
    for k, tol in ((0, mean(t_r) + kl * mean(t_k)), (1, mean(t_r)), (2, mean(t_k) if kl else zero), (3, zero)):
        _close(out[k], want[k].detach(), tol + 4 * U * (want[k].detach().abs() + mean(wide.abs())), "out%d" % k)
    w = (wide.abs() * ratio + (kl * (1 + torch.exp(q)) if kl else 0)) * share * scale
    dw = (t_r + kl * t_k + 4 * U * w / share / scale) * share * scale
    _close(grad, g64, _grad_tol(x, g64, torch.where(keep, w, zero), d, t)
           + (torch.where(keep, dw, zero) / t).unsqueeze(d if d == 1 else -1), "grad")
    plain = ops.policy_loss(*args, ref_logprobs=refd, **opts)
    if shape[0] != "channels last":     # (there the pass with a gradient, whose order is another one, is another kernel)
        assert torch.equal(plain[0], out) and torch.equal(plain[1], logp)
    _close(plain[1], lp, tl, "logp without a gradient")
    assert plain[2] is None
    # the module: the same gradient for an upstream factor of 1 and of `scale`, and from a second backward
    loss = ClippedPolicyLoss(clip_low=0.2, clip_high=0.3, kl_weight=kl, reduction=reduction, **how)
    leaf = x.to(dev).requires_grad_(True)
    res = loss(leaf, *args[1:], ref_logprobs=refd)
    for k, key in enumerate(("total", "surrogate", "kl", "clipped")):
        assert torch.equal(res[key].detach(), out[k]) and res[key].requires_grad == (k == 0)
    (scale * res["total"]).backward(retain_graph=True)
    assert torch.equal(leaf.grad, grad) or (leaf.grad.double() - grad.double()).abs().max() <= 2 * _grad_tol(
        x, g64, torch.where(keep, w, zero), d, t).max()
    leaf.grad = None
    res["total"].backward()
    one = ops.policy_loss(*args, ref_logprobs=refd, want_grad=True, **opts)[2]
    _close(leaf.grad, one.cpu(), 2 * _grad_tol(x, g64 / scale, torch.where(keep, w, zero) / scale, d, t), "second backward")


def test_policy_branches_by_hand(dev):
    """Advantage and ratio on each side of each bound: (ratio, A) -> the gradient of -min(r A, clip(r) A) by logp."""
    x = torch.zeros(1, 6, 2, device=dev)
    y = torch.zeros(1, 6, dtype=torch.int64, device=dev)
    lp = math.log(0.5)
    r = torch.tensor([[0.5, 0.5, 1.0, 1.0, 2.0, 2.0]])
    a = torch.tensor([[1.0, -1.0, 1.0, -1.0, 1.0, -1.0]])
    old = (lp - torch.log(r.double())).float()
    out, _, grad = ops.policy_loss(x, y, old.to(dev), a.to(dev), class_dim=-1, want_grad=True)
    dl = torch.tensor([-0.5, 0.0, -1.0, 1.0, 0.0, 2.0])     # clipped: r < 0.8 with A < 0, r > 1.2 with A > 0
    want = torch.stack([dl, -dl], -1) * 0.5 / 6
    assert (grad[0].cpu() - want).abs().max() <= 16 * U
    loss = torch.tensor([-0.5, 0.8, -1.0, 1.0, -1.2, 2.0]).mean()
    assert abs(out[0].item() - loss.item()) <= 16 * U and abs(out[3].item() - 2 / 6) <= 2 * U


def test_nothing_counted_and_no_positions(dev):
    for d, shape in ((-1, (2, 3, 40)), (1, (2, 4, 6)), (-1, (2, 3, 5000))):
        x = torch.randn(shape, device=dev)
        y = torch.full(_last(x, d).shape[:-1], 255 if x.shape[d] < 255 else -1, device=dev)
        how = dict(class_dim=d, ignore_index=int(y.flatten()[0]))
        f = torch.full(y.shape, math.nan, device=dev)
        for reduction in ("token", "sequence"):
            out, logp, grad = ops.policy_loss(x, y, f, torch.ones(2, device=dev), ref_logprobs=f, kl_weight=0.1,
                                              reduction=reduction, want_grad=True, **how)
            assert (out == 0).all() and (logp == 0).all() and (grad == 0).all()
        total, rewards, grad = ops.preference_loss(x, y, f, want_grad=True, average=True, **how)
        assert abs(total.item() - math.log(2)) <= 2 * U and (rewards == 0).all() and (grad == 0).all()
    out, logp, grad = ops.policy_loss(torch.zeros(0, 3, 9, device=dev), torch.zeros(0, 3, dtype=torch.int64, device=dev),
                                      torch.zeros(0, 3, device=dev), torch.ones(0, device=dev), class_dim=-1, want_grad=True)
    assert (out == 0).all() and logp.shape == (0, 3) and grad.shape == (0, 3, 9)
    x, y, f = torch.zeros(2, 0, 9, device=dev), torch.zeros(2, 0, dtype=torch.int64, device=dev), torch.zeros(2, 0, device=dev)
    assert ops.token_logprobs(x, y, class_dim=-1)[0].shape == (2, 0)
    out, _, grad = ops.policy_loss(x, y, f, torch.ones(2, device=dev), class_dim=-1, want_grad=True)
    assert (out == 0).all() and grad.shape == x.shape
    total, _, grad = ops.preference_loss(x, y, f, class_dim=-1, want_grad=True)
    assert abs(total.item() - math.log(2)) <= 2 * U and grad.shape == x.shape


def test_gradient_against_differences(dev):
    """Central differences of the losses themselves in fp32: a step of 1/16 changes a loss of order 1 by about 1/16; its
    rounding, 2^-22 at most, counts 8 times, the third derivative (order 1) times step^2 / 6 < 1e-3 the rest."""
    x = torch.randn(2, 3, 4, generator=torch.Generator().manual_seed(1)).to(dev)
    y = torch.tensor([[0, 2, 1, 255], [1, 255, 0, 2]], device=dev)
    ref = torch.full((2, 4), -1.0, device=dev)
    old = ops.token_logprobs(x, y)[0] - 0.05
    adv = torch.tensor([1.0, -0.5], device=dev)
    for f in (lambda v, **k: ops.preference_loss(v, y, ref, beta=0.5, **k),
              lambda v, **k: ops.policy_loss(v, y, old, adv, ref_logprobs=ref, kl_weight=0.3, clip_low=0.9, clip_high=9.0, **k)):
        grad = f(x, want_grad=True)[2]
        for i in range(x.numel()):
            step = torch.zeros_like(x)
            step.view(-1)[i] = 1 / 16
            up, down = (f(x + s * step)[0].reshape(-1)[0].item() for s in (1, -1))
            assert abs((up - down) * 8 - grad.view(-1)[i].item()) <= 1e-3 + 16 * 2.0 ** -22


def test_differentiable_logprobs_and_their_views(dev):
    """pruning.losses.token_logprobs: the label term of a cross-entropy, by autograd; views that ops refuses are copied."""
    x = torch.randn(2, 6, 5, 30, generator=torch.Generator().manual_seed(4)).to(dev).transpose(1, 2).requires_grad_(True)
    y = torch.randint(0, 30, (2, 5, 6), generator=torch.Generator().manual_seed(5)).to(dev)
    logp = token_logprobs(x, y.int(), class_dim=-1)
    assert logp.requires_grad
    v = x.detach().cpu().double().requires_grad_(True)
    want = -ot.token_logprobs(v, y.cpu(), class_dim=-1)[0].mean()
    g64, = torch.autograd.grad(want, v)
    _close(torch.autograd.grad(-token_logprobs(x, y, class_dim=-1).mean(), x)[0], g64,
           _grad_tol(v.detach().float(), g64, torch.full(y.shape, 1 / 60, dtype=torch.float64), -1, 1.0))
    with torch.no_grad():
        assert not token_logprobs(x, y, class_dim=-1).requires_grad


def test_another_stream_and_a_captured_run(dev):
    """The calls on a stream of their own, two calls with tensors of their own on two streams at once, and captured into a
    graph: every replay, eager work between them, repeats the eager results."""
    sets = []
    for seed in (31, 32):
        x, y, d, ignore = _inputs("last", 4, (50,), 5000, torch.bfloat16, seed=seed)
        x, y = x.to(dev), y.to(dev)
        old = ops.token_logprobs(x, y, class_dim=-1, ignore_index=ignore)[0] - 0.03
        sets.append((x, y, old, torch.randn(4, device=dev)))

    def both(x, y, old, adv):
        a = ops.policy_loss(x, y, old, adv, ref_logprobs=old, kl_weight=0.1, class_dim=-1, ignore_index=-100, want_grad=True)
        b = ops.preference_loss(x, y, old, class_dim=-1, ignore_index=-100, want_grad=True)
        return (*a, *b)

    eager = [both(*s) for s in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = []
    for s, args in zip(streams, sets):
        with torch.cuda.stream(s):
            got.append(both(*args))
    torch.cuda.synchronize()
    for g, e in zip(got, eager):
        assert all(torch.equal(a, b) for a, b in zip(g, e))
    side = torch.cuda.Stream()
    graphs = []
    for args in sets:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = both(*args)
        graphs.append((graph, out))
    for turn in range(3):
        for args, (graph, out) in zip(sets, graphs):
            args[0].mul_(0.9)
            graph.replay()
            torch.cuda.synchronize()
            kept = [o.clone() for o in out]
            assert all(torch.equal(a, b) for a, b in zip(kept, both(*args))), turn


def test_refusals_on_the_device(dev):
    x, y, f = torch.zeros(2, 3, 9, device=dev), torch.zeros(2, 3, dtype=torch.int64, device=dev), torch.zeros(2, 3, device=dev)
    how = dict(class_dim=-1)
    for call, kind, text in [
        (lambda: ops.token_logprobs(x.double(), y, **how), TypeError, "dtype"),
        (lambda: ops.token_logprobs(x, y.int(), **how), TypeError, "labels"),
        (lambda: ops.token_logprobs(x, y.cpu(), **how), RuntimeError, "labels"),
        (lambda: ops.token_logprobs(x, y[:, :2], **how), ValueError, "shape"),
        (lambda: ops.token_logprobs(x, y, class_dim=0), ValueError, "class_dim"),
        (lambda: ops.token_logprobs(x, y, class_dim=1), ValueError, "shape"),
        (lambda: ops.token_logprobs(x, y, ignore_index=3, **how), ValueError, "ignore_index"),
        (lambda: ops.token_logprobs(x, y, temperature=0.0, **how), ValueError, "temperature"),
        (lambda: ops.token_logprobs(x, y, temperature=math.nan, **how), ValueError, "temperature"),
        (lambda: ops.token_logprobs(x[..., :0], y, **how), ValueError, "no classes"),
        (lambda: ops.token_logprobs(x[0, 0], y[0, 0], **how), ValueError, "axis"),
        (lambda: ops.token_logprobs_grad(x, y, torch.zeros(5, device=dev), f, **how), ValueError, "stats"),
        (lambda: ops.token_logprobs_grad(x, y, torch.zeros(2, 3, 2, device=dev), f[:, :1], **how), ValueError, "weight|contiguous"),
        (lambda: ops.token_logprobs_grad(x, y, torch.zeros(2, 3, 2, device=dev), f, out=x, **how), ValueError, "device_scale"),
        (lambda: ops.preference_loss(x[:1], y[:1], f[:1], **how), ValueError, "half"),
        (lambda: ops.preference_loss(x, y, f[:1], **how), ValueError, "ref_logprobs"),
        (lambda: ops.preference_loss(x, y, f.half(), **how), TypeError, "ref_logprobs"),
        (lambda: ops.preference_loss(x, y, f, beta=0.0, **how), ValueError, "beta"),
        (lambda: ops.preference_loss(x, y, f, label_smoothing=0.5, **how), ValueError, "label_smoothing"),
        (lambda: ops.preference_loss(x, y, f, label_smoothing=0.1, loss_type="ipo", **how), ValueError, "ipo"),
        (lambda: ops.policy_loss(x, y, f, f[:1], **how), ValueError, "advantages"),
        (lambda: ops.policy_loss(x, y, f, f, clip_low=1.5, **how), ValueError, "clip_low"),
        (lambda: ops.policy_loss(x, y, f, f, kl_weight=0.1, **how), ValueError, "ref_logprobs"),
    ]:
        with pytest.raises(kind, match=text):
            call()


# both sides of the row width where each form of the row kernels ends (full 16-byte vectors of 4, 16, 64, 256 lanes ...),
# in sequences short enough that a wave's rows belong to several of them
WIDTHS = [31, 32, 33, 63, 64, 127, 128, 143, 144, 287, 288, 447, 448, 895, 896, 1279, 1280, 2303, 2304, 2559, 2560, 4607, 4608,
          9215, 9216, 18431, 18432, 36863, 36864]


@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_the_ends_of_their_forms(dev, c, dtype):
    shape = ("last", 5, (7,), c, dtype) if c < 2000 else ("last", 2, (3,), c, dtype)
    test_token_logprobs_and_gradient(dev, shape, 0.7)
    test_policy_loss(dev, shape, "sequence", 0.2, 0.7, True)
    test_policy_loss(dev, shape, "token", 0.0, 1.0, False)


# logits whose classes lie next to each other and whose gradient's positions do: one position a lane, or a workgroup
@pytest.mark.parametrize("n, positions, c", [(2, (20, 30), 21), (2, (1, 7), 21), (4, (9,), 6), (2, (17, 31), 40), (2, (300,), 300),
                                             (2, (8, 16), 150), (2, (301,), 1000)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_channels_last_logits(dev, n, positions, c, dtype):
    shape = ("channels last", n, positions, c, dtype)
    x = _inputs(*shape)[0]
    assert x.to(dev).stride() == x.stride() and not x.to(dev).is_contiguous()
    test_token_logprobs_and_gradient(dev, shape, 0.7)
    test_preference_loss(dev, shape, "sigmoid", 0.1, True)
    test_policy_loss(dev, shape, "token", 0.0, 1.0, False)
    test_policy_loss(dev, shape, "sequence", 0.2, 0.7, True)


@pytest.mark.parametrize("c", [5, 21, 40, 300])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_every_second_position_of_many(dev, c, dtype):
    """Planes whose positions lie two apart: the same bounds as the dense tensor's."""
    wide = (2.0 * torch.randn(2, c, 403, 2, generator=torch.Generator().manual_seed(31))).to(dtype)
    y = torch.randint(0, c, (2, 403), generator=torch.Generator().manual_seed(32))
    y[1, ::5] = -100
    how = dict(class_dim=1, ignore_index=-100)
    x, view = wide[..., 0].contiguous(), wide.to(dev)[..., 0]
    assert view.stride(2) == 2
    v = x.double().requires_grad_(True)
    want, _ = ot.token_logprobs(v, y, **how)
    g64, = torch.autograd.grad(want.sum(), v)
    logp, stats = ops.token_logprobs(view, y.to(dev), **how)
    _close(logp, want.detach(), _bounds(x, 1, 1.0)[1] + 2 * U * want.detach().abs(), "logp")
    grad = ops.token_logprobs_grad(view, y.to(dev), stats, torch.ones(2, device=dev), **how)
    _close(grad, g64, _grad_tol(x, g64, torch.ones(y.shape, dtype=torch.float64), 1, 1.0), "grad")
    # the policy loss at its own sample: ratio 1, so total = -mean A and the gradient -A logp's share of the mean
    adv = torch.tensor([0.5, -2.0], device=dev)
    out, again, pg = ops.policy_loss(view, y.to(dev), logp, adv, want_grad=True, **how)
    # (the ratio of two passes' logp is off by their difference, which both bounds hold)
    tl = _bounds(x, 1, 1.0)[1] + 2 * U * want.detach().abs()
    _close(again, want.detach(), tl, "policy logp")
    keep = (y != -100).double()
    a64 = adv.cpu().double()[:, None] * keep / keep.sum()
    _close(out[0], -a64.sum(), (a64.abs() * (2 * tl + 4 * U)).sum() + 4 * U, "total")
    p64, = torch.autograd.grad(-(ot.token_logprobs(v, y, **how)[0] * a64).sum(), v)
    _close(pg, p64, _grad_tol(x, p64, a64.abs() * (1 + 2 * tl + 4 * U), 1, 1.0) + (a64.abs() * (2 * tl + 4 * U)).unsqueeze(1), "policy grad")


@pytest.mark.parametrize("layout, positions, c", [("last", (6,), 5000), ("last", (40,), 9), ("last", (5,), 700), ("last", (4,), 90001),
                                                  ("planes", (8, 12), 21), ("planes", (5, 7), 70), ("planes", (6,), 3001)])
@pytest.mark.parametrize("factor", [math.inf, math.nan])
def test_ignored_positions_stay_zero_under_any_factor(dev, layout, positions, c, factor):
    """An infinite or NaN factor from above (a loss scale that ran over) reaches the counted positions alone, in every kernel."""
    x, y, d, ignore = _inputs(layout, 2, positions, c, torch.float32, seed=41)
    y.reshape(-1)[:3] = torch.tensor([ignore, 1, ignore])
    keep = y != ignore
    how = dict(class_dim=d, ignore_index=ignore)
    xd, yd = x.to(dev), y.to(dev)
    _, stats = ops.token_logprobs(xd, yd, **how)
    old, adv = torch.zeros(y.shape, device=dev), torch.ones(2, device=dev)
    far = torch.full((1,), factor, device=dev)
    leaf = xd.clone().requires_grad_(True)
    total = ClippedPolicyLoss(kl_weight=0.1, **how)(leaf, yd, old, adv, ref_logprobs=old)["total"]
    grads = [ops.token_logprobs_grad(xd, yd, stats, torch.ones(y.shape, device=dev), device_scale=far, **how),
             ops.token_logprobs_grad(xd, yd, stats, adv, scale=factor, **how),
             ops.policy_loss(xd, yd, old, adv, ref_logprobs=old, kl_weight=0.1, want_grad=True, grad_scale=factor, **how)[2],
             ops.preference_loss(xd, yd, old, want_grad=True, grad_scale=factor, **how)[2],
             torch.autograd.grad(far[0] * total, leaf)[0]]
    for k, g in enumerate(grads):
        g = _last(g, d).cpu()
        assert (g[~keep] == 0).all(), k
        assert not torch.isfinite(g[keep]).all(-1).any(), k


def _long_tail(layout, n, positions, c, t=17.0):
    """One class at 0 and the others at -t in every position, and what the label's log-probability and a tail class's softmax are:
    every tail class is below half a step of a sum that has reached 1."""
    x = torch.full((n, *positions, c), -t)
    top = torch.randint(0, c, (n, *positions), generator=torch.Generator().manual_seed(c))
    x.scatter_(-1, top.unsqueeze(-1), 0.0)
    tail = math.exp(-t)
    return (x.movedim(-1, 1).contiguous() if layout == "planes" else x), top, -math.log1p((c - 1) * tail), tail / (1 + (c - 1) * tail)


# A tail class's exponential: exponent t log2(e) rounds by u of 24.5 (17 u of the value), the instruction 2 u: 20 u; trees of
# them, a rescaling and the joins 7 u: the tail's sum T, and with it log(1 + T), is off by at most 27 u of itself, and rounds
# to fp32 by u.  The tree of at most 16 exponentials that holds the 1 rounds four times at values below 2: 4 u.  What a chain of
# fp32 additions holds back shows as hundreds of u.
TAIL, TREE = 32, 4


def _check_long_tail(dev, x, y, d, logp, p):
    """x on the host, or a view on the device."""
    x = x.to(dev)
    how = dict(class_dim=d, ignore_index=-100)
    got, stats = ops.token_logprobs(x, y.to(dev), **how)
    assert (got.double() - logp).abs().max().item() <= TAIL * U * abs(logp) + TREE * U
    out, again, _ = ops.policy_loss(x, y.to(dev), torch.full(y.shape, logp, device=dev), torch.ones(x.shape[0], device=dev), **how)
    assert (again.double() - logp).abs().max().item() <= TAIL * U * abs(logp) + TREE * U
    # the statistics' sum: the tree's error, that of the tail (less than u) and its rounding; a class's softmax by its exponential's
    # 20 u, the sum's, the quotient's and the product's
    s = stats[..., 1].double() * torch.exp(stats[..., 0].double())
    assert (s * math.exp(logp) - 1).abs().max().item() <= (TREE + 2) * U
    grad = _last(ops.token_logprobs_grad(x, y.to(dev), stats, torch.ones(y.shape, device=dev), **how), d)
    want = torch.full((x.shape[0] * y[0].numel(), grad.shape[-1]), -p, device=dev, dtype=torch.float64)
    want.scatter_(-1, y.to(dev).reshape(-1, 1), -math.expm1(logp))
    # (at the label 1 - p is taken in fp32: the sum's error and 2 u of 1)
    assert ((grad.double().reshape(want.shape) - want).abs() <= (TAIL + TREE) * U * p + (want > 0) * (TREE + 4) * U).all()


@pytest.mark.parametrize("c, l, step", [(32000, 520, 1), (32001, 260, 2), (5000, 600, 1), (5000, 600, 2), (150, 600, 1), (250, 600, 1),
                                        (60, 600, 2), (40, 600, 2)])
def test_planes_of_many_classes_keep_a_long_tail(dev, c, l, step):
    """More positions than a workgroup each would take, neighbouring ones and every second one."""
    n = 1 if l > 512 else 2
    x, y, logp, p = _long_tail("planes", n, (l,), c)
    x = x.to(dev)
    if step > 1:
        x = torch.stack([x, torch.zeros_like(x)], -1)[..., 0]
    _check_long_tail(dev, x, y, 1, logp, p)


@pytest.mark.parametrize("layout, positions, c", [("last", (4000,), 9), ("last", (500,), 1000), ("last", (3,), 90001), ("planes", (80, 90), 21),
                                                  ("planes", (40, 50), 150), ("planes", (5,), 3001)])
@pytest.mark.parametrize("apart", [1e-5, 1e-4, 1e-2, 0.5, 3.0])
def test_kl_of_a_policy_near_its_reference(dev, layout, positions, c, apart):
    """exp(q) - q - 1 is about q^2 / 2: a policy that has hardly left its reference.  Against the formula in 64 bits at the
    log-probabilities that the call gives back: q = ref - logp rounds by u of itself, which the derivative exp(q) - 1 carries;
    the value itself by at most 14 u (ten steps of a series whose terms shrink, or the exponential's 3 u and two differences);
    exp(q) - 1 by u q exp(q) and 10 u."""
    x, y, d, ignore = _inputs(layout, 2, positions, c, torch.float32, seed=51)
    how = dict(class_dim=d, ignore_index=ignore)
    keep = y != ignore
    xd, yd = x.to(dev), y.to(dev)
    logp = ops.token_logprobs(xd, yd, **how)[0].cpu()
    ref = (logp.double() + apart * torch.randn(y.shape, generator=torch.Generator().manual_seed(52), dtype=torch.float64)).float()
    out, again, grad = ops.policy_loss(xd, yd, logp.to(dev), torch.zeros(2, device=dev), ref_logprobs=ref.to(dev), kl_weight=0.5,
                                       want_grad=True, grad_scale=float(keep.sum()), **how)
    q = torch.where(keep, ref.double() - again.cpu().double(), 0.0)
    far = torch.expm1(q) - q
    rough = 2.0 ** -52 * q.abs()         # (of this line's own subtraction)
    want = far.sum() / keep.sum()
    assert out[2] >= 0 and abs(out[2].item() - want.item()) <= ((14 * U * far + U * (q * torch.expm1(q)).abs() + rough).sum() / keep.sum()).item() + U * want.item()
    w = -0.5 * torch.expm1(q)
    v = x.double().requires_grad_(True)
    g64, = torch.autograd.grad((ot.token_logprobs(v, y, **how)[0] * w).sum(), v)
    # the weight: 0.5 (1 - exp(q)) and the share's product and rounding
    extra = (w.abs() * 10 * U + 0.5 * U * q.abs() * torch.exp(q)).unsqueeze(d if d == 1 else -1)
    _close(grad, g64, _grad_tol(x, g64, w.abs(), d, 1.0) + extra, "grad")


def test_an_out_that_shares_memory_is_refused(dev):
    """Before anything is launched; a separate one's version tells autograd of the write."""
    x = torch.randn(2, 3, 40, generator=torch.Generator().manual_seed(1)).to(dev)
    y = torch.zeros(2, 3, dtype=torch.int64, device=dev)
    how = dict(class_dim=-1, ignore_index=-100)
    _, stats = ops.token_logprobs(x, y, **how)
    w, half = torch.ones(2, 3, device=dev), torch.full((1,), 0.5, device=dev)
    buf = torch.zeros(1000, device=dev)

    def grad(out, x=x, y=y, stats=stats, w=w, scale=half):
        return ops.token_logprobs_grad(x, y, stats, w, device_scale=scale, out=out, **how)

    want = ops.token_logprobs_grad(x, y, stats, w, scale=0.5, **how)
    here, wide = buf[100:340].view(2, 3, 40), torch.zeros(2, 4, 40, device=dev)
    for call in (lambda: grad(x), lambda: grad(here, stats=buf[330:342].view(2, 3, 2)), lambda: grad(here, w=buf[95:101].view(2, 3)),
                 lambda: grad(here, scale=buf[339:340]), lambda: grad(wide.view(-1)[:240].view(2, 3, 40), x=wide[:, 1:]),
                 lambda: grad(here, y=buf[90:102].view(torch.int64).view(2, 3))):
        with pytest.raises(ValueError, match="share memory"):
            call()
    assert (buf == 0).all() and (wide == 0).all()
    version = buf._version
    assert torch.equal(grad(here, stats=buf[340:352].view(2, 3, 2).copy_(stats)), want) and buf._version > version + 1


@pytest.mark.parametrize("layout, n, positions, c", [
    ("planes", 2, (300,), 2), ("planes", 2, (300,), 8), ("planes", 2, (300,), 21), ("planes", 2, (301,), 32), ("planes", 1, (3,), 19)])
def test_planes_of_few_classes_keep_a_tail(dev, layout, n, positions, c):
    x, y, logp, p = _long_tail(layout, n, positions, c)
    _check_long_tail(dev, x, y, 1, logp, p)
    if len(positions) == 1:      # one position a lane
        wide = x.to(dev)
        _check_long_tail(dev, torch.stack([wide, torch.zeros_like(wide)], -1)[..., 0], y, 1, logp, p)


@pytest.mark.parametrize("layout, n, positions, c", [
    ("last", 2, (9,), 7), ("last", 2, (40,), 31), ("last", 2, (40,), 150), ("last", 2, (20,), 255), ("last", 2, (20,), 447),
    ("last", 2, (20,), 895), ("last", 2, (9,), 2000), ("last", 2, (9,), 8000), ("last", 2, (3,), 32000), ("last", 2, (3,), 50001),
    ("last", 1, (2,), 131072), ("last", 1, (2,), 200003), ("planes", 2, (5,), 3001), ("planes", 2, (3,), 100001)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_keep_a_long_tail(dev, layout, n, positions, c, dtype):
    x, y, logp, p = _long_tail(layout, n, positions, c)
    d = -1 if layout == "last" else 1
    if dtype == torch.float32:
        _check_long_tail(dev, x, y, d, logp, p)
    else:
        got = ops.token_logprobs(x.to(dtype).to(dev), y.to(dev), class_dim=d, ignore_index=-100)[0]
        assert (got.double() - logp).abs().max().item() <= TAIL * U * abs(logp) + TREE * U


@pytest.mark.parametrize("layout, positions, c", [("last", (1000,), 2), ("last", (1000,), 300), ("last", (100,), 5000), ("last", (100,), 90000),
                                                  ("planes", (1000,), 2), ("planes", (1000,), 40), ("planes", (200,), 300)])
@pytest.mark.parametrize("t", [1.0, 0.7])
def test_log_ratios_of_many_positions_that_round_alike(dev, layout, positions, c, t):
    """Every position's label lies 8 - 0.4 steps below the maximum, which a subtraction in fp32 rounds to 8, and all the same way:
    a sequence's log ratio adds that up.  Nor may T = 0.7 be its neighbour in fp32.  Two classes count (the rest are -inf): the
    other one's exp(-8 / T) is off by 24 u at most (its distance, the product of up to 16.5, the instruction), its addition to
    the maximum's 1 rounds by half a step at 1, which is u (all further ones add zeros), and a position's log ratio, where it
    is kept in fp32, by u."""
    n, low32 = 2, torch.tensor(0.4 * 2.0 ** -21)
    x = torch.full((n, *positions, c), -math.inf)
    x[..., 0], x[..., c - 1] = 8.0, low32
    y = torch.full((n, *positions), c - 1)
    y[1, ::3] = 0
    if layout == "planes":
        x = x.movedim(-1, 1).contiguous()
    d = -1 if layout == "last" else 1
    how = dict(class_dim=d, ignore_index=-100, temperature=t)
    z = -(8.0 - low32.double().item()) / t
    norm = math.log1p(math.exp(z))
    logp = torch.where(y == 0, torch.tensor(-norm, dtype=torch.float64), torch.tensor(z - norm, dtype=torch.float64))
    ref = logp.float()
    per = (logp - ref.double())
    want = per.sum(1)
    _, rewards, _ = ops.preference_loss(x.to(dev), y.to(dev), ref.to(dev), beta=1.0, **how)
    tol = positions[0] * (24 * U * math.exp(z) + U) + U * per.abs().sum(1) + U * want.abs()
    assert ((rewards.cpu().double() - want).abs() <= tol).all(), (rewards, want, tol)


@pytest.mark.parametrize("layout, c, l", [("last", 2, 1), ("last", 2, 5000), ("planes", 2, 1), ("planes", 2, 600), ("planes", 2000, 7),
                                          ("last", 90000, 3)])
def test_log_ratios_are_held_in_64_bits(dev, layout, c, l):
    """ipo: h - 1 / (2 beta), h the difference of two sequences' log ratios.  Two equal classes (the others -inf): logp = -log 2 up
    to 2^-50, every log ratio is exact up to that, the loss rounds to fp32 once."""
    x = torch.full((2, l, c), -math.inf)
    x[..., 0] = x[..., 1] = 0.0
    d = -1 if layout == "last" else 1
    x = (x if d == -1 else x.movedim(-1, 1).contiguous()).to(dev)
    y = torch.zeros(2, l, dtype=torch.int64, device=dev)
    ref = torch.full((2, l), -math.log(2.0))
    ref[0] -= 4.0 + 1e-4
    ref[1, ::2] += 1e-3
    s = (-math.log(2.0) - ref.double()).mean(1)
    off = (s[0] - s[1]).item() - 4.0
    total, rewards, _ = ops.preference_loss(x, y, ref.to(dev), beta=0.125, loss_type="ipo", average=True, class_dim=d, ignore_index=-100)
    # (h is off by 2^-47 at most, the square by twice that of its root)
    assert abs(total.item() - off * off) <= U * off * off + 2 * 2.0 ** -47 * abs(off)
    assert ((rewards.cpu().double() - 0.125 * s).abs() <= U * 0.125 * s.abs() + 2.0 ** -50).all()


def test_preference_options_keep_their_precision(dev):
    """ipo: h - 1 / (2 beta) is a difference: beta = 0.1 may not be its neighbour in fp32.  Two equal classes: logp =
    -log 2 up to 2^-50, h is exact, the loss rounds to fp32 once."""
    x = torch.zeros(2, 2, 1, device=dev)
    y = torch.zeros(2, 1, dtype=torch.int64, device=dev)
    for beta, off in ((0.1, 1e-4), (0.3, -3e-5), (0.7, 1e-3)):
        ref = torch.tensor([[-math.log(2.0) - 0.5 / beta - off], [-math.log(2.0)]]).float()
        h = ref[1].double().item() - ref[0].double().item()
        want = (h - 0.5 / beta) ** 2
        total, rewards, grad = ops.preference_loss(x, y, ref.to(dev), beta=beta, loss_type="ipo", want_grad=True)
        # (h is off by 2^-48 at most, the square by twice that of its root)
        assert abs(total.item() - want) <= U * want + 2 * 2.0 ** -48 * math.sqrt(want)
        slope = 2 * (h - 0.5 / beta)
        assert abs(grad[0, 0, 0].item() - 0.5 * slope) <= 4 * U * abs(slope) + 2.0 ** -48


@pytest.mark.parametrize("layout, l, c", [("last", 3, 13), ("last", 3, 29), ("last", 5, 150), ("last", 2, 1001), ("last", 2, 5003),
                                          ("last", 2, 50001), ("last", 1, 200003), ("planes", 9, 13), ("planes", 70, 45), ("planes", 2, 700)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zeros_carry_one_sign(dev, layout, l, c, dtype):
    """An excluded class's gradient is -w p with p = 0: minus zero for a positive weight, plus zero for a negative one, wherever
    the label lies and whichever lane stores it (a row's last classes belong to two vectors)."""
    d = -1 if layout == "last" else 1
    for label in (0, c // 2, c - 9 if c > 9 else 1, c - 1):
        x = torch.randn(2, l, c, generator=torch.Generator().manual_seed(label))
        x[..., torch.arange(c) % 3 == (label + 1) % 3] = -math.inf
        y = torch.full((2, l), label)
        x = (x if d == -1 else x.movedim(-1, 1).contiguous()).to(dtype).to(dev)
        y, weight = y.to(dev), torch.tensor([1.0, -2.0], device=dev)
        how = dict(class_dim=d, ignore_index=-100)
        logp, stats = ops.token_logprobs(x, y, **how)
        grads = [ops.token_logprobs_grad(x, y, stats, weight, **how), ops.policy_loss(x, y, logp, -weight, want_grad=True, **how)[2]]
        zero = torch.isinf(_last(x, d))
        for k, g in enumerate(grads):      # (the surrogate -r A at A = -weight and r = 1: d / d logp = weight)
            g = _last(g, d)
            assert (g[zero] == 0).all()
            right = torch.signbit(g) == (weight > 0).view(2, 1, 1)
            assert right[zero].all(), (k, label)


def test_policy_gradients_of_captured_passes(dev):
    """The forward pass leaves a gradient for a factor of 1.  Captured with its backward pass, apart from it, or a captured
    backward pass of an eager forward: every replay, at another factor and with its last result overwritten, is the eager one."""
    x, y, d, ignore = _inputs("last", 3, (20,), 1000, torch.bfloat16, seed=61)
    y, adv = y.to(dev), torch.randn(3, generator=torch.Generator().manual_seed(1)).to(dev)
    old = ops.token_logprobs(x.to(dev), y, class_dim=d, ignore_index=ignore)[0] - 0.05
    loss = ClippedPolicyLoss(kl_weight=0.1, class_dim=d, ignore_index=ignore)
    want = [ops.policy_loss(x.to(dev), y, old, adv, ref_logprobs=old, kl_weight=0.1, clip_low=0.2, clip_high=0.2, class_dim=d,
                            ignore_index=ignore, want_grad=True, grad_scale=s)[2] for s in (1.0, 2.0)]
    side = torch.cuda.Stream()

    for how in ("one capture", "two captures", "eager forward"):
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            factor, base = torch.ones((), device=dev), x.to(dev).requires_grad_(True)
        graphs = [torch.cuda.CUDAGraph() for _ in range(2)]

        def ahead():
            logits = base * 1      # (no leaf's accumulator takes part)
            return logits, loss(logits, y, old, adv, ref_logprobs=old)["total"]

        if how == "one capture":
            with torch.cuda.graph(graphs[1], stream=side):
                logits, total = ahead()
                got, = torch.autograd.grad(total, logits, factor)
            graphs = graphs[1:]
        else:
            if how == "two captures":
                with torch.cuda.graph(graphs[0], stream=side):
                    logits, total = ahead()
            else:
                with torch.cuda.stream(side):
                    logits, total = ahead()
                graphs = graphs[1:]
            side.synchronize()
            with torch.cuda.graph(graphs[-1], stream=side):
                got, = torch.autograd.grad(total, logits, factor)
        for g in graphs[:-1]:
            g.replay()
        for turn, k in enumerate((0, 1, 0, 0, 1)):
            factor.fill_(1.0 + k)
            got.zero_()
            graphs[-1].replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want[k]), (how, turn)
        del got, total, logits


@pytest.mark.parametrize("d, shape", [(-1, (2, 3, 0, 5)), (-1, (2, 0, 4, 5)), (1, (2, 5, 3, 0)), (1, (2, 5, 0, 3)), (-1, (0, 3, 4, 5)), (1, (2, 300, 0, 3))])
def test_no_positions_on_several_axes(dev, d, shape):
    x = torch.zeros(shape, device=dev, dtype=torch.bfloat16)
    lab = _last(x, d).shape[:-1]
    y, f = torch.zeros(lab, dtype=torch.int64, device=dev), torch.zeros(lab, device=dev)
    how = dict(class_dim=d, ignore_index=-100)
    logp, stats = ops.token_logprobs(x, y, **how)
    assert logp.shape == lab and ops.token_logprobs_grad(x, y, stats, f, **how).shape == shape
    out, _, grad = ops.policy_loss(x, y, f, f, want_grad=True, **how)
    assert (out == 0).all() and grad.shape == shape
    leaf = x.clone().requires_grad_(True)
    (token_logprobs(leaf, y, **how).sum() + ClippedPolicyLoss(**how)(leaf, y, f, f)["total"]).backward()
    assert leaf.grad.shape == shape
    if shape[0]:
        total, rewards, grad = ops.preference_loss(x, y, f, want_grad=True, **how)
        assert abs(total.item() - math.log(2)) <= 2 * U and (rewards == 0).all() and grad.shape == shape


@pytest.mark.parametrize("layout, positions, c", [("last", (6,), 1000), ("last", (40,), 9), ("last", (3,), 90001), ("planes", (8, 12), 21),
                                                  ("planes", (5, 7), 70), ("planes", (6,), 3001)])
@pytest.mark.parametrize("reduction", ["token", "sequence"])
def test_positions_without_an_advantage_add_nothing(dev, layout, positions, c, reduction):
    """r A = 0 for A = 0, however far the policy has moved: r = exp(200) is no fp32 value, and yet finite; a place holder of -1e9
    as the old log-probability alike."""
    x, y, d, ignore = _inputs(layout, 2, positions, c, torch.float32, seed=71)
    how = dict(class_dim=d, ignore_index=ignore, reduction=reduction)
    xd, yd = x.to(dev), y.to(dev)
    old = ops.token_logprobs(xd, yd, class_dim=d, ignore_index=ignore)[0] - 0.05
    adv = torch.randn(y.shape, generator=torch.Generator().manual_seed(72)).to(dev)
    adv.view(-1)[::3] = 0.0
    want = ops.policy_loss(xd, yd, old, adv, want_grad=True, **how)
    far = old.clone()
    far.view(-1)[::3] = -200.0
    far.view(-1)[::6] = -1e9
    got = ops.policy_loss(xd, yd, far, adv, want_grad=True, **how)
    for a, b in zip(want, got):
        assert torch.isfinite(a).all() and torch.equal(a, b)
    far.view(-1)[3] = -math.inf        # an excluded label's: its ratio is infinite, the product undefined
    if y.view(-1)[3] != ignore:
        assert torch.isnan(ops.policy_loss(xd, yd, far, adv, **how)[0][0])


@pytest.mark.parametrize("t", [0.7, 1.3])
@pytest.mark.parametrize("shape", [("last", 4, (37,), 1031, torch.bfloat16), ("last", 6, (3000,), 7, torch.float32), ("last", 2, (9,), 50001, torch.float16),
                                   ("planes", 4, (24, 20), 21, torch.float32), ("planes", 2, (30, 22), 150, torch.float32)],
                         ids=lambda s: "%s-%d" % (s[0], s[3]))
@pytest.mark.parametrize("average", [False, True])
def test_preference_loss_at_a_temperature(dev, shape, t, average):
    """The bounds of test_preference_loss, at T != 1."""
    x, y, d, ignore = _inputs(*shape, seed=81)
    beta, n = 0.3, x.shape[0]
    how = dict(class_dim=d, ignore_index=ignore, temperature=t)
    lp, keep = ot.token_logprobs(x.double(), y, **how)
    ref = (lp + 0.3 * torch.randn(y.shape, generator=torch.Generator().manual_seed(82), dtype=torch.float64)).float()
    v = x.double().requires_grad_(True)
    total, rewards = ot.preference(v, y, ref, beta=beta, average=average, **how)
    g64, = torch.autograd.grad(total, v)
    got, rew, grad = ops.preference_loss(x.to(dev), y.to(dev), ref.to(dev), beta=beta, average=average, want_grad=True, **how)
    tr = _ratio_tol(x, lp, keep, d, t, average)
    _close(rew, rewards.detach(), beta * tr + 2 * U * rewards.detach().abs(), "rewards")
    th = tr[: n // 2] + tr[n // 2:]
    _close(got, total.detach(), (beta * th).mean() + 2 * U * total.detach().abs(), "total")
    r = rewards.detach() / beta
    dh = -beta * torch.sigmoid(-beta * (r[: n // 2] - r[n // 2:]))
    ddh = beta * beta / 4 * th + 4 * U * dh.abs()
    counts = keep.reshape(n, -1).sum(1).clamp(min=1).double() if average else torch.ones(n, dtype=torch.float64)
    wide = lambda s: (torch.cat([s, s]).abs() / (n // 2) / counts).view(-1, *([1] * (y.dim() - 1))).expand(y.shape)  # noqa: E731
    _close(grad, g64, _grad_tol(x, g64, wide(dh), d, t) + (wide(ddh) / t).unsqueeze(d if d == 1 else -1), "grad")


@pytest.mark.parametrize("shape", [("last", 3, (41,), 1025, torch.bfloat16), ("last", 2, (7,), 50001, torch.float16), ("last", 4, (40,), 6, torch.float32),
                                   ("last", 2, (3,), 140001, torch.bfloat16), ("planes", 3, (24, 20), 21, torch.float32),
                                   ("planes", 2, (30, 22), 150, torch.float32), ("planes", 2, (6,), 3001, torch.float32)],
                         ids=lambda s: "%s-%d" % (s[0], s[3]))
def test_policy_module_gradients_under_a_factor(dev, shape):
    """Upstream factors of 1, 4 and 1/8, value by value: old = logp, so r = 1 up to logp's error and d / d logp = -A share."""
    x, y, d, ignore = _inputs(*shape, seed=91)
    how = dict(class_dim=d, ignore_index=ignore)
    lp, keep = ot.token_logprobs(x.double(), y, **how)
    adv = torch.randn(x.shape[0], generator=torch.Generator().manual_seed(92))
    wide = torch.where(keep, adv.double().view(-1, *([1] * (y.dim() - 1))).expand(y.shape), 0.0)
    tl = _bounds(x, d, 1.0)[1] + 3 * U * lp.abs()
    for factor in (1.0, 4.0, 0.125):
        v = x.double().requires_grad_(True)
        w = -factor * wide / keep.sum()
        g64, = torch.autograd.grad((ot.token_logprobs(v, y, **how)[0] * w).sum(), v)
        leaf = x.to(dev).requires_grad_(True)
        (factor * ClippedPolicyLoss(**how)(leaf, y.to(dev), lp.float().to(dev), adv.to(dev))["total"]).backward()
        # the weight: the ratio is off by logp's error and old's rounding, the exponential 3 u, the products and the share 4 u
        extra = (w.abs() * (2 * tl + 8 * U)).unsqueeze(d if d == 1 else -1)
        _close(leaf.grad, g64, _grad_tol(x, g64, w.abs(), d, 1.0) + extra, factor)


@pytest.mark.parametrize("shape", SHAPES + [("planes", 2, (300,), 5001, torch.float32), ("channels last", 1, (700,), 2000, torch.bfloat16)],
                         ids=IDS + ["planes-2-300-5001-float32", "channels last-1-700-2000-bfloat16"])
@pytest.mark.parametrize("t", [1.0, 0.7])
def test_long_sums_stay_within_short_chains(dev, shape, t):
    """The bound of sums in short trees joined in fp64: no chain grows with the classes.  An exponential is off by 2 u D + 2 u, its
    tree by 4 u; a running maximum's rescalings by 2 u each, 12 of them at most here (256 threads over 3001 classes at random,
    six steps of the long rows), the last one's distance part of D: R = u (2 D + 32).  logp = d / T - log s, d / T and the
    logarithm in fp64: R and its own rounding.  A gradient w (1[label] - p) / T: p off by R and the exponential's 2 u D + 6 u
    again, 4 u of w, half a step."""
    x, y, d, ignore = _inputs(*shape, seed=101)
    how = dict(class_dim=d, temperature=t, ignore_index=ignore)
    v = x.double().requires_grad_(True)
    want, keep = ot.token_logprobs(v, y, **how)
    weight = torch.randn(y.shape, generator=torch.Generator().manual_seed(102))
    g64, = torch.autograd.grad((want * weight.double()).sum(), v)
    z = _last(x.double(), d) / t
    r = U * (2 * (z.amax(-1) - z.amin(-1)) + 32)
    logp, stats = ops.token_logprobs(x.to(dev), y.to(dev), **how)
    _close(logp, want.detach(), torch.where(keep, r + U * want.detach().abs(), 0.0), "logp")
    grad = ops.token_logprobs_grad(x.to(dev), y.to(dev), stats, weight.to(dev), **how)
    p, w = torch.softmax(z, -1), (weight.double().abs() / t).unsqueeze(-1)
    tol = (w * (p * 2 * r.unsqueeze(-1) + 4 * U)).movedim(-1, d if d == 1 else -1)
    _close(grad, g64, tol + HALF_STEP[x.dtype] * (g64.abs() + tol) + LEAST[x.dtype] / 2, "grad")
