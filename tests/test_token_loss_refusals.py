"""What the loss and update entry points refuse, and what runs without a device."""
import copy
import ctypes
import pickle

import pytest
import torch

from oracle import tokenloss as ot
from spice_amd import _native as nat
from spice_amd import ops
from spice_amd.pruning.cli_helpers import build_config_from_args, create_parser, validate_args
from spice_amd.pruning.losses import ClippedPolicyLoss, PreferenceLoss, token_logprobs
from spice_amd.pruning.optim import ClippedAdam

X, Y, F = torch.zeros(2, 5, 3), torch.zeros(2, 3, dtype=torch.int64), torch.zeros(2, 3)


@pytest.mark.parametrize("call", [
    lambda: ops.token_logprobs(X, Y),
    lambda: ops.token_logprobs_grad(X, Y, torch.zeros(2, 3, 2), F),
    lambda: ops.preference_loss(X, Y, F),
    lambda: ops.policy_loss(X, Y, F, torch.zeros(2)),
    lambda: token_logprobs(X, Y),
    lambda: PreferenceLoss()(X, Y, F),
    lambda: ClippedPolicyLoss()(X, Y, F, torch.zeros(2)),
    lambda: ops.grad_norm([F]),
    lambda: ops.clip_grad_norm([F], 1.0),
    lambda: ops.adam_step([F], [F], [F], [F], 1, lr=1e-3),
])
def test_host_tensors_are_refused(call):
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        call()


def test_choices_and_empty_lists_are_refused():
    with pytest.raises(ValueError, match="loss_type"):
        ops.preference_loss(X, Y, F, loss_type="hinge")
    with pytest.raises(ValueError, match="reduction"):
        ops.policy_loss(X, Y, F, F, reduction="sum")
    with pytest.raises(ValueError, match="norm_type"):
        ops.grad_norm([F], norm_type=1.0)
    for call in (lambda: ops.grad_norm([]), lambda: ops.clip_grad_norm([], 1.0),
                 lambda: ops.adam_step([], [], [], [], 1, lr=1e-3)):
        with pytest.raises(ValueError, match="no tensors"):
            call()
    with pytest.raises(ValueError, match="max_norm"):
        ops.adam_step([F], [F], [F], [F], 1, lr=1e-3, max_norm=-1.0)
    with pytest.raises(ValueError, match="max_norm"):
        ops.adam_step([F], [F], [F], [F], 1, lr=1e-3, norm=torch.zeros(()))


def _logits(**over):
    f = dict(data=16, dtype=0, pad_=0, n=2, l=3, c=5, n_stride=15, l_stride=5, c_stride=1)
    f.update(over)
    return nat.Logits(*[f[k] for k, _ in nat.Logits._fields_])


def _labels(**over):
    f = dict(data=16, n_stride=3, l_stride=1, ignore_index=255)
    f.update(over)
    return nat.Labels(*[f[k] for k, _ in nat.Labels._fields_])


@pytest.mark.parametrize("x, y, t", [
    (_logits(data=None), _labels(), 1.0), (_logits(dtype=3), _labels(), 1.0), (_logits(c=0), _labels(), 1.0),
    (_logits(n=-1), _labels(), 1.0), (_logits(n=1 << 30, l=1 << 30), _labels(), 1.0), (_logits(), _labels(data=None), 1.0),
    (_logits(), _labels(ignore_index=4), 1.0), (_logits(), _labels(), 0.0), (_logits(), _labels(), -1.0),
    (_logits(), _labels(), float("nan")), (_logits(), _labels(), float("inf"))])
def test_c_abi_checks_the_logits_before_anything_is_queued(x, y, t):
    assert nat.lib().spice_token_logprobs(x, y, t, 16, 16, None) == nat.ERR_ARG
    assert nat.lib().spice_token_logprobs_grad(x, y, t, 16, 16, 3, 1, 1.0, None, 0, 1, 16, None) == nat.ERR_ARG
    p = nat.PreferenceParams(t, 0.1, 0.0, 0, 0)
    assert nat.lib().spice_preference_loss(x, y, 16, p, 16, 16, 16, 16, 16, 16, 1 << 20, None) == nat.ERR_ARG
    q = nat.PolicyParams(t, 0.2, 0.2, 0.0, 1.0, 0)
    assert nat.lib().spice_policy_loss(x, y, 16, 16, 1, 0, None, q, 16, 16, None, None, 1, None, 16, 1 << 20, None) == nat.ERR_ARG


def test_c_abi_checks_the_losses_options():
    L = nat.lib()
    need = L.spice_token_loss_workspace_bytes(2, 3)
    good = nat.PreferenceParams(1.0, 0.1, 0.0, 0, 0)

    def pref(p=good, x=None, ref=16, total=16, ws=16, size=need):
        return L.spice_preference_loss(x or _logits(), _labels(), ref, p, total, 16, 16, 16, 16, ws, size, None)

    assert pref(x=_logits(n=3)) == nat.ERR_ARG and pref(x=_logits(n=0)) == nat.ERR_ARG
    assert pref(ref=None) == nat.ERR_ARG and pref(total=None) == nat.ERR_ARG and pref(ws=None) == nat.ERR_ARG
    assert pref(ws=20) == nat.ERR_ARG and pref(size=need - 1) == nat.ERR_WORKSPACE
    for bad in ((1.0, 0.0, 0.0, 0, 0), (1.0, 0.1, 0.5, 0, 0), (1.0, 0.1, -0.1, 0, 0), (1.0, 0.1, 0.0, 2, 0), (1.0, 0.1, 0.1, 1, 0),
                (1.0, float("nan"), 0.0, 0, 0)):
        assert pref(nat.PreferenceParams(*bad)) == nat.ERR_ARG

    def pol(*p, ref=None, size=need):
        return L.spice_policy_loss(_logits(), _labels(), 16, 16, 1, 0, ref, nat.PolicyParams(*p), 16, 16, None, None, 1, None, 16,
                                   size, None)

    for bad in ((1.0, -0.1, 0.2, 0.0, 1.0, 0), (1.0, 1.1, 0.2, 0.0, 1.0, 0), (1.0, 0.2, -0.2, 0.0, 1.0, 0),
                (1.0, 0.2, 0.2, 0.1, 1.0, 0), (1.0, 0.2, 0.2, 0.0, 1.0, 2), (1.0, 0.2, 0.2, -1.0, 1.0, 0)):
        assert pol(*bad) == nat.ERR_ARG
    assert pol(1.0, 0.2, 0.2, 0.0, 1.0, 0, size=need - 1) == nat.ERR_WORKSPACE


def _table(*p):
    return (ctypes.c_void_p * len(p))(*p)


def _counts(*n):
    return (ctypes.c_int64 * len(n))(*n)


def test_c_abi_checks_the_tensor_tables():
    L = nat.lib()
    n = _counts(8, 8)
    need = L.spice_grad_norm_workspace_bytes(n, 2)
    assert L.spice_grad_norm_workspace_bytes(_counts(8, -1), 2) == 0

    def norm(p=(16, 64), n=n, dtype=0, kind=0, limit=1.0, record=16, ws=16, size=need):
        return L.spice_grad_norm(_table(*p), n, 2, dtype, kind, limit, record, ws, size, None)

    for bad in (dict(p=(16, None)), dict(p=(16, 18)), dict(n=_counts(8, -8)), dict(dtype=3), dict(kind=2), dict(limit=-1.0),
                dict(limit=float("nan")), dict(record=None), dict(ws=None), dict(ws=12)):
        assert norm(**bad) == nat.ERR_ARG, bad
    assert norm(size=need - 1) == nat.ERR_WORKSPACE
    assert L.spice_grad_clip(_table(16, 64), 0, _table(16, 64), 1, n, 2, 16, None) == nat.ERR_ARG
    assert L.spice_grad_clip(_table(16, 64), 0, _table(16, None), 0, n, 2, 16, None) == nat.ERR_ARG

    def adam(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, step=1, limit=1.0, p=(16, 64), size=need):
        t = _table(16, 64)
        return L.spice_adam_step(_table(*p), t, t, t, n, 2, 0, nat.AdamParams(lr, b1, b2, eps, wd, step, limit, 0), None, None, 16,
                                 16, size, None)

    for bad in (dict(lr=-1.0), dict(b1=1.0), dict(b2=1.0), dict(b1=-0.1), dict(eps=-1.0), dict(wd=-1.0), dict(step=0),
                dict(limit=float("nan")), dict(p=(16, None)), dict(lr=float("nan"))):
        assert adam(**bad) == nat.ERR_ARG, bad
    assert adam(size=need - 1) == nat.ERR_WORKSPACE


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(nat.Logits) == 64 and ctypes.sizeof(nat.Labels) == 32
    assert ctypes.sizeof(nat.PreferenceParams) == 20 and ctypes.sizeof(nat.PolicyParams) == 24
    assert ctypes.sizeof(nat.AdamParams) == 56


def test_optimizer_checks_its_options():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for bad in (dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-1.0), dict(max_grad_norm=0.0)):
        with pytest.raises(ValueError):
            ClippedAdam(p, **bad)


def test_max_grad_norm_flag(tmp_path):
    base = ["--model", "DeepLabV3Plus_resnet", "--strategy", "magnitude", "--ratio", "0.5", "--output-dir", str(tmp_path)]
    args = create_parser().parse_args(base + ["--max-grad-norm", "0.5"])
    validate_args(args)
    assert build_config_from_args(args).max_grad_norm == 0.5
    assert build_config_from_args(create_parser().parse_args(base)).max_grad_norm is None
    with pytest.raises(ValueError, match="norm limit"):
        validate_args(create_parser().parse_args(base + ["--max-grad-norm", "0"]))


def _differences(f, x, eps=1e-6):
    got = torch.zeros_like(x)
    for i in range(x.numel()):
        d = torch.zeros_like(x)
        d.view(-1)[i] = eps
        got.view(-1)[i] = (f(x + d) - f(x - d)) / (2 * eps)
    return got


@pytest.mark.parametrize("loss", ["sigmoid", "ipo", "policy"])
def test_oracle_gradients_against_differences(loss):
    """Central differences in 64 bits: their error is eps^2/6 of a third derivative (order 1 here) plus 2^-53 / eps."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 3, 4, dtype=torch.float64, generator=g)
    y = torch.tensor([[0, 2, 1, 255], [1, 255, 0, 2]])
    aux = torch.randn(2, 4, generator=g).double() - 1.0
    adv = torch.randn(2, 4, generator=g)

    def f(v):
        if loss == "policy":
            old = ot.token_logprobs(x, y)[0] - 0.1
            return ot.policy(v, y, old, adv, ref=aux, kl_weight=0.3, reduction="sequence")[0]
        return ot.preference(v, y, aux, beta=0.5, loss_type=loss)[0]

    v = x.clone().requires_grad_(True)
    got, = torch.autograd.grad(f(v), v)
    assert (got - _differences(f, x)).abs().max() <= 1e-8


def test_c_abi_checks_the_types_of_a_mixed_norm():
    L = nat.lib()
    n = _counts(8, 8, 8)
    need = L.spice_grad_norm_workspace_bytes(n, 3)

    def norm(p=(16, 66, 130), types=(0, 1, 2), kind=0, limit=1.0, record=16, ws=16, size=need):
        return L.spice_grad_norm_of_types(_table(*p), (ctypes.c_int32 * 3)(*types) if types else None, n, 3, kind, limit, record, ws,
                                          size, None)

    for bad in (dict(types=(0, 1, 3)), dict(types=(-1, 1, 2)), dict(types=None), dict(p=(18, 66, 130)), dict(p=(16, 67, 130)),
                dict(p=(16, None, 130)), dict(kind=2), dict(limit=-1.0), dict(record=None), dict(ws=None), dict(ws=12)):
        assert norm(**bad) == nat.ERR_ARG, bad
    assert norm(size=need - 1) == nat.ERR_WORKSPACE
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        ops.grad_norm([F, F.half()], any_type=True)


def _with_state(params, **options):
    opt = ClippedAdam(params, **options)
    for k, p in enumerate(params):
        state = opt._state_of(p)
        state["step"] = 3 + k
        for j, key in enumerate(("exp_avg", "exp_avg_sq")):
            state[key].copy_(torch.rand(p.shape, generator=torch.Generator().manual_seed(7 * k + j)))
    return opt


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_loaded_moments_keep_their_precision_and_take_their_parameters_order(dtype):
    make = lambda **how: [torch.nn.Parameter(torch.ones(4, 3, 2, 5, dtype=dtype).contiguous(**how)), torch.nn.Parameter(torch.ones(7, dtype=dtype))]  # noqa: E731
    old, new = make(), make(memory_format=torch.channels_last)
    a, b = _with_state(old, lr=2e-3, weight_decay=0.1, decoupled=True), ClippedAdam(new)
    b.load_state_dict(a.state_dict())
    for k, (p, q) in enumerate(zip(old, new)):
        assert b.state[q]["step"] == 3 + k
        for key in ("exp_avg", "exp_avg_sq"):
            x, y = a.state[p][key], b.state[q][key]
            assert y.dtype == torch.float32 and y.stride() == q.stride() and torch.equal(x, y) and x.data_ptr() != y.data_ptr()
    assert b.param_groups[0]["lr"] == 2e-3 and b.param_groups[0]["decoupled"] and b.param_groups[0]["weight_decay"] == 0.1


@pytest.mark.parametrize("kind, decoupled", [(torch.optim.Adam, False), (torch.optim.AdamW, True)])
def test_a_state_of_torch_adam_is_taken_up(kind, decoupled):
    p, q = torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(5))
    a = kind([p], lr=5e-3, betas=(0.8, 0.95), weight_decay=0.2)
    for k in range(3):
        p.grad = torch.arange(5.0) + k
        a.step()
    torch.optim.lr_scheduler.ExponentialLR(a, 0.9)     # (its initial_lr stays in the groups)
    b = ClippedAdam([q], max_grad_norm=1.0)
    b.load_state_dict(a.state_dict())
    assert b.state[q]["step"] == 3 and isinstance(b.state[q]["step"], int)
    assert torch.equal(b.state[q]["exp_avg"], a.state[p]["exp_avg"]) and torch.equal(b.state[q]["exp_avg_sq"], a.state[p]["exp_avg_sq"])
    group = b.param_groups[0]
    assert (group["lr"], group["betas"], group["weight_decay"], group["decoupled"], group["initial_lr"]) == (5e-3, (0.8, 0.95), 0.2, decoupled, 5e-3)
    assert not {"amsgrad", "maximize", "fused", "decoupled_weight_decay"} & set(group)


def test_states_that_are_not_its_own_are_refused_as_a_whole():
    p, q = torch.nn.Parameter(torch.ones(5)), torch.nn.Parameter(torch.ones(5))
    sgd = torch.optim.SGD([p], lr=0.5, momentum=0.9)
    p.grad = torch.ones(5)
    sgd.step()
    for state, text in ((sgd.state_dict(), "not Adam's"), (torch.optim.Adam([p], amsgrad=True).state_dict(), "amsgrad"),
                        (torch.optim.Adam([p], maximize=True).state_dict(), "maximize"),
                        (_with_state([torch.nn.Parameter(torch.ones(6))], lr=0.5).state_dict(), "shape"),
                        (_with_state([p, torch.nn.Parameter(torch.ones(5))], lr=0.5).state_dict(), "parameter group")):
        opt = ClippedAdam([q], lr=0.25)
        with pytest.raises(ValueError, match=text):
            opt.load_state_dict(state)
        assert opt.param_groups[0]["lr"] == 0.25 and not opt.state[q]


def test_c_abi_checks_the_options_in_full_precision():
    L = nat.lib()
    assert ctypes.sizeof(nat.PreferenceOptions) == 32 and ctypes.sizeof(nat.PolicyOptions) == 48
    need = L.spice_token_loss_workspace_bytes(2, 3)

    def pref(*p, size=need):
        return L.spice_preference_loss_opts(_logits(), _labels(), 16, nat.PreferenceOptions(*p), 16, 16, 16, 16, 16, size, None)

    def pol(*p, ref=None, size=need):
        return L.spice_policy_loss_opts(_logits(), _labels(), 16, 16, 1, 0, ref, nat.PolicyOptions(*p), 16, 16, None, None, 1, None, 16,
                                        size, None)

    nan, inf = float("nan"), float("inf")
    for bad in ((0.0, 0.1, 0.0, 0, 0), (nan, 0.1, 0.0, 0, 0), (inf, 0.1, 0.0, 0, 0), (1e-39, 0.1, 0.0, 0, 0), (1.0, 0.0, 0.0, 0, 0),
                (1.0, nan, 0.0, 0, 0), (1.0, inf, 0.0, 0, 0), (1.0, 0.1, 0.5, 0, 0), (1.0, 0.1, -0.1, 0, 0), (1.0, 0.1, 0.0, 2, 0),
                (1.0, 0.1, 0.1, 1, 0)):
        assert pref(*bad) == nat.ERR_ARG, bad
    assert pref(1.0, 0.1, 0.0, 0, 0, size=need - 1) == nat.ERR_WORKSPACE
    for bad in ((nan, 0.2, 0.2, 0.0, 1.0, 0), (1.0, -0.1, 0.2, 0.0, 1.0, 0), (1.0, 1.1, 0.2, 0.0, 1.0, 0), (1.0, 0.2, nan, 0.0, 1.0, 0),
                (1.0, 0.2, 0.2, 0.1, 1.0, 0), (1.0, 0.2, 0.2, -1.0, 1.0, 0), (1.0, 0.2, 0.2, 0.0, 1.0, 2)):
        assert pol(*bad) == nat.ERR_ARG, bad
    assert pol(1.0, 0.2, 0.2, 0.0, 1.0, 0, size=need - 1) == nat.ERR_WORKSPACE


def test_c_abi_checks_the_adam_options():
    L = nat.lib()
    assert ctypes.sizeof(nat.AdamOptions) == 64
    n, t = _counts(8, 8), _table(16, 64)
    need = L.spice_grad_norm_workspace_bytes(n, 2)

    def adam(lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, wd=0.0, limit=1.0, step=1, ws=16, size=need):
        return L.spice_adam_step_opts(t, t, t, t, n, 2, 0, nat.AdamOptions(lr, b1, b2, eps, wd, limit, step, 0), None, None, 16, ws, size,
                                      None)

    for bad in (dict(lr=-1.0), dict(b1=1.0), dict(b2=float("nan")), dict(eps=-1.0), dict(wd=-1.0), dict(limit=float("nan")), dict(step=0),
                dict(ws=None), dict(ws=12)):
        assert adam(**bad) == nat.ERR_ARG, bad
    assert adam(size=need - 1) == nat.ERR_WORKSPACE


def test_c_abi_checks_every_pointers_alignment():
    """Before anything is queued: an address between two elements would fault on the device, or read half of each."""
    L = nat.lib()
    need, odd = L.spice_token_loss_workspace_bytes(2, 3), 18
    pref_opts, pol_opts = nat.PreferenceOptions(1.0, 0.1, 0.0, 0, 0), nat.PolicyOptions(1.0, 0.2, 0.2, 0.1, 1.0, 0)

    def logp(x=_logits(), y=_labels(), out=16, stats=16):
        return L.spice_token_logprobs(x, y, 1.0, out, stats, None)

    def grad(x=_logits(), y=_labels(), stats=16, weight=16, scale=16, out=16):
        return L.spice_token_logprobs_grad(x, y, 1.0, stats, weight, 3, 1, 1.0, scale, 0, 1, out, None)

    def pref(x=_logits(), y=_labels(), ref=16, total=16, rewards=16, weight=16, stats=16, ws=16):
        return L.spice_preference_loss_opts(x, y, ref, pref_opts, total, rewards, weight, stats, ws, need, None)

    def pol(x=_logits(), y=_labels(), old=16, adv=16, ref=16, out=16, logp=16, stats=16, weight=16, g=16, ws=16):
        return L.spice_policy_loss_opts(x, y, old, adv, 1, 0, ref, pol_opts, out, logp, stats, weight, 1, g, ws, need, None)

    for call, names in ((logp, ("out", "stats")), (grad, ("stats", "weight", "scale", "out")),
                        (pref, ("ref", "total", "rewards", "weight", "stats", "ws")),
                        (pol, ("old", "adv", "ref", "out", "logp", "stats", "weight", "g", "ws"))):
        for name in names:
            assert call(**{name: odd}) == nat.ERR_ARG, (call.__name__, name)
        assert call(x=_logits(data=18)) == call(x=_logits(data=17, dtype=1)) == call(y=_labels(data=20)) == nat.ERR_ARG, call.__name__
    assert grad(x=_logits(dtype=2), out=17) == pol(x=_logits(dtype=2), g=17) == nat.ERR_ARG
    n, t = _counts(8, 8), _table(16, 64)
    size = L.spice_grad_norm_workspace_bytes(n, 2)
    a = nat.AdamOptions(1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, 1, 0)
    assert L.spice_grad_norm(t, n, 2, 0, 0, 1.0, odd, 16, size, None) == nat.ERR_ARG
    assert L.spice_grad_clip(t, 0, t, 0, n, 2, odd, None) == nat.ERR_ARG
    assert L.spice_grad_norm_clip(t, 0, t, 0, n, 2, 0, 1.0, odd, 16, size, None) == nat.ERR_ARG
    for norm, step, record in ((odd, None, 16), (None, 20, 16), (None, None, odd)):
        assert L.spice_adam_step_opts(t, t, t, t, n, 2, 0, a, norm, step, record, 16, size, None) == nat.ERR_ARG


def test_copies_of_the_optimizer_keep_its_limit():
    p = torch.nn.Parameter(torch.ones(5))
    opt = _with_state([p], lr=0.5, max_grad_norm=0.25)
    for again in (copy.deepcopy(opt), pickle.loads(pickle.dumps(opt))):
        assert again.max_grad_norm == 0.25 and again.last_grad_norm is None and again.param_groups[0]["lr"] == 0.5
        q, = again.param_groups[0]["params"]
        assert again.state[q]["step"] == 3 and torch.equal(again.state[q]["exp_avg"], opt.state[p]["exp_avg"])


@pytest.mark.parametrize("types", [(torch.float32,), (torch.float32, torch.bfloat16)])
def test_the_optimizer_refuses_host_parameters(types):
    params = [torch.nn.Parameter(torch.ones(5, dtype=t)) for t in types]
    for p in params:
        p.grad = torch.ones_like(p)
    opt = ClippedAdam(params, lr=0.5, max_grad_norm=1.0)
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        opt.step()
    assert all((p == 1).all() for p in params)
