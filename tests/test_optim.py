"""The optimiser step's host side and oracle, without a GPU: the 8-bit code's properties, the
oracle against torch.optim.AdamW, and every refusal."""

from __future__ import annotations

import copy
import ctypes

import numpy as np
import pytest
import torch

from card_playing_gym_amd import _native as nat
from card_playing_gym_amd.nn import AdamW, AdamWPlan, grad_norm, moment_values
from card_playing_gym_amd.nn import optim as O
from oracle import optim as ref


@pytest.fixture
def anywhere(monkeypatch):
    """Argument checks on CPU tensors: they come before anything is launched."""

    monkeypatch.setattr(O, "require_device", lambda *tensors: None)


def test_oracle_is_torchs_adamw():
    gen = torch.Generator().manual_seed(0)
    p = torch.randn(300, generator=gen, dtype=torch.float64).requires_grad_()
    theirs = torch.optim.AdamW([p], lr=3e-3, betas=(0.8, 0.95), eps=1e-7, weight_decay=0.1)
    x, m, v = p.detach().numpy().copy(), np.zeros(300), np.zeros(300)
    for t in range(1, 6):
        p.grad = torch.randn(300, generator=gen, dtype=torch.float64) * 3
        g = p.grad.numpy().copy()
        norm = torch.nn.utils.clip_grad_norm_([p], 10.0)
        theirs.step()
        x, m, v = ref.adamw(x, g * ref.clip_factor(float(norm), 10.0), m, v, t, 3e-3, (0.8, 0.95), 1e-7, 0.1)
        np.testing.assert_allclose(x, p.detach().numpy(), rtol=1e-12, atol=1e-14)


@pytest.mark.parametrize("signed, octaves", [(True, 16), (False, 32)])
def test_codes_cover_their_octaves_in_eighths(signed, octaves):
    f = ref.code_values(signed)[: 128 if signed else 256]
    assert f[0] == 0 and f[-1] == 1 and (np.diff(f) > 0).all()
    assert f[1] == 1.25 * 2.0**-octaves
    assert (np.diff(f)[1:] / f[1:-1] <= 1 / 8).all()


@pytest.mark.parametrize("signed", [True, False])
def test_rounding_of_codes_is_unbiased_and_keeps_held_values(signed):
    """Every code's value is kept whatever the random number; between two codes the mean over all 65536
    random numbers is the value, up to half a random number's step."""

    f = ref.code_values(signed)[: 128 if signed else 256]
    noise = np.arange(65536)
    for q in (1, 2, 7, 40, 126):
        row = np.array([f[q], 1.0])
        for r in (0, 32768, 65535):
            codes, scales = ref.encode(row, np.array([r, 0]), signed)
            assert codes[0] == q and scales[0] == 1
        x = f[q] + 0.3 * (f[q + 1] - f[q])
        codes = np.array([ref.encode(np.array([x, 1.0]), np.array([r, 0]), signed)[0][0] for r in noise[::16]])
        mean = f[codes].mean()
        assert abs(mean - x) <= (f[q + 1] - f[q]) / 4096


def test_random_words_differ_by_step_tensor_and_element():
    e = np.arange(4096)
    rows = [ref.words(s, t, i, e) for s, t, i in ((0, 1, 0), (0, 2, 0), (0, 1, 1), (1, 1, 0))]
    rows.append(ref.words(0, 1, 0, e + 2**32))
    for a in range(len(rows)):
        assert len(np.unique(rows[a])) == e.size
        for b in range(a):
            assert (rows[a] == rows[b]).mean() < 0.01
        for part in (rows[a] & np.uint64(0xFFFF), rows[a] >> np.uint64(16)):
            # mean of 4096 uniform 16-bit numbers: standard error 0.0045 of the range
            assert abs(part.mean() / 65536 - 0.5) < 0.02


# ---- refusals ----------------------------------------------------------------------------------


def _lists(bits=32, sizes=(5, 300), dtype=torch.float32):
    params = [torch.zeros(n, dtype=dtype) for n in sizes]
    moment = torch.float32 if bits == 32 else torch.uint8
    state = [[torch.zeros(n, dtype=moment) for n in sizes] for _ in range(2)]
    steps = [torch.zeros(()) for _ in sizes]
    scales = {} if bits == 32 else {
        name: [torch.zeros(-(-n // 256)) for n in sizes] for name in ("exp_avg_scales", "exp_avg_sq_scales")}
    return params, *state, steps, scales


@pytest.mark.parametrize("bits", [32, 8])
def test_plan_takes_matching_lists(anywhere, bits):
    params, m, v, steps, scales = _lists(bits)
    plan = AdamWPlan(params, m, v, steps, **scales)
    assert plan.state_bits == bits


def test_plan_refusals(anywhere):
    params, m, v, steps, scales = _lists(8)
    with pytest.raises(ValueError, match="at least one"):
        AdamWPlan([], [], [], [])
    with pytest.raises(ValueError, match="both lists"):
        AdamWPlan(params, m, v, steps, exp_avg_scales=scales["exp_avg_scales"])
    with pytest.raises(ValueError, match="contiguous torch.float32"):
        AdamWPlan(params, m, v, steps)  # codes without scales
    with pytest.raises(ValueError, match=r"\[2\]"):
        AdamWPlan(params, m, v, steps, exp_avg_scales=scales["exp_avg_scales"],
                  exp_avg_sq_scales=[torch.zeros(1), torch.zeros(3)])
    params, m, v, steps, _ = _lists()
    with pytest.raises(ValueError, match="differ in length"):
        AdamWPlan(params, m[:1], v, steps)
    with pytest.raises(ValueError, match="one type"):
        AdamWPlan([params[0], params[1].bfloat16()], m, v, steps)
    with pytest.raises(ValueError, match="Unsupported dtype"):
        AdamWPlan([p.double() for p in params], m, v, steps)
    with pytest.raises(ValueError, match="contiguous"):
        AdamWPlan([params[0], torch.zeros(600)[::2]], m, v, steps)
    with pytest.raises(ValueError, match="exp_avg_sqs"):
        AdamWPlan(params, m, [v[0], torch.zeros(299)], steps)
    with pytest.raises(ValueError, match=r"steps\[1\]"):
        AdamWPlan(params, m, v, [steps[0], torch.zeros((), dtype=torch.int64)])
    with pytest.raises(ValueError, match="share memory"):
        AdamWPlan([params[1], params[1]], [m[1], m[0].new_zeros(300)], [v[1], v[1].clone()], steps)
    with pytest.raises(ValueError, match="share memory"):  # the moments of one tensor inside another's
        AdamWPlan(params, [m[1][:5], m[1]], v, steps)
    with pytest.raises(ValueError, match="first"):
        AdamWPlan(params, m, v, steps, first=-1)


def test_step_refusals(anywhere):
    params, m, v, steps, _ = _lists()
    plan = AdamWPlan(params, m, v, steps)
    grads = [torch.ones(5), torch.ones(300)]
    with pytest.raises(ValueError, match="2 parameters but 1"):
        plan.step(grads[:1], lr=1e-3)
    with pytest.raises(ValueError, match="shape"):
        plan.step([torch.ones(1, 5), grads[1]], lr=1e-3)
    with pytest.raises(ValueError, match="type or device"):
        plan.step([grads[0].double(), None], lr=1e-3)
    with pytest.raises(ValueError, match="sparse"):
        plan.step([grads[0].to_sparse(), None], lr=1e-3)
    with pytest.raises(ValueError, match="without max_norm"):
        plan.step(grads, lr=1e-3, norm=torch.zeros((), dtype=torch.float64))
    with pytest.raises(ValueError, match="norm must be"):
        plan.step(grads, lr=1e-3, max_norm=1.0, norm=torch.zeros(()))
    with pytest.raises(ValueError, match="non-negative"):
        plan.step(grads, lr=1e-3, max_norm=-1.0)
    with pytest.raises(ValueError, match="lr must be"):
        plan.step(grads, lr=torch.zeros((), dtype=torch.float64))
    params[0].data = torch.zeros(5)
    with pytest.raises(ValueError, match="moved"):
        plan.step(grads, lr=1e-3)
    assert not any(t.any() for t in (*params, *m, *v, *steps))


def test_cpu_tensors_are_refused():
    params, m, v, steps, _ = _lists()
    with pytest.raises(RuntimeError, match="ROCm"):
        AdamWPlan(params, m, v, steps)
    with pytest.raises(RuntimeError, match="ROCm"):
        grad_norm(params)
    with pytest.raises(RuntimeError, match="ROCm"):
        moment_values(torch.zeros(4, dtype=torch.uint8), torch.zeros(1), True)


def test_norm_and_values_refusals(anywhere):
    with pytest.raises(ValueError, match="at least one"):
        grad_norm([None])
    with pytest.raises(ValueError, match="Unsupported dtype"):
        grad_norm([torch.zeros(3, dtype=torch.float64)])
    with pytest.raises(ValueError, match="uint8"):
        moment_values(torch.zeros(4), torch.zeros(1), True)
    with pytest.raises(ValueError, match=r"\[2\]"):
        moment_values(torch.zeros(257, dtype=torch.uint8), torch.zeros(1), False)


def test_native_refusals():
    """Fake addresses: every check comes before a launch."""

    lib = nat.lib()
    tensors = (nat.AdamWTensor * 1)(nat.AdamWTensor(16, 16, 16, None, None, 16, 8))
    grads = (ctypes.c_void_p * 1)(16)
    need = lib.cg_adamw_workspace_size(1)

    def status(size=need, workspace=16, norm=None, n=1, **options):
        config = nat.AdamWConfig(1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None, 0, 0, nat.CG_F32, 32, nat.CG_CLIP_NONE)
        for name, value in options.items():
            setattr(config, name, value)
        return lib.cg_adamw_step(tensors, grads, n, ctypes.byref(config), norm, workspace, size, None)

    for options in ({"size": need - 1}, {"workspace": None}, {"workspace": 8}, {"n": -1}, {"dtype": 7},
                    {"state_bits": 16}, {"beta1": 1.0}, {"beta2": -0.1}, {"clip": 3}, {"clip": nat.CG_CLIP_OWN_NORM},
                    {"clip": nat.CG_CLIP_GIVEN_NORM}, {"state_bits": 8}):
        assert status(**options) == nat.CG_ERR_INVALID, options
    tensors[0].step = None
    assert status() == nat.CG_ERR_INVALID
    for n in (-1, 2**33 + 1):
        tensors[0].n = n
        assert status() == nat.CG_ERR_RANGE
    assert lib.cg_adamw_step(tensors, grads, 1, None, None, 16, need, None) == nat.CG_ERR_INVALID
    sizes, dtypes = (ctypes.c_int64 * 1)(4), (ctypes.c_int32 * 1)(9)
    need = lib.cg_grad_norm_workspace_size(1)
    assert lib.cg_grad_norm(grads, sizes, dtypes, 1, 16, 16, need, None) == nat.CG_ERR_INVALID
    dtypes[0] = 0
    assert lib.cg_grad_norm(grads, sizes, dtypes, 1, None, 16, need, None) == nat.CG_ERR_INVALID
    assert lib.cg_grad_norm(grads, sizes, dtypes, 1, 16, 16, need - 1, None) == nat.CG_ERR_INVALID
    sizes[0] = 2**33 + 1
    assert lib.cg_grad_norm(grads, sizes, dtypes, 1, 16, 16, need, None) == nat.CG_ERR_RANGE
    assert lib.cg_moment_values(None, None, 1, None, 4, None) == nat.CG_ERR_INVALID
    assert lib.cg_moment_values(None, None, 1, None, -4, None) == nat.CG_ERR_RANGE


def test_optimizer_options():
    p = torch.nn.Parameter(torch.zeros(3))
    for options in ({"lr": -1.0}, {"betas": (1.0, 0.9)}, {"eps": -1e-8}, {"weight_decay": -0.1}, {"max_norm": -1.0},
                    {"state_bits": 16}):
        with pytest.raises(ValueError):
            AdamW([p], **options)
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="ROCm"):
        AdamW([p]).step()


def test_state_dict_refusals(anywhere):
    p = torch.nn.Parameter(torch.zeros(300))
    theirs = torch.optim.AdamW([p])
    p.grad = torch.ones(300)
    theirs.step()
    eight = AdamW([p], state_bits=8)
    with pytest.raises(ValueError, match="8-bit"):
        eight.load_state_dict(theirs.state_dict())
    wide = AdamW([p])
    wide.load_state_dict(theirs.state_dict())
    assert float(wide.state[p]["step"]) == 1 and torch.equal(wide.state[p]["exp_avg"], theirs.state[p]["exp_avg"])
    with pytest.raises(ValueError, match="32-bit"):
        wide.load_state_dict({**eight.state_dict(), "state": {0: eight._new_state(p)}})
    other = AdamW([torch.nn.Parameter(torch.zeros(299))])
    with pytest.raises(ValueError, match="shape"):
        other.load_state_dict(theirs.state_dict())


def test_state_dicts_of_other_steps_are_refused(anywhere):
    """Options that change the step, which it would leave out without a word."""

    p = torch.nn.Parameter(torch.zeros(300))
    p.grad = torch.ones(300)
    for theirs in (torch.optim.AdamW([p], amsgrad=True), torch.optim.AdamW([p], maximize=True),
                   torch.optim.Adam([p], weight_decay=0.1)):
        theirs.step()
        with pytest.raises(ValueError, match="options"):
            AdamW([p]).load_state_dict(theirs.state_dict())
    theirs = torch.optim.Adam([p])
    theirs.step()
    ours = AdamW([p])
    ours.load_state_dict(theirs.state_dict())
    assert ours.param_groups[0]["weight_decay"] == 0 and float(ours.state[p]["step"]) == 1


def test_a_loaded_learning_rate_goes_into_the_one_that_is_there(anywhere):
    """A captured step reads it there; a state dict's may lie on another device."""

    p, lr = torch.nn.Parameter(torch.zeros(3)), torch.tensor(0.5)
    ours = AdamW([p], lr=lr)
    for given in (0.25, torch.tensor(0.125), torch.tensor([0.0625])):
        ours.load_state_dict(AdamW([torch.nn.Parameter(torch.zeros(3))], lr=given).state_dict())
        assert ours.param_groups[0]["lr"] is lr and lr == given


def _stepped(optimizer):
    """A parameter of ones with one step of torch's, and its optimiser's state dict."""

    p = torch.nn.Parameter(torch.zeros(300))
    p.grad = torch.ones(300)
    theirs = optimizer([p])
    theirs.step()
    return p, theirs.state_dict()


@pytest.mark.parametrize("in_place", [False, True])
def test_load_hooks_are_obeyed(anywhere, in_place):
    """What a pre-hook makes of the dict is what is checked and loaded, state and options; a post-hook finds the state
    loaded and what it sets stays.  As torch.optim.AdamW does it."""

    p, saved = _stepped(torch.optim.AdamW)
    seen = []

    def before(optimizer, given):
        entry = {**given["state"][0], "exp_avg": torch.full((300,), 7.0)}
        groups = [{**group, "lr": 0.5} for group in given["param_groups"]]
        if in_place:
            given["state"], given["param_groups"] = {0: entry}, groups
            return None
        return {"state": {0: entry}, "param_groups": groups}

    def after(optimizer):
        state = optimizer.state[p]
        seen.append((float(state["exp_avg"][0]), float(state["step"]), optimizer.param_groups[0]["lr"]))
        state["exp_avg_sq"].fill_(3)
        optimizer.param_groups[0]["eps"] = 0.25

    for kind in (torch.optim.AdamW, AdamW):
        optimizer = kind([p])
        optimizer.register_load_state_dict_pre_hook(before)
        optimizer.register_load_state_dict_post_hook(after)
        for _ in range(2):  # (the second into state that is there)
            given = copy.deepcopy(saved)
            optimizer.load_state_dict(given)
            state = optimizer.state[p]
            assert (state["exp_avg"] == 7).all() and (state["exp_avg_sq"] == 3).all() and float(state["step"]) == 1
            assert optimizer.param_groups[0]["lr"] == 0.5 and optimizer.param_groups[0]["eps"] == 0.25
    assert seen == [(7.0, 1.0, 0.5)] * 4
    assert torch.equal(given["state"][0]["exp_avg_sq"], saved["state"][0]["exp_avg_sq"])  # (the caller's, not ours)


def test_hooks_see_moments_as_they_are_saved(anywhere):
    """Not by way of the parameter's type: 1 + 2^-20 has no bf16, code 200 of uint8 stays a code."""

    p = torch.nn.Parameter(torch.zeros(300, dtype=torch.bfloat16))
    seen = []
    for bits, value in ((32, 1 + 2.0**-20), (8, 200)):
        optimizer = AdamW([p], state_bits=bits)
        optimizer.register_load_state_dict_post_hook(lambda o: seen.append(o.state[p]["exp_avg"].clone()))
        state = {name: x + (value if name == "exp_avg" else 0) for name, x in optimizer._new_state(p).items()}
        optimizer.load_state_dict({**optimizer.state_dict(), "state": {0: state}})
        assert seen[-1].dtype == state["exp_avg"].dtype and (seen[-1] == value).all()


def test_dicts_that_hooks_make_are_checked(anywhere):
    """Before anything is loaded: a hook may repair a dict, and one that breaks it changes nothing."""

    p, saved = _stepped(lambda params: torch.optim.AdamW(params, amsgrad=True))
    repaired = AdamW([p])
    repaired.register_load_state_dict_pre_hook(
        lambda o, given: {**given, "param_groups": [{**g, "amsgrad": False} for g in given["param_groups"]]})
    repaired.load_state_dict(saved)
    assert float(repaired.state[p]["step"]) == 1
    lr = torch.tensor(0.5)
    ours = AdamW([p], lr=lr)
    ours.load_state_dict({**repaired.state_dict(), "param_groups": ours.state_dict()["param_groups"]})
    held = ours.state[p]
    kept = {name: x.clone() for name, x in held.items()}
    handle = ours.register_load_state_dict_pre_hook(
        lambda o, given: {**given, "state": {0: {**given["state"][0], "exp_avg": torch.zeros(299)}}})
    groups = ours.param_groups
    given = repaired.state_dict()
    for _ in range(2):
        with pytest.raises(ValueError, match="shape"):
            ours.load_state_dict(given)
        assert ours.state[p] is held and all(torch.equal(held[name], x) for name, x in kept.items())
        assert ours.param_groups is groups and groups[0]["lr"] is lr and lr == 0.5
    handle.remove()
    ours.load_state_dict(given)
    assert lr == 1e-3


def test_a_learning_rate_on_the_host_is_a_number(anywhere, monkeypatch):
    """The step's launch gets its value as it is by then."""

    given = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(AdamWPlan, "_step", lambda self, grads, *, lr, **_: given.append(lr), raising=False)
    monkeypatch.setattr(AdamWPlan, "step", lambda self, grads, *, lr, **_: given.append(lr))
    p, lr = torch.nn.Parameter(torch.zeros(3)), torch.tensor(0.5, dtype=torch.float64)
    p.grad = torch.ones(3)
    optimizer = AdamW([p], lr=lr)
    for value in (0.5, 0.25):
        lr.fill_(value)
        optimizer.step()
    assert given == [0.5, 0.25] and all(isinstance(x, float) for x in given)


@pytest.fixture
def recorded(anywhere, monkeypatch):
    """Steps on CPU tensors up to their launch: the parameters, rates and gradients of each launch."""

    launches = []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(AdamWPlan, "_step", lambda self, grads, *, lr, **_: launches.append((self, list(grads), lr)))
    return launches


def test_a_look_at_state_makes_none(recorded):
    """An entry that reading `state` left there, empty, is no state."""

    params = [torch.nn.Parameter(torch.ones(n)) for n in (3, 5)]
    optimizer = AdamW(params, lr=1e-2)
    assert not optimizer.state[params[0]] and not optimizer.state[params[1]].get("exp_avg")
    params[0].grad = torch.ones(3)
    optimizer.step()
    params[1].grad = torch.ones(5)
    optimizer.step()
    assert [[p.numel() for p in plan.params] for plan, _, _ in recorded] == [[3], [3, 5]]
    assert optimizer.state[params[1]]["exp_avg"].shape == (5,)
    twin = AdamW([torch.nn.Parameter(torch.ones(n)) for n in (3, 5)], lr=1e-2)
    for p in twin.param_groups[0]["params"]:
        assert not twin.state[p]
    saved = optimizer.state_dict()
    saved["state"][1] = {}
    twin.load_state_dict(saved)
    for p in twin.param_groups[0]["params"]:
        p.grad = torch.ones_like(p)
    twin.step()
    assert [p.numel() for p in recorded[-1][0].params] == [3, 5]


def test_parameters_exchanged_in_their_group(recorded):
    """Groups edited in place, as programs that grow or prune tensors do: the step follows them."""

    a, b, c, d = (torch.nn.Parameter(torch.ones(n)) for n in (3, 5, 7, 9))
    optimizer = AdamW([{"params": [a, b], "lr": 0.5}, {"params": [c], "lr": 0.25}])
    for p in (a, b, c, d):
        p.grad = torch.ones_like(p)
    optimizer.step()
    # b's place goes to d, with b's state cut to its size
    held = optimizer.state.pop(b)
    optimizer.state[d] = {name: x if name == "step" else torch.zeros(9) for name, x in held.items()}
    optimizer.param_groups[0]["params"][1] = d
    optimizer.step()
    # c to the other group, in the same order
    optimizer.param_groups[0]["params"].append(optimizer.param_groups[1]["params"].pop())
    optimizer.step()
    # a parameter more without add_param_group, one less
    optimizer.param_groups[1]["params"].append(b)
    optimizer.param_groups[0]["params"].remove(a)
    optimizer.step()
    sizes = [([p.numel() for p in plan.params], [g.numel() for g in grads], lr) for plan, grads, lr in recorded]
    assert sizes == [([3, 5], [3, 5], 0.5), ([7], [7], 0.25), ([3, 9], [3, 9], 0.5), ([7], [7], 0.25),
                     ([3, 9, 7], [3, 9, 7], 0.5), ([9, 7], [9, 7], 0.5), ([5], [5], 0.25)]
    assert recorded[3][0].params[0] is c and recorded[-1][0].params[0] is b and b in optimizer.state
