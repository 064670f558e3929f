"""The policy loss's host side and oracle, without a GPU: the oracle against torch's autograd in
float64 and against differences, and every refusal."""

from __future__ import annotations

import ctypes
import shutil
import subprocess

import numpy as np
import pytest
import torch

from card_playing_gym_amd import _native as nat
from card_playing_gym_amd.rl import policy, policy_loss
from oracle import policy as ref
from tests.conftest import ROOT


def _inputs(rows=40, width=9, seed=0):
    rng = np.random.default_rng(seed)
    logits = rng.normal(size=(rows, width)) * 2
    mask = rng.random((rows, width)) < 0.6
    actions = rng.integers(0, width, rows)
    mask[np.arange(rows), actions] = True
    logp = ref.log_softmax(logits, mask)[np.arange(rows), actions]
    old = logp + rng.normal(size=rows) * 0.3
    return logits, actions, old, rng.normal(size=rows), mask, rng


@pytest.mark.parametrize("reference", ["none", "logits", "sampled"])
@pytest.mark.parametrize("masked", [False, True])
def test_oracle_is_autograds(masked, reference):
    logits, actions, old, adv, mask, rng = _inputs(seed=masked)
    weights = rng.random(len(adv)) * (rng.random(len(adv)) < 0.8)
    options = {"weights": weights, "clip": 0.1, "clip_high": 0.3, "entropy_coef": 0.05, "normalizer": 17.0}
    if masked:
        mask[3] = False  # a row without a legal entry
        options["mask"] = mask
    if reference != "none":
        options["kl_coef"] = 0.2
    if reference == "logits":
        options["reference_logits"] = logits + rng.normal(size=logits.shape) * 0.3
    elif reference == "sampled":
        options["reference_log_probs"] = old + rng.normal(size=len(old)) * 0.2
    got = ref.policy_loss(logits, actions, old, adv, **options)

    z = torch.from_numpy(logits).requires_grad_()
    legal = torch.from_numpy(mask) if masked else torch.ones(logits.shape, dtype=torch.bool)
    fill = lambda t: torch.log_softmax(t.masked_fill(~legal, -1e300), 1)  # noqa: E731
    logp = fill(z)
    p = logp.exp()
    lp = logp.gather(1, torch.from_numpy(actions)[:, None])[:, 0]
    ratio = (lp - torch.from_numpy(old)).exp()
    a = torch.from_numpy(adv)
    loss = -torch.minimum(ratio * a, ratio.clamp(0.9, 1.3) * a) + 0.05 * (p * logp).where(legal, torch.zeros(())).sum(1)
    if reference == "logits":
        logq = fill(torch.from_numpy(options["reference_logits"]))
        loss = loss + 0.2 * (p * (logp - logq)).where(legal, torch.zeros(())).sum(1)
    elif reference == "sampled":
        d = torch.from_numpy(options["reference_log_probs"]) - lp
        loss = loss + 0.2 * (torch.expm1(d) - d)
    w = torch.from_numpy(weights) * legal.any(1)
    total = (w * loss.where(legal.any(1), torch.zeros(()))).sum() / 17.0
    total.backward()
    assert abs(got["loss"] - total.item()) <= 1e-12
    np.testing.assert_allclose(got["grad"], z.grad.numpy(), atol=1e-12)


def test_oracles_gradient_is_the_difference_quotient():
    logits, actions, old, adv, mask, rng = _inputs(rows=6, width=5, seed=4)
    options = {"mask": mask, "entropy_coef": 0.1, "kl_coef": 0.3, "reference_logits": logits + 0.2 * rng.normal(size=logits.shape)}
    grad = ref.policy_loss(logits, actions, old, adv, **options)["grad"]
    h = 1e-6
    for i in range(6):
        for j in range(5):
            up, down = logits.copy(), logits.copy()
            up[i, j] += h
            down[i, j] -= h
            slope = (ref.policy_loss(up, actions, old, adv, **options)["loss"]
                     - ref.policy_loss(down, actions, old, adv, **options)["loss"]) / (2 * h)
            assert abs(slope - grad[i, j]) < 1e-8


# ---- refusals -------------------------------------------------------------------------------


@pytest.fixture
def anywhere(monkeypatch):
    """Argument checks on CPU tensors; nothing may be launched."""

    monkeypatch.setattr(policy, "require_device", lambda *tensors: None)
    monkeypatch.setattr(policy._Call, "forward", lambda *args: pytest.fail("a bad call was launched"))


def _call(**changes):
    given = {"logits": torch.zeros(4, 6), "actions": torch.zeros(4, dtype=torch.int64), "old_log_probs": torch.zeros(4),
             "advantages": torch.zeros(4)} | changes
    return policy_loss(given.pop("logits"), given.pop("actions"), given.pop("old_log_probs"), given.pop("advantages"),
                       **given)


@pytest.mark.parametrize("changes, message", [
    ({"logits": torch.zeros(4)}, "logits must be"),
    ({"logits": torch.zeros(4, 0)}, "at least one entry"),
    ({"logits": torch.zeros(4, 6, dtype=torch.float64)}, "Unsupported dtype"),
    ({"actions": torch.zeros(4, dtype=torch.int32)}, "actions must be"),
    ({"actions": torch.zeros(5, dtype=torch.int64)}, "actions must be"),
    ({"old_log_probs": torch.zeros(4, dtype=torch.float64)}, "old_log_probs must be"),
    ({"advantages": torch.zeros(4, 1)}, "advantages must be"),
    ({"advantages": torch.zeros(4, requires_grad=True)}, "detach"),
    ({"weights": torch.zeros(3)}, "weights must be"),
    ({"mask": torch.ones(4, 5, dtype=torch.bool)}, "mask must be"),
    ({"mask": torch.ones(4, 6)}, "mask must be"),
    ({"reference_logits": torch.zeros(4, 6).half()}, "reference_logits must be"),
    ({"reference_log_probs": torch.zeros(4, 6)}, "reference_log_probs must be"),
    ({"reference_logits": torch.zeros(4, 6), "reference_log_probs": torch.zeros(4)}, "not both"),
    ({"kl_coef": 0.1}, "needs a reference"),
    ({"kl_coef": torch.zeros(())}, "needs a reference"),
    ({"clip": -0.1}, "non-negative"),
    ({"clip_high": -0.1}, "non-negative"),
    ({"normalizer": 0.0}, "positive"),
    ({"normalizer": torch.zeros((), dtype=torch.float64)}, "normalizer must be"),
    ({"entropy_coef": torch.zeros(1)}, "entropy_coef must be"),
    ({"entropy_coef": torch.zeros((), requires_grad=True)}, "detach"),
])
def test_refusals(anywhere, changes, message):
    with pytest.raises(ValueError, match=message):
        _call(**changes)


@pytest.mark.parametrize("rows, width", [(2**32 + 4, 6), (2**31, 1), (4, 2**32 + 6), (4, 2**30 + 1)])
def test_sizes_past_the_descriptors_are_refused(anywhere, rows, width):
    """2^32 + 4 rows must not become 4."""

    vector = lambda dtype=torch.float32: torch.zeros((), dtype=dtype).expand(rows)  # noqa: E731
    with pytest.raises(ValueError, match="up to"):
        _call(logits=torch.zeros(()).expand(rows, width), actions=vector(torch.int64), old_log_probs=vector(),
              advantages=vector())


def test_cpu_tensors_are_refused():
    with pytest.raises(RuntimeError, match="ROCm"):
        _call()


def test_native_refusals():
    """Fake addresses: every check comes before a launch."""

    lib = nat.lib()
    zero = nat.Scalar(0.0, None)
    size = 1 << 20

    def call(value=16, log_probs=16, entropy=16, kl=None, workspace=16, size=size, upstream=None, grad=16, **changes):
        d = nat.PolicyLoss(16, None, 16, 16, 16, None, None, None, 6, 6, 6, 4, 6, nat.CG_F32, 0.8, 1.2,
                           nat.Scalar(4.0, None), zero, zero)
        for name, x in changes.items():
            setattr(d, name, x)
        if size < 0:  # short by that much
            size += (lib.cg_policy_loss_workspace_size if upstream is None else lib.cg_policy_loss_backward_workspace_size)(
                ctypes.byref(d))
        if upstream is not None:
            return lib.cg_policy_loss_backward(ctypes.byref(d), upstream or None, 0, grad, workspace, size, None)
        return lib.cg_policy_loss_forward(ctypes.byref(d), value, log_probs, entropy, kl, None, workspace, size, None)

    for changes in ({"value": None}, {"workspace": None}, {"size": -1}, {"rows": 3, "width": 20000, "size": -1}, {"log_probs": None}, {"entropy": None},
                    {"kl": 16}, {"rows": -1}, {"width": 0}, {"dtype": 5}, {"logits": None}, {"actions": None},
                    {"old_log_probs": None}, {"advantages": None}, {"ld_logits": -1}, {"reference_logits": 16},
                    {"reference_logits": 16, "reference_log_probs": 16, "kl": 16}, {"upstream": 0}, {"upstream": 16, "grad": None},
                    {"upstream": 16, "width": 40000, "workspace": None}, {"upstream": 16, "width": 40000, "size": -1}):
        assert call(**changes) == nat.CG_ERR_INVALID, changes
    assert lib.cg_policy_loss_forward(None, 16, 16, 16, None, None, 16, size, None) == nat.CG_ERR_INVALID
    assert call(width=(1 << 30) + 1) == nat.CG_ERR_UNSUPPORTED


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_of_the_update_match_the_header(tmp_path):
    structs = {"cg_scalar": nat.Scalar, "cg_policy_loss": nat.PolicyLoss, "cg_adamw_tensor": nat.AdamWTensor,
               "cg_adamw_config": nat.AdamWConfig}
    lines = []
    for cname, py in structs.items():
        lines.append(f'printf("{cname} size %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {field} %zu\\n", offsetof({cname}, {field}));' for field, _ in py._fields_]
    source, exe = tmp_path / "layout.c", tmp_path / "layout"
    source.write_text("#include <stdio.h>\n#include <stddef.h>\n#include \"cardgym_hip.h\"\nint main(void){\n"
                      + "\n".join(lines) + "\nreturn 0;}\n")
    subprocess.run(["gcc", "-I", str(ROOT / "include"), str(source), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        cname, field, value = line.split()
        py = structs[cname]
        assert int(value) == (ctypes.sizeof(py) if field == "size" else getattr(py, field).offset), line


@pytest.mark.parametrize("name", ["logits", "old_log_probs", "advantages", "weights", "reference_logits",
                                  "reference_log_probs", "normalizer", "entropy_coef", "kl_coef"])
@pytest.mark.parametrize("wanted", [False, True])
def test_forward_derivatives_are_refused(anywhere, name, wanted):
    """The loss would come back without the derivative that was asked for; with its own gradient wanted or not."""

    from torch.autograd import forward_ad

    shape = {"logits": (4, 6), "reference_logits": (4, 6), "normalizer": (), "entropy_coef": (), "kl_coef": ()}.get(name, (4,))
    changes = {"logits": torch.zeros(4, 6, requires_grad=wanted and name != "logits")}
    if name == "kl_coef":
        changes["reference_log_probs"] = torch.zeros(4)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="forward"):
            _call(**(changes | {name: forward_ad.make_dual(torch.ones(shape), torch.ones(shape))}))
