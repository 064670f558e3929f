"""Sampling under controls, the record of top entries and the distillation loss, without a GPU: the oracles against
closed forms, torch's autograd in float64 and differences, and every refusal."""

from __future__ import annotations

import ctypes
import shutil
import subprocess

import numpy as np
import pytest
import torch

from card_playing_gym_amd import _native as nat
from card_playing_gym_amd.rl import choose, distill_loss, sample_logits, top_logits
from oracle import choose as ref
from oracle import distill as ref_distill
from tests.conftest import ROOT


# ---- the oracles -----------------------------------------------------------------------------------------------------


def test_sampling_closed_forms():
    z = np.log(np.array([[0.1, 0.4, 0.2, 0.3]]))
    grid = np.arange(1000) / 1000 + 0.0005
    share = lambda **c: np.bincount(ref.sample(z.repeat(1000, 0), grid, **c)[0], minlength=4) / 1000  # noqa: E731
    np.testing.assert_allclose(share(), [0.1, 0.4, 0.2, 0.3], atol=1e-3)
    np.testing.assert_allclose(share(top_k=2), [0, 4 / 7, 0, 3 / 7], atol=1e-3)
    np.testing.assert_allclose(share(top_p=0.71), [0, 4 / 9, 2 / 9, 3 / 9], atol=1e-3)
    np.testing.assert_allclose(share(top_p=0.69), [0, 4 / 7, 0, 3 / 7], atol=1e-3)
    np.testing.assert_allclose(share(min_p=0.51), [0, 4 / 7, 0, 3 / 7], atol=1e-3)
    np.testing.assert_allclose(share(temperature=0.5), np.array([1, 16, 4, 9]) / 30, atol=1e-3)
    # top_p is of what top_k has left: 4/7 < 0.6
    np.testing.assert_allclose(share(top_k=2, top_p=0.57), [0, 1, 0, 0], atol=1e-3)
    for controls in ({"top_k": 1}, {"top_p": 0.0}, {"min_p": 1.0}, {"temperature": 0.0}):
        assert share(**controls)[1] == 1
    actions, log_probs, _ = ref.sample(z, np.array([0.35]))  # the order is 1, 3, 2, 0: 0.4 covers 0.35
    assert actions[0] == 1 and abs(log_probs[0] - np.log(0.4)) < 1e-12


def test_ties_and_signs_of_zero_go_by_their_index():
    z = np.array([[1.0, 2.0, -0.0, 2.0, 0.0]])
    assert list(ref.ordered(z[0], np.ones(5, dtype=bool))) == [1, 3, 0, 2, 4]
    log_probs, indices, rest = ref.top(z, 3)
    assert indices.tolist() == [[1, 3, 0]]
    p = torch.from_numpy(z).softmax(1)[0].numpy()
    np.testing.assert_allclose(np.exp(log_probs[0]), p[[1, 3, 0]])
    np.testing.assert_allclose(np.exp(rest[0]), p[[2, 4]].sum())


@pytest.mark.parametrize("rest", [False, True])
@pytest.mark.parametrize("masked", [False, True])
def test_distillation_is_autograds(masked, rest):
    rng = np.random.default_rng(5)
    rows, width, k, t = 12, 9, 4, 1.7
    logits, teacher = rng.normal(size=(rows, width)) * 2, rng.normal(size=(rows, width)) * 2
    mask = rng.random((rows, width)) < 0.7 if masked else np.ones((rows, width), dtype=bool)
    mask[:, 2:8] = True
    log_probs, indices, log_rest = ref.top(teacher, k, mask, t)
    weights = rng.random(rows) * (rng.random(rows) < 0.8)
    got = ref_distill.distill(logits, indices, log_probs, log_rest if rest else None, mask if masked else None, weights, 7.0, t)

    z = torch.from_numpy(logits).requires_grad_()
    legal, at, logq = torch.from_numpy(mask), torch.from_numpy(indices), torch.from_numpy(log_probs)
    logp = torch.log_softmax((z / t).masked_fill(~legal, -1e300), 1)
    if not rest:
        logq = logq.log_softmax(1)
    kl = (logq.exp() * (logq - logp.gather(1, at))).sum(1)
    if rest:
        outside = legal.scatter(1, at, False)
        log_rest = torch.from_numpy(log_rest)
        some = outside.any(1)
        beside = logp.masked_fill(~outside, -1e300).logsumexp(1)
        kl = kl + torch.where(some, log_rest.exp() * (log_rest - beside), 0.0)
    loss = (torch.from_numpy(weights) * kl).sum() / 7.0
    loss.backward()
    assert abs(got["loss"] - loss.item()) < 1e-12
    np.testing.assert_allclose(got["grad"], z.grad.numpy(), atol=1e-12)
    step = 1e-6
    for r, j in ((0, 0), (3, 2), (7, 8)):
        moved = [logits.copy(), logits.copy()]
        moved[0][r, j] += step
        moved[1][r, j] -= step
        up, down = (ref_distill.distill(m, indices, log_probs, None if not rest else np.asarray(log_rest),
                                        mask if masked else None, weights, 7.0, t)["loss"] for m in moved)
        assert abs((up - down) / (2 * step) - got["grad"][r, j]) < 1e-8


def test_rows_of_the_distillation_oracle_that_do_not_count():
    logits = np.zeros((6, 4))
    logits[0, 1], logits[1, 2] = np.nan, np.inf
    indices = np.array([[-1, -1], [0, -1], [1, 1], [4, -1], [0, -2], [0, 1]])
    log_probs = np.full((6, 2), -1.0)
    log_probs[:5] = -np.inf
    out = ref_distill.distill(logits, indices, log_probs)
    assert (out["kl"][:2] == 0).all() and (out["grad"][:2] == 0).all()  # no record
    assert np.isnan(out["kl"][2:5]).all() and np.isnan(out["grad"][2:5]).all()  # one out of order
    assert np.isfinite(out["kl"][5])
    assert np.isnan(ref_distill.distill(logits, indices, log_probs, np.zeros(6))["kl"][:5]).all()
    nothing = ref_distill.distill(logits, indices, log_probs, mask=np.zeros((6, 4), dtype=bool))
    assert (nothing["kl"] == 0).all() and (nothing["grad"] == 0).all()


# ---- refusals --------------------------------------------------------------------------------------------------------


@pytest.fixture
def anywhere(monkeypatch):
    """Argument checks without a GPU: nothing past them is reached."""

    monkeypatch.setattr(choose, "require_device", lambda *tensors: None)


def _sample(**changes):
    given = {"logits": torch.zeros(4, 6), "uniforms": torch.zeros(4, dtype=torch.float64)} | changes
    return sample_logits(given.pop("logits"), given.pop("uniforms"), **given)


def _distill(**changes):
    given = {"logits": torch.zeros(4, 6), "indices": torch.zeros(4, 2, dtype=torch.int64), "log_probs": torch.zeros(4, 2)} | changes
    return distill_loss(given.pop("logits"), given.pop("indices"), given.pop("log_probs"), **given)


ROWS = [
    ({"logits": torch.zeros(4)}, "logits must be"),
    ({"logits": torch.zeros(4, 0)}, "at least one entry"),
    ({"logits": torch.zeros(4, 6, dtype=torch.float64)}, "Unsupported dtype"),
    ({"logits": torch.zeros(()).expand(4, 2**18 + 1)}, "up to"),
    ({"logits": torch.zeros(()).expand(2**31, 6)}, "up to"),
    ({"mask": torch.ones(4, 5, dtype=torch.bool)}, "mask must be"),
    ({"mask": torch.ones(4, 6)}, "mask must be"),
]


@pytest.mark.parametrize("changes, message", ROWS + [
    ({"uniforms": torch.zeros(4)}, "uniforms must be"),
    ({"uniforms": torch.zeros(5, dtype=torch.float64)}, "uniforms must be"),
    ({"temperature": -0.5}, "temperature must be"),
    ({"temperature": float("nan")}, "temperature must be"),
    ({"temperature": float("inf")}, "temperature must be"),
    ({"temperature": torch.ones(4, dtype=torch.float64)}, "temperature must be a number or"),
    ({"temperature": torch.ones(())}, "temperature must be a number or"),
    ({"top_p": -0.1}, "top_p must not"),
    ({"top_p": float("nan")}, "top_p must not"),
    ({"top_p": torch.ones(3)}, "top_p must be a number or"),
    ({"min_p": 1.5}, "min_p may be"),
    ({"min_p": float("nan")}, "min_p may be"),
    ({"min_p": torch.ones(4).half()}, "min_p must be a number or"),
    ({"top_k": torch.ones(4, dtype=torch.int32)}, "top_k must be a number or"),
    ({"top_k": torch.ones(4)}, "top_k must be a number or"),
])
def test_sampling_refusals(anywhere, changes, message):
    with pytest.raises(ValueError, match=message):
        _sample(**changes)


@pytest.mark.parametrize("changes, message", ROWS + [
    ({"k": 0}, "k must be"),
    ({"k": 257}, "k must be"),
    ({"temperature": 0.0}, "temperature must be"),
    ({"temperature": -1.0}, "temperature must be"),
    ({"temperature": float("nan")}, "temperature must be"),
    ({"temperature": 1e31}, "temperature must be"),
])
def test_record_refusals(anywhere, changes, message):
    given = {"logits": torch.zeros(4, 6), "k": 3} | changes
    with pytest.raises(ValueError, match=message):
        top_logits(given.pop("logits"), given.pop("k"), **given)


@pytest.mark.parametrize("changes, message", ROWS + [
    ({"indices": torch.zeros(4, 2, dtype=torch.int32)}, "indices must be"),
    ({"indices": torch.zeros(4, dtype=torch.int64)}, "indices must be"),
    ({"indices": torch.zeros(4, 0, dtype=torch.int64)}, "k from 1"),
    ({"indices": torch.zeros(4, 257, dtype=torch.int64)}, "k from 1"),
    ({"indices": torch.zeros(5, 2, dtype=torch.int64)}, "indices must be"),
    ({"log_probs": torch.zeros(4, 3)}, "log_probs must be"),
    ({"log_probs": torch.zeros(4, 2, dtype=torch.float64)}, "log_probs must be"),
    ({"log_probs": torch.zeros(4, 2, requires_grad=True)}, "detach"),
    ({"log_rest": torch.zeros(4, 1)}, "log_rest must be"),
    ({"log_rest": torch.zeros(4, requires_grad=True)}, "detach"),
    ({"weights": torch.zeros(3)}, "weights must be"),
    ({"normalizer": 0.0}, "positive"),
    ({"normalizer": torch.zeros((), dtype=torch.float64)}, "normalizer must be"),
    ({"temperature": 0.0}, "temperature must be"),
    ({"temperature": float("inf")}, "temperature must be"),
])
def test_distillation_refusals(anywhere, changes, message):
    with pytest.raises(ValueError, match=message):
        _distill(**changes)


def test_cpu_tensors_are_refused():
    for call in (_sample, _distill, lambda: top_logits(torch.zeros(4, 6), 2)):
        with pytest.raises(RuntimeError, match="ROCm"):
            call()


@pytest.mark.parametrize("name", ["logits", "log_probs", "log_rest", "weights", "normalizer"])
def test_forward_derivatives_are_refused(anywhere, name):
    from torch.autograd import forward_ad

    shape = {"logits": (4, 6), "log_probs": (4, 2), "normalizer": ()}.get(name, (4,))
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="distill_loss has no forward"):
            _distill(**{name: forward_ad.make_dual(torch.ones(shape), torch.ones(shape))})


@pytest.mark.parametrize("k", [0.5, 2.7, float("nan"), float("inf"), -0.5])
def test_a_top_k_that_is_no_whole_number_is_refused(anywhere, k):
    with pytest.raises(ValueError, match="top_k must be a whole number"):
        _sample(top_k=k)


@pytest.mark.parametrize("name", ["logits", "uniforms", "temperature", "top_p", "min_p"])
def test_forward_derivatives_of_answers_are_refused(anywhere, name):
    from torch.autograd import forward_ad

    dtype = torch.float64 if name == "uniforms" else torch.float32
    x = torch.ones((4, 6) if name == "logits" else (4,), dtype=dtype)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match="sample_logits has no forward"):
            _sample(**{name: dual})
        if name == "logits":
            with pytest.raises(RuntimeError, match="top_logits has no forward"):
                top_logits(dual, 3)


def test_native_refusals():
    """Fake addresses: every check comes before a launch."""

    lib = nat.lib()
    invalid, unsupported = nat.CG_ERR_INVALID, nat.CG_ERR_UNSUPPORTED

    def rows(**changes):
        d = nat.PolicyRows(16, None, 6, 0, 4, 6, nat.CG_F32)
        for name, x in changes.items():
            setattr(d, name, x)
        return d

    bad = [{"logits": None}, {"rows": -1}, {"width": 0}, {"dtype": 5}, {"ld_logits": -1}, {"ld_mask": -1}]

    def sample(d, uniforms=16, actions=16, log_probs=16, **controls):
        c = nat.SampleControls(1.0, 1.0, 0.0, 0, None, None, None, None)
        for name, x in controls.items():
            setattr(c, name, x)
        return lib.cg_sample_logits(d, uniforms, ctypes.byref(c), actions, log_probs, None)

    def top(d, k=3, temperature=1.0, log_probs=16, indices=16, log_rest=16):
        return lib.cg_top_logits(d, k, temperature, log_probs, indices, log_rest, None)

    def distill(d, value=16, kl=16, workspace=16, size=1 << 20, upstream=None, grad=16, **changes):
        loss = nat.DistillLoss(d, 16, 16, None, None, 3, 1.0, nat.Scalar(4.0, None))
        for name, x in changes.items():
            setattr(loss, name, x)
        if upstream is not None:
            return lib.cg_distill_loss_backward(ctypes.byref(loss), upstream or None, 0, grad, None)
        if size < 0:  # short by that much
            size += lib.cg_distill_loss_workspace_size(ctypes.byref(loss))
        return lib.cg_distill_loss_forward(ctypes.byref(loss), value, kl, None, workspace, size, None)

    for call in (sample, top, distill):
        for changes in bad:
            assert call(rows(**changes)) == invalid, changes
        assert call(rows(width=(1 << 18) + 1)) == unsupported
    for changes in ({"uniforms": None}, {"actions": None}, {"log_probs": None}, {"temperature": -1.0},
                    {"temperature": float("nan")}, {"temperature": float("inf")}):
        assert sample(rows(), **changes) == invalid, changes
    for changes in ({"k": 0}, {"k": 257}, {"temperature": 0.0}, {"temperature": float("nan")}, {"log_probs": None},
                    {"indices": None}, {"log_rest": None}):
        assert top(rows(), **changes) == invalid, changes
    for changes in ({"value": None}, {"kl": None}, {"workspace": None}, {"size": -1},
                    {"k": 0}, {"k": 257}, {"temperature": 0.0}, {"indices": None}, {"log_probs": None}, {"upstream": 0},
                    {"upstream": 16, "grad": None}):
        assert distill(rows(), **changes) == invalid, changes
    # A launch has fewer than 2^32 threads.
    many = {"rows": 2**31 - 1, "width": 9000}
    assert sample(rows(**many)) == top(rows(**many)) == distill(rows(**many), upstream=16) == unsupported
    assert distill(rows(**many), size=1 << 40) == unsupported
    assert lib.cg_sample_logits(None, 16, None, 16, 16, None) == invalid
    assert lib.cg_sample_logits(ctypes.byref(rows()), 16, None, 16, 16, None) == invalid
    assert lib.cg_top_logits(None, 3, 1.0, 16, 16, 16, None) == invalid
    assert lib.cg_distill_loss_forward(None, 16, 16, None, 16, 1 << 20, None) == invalid
    assert lib.cg_distill_loss_backward(None, 16, 0, 16, None) == invalid


@pytest.mark.skipif(shutil.which("gcc") is None, reason="needs gcc")
def test_struct_layouts_match_the_header(tmp_path):
    structs = {"cg_policy_rows": nat.PolicyRows, "cg_sample_controls": nat.SampleControls, "cg_distill_loss": nat.DistillLoss}
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
