"""The policy loss over more rows than its launches take at a time, and its kernels that only long calls reach
(csrc/loss.hip): 2048 blocks at most of 64 (rows of up to 128 entries), 32, 16, 8, 4 or one row each, 512 of the
wide rows' blocks; 16 lanes a row of 257 to 512 entries and 32 of up to 1024 from 8193 rows on.

Most rows of a call are compared with the same call in which only a few spread ones have weight, bit for bit (a row's
numbers are its own); those few with float64.  The loss is compared with the sum over the reported rows."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from card_playing_gym_amd.rl import policy_loss
from tests.test_gpu_policy_loss import DTYPES, HALF_STEP, TINY, U, check, expected, host

pytestmark = pytest.mark.gpu

CLIP, ENTROPY, KL = 0.2, 0.03, 0.2


def inputs(device, rows, width, dtype, reference, masked, seed):
    """Made on the device; the ratios are near 1, on either side of the clip range."""

    gen = torch.Generator(device=device).manual_seed(seed)
    normal = lambda *shape: torch.randn(shape, generator=gen, device=device)  # noqa: E731
    logits = (2 * normal(rows, width)).to(dtype)
    actions = torch.randint(0, width, (rows,), generator=gen, device=device)
    options = {"entropy_coef": ENTROPY, "normalizer": float(rows)}
    legal = torch.ones((), dtype=torch.bool, device=device)
    if masked:
        legal = torch.rand((rows, width), generator=gen, device=device) < 0.5
        legal.scatter_(1, actions[:, None], True)
        options["mask"] = legal
    log_p = logits.float().masked_fill(~legal, -torch.inf).log_softmax(1).gather(1, actions[:, None])[:, 0]
    given = {"logits": logits, "actions": actions, "old": log_p + 0.15 * normal(rows), "advantages": normal(rows)}
    options["weights"] = 0.5 + torch.rand(rows, generator=gen, device=device)
    if reference:
        options["kl_coef"] = KL
    if reference == "logits":
        options["reference_logits"] = (logits.float() + 0.3 * normal(rows, width)).to(dtype)
    if reference == "sampled":
        options["reference_log_probs"] = log_p + 0.2 * normal(rows)
    return given, options


def call(given, options):
    leaf = given["logits"].detach().requires_grad_()
    out = policy_loss(leaf, given["actions"], given["old"], given["advantages"], **options)
    return out, torch.autograd.grad(out.loss, leaf)[0]


def loss_of_rows(given, options, out):
    """The loss from what the rows report, and how far the reports' roundings to fp32 may take it."""

    log_p, a, w = out.log_probs.double(), given["advantages"].double(), options["weights"].double()
    r = (log_p - given["old"].double()).exp()
    kl = torch.zeros_like(r) if out.kl is None else out.kl.double()
    rows = -torch.minimum(r * a, r.clamp(1 - CLIP, 1 + CLIP) * a) + KL * kl - ENTROPY * out.entropy.double()
    off = U * (r * a.abs() * (log_p.abs() + 1) + KL * kl + ENTROPY * out.entropy.double())
    return (w * rows).sum().item() / options["normalizer"], 2 * (w * off).sum().item() / options["normalizer"]


def spread(rows, device, count):
    """The first and last rows, and some between: of every turn and place in a block."""

    picks = np.unique(np.r_[np.arange(8), rows - 1 - np.arange(8), np.random.default_rng(0).integers(0, rows, count)])
    return torch.from_numpy(picks).to(device)


def compare(device, rows, width, dtype, reference, masked, count=200, check=check):
    given, options = inputs(device, rows, width, dtype, reference, masked, seed=rows + width)
    out, grad = call(given, options)
    value, off = loss_of_rows(given, options, out)
    assert abs(out.loss.item() - value) <= off + U * abs(value)
    some = spread(rows, device, count)
    weights = torch.zeros_like(options["weights"])
    weights[some] = options["weights"][some]
    few, few_grad = call(given, {**options, "weights": weights})
    fields = [name for name in ("log_probs", "entropy", "kl") if getattr(out, name) is not None]
    for all_of, part in [(getattr(out, name), getattr(few, name)) for name in fields] + [(grad, few_grad)]:
        assert torch.equal(all_of[some], part[some])
        part = part.clone()
        part[some] = 0
        assert not part.any()
    cut = lambda x: x[some] if isinstance(x, torch.Tensor) and x.dim() else x  # noqa: E731
    check({k: cut(v) for k, v in given.items()}, {k: cut(v) for k, v in options.items()},
          few._replace(**{name: getattr(few, name)[some] for name in fields}), few_grad[some])


REFERENCES = [None, "logits", "sampled"]


# Two turns and a few rows of a third's block (or of the second's): a block that is part empty, one that has a turn less.
@pytest.mark.parametrize("rows, width, dtype", [
    (65536 + 32 * 40 + 5, 3, torch.float32), (65536 * 2 + 32 + 1, 5, torch.bfloat16), (65536 + 31, 7, torch.float16),
    (131072 + 64 * 700 + 13, 40, torch.bfloat16), (131072 * 2 + 64 + 1, 9, torch.float16), (131072 + 63, 77, torch.float32),
    (131072 + 1, 100, torch.bfloat16), (65536 + 32 * 9 + 3, 130, torch.bfloat16), (65536 + 1, 200, torch.float16),
    (32768 + 16 * 300 + 7, 300, torch.float32), (32768 * 2 + 1, 512, torch.bfloat16), (16384 + 8 * 100 + 3, 600, torch.bfloat16),
    (16384 + 7, 1024, torch.float16), (8192 + 4 * 50 + 3, 1100, torch.float32), (2048 * 2 + 5, 2100, torch.bfloat16),
    (2048 + 9, 5000, torch.float16),
])
def test_rows_of_several_turns(device, rows, width, dtype):
    for k, reference in enumerate(REFERENCES):
        compare(device, rows, width, dtype, reference, masked=k != 2)


@pytest.mark.parametrize("width", [257, 511, 512, 513, 1023])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_few_lanes_a_row(device, dtype, width):
    for k, reference in enumerate(REFERENCES):
        compare(device, 8193 + k, width, dtype, reference, masked=k != 1)


def check_wide(given, options, out, grad):
    """Where a lane adds 64 entries in fp32, so that S is off by (3 m1 + 68) u; without a reference."""

    want = expected(given, options)
    p, x = want["p"], np.abs(want["x"])
    m1, m2 = (p * x).sum(1), 3 * (p * x * x).sum(1)
    s = (3 * m1 + 68) * U
    assert (np.abs(host(out.log_probs) - want["log_probs"]) <= s + U * np.abs(want["log_probs"])).all()
    entropy = (m2 + 72 * m1 + 72) * U
    assert (np.abs(host(out.entropy) - want["entropy"]) <= entropy + U * want["entropy"]).all()
    f = (host(options["weights"]) / options["normalizer"])[:, None]
    own = np.abs(want["own"])[:, None]
    own_off = s[:, None] * np.abs(host(given["advantages"]) * want["ratio"])[:, None] + 16 * U * own
    bracket = ENTROPY * (x + 2 * want["entropy"][:, None] + m1[:, None]) + own
    off = f * p * (bracket * ((3 * x + 40) * U + 3 * s[:, None]) + ENTROPY * entropy[:, None] + own_off)
    off[np.arange(len(s)), host(given["actions"])] += (f * own_off)[:, 0]
    target = want["grad"]
    bar = off + HALF_STEP[given["logits"].dtype] * (np.abs(target) + off) + TINY[given["logits"].dtype]
    assert (np.abs(host(grad) - target) <= bar).all()
    if "mask" in options:
        assert (host(grad)[~host(options["mask"])] == 0).all()


# 512 lanes of 32 and 64 entries, 1024 of 32 (fp32) and 64, and rows read again for each pass; over 512 rows.
@pytest.mark.parametrize("rows, width", [(520, 9001), (1030, 8200), (515, 16391), (513, 32771), (70, 33000), (70, 65536), (514, 65543)])
@pytest.mark.parametrize("dtype", DTYPES, ids=["fp32", "bf16", "fp16"])
def test_wide_rows_of_several_turns(device, dtype, rows, width):
    compare(device, rows, width, dtype, None, masked=rows % 2 == 0, count=8, check=check_wide)
    compare(device, rows, width, dtype, "logits", masked=rows % 2 == 1, count=8)


@pytest.mark.parametrize("rows, width, dtype", [(4096, 32768, torch.bfloat16), (4096, 16384, torch.float32)])
def test_a_loss_of_as_many_bytes_as_go_past_the_caches(device, rows, width, dtype):
    """512 MB of logits and gradient to the byte."""

    compare(device, rows, width, dtype, None, masked=False, count=8, check=check_wide)
