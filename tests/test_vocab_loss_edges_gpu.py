"""The losses over a large vocabulary where a logit, a teacher or a temperature is out of the ordinary, and how near their
results come in norms (``test_vocab_loss_gpu.py`` bounds them number by number)."""
import math

import pytest
import torch

from supertoken_b200 import ops
from test_vocab_loss_gpu import E32, formula, make, near

pytestmark = pytest.mark.gpu

# (rows, vocabulary) of the two ways that a bf16 call for loss and gradients goes: E about each part's maximum, and (more than 48 MB
# of it) about a fixed reference
BOTH_WAYS = [(40, 300), (900, 32_000)]


@pytest.mark.parametrize("K", [0, 3])
@pytest.mark.parametrize("D", [64, 1024])
@pytest.mark.parametrize("rows,V", BOTH_WAYS)
def test_a_target_of_minus_infinity(rows, V, D, K):
    """Its loss is +inf; shares are those of the other ids, so the row's gradients are as finite as any."""
    hidden, weight, targets = make(1, rows, D, V)
    hidden[..., 0] = 1.0
    weight[V - 50:, 0] = -math.inf
    targets.clamp_(max=V - 51)
    targets[0, 7] = V - 20
    if K:  # more than half of the share, as that is summed once more
        ids, logits = targets[..., None].repeat(1, 1, K), torch.full((1, rows, K), -2.0, device="cuda")
        ids[..., 1:], logits[..., 0] = 5, 0.0
        rest, loss_of, grads_of = (ids, logits), ops.vocab_distillation, ops.vocab_distillation_grads
    else:
        rest, loss_of, grads_of = (targets,), ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads
    others = torch.arange(rows, device="cuda")[None] != 7
    want = formula(hidden, weight[:V - 50], rest[0].clamp(max=V - 51), *rest[1:], valid=others, reduction="none")
    for loss in (loss_of(hidden, weight, *rest, reduction="none"), grads_of(hidden, weight, *rest, reduction="none")[0]):
        assert float(loss[0, 7]) == math.inf
        near(torch.where(others, loss, 0.0), want, "loss")
    gw = grads_of(hidden, weight, *rest, reduction="none")[2]
    assert not bool(gw[:V - 50].isnan().any())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [0.01, 0.7, 1.0, 2.5])
def test_a_teachers_lowest_and_largest_numbers(T, dtype):
    """A logit above -inf is an entry, whatever the temperature: rows of the type's lowest and largest numbers are uniform."""
    hidden, weight, ids, logits = make(2, 40, 64, 500, 40)
    logits = logits.to(dtype)
    low, high = torch.finfo(dtype).min, torch.finfo(dtype).max
    logits[0, 1], logits[0, 2], logits[0, 3], logits[0, 4, 1:] = low, high, low, low
    logits[0, 3, 5], logits[0, 5, ::2], logits[0, 6, 1::2] = high, -math.inf, high
    want = formula(hidden, weight, ids, logits, T=T, reduction="none")
    assert not bool(want["loss"].isnan().any())
    loss, gh, gw = ops.vocab_distillation_grads(hidden, weight, ids, logits, temperature=T, reduction="none")
    near(loss, want, "loss"), near(gh, want, "gh"), near(gw, want, "gw")
    mean = ops.vocab_distillation(hidden, weight, ids, logits, temperature=T)
    near(mean, formula(hidden, weight, ids, logits, T=T), "loss")
