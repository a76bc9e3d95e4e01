"""The losses over a large vocabulary where a logit, a teacher or a temperature is out of the ordinary, and how near their
results come in norms (``test_vocab_loss_gpu.py`` bounds them number by number)."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fw

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


def sure(rows, D, V, lean, dtype, K=0, twice=False):
    """Rows that point to their target: losses far below 1.  A teacher has most of its share there, ``twice``: in two entries."""
    hidden, weight, targets = make(1, rows, D, V, dtype=dtype)
    hidden = (0.3 * hidden.float() + 40 * lean * weight[targets.long()].float()).to(dtype)
    if not K:
        return hidden, weight, targets
    ids = torch.randint(0, V, (1, rows, K), device="cuda", generator=torch.Generator("cuda").manual_seed(0), dtype=torch.int32)
    logits = torch.full((1, rows, K), -9.0, device="cuda")
    ids[..., K // 2], logits[..., K // 2] = targets, 0.0
    if twice:
        ids[..., 0], logits[..., 0] = targets, -2.0
    return hidden, weight, ids, logits


def norms(hidden, weight, args, want, T, up):
    """Bounds of the loss of a row and of the gradients' 2-norms.
    A share q is off by 8 roundings of 32 bits of an exponent of |lse| / ln 2 + 1 at the most (the logit that is summed in 32 bits, its scaling, lse and its
    logarithm, the difference, exp2, and what lse is saved in), and that is what the target's dlogit, a difference of shares, is off by beside
    its own rounding.  Logits that are summed by the tensor cores are off by (D / 16 + 4) 2^-23 of the largest of a row: D / 16 steps, cut off at 32 bits, and
    that is what the other shares are off by, of themselves.  In both gradients up to three roundings to 16 bits (E, G or a H, the result) count,
    each of at most u / sqrt(3) in the 2-norm as errors are spread evenly over a step, together u."""
    u = torch.finfo(hidden.dtype).eps / 2
    n, D = hidden.shape[1], hidden.shape[2]
    h, w, ids = hidden[0].double(), weight.double(), args[0].reshape(n, -1).long()
    z = h @ w.T / T
    lse = torch.logsumexp(z, 1)
    off = 8 * 2.0 ** -24 * (lse.abs() / math.log(2) + 1)
    cut = (D / 16 + 4) * E32 * z.abs().amax(1)
    t = ids[:, -1] if len(args) == 1 else ids[:, ids.shape[1] // 2]
    rest = -torch.expm1(z.gather(1, t[:, None])[:, 0] - lse)  # shares of all but the target
    loss_tol = T * T * (off + cut * rest + 16 * E32)
    f = up.double() * T
    dG = f * (off + cut * rest)
    gh = (dG[:, None] * w[t]).norm()
    gw = torch.zeros_like(w).index_add_(0, t, dG[:, None] * h).norm()
    # (a teacher's other entries are not summed again)
    if len(args) == 2:
        gh, gw = 2 * gh, 2 * gw
    return loss_tol, u, float(gh / want["gh"].norm()), float(gw / want["gw"].norm())


def near_in_norm(got, want, u, extra, name):
    got, want = got.double().flatten(), want.flatten()
    off, along = float((got - want).norm() / want.norm()), float(got @ want / (want @ want)) - 1
    assert off <= u + extra, f"{name}: {off:.3g} off in the 2-norm, {u + extra:.3g} allowed"
    # a value rounds to 16 bits with all of its likes, but by less than half of u where it lies just below a power of two as a target's dlogit does
    assert abs(along) <= u / 2 + extra, f"{name}: too large by {along:.3g}, {u / 2 + extra:.3g} allowed"


@pytest.mark.parametrize("K,twice", [(0, False), (6, False), (6, True)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V,lean", [(300, 2048, 5000, 0.3), (300, 4096, 5000, 0.3), (300, 4096, 5000, 0.4), (1000, 2056, 30_000, 0.3)])
def test_rows_that_are_sure_of_their_target(rows, D, V, lean, dtype, K, twice):
    """Losses and dlogits are small differences there, for which the target's logit is summed in 32 bits, in every way to the gradients."""
    hidden, weight, *args = sure(rows, D, V, lean, dtype, K, twice)
    loss_of, grads_of = (ops.vocab_distillation, ops.vocab_distillation_grads) if K else (ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads)
    for reduction, up in (("mean", torch.full((rows,), 4096.0 / rows, device="cuda")),
                          ("none", torch.linspace(256.0, 4096.0, rows, device="cuda"))):
        grad = 4096.0 if reduction == "mean" else up[None]
        want = formula(hidden, weight, *args, reduction=reduction, grad=grad)
        each = formula(hidden, weight, *args, reduction="none")["loss"][0]
        loss_tol, u, gh_extra, gw_extra = norms(hidden, weight, args, want, 1.0, up)
        loss, gh, gw = grads_of(hidden, weight, *args, None, grad, reduction=reduction)
        h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        auto = loss_of(h, w, *args, reduction=reduction)
        ah, aw = torch.autograd.grad(auto, (h, w), torch.as_tensor(grad, device="cuda").expand_as(auto))
        for x in (loss, auto.detach(), loss_of(hidden, weight, *args, reduction=reduction)):
            if reduction == "none":
                assert bool(((x[0].double() - each).abs() <= loss_tol).all())
            else:
                assert abs(float(x) - float(each.mean())) <= float(loss_tol.mean()) + 64 * E32 * float(each.abs().mean())
        for name, x in (("gh", gh), ("gh", ah), ("gw", gw), ("gw", aw)):
            near_in_norm(x, want[name], u, gh_extra if name == "gh" else gw_extra, f"{name}, {reduction}")


@pytest.mark.parametrize("K", [0, 3])
@pytest.mark.parametrize("far", [0.0, 200.0])  # (a row beside it that has the tile made again)
@pytest.mark.parametrize("rows,V", BOTH_WAYS)
def test_a_logit_of_plus_infinity(rows, V, far, K):
    """There are no shares then: loss, the row's gradient and the weight's are NaN by every call, whichever the target is."""
    hidden, weight, *rest = make(1, rows, 64, V, K)
    hidden[..., 0], weight[:, 0] = 0.0, -1.0
    hidden[0, 5, 0], hidden[0, 9, 0], weight[V // 2, 0] = math.inf, far, 1.0
    loss_of, grads_of = (ops.vocab_distillation, ops.vocab_distillation_grads) if K else (ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads)
    for target in (V // 2, V // 2 + 1):
        rest[0][0, 5] = target
        loss, gh, gw = grads_of(hidden, weight, *rest, reduction="none")
        assert loss.isnan().nonzero().tolist() == [[0, 5]] and bool(gh[0, 5].isnan().all()) and bool(gw.isnan().all())
        assert not bool(gh[0, :5].isnan().any()) and not bool(gh[0, 6:].isnan().any())
        assert loss_of(hidden, weight, *rest, reduction="none").isnan().nonzero().tolist() == [[0, 5]]
        h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        for reduction in ("none", "mean"):
            ah, aw = torch.autograd.grad(loss_of(h, w, *rest, reduction=reduction).sum(), (h, w))
            assert ah[0].isnan().any(1).nonzero().tolist() == [[5]] and bool(ah[0, 5].isnan().all()) and bool(aw.isnan().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [0, 3])
@pytest.mark.parametrize("rows,V", BOTH_WAYS + [(256, 300)])
def test_ids_that_the_weight_rules_out(rows, V, K, dtype):
    """Logits of -inf by way of the weight: those ids' rows of its gradient are 0, the others as if they were not there."""
    hidden, weight, *rest = make(1, rows, 64, V, K, dtype=dtype)
    hidden[..., 0] = 1.0
    weight[V - 50:, 0] = -math.inf
    rest[0].clamp_(max=V - 51)
    want = formula(hidden, weight[:V - 50], *rest, reduction="sum", grad=64.0)
    loss_of, grads_of = (ops.vocab_distillation, ops.vocab_distillation_grads) if K else (ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads)
    loss, _, gw = grads_of(hidden, weight, *rest, None, 64.0, reduction="sum")
    near(loss, want, "loss"), near(gw[:V - 50], want, "gw")
    w = weight.clone().requires_grad_(True)
    aw, = torch.autograd.grad(loss_of(hidden, w, *rest, reduction="none").sum(), w, torch.tensor(64.0, device="cuda"))
    near(aw[:V - 50], want, "gw")
    assert not bool(gw[V - 50:].any()) and not bool(aw[V - 50:].any())


@pytest.mark.parametrize("top,low", [(-66.0, -87.5), (-60.0, -80.0), (-56.0, -76.0), (-55.0, -75.0), (0.0, -20.0), (66.0, 46.0), (68.0, 48.0)])
def test_small_shares_of_many_ids(top, low):
    """One id far above 300 000 others, which together are a small part of the row wherever its logits lie.  One product a logit, exact in 32
    bits; lse is off by 8 roundings of its exponent at the most, and by those of its sum: at most 128 columns of a part to the sum with the large one in
    it, two at a time and four sums at the end, less than 70 additions, then every 32nd of 2 344 or 4 688 parts, 147 at most, and 10 to
    bring those sums together; 227 times half a step of a sum of 1 to 2, 2^-24.  Gradients: three roundings to 16 bits and that."""
    V, rows = 300_001, 100
    hidden = torch.zeros(1, rows, 64, device="cuda", dtype=torch.bfloat16)
    weight = torch.zeros(V, 64, device="cuda", dtype=torch.bfloat16)
    hidden[..., 0], weight[:, 0], weight[77, 0] = 1.0, low, top
    targets = torch.full((1, rows), 77, device="cuda")
    rest = (V - 1) * math.exp(low - top)
    off = 8 * 2.0 ** -24 * (abs(top) / math.log(2) + 1) + 227 * 2.0 ** -24
    loss, gh, gw = ops.vocab_cross_entropy_grads(hidden, weight, targets)
    for x in (loss, ops.vocab_cross_entropy(hidden, weight, targets)):
        assert abs(float(x) - math.log1p(rest)) <= off
    q = math.exp(low - top) / (1 + rest)
    others = torch.cat([gw[:77, 0], gw[78:, 0]]).double() / q - 1
    assert float(others.abs().max()) <= 3.1 * 2.0 ** -8 + 2 * off


@pytest.mark.parametrize("V", [11, 1000])
@pytest.mark.parametrize("rows", [300, 8192, 1 << 20])
def test_the_mean_of_many_equal_losses(rows, V):
    """Logits of 0: every row's loss is log V by four roundings of 32 bits at the most (log2 of the sum, its product with ln 2, ln 2 itself, the difference
    to the target's 0), and so is their mean, with one rounding more."""
    hidden = torch.zeros(rows, 8, device="cuda", dtype=torch.bfloat16)
    weight, targets = torch.zeros(V, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(rows, device="cuda", dtype=torch.int32)
    for reduction, by in (("mean", 1), ("sum", rows)):
        for loss in (ops.vocab_cross_entropy(hidden, weight, targets, reduction=reduction),
                     ops.vocab_cross_entropy_grads(hidden, weight, targets, reduction=reduction)[0]):
            assert abs(float(loss) / by / math.log(V) - 1) <= 5 * 2.0 ** -24


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [1.0, 2.0 ** 15, 2.0 ** 16])
def test_nothing_comes_down_to_the_loss(T, dtype):
    hidden, weight, ids, logits = make(2, 70, 64, 500, 4, dtype=dtype)
    for reduction, grad in (("none", torch.zeros(2, 70, device="cuda")), ("sum", 0.0), ("mean", 0.0)):
        loss, gh, gw = ops.vocab_distillation_grads(hidden, weight, ids, logits, None, grad, temperature=T, reduction=reduction)
        near(loss, formula(hidden, weight, ids, logits, T=T, reduction=reduction), "loss")
        assert bool((gh == 0).all()) and bool((gw == 0).all())
        h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        auto = ops.vocab_distillation(h, w, ids, logits, temperature=T, reduction=reduction)
        assert all(bool((x == 0).all()) for x in torch.autograd.grad(auto, (h, w), torch.zeros_like(auto)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("T", [2.0 ** -16, 2.0 ** -10, 2.0 ** 16])
def test_the_range_of_temperatures(T, dtype):
    args = make(2, 70, 64, 500, 4, dtype=dtype)
    for reduction in ("none", "mean"):
        want = formula(*args, T=T, reduction=reduction)
        out = ops.vocab_distillation_grads(*args, temperature=T, reduction=reduction)
        for name, x in zip(("loss", "gh", "gw"), out):
            over = want[name].abs() > torch.finfo(x.dtype).max  # (65 536 times what a gradient is at a temperature of 1, in fp16: rounds to infinity)
            assert bool((x[over] == want[name][over].sign() * math.inf).all())
            want[name + "_tol"] = torch.where(over, math.inf, want[name + "_tol"])
            near(torch.where(over, 0.0, x), want, name)
    empty = [x[:, :0] for x in (args[0], args[2], args[3])]
    for t in (2.0 ** -17, 1e-10, 2.0 ** 17, 1e20):
        for h, ids, logits in ((args[0], *args[2:]), empty):
            with pytest.raises(ValueError, match="temperature"):
                ops.vocab_distillation(h, args[1], ids, logits, temperature=t, reduction="none")
            with pytest.raises(ValueError, match="temperature"):
                ops.vocab_distillation_grads(h, args[1], ids, logits, temperature=t, reduction="none")


@pytest.mark.parametrize("K", [0, 4])
def test_forward_mode_is_refused(K):
    """A tangent is not dropped: by the losses, by the calls for gradients, and on its way down to a loss."""
    args = make(2, 20, 64, 500, K)
    loss_of, grads_of = (ops.vocab_distillation, ops.vocab_distillation_grads) if K else (ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads)
    h = args[0].clone().requires_grad_(True)
    eager = {r: loss_of(h, *args[1:], reduction=r) for r in ("sum", "none")}
    with fw.dual_level():
        for which in (0, 1, 3) if K else (0, 1):
            dual = list(args)
            dual[which] = fw.make_dual(args[which], torch.ones_like(args[which]))
            for call in (loss_of, grads_of):
                with pytest.raises(RuntimeError, match="forward-mode"):
                    call(*dual)
        for loss in eager.values():
            up = fw.make_dual(torch.ones_like(loss), torch.ones_like(loss))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(loss, h, up, retain_graph=True)
            with pytest.raises(RuntimeError, match="forward-mode"):
                grads_of(*args, None, up, reduction="sum" if loss.dim() == 0 else "none")
        plain = loss_of(*args)  # nothing has a tangent
    assert torch.equal(plain, loss_of(*args))
    for reduction, loss in eager.items():  # as good as before the refusals
        near(torch.autograd.grad(loss.sum(), h)[0], formula(*args, reduction=reduction), "gh")


def test_a_teacher_that_wants_a_gradient_is_refused():
    hidden, weight, ids, logits = make(2, 20, 64, 500, 4)
    plain = ops.vocab_distillation(hidden, weight, ids, logits)
    logits.requires_grad_(True)
    for h in (hidden, hidden.clone().requires_grad_(True)):
        with pytest.raises(RuntimeError, match="detach"):
            ops.vocab_distillation(h, weight, ids, logits)
    assert torch.equal(ops.vocab_distillation(hidden, weight, ids, logits.detach()), plain)
    with torch.no_grad():
        assert torch.equal(ops.vocab_distillation(hidden, weight, ids, logits), plain)
    assert ops.vocab_distillation_grads(hidden, weight, ids, logits)[1].shape == hidden.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("frozen", [0, 1])
def test_one_gradient_of_more_than_is_held_at_a_time(frozen, dtype):
    """Two chunks of rows or two pieces of the vocabulary, one gradient wanted."""
    hidden, weight, targets = make(1, 2300, 64, 300_001, dtype=dtype)
    for reduction in ("mean", "none"):
        want = formula(hidden, weight, targets, reduction=reduction, grad=64.0)
        for name in ("gh_tol", "gw_tol"):  # what comes down is multiplied onto them once they are rounded
            want[name] = want[name] * (1 + 2 ** -8) + torch.finfo(dtype).eps / 2 * want[name[:2]].abs()
        h, w = hidden.clone().requires_grad_(frozen == 1), weight.clone().requires_grad_(frozen == 0)
        loss = ops.vocab_cross_entropy(h, w, targets, reduction=reduction)
        near(loss.detach(), want, "loss")
        got, = torch.autograd.grad(loss, h if frozen else w, torch.tensor(64.0, device="cuda").expand_as(loss))
        near(got, want, "gh" if frozen else "gw")


@pytest.mark.parametrize("K", [0, 5])
def test_more_rows_are_scored_than_are_held_at_a_time(K):
    """Two chunks of rows; some of both by their formula, and their sum."""
    rows, V = 9000, 1_000_003
    args = list(make(1, rows, 8, V, K))
    some = torch.tensor([0, 1, 255, 8191, 8447, 8448, 8449, 8703, 8704, 8999], device="cuda")
    loss_of = ops.vocab_distillation if K else ops.vocab_cross_entropy
    each = loss_of(*args, reduction="none")
    for at in some:
        one = [args[0][:, at:at + 1], args[1], *(x[:, at:at + 1] for x in args[2:])]
        near(each[:, at:at + 1], formula(*one, reduction="none"), "loss")
    mean = float(each.double().mean())
    assert abs(float(loss_of(*args)) / mean - 1) <= 2.0 ** -24
    few = torch.arange(rows, device="cuda")[None] % 3 == 0  # fewer than a chunk count
    kept = loss_of(*args, few, reduction="none")
    assert bool((kept[~few] == 0).all())
    # (the rows have other places in their tiles, which changes no row's sums)
    assert torch.equal(kept[few], each[few])
    assert abs(float(loss_of(*args, few, reduction="sum")) / float(kept.double().sum()) - 1) <= 2.0 ** -24


def loss_bound(hidden, weight, args, T=1.0):
    """Per row: the bounds of ``norms`` for any row, that is, cut sums of the tensor cores in the target's logit and in lse, and 16 e (1 + |log p|) for a
    teacher's shares.  About 1e-5 of the loss, where the sum of |h w| that bounds any order of the terms allows a thousand times as much."""
    n, D = math.prod(hidden.shape[:-1]), hidden.shape[-1]
    z = hidden.reshape(n, D).double() @ weight.double().T / T
    bound = 8 * 2.0 ** -24 * (torch.logsumexp(z, 1).abs() / math.log(2) + 1) + 2 * (D / 16 + 4) * E32 * z.abs().amax(1) + 16 * E32
    if len(args) == 2:
        logp = torch.log_softmax(args[1].reshape(n, -1).double() / T, 1)
        bound = bound + 16 * E32 * (logp.exp() * logp.abs()).sum(1)
    return T * T * bound


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,L,D,V,K,T", [(2, 300, 770, 4099, 0, 1.0), (8, 64, 1024, 8256, 0, 1.0), (3, 171, 136, 513, 7, 1.0), (1, 300, 520, 20_000, 3, 2.0),
                                         (3, 900, 64, 10_000, 0, 1.0), (1, 1000, 1032, 30_000, 7, 1.5), (1, 1000, 771, 30_000, 0, 1.0)])
def test_how_near_in_norms(B, L, D, V, K, T, dtype):
    """Losses row by row at about 1e-5 of them, gradients at what three roundings to 16 bits leave, and no factor on them."""
    hidden, weight, *args = make(B, L, D, V, K, dtype=dtype)
    kd = {"temperature": T} if K else {}
    loss_of, grads_of = (ops.vocab_distillation, ops.vocab_distillation_grads) if K else (ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads)
    bound, u = loss_bound(hidden, weight, args, T), torch.finfo(dtype).eps / 2
    up = torch.linspace(1024.0, 4096.0, B * L, device="cuda").view(B, L)
    for reduction, grad in (("mean", 4096.0), ("none", up)):
        want = formula(hidden, weight, *args, T=T, reduction=reduction, grad=grad)
        each = formula(hidden, weight, *args, T=T, reduction="none")["loss"].flatten()
        loss, gh, gw = grads_of(hidden, weight, *args, None, grad, reduction=reduction, **kd)
        h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
        auto = loss_of(h, w, *args, reduction=reduction, **kd)
        ah, aw = torch.autograd.grad(auto, (h, w), torch.as_tensor(grad, device="cuda").expand_as(auto))
        for x in (loss, auto.detach(), loss_of(hidden, weight, *args, reduction=reduction, **kd)):
            if reduction == "none":
                assert bool(((x.flatten().double() - each).abs() <= bound).all())
            else:
                assert abs(float(x) - float(each.mean())) <= float(bound.mean())
        for name, x in (("gh", gh), ("gh", ah), ("gw", gw), ("gw", aw)):
            near_in_norm(x, want[name], u, 0.0, f"{name}, {reduction}")


@pytest.mark.parametrize("K", [0, 7])
@pytest.mark.parametrize("D", [770, 1032])
def test_large_steps_with_rows_of_any_height(D, K):
    """As much of E as has a fixed reference, at widths whose targets are summed again: rows above and below it that are made again, a teacher that is
    sure, rows that do not count between them."""
    hidden, weight, *args = make(1, 1000, D, 30_000, K)
    weight[:, 0], hidden[..., 0] = 1.0, 0.0
    for at, height in ((17, 90.0), (18, -90.0), (300, 70.0), (301, -70.0), (302, -50.0), (700, 200.0), (999, -300.0)):
        hidden[0, at, 0] = height
    if K:
        args[1][0, ::2, 3] = 9.0
    valid = torch.arange(1000, device="cuda")[None] % 5 != 2
    valid[0, 512:768] &= torch.arange(256, device="cuda") < 100
    hidden = torch.where(valid[..., None], hidden, math.nan)
    clean = torch.where(valid[..., None], hidden, 0.0)
    kd = {"temperature": 1.5} if K else {}
    grads_of = ops.vocab_distillation_grads if K else ops.vocab_cross_entropy_grads
    bound = torch.where(valid[0], loss_bound(clean, weight, args, 1.5 if K else 1.0), 0.0)
    for reduction in ("mean", "none"):
        want = formula(clean, weight, *args, valid=valid, T=1.5 if K else 1.0, reduction=reduction, grad=64.0)
        loss, gh, gw = grads_of(hidden, weight, *args, valid, 64.0, reduction=reduction, **kd)
        near(loss, want, "loss"), near(gh, want, "gh"), near(gw, want, "gw")
        assert bool((gh[~valid] == 0).all())
        if reduction == "none":
            assert bool(((loss[0].double() - want["loss"][0]).abs() <= bound).all())
        # (the column that the heights go through cancels in dH and is made of a few rows in dW)
        near_in_norm(gh[..., 1:], want["gh"][..., 1:], 2.0 ** -8, 0.0, "gh"), near_in_norm(gw[:, 1:], want["gw"][:, 1:], 2.0 ** -8, 0.0, "gw")
    args[0][0, 18 if not K else slice(18, 19)] = 30_000  # an id outside, in a row that is made again
    loss, gh, gw = grads_of(hidden, weight, *args, valid, reduction="none", **kd)
    assert loss.isnan().nonzero().tolist() == [[0, 18]] and bool(gh[0, 18].isnan().all()) and bool(gw.isnan().all())
    assert not bool(gh[0, :18].isnan().any()) and not bool(gh[0, 19:].isnan().any())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [0, 4])
@pytest.mark.parametrize("D", [1024, 4096])
@pytest.mark.parametrize("offset", [20.0, -20.0])
def test_logits_with_an_offset_in_common(offset, D, K, dtype):
    """The target's logit is not summed once more at the cost of the others'.  Sums of 16 to 32 are cut off by half a step of 2^-19 on average in each of D / 16
    steps; what the target was cut by, of itself, times a mean of normally distributed logits that is off by at most 1 / 2, and by the target's own
    logit, 1 on average, leaves that by 1.5 / 20; and the roundings of ``norms``.  A teacher's entries but the one with 0.51 of the share are off by
    as much as the target's own logit is, 1 / 20 of the cut."""
    hidden, weight, *args = make(1, 500, D, 8000, K, dtype=dtype)
    weight[:, 0], hidden[..., 0] = 1.0, offset
    if K:
        args[1][:] = torch.tensor([0.18, 0.51, 0.16, 0.15], device="cuda").log()
    loss_of, grads_of = (ops.vocab_distillation, ops.vocab_distillation_grads) if K else (ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads)
    want = formula(hidden, weight, *args, reduction="none")
    left = D / 16 * 2.0 ** -20 * (1.5 + (0.49 if K else 0.0)) / 20
    off = float(8 * 2.0 ** -24 * (torch.logsumexp(hidden[0].double() @ weight.double().T, 1).abs() / math.log(2) + 1).mean())
    for loss in (loss_of(hidden, weight, *args, reduction="none"), grads_of(hidden, weight, *args, reduction="none")[0]):
        assert abs(float((loss.double() - want["loss"]).mean())) <= left + off


@pytest.mark.parametrize("down", [1.0, 1e-3, 1e-5, 1e-6])
def test_rows_of_small_weight_in_half_precision(down):
    """Without a reduction fp16 dlogits have the scale of the largest |grad_loss|, 16376.  In a row's gradient, of itself: its target's dlogit is off by u at the
    most, everything else by roundings of u / sqrt(3) in the 2-norm, together less than 2 u; below 2^-14 all dlogits are rounded to 2^-24, that is
    2^-25 / sqrt(3) each in the 2-norm, and so are the results; a row of them by half as much again at the most."""
    rows, D, V = 300, 256, 3000
    hidden, weight, targets = make(1, rows, D, V, dtype=torch.float16)
    up = torch.full((1, rows), 65536.0 * down, device="cuda")
    up[0, 0] = 65536.0
    want = formula(hidden, weight, targets, reduction="none", grad=up)["gh"][0]
    size, u = want.norm(dim=1), 2.0 ** -11
    coarse = 2.0 ** -25 / math.sqrt(3) * (65536 / 16376 * float(weight.double().norm()) + math.sqrt(D))
    h = hidden.clone().requires_grad_(True)
    auto, = torch.autograd.grad(ops.vocab_cross_entropy(h, weight, targets, reduction="none"), h, up)
    for gh in (ops.vocab_cross_entropy_grads(hidden, weight, targets, None, up, reduction="none")[1], auto):
        assert bool(((gh[0].double() - want).norm(dim=1) <= 2 * u * size + 1.5 * coarse).all())


@pytest.mark.parametrize("D", [770, 1024])
def test_a_targets_dlogit_is_not_rounded_on_large_steps(D):
    """Cross entropy in bf16 with more than 48 MB of E: the row's factor takes back what its target's entry lost.  Numbers with mantissas that are spread evenly
    over their logarithm round by 0.425 u in the 2-norm (the root of a third of the mean of 1 / m^2); dH has the result's own rounding, dW that and a H's, and
    a tenth more is left to the other ids' shares, whose rows of the weight hardly add up."""
    hidden, weight, targets = make(1, 1000, D, 30_000)
    want = formula(hidden, weight, targets)
    _, gh, gw = ops.vocab_cross_entropy_grads(hidden, weight, targets)
    one = 1.1 * 0.425 * 2.0 ** -8
    assert float((gh.double() - want["gh"]).norm() / want["gh"].norm()) <= one
    assert float((gw.double() - want["gw"]).norm() / want["gw"].norm()) <= math.sqrt(2) * one
