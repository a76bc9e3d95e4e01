"""Losses over a large vocabulary against their formulas in 64 bits.

Bounds, with u half a step of the 16-bit type (``finfo.eps / 2``) and e = 2^-23, twice the half step of 32 bits (room
for sums that truncate):
  logits     |dz| <= (D + 4) e sum_d |h_d w_d|, since the products of two 16-bit numbers are exact in 32
  loss       T^2 (2 s max|dz| + 16 e (1 + |lse| + |log p|)), the sums of V and K terms taken in 32 bits by trees and pieces
             of at most 256 terms
  G          u |G| for its rounding, and (2 s max|dz| + 16 e (1 + |lse|)) (q + p) for the logits; fp16 steps are 2^-25 of the
             largest |g T| at least
  gradients  sums of |dG| times the other factor, (terms) e of the sum of |G| times it, and u of the result's own rounding; in dW
             of the call that returns loss and gradients h times its row's factor is rounded to 16 bits, too:
             G (1 + a) h (1 + b) with |a|, |b| <= u is off by at most (u + u + u^2) |G h|; what comes down through autograd may be
             multiplied onto them once they are rounded, by at most u of the result again
"""
import math

import pytest
import torch

from supertoken_b200 import GPUBPETrainer, ops

pytestmark = pytest.mark.gpu
E32 = 2.0 ** -23


def make(B, L, D, V, K=0, dtype=torch.bfloat16, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    hidden = torch.randn(B, L, D, generator=g, device="cuda").to(dtype)
    weight = (torch.randn(V, D, generator=g, device="cuda") * spread / math.sqrt(D)).to(dtype)
    if not K:
        return hidden, weight, torch.randint(0, V, (B, L), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.randint(0, V, (B, L, K), generator=g, device="cuda", dtype=torch.int32)
    return hidden, weight, ids, torch.randn(B, L, K, generator=g, device="cuda") * 2


def formula(hidden, weight, ids, logits=None, valid=None, T=1.0, reduction="mean", grad=None):
    """Loss and gradients in 64 bits with the bounds above: {"loss", "gh", "gw"} and the same names with "_tol"."""
    dtype = hidden.dtype
    u = torch.finfo(dtype).eps / 2
    tiny = 2.0 ** -25 if dtype == torch.float16 else 2.0 ** -133
    shape, D = hidden.shape[:-1], hidden.shape[-1]
    V, n = weight.shape[0], math.prod(hidden.shape[:-1])
    live = torch.ones(n, dtype=torch.bool, device="cuda") if valid is None else valid.reshape(n) != 0
    if logits is None:
        ids, t = ids.reshape(n, 1).long(), torch.zeros(n, 1, dtype=torch.float64, device="cuda")
    else:
        ids, t = ids.reshape(n, -1).long(), logits.reshape(n, -1).double() / T
    t = t.masked_fill(ids < 0, -math.inf)
    live = live & (t > -math.inf).any(1)
    h = torch.where(live[:, None], hidden.detach().reshape(n, D).double(), 0.0)
    w, ids = weight.detach().double(), ids.clamp_min(0)
    z = h @ w.T / T
    dz = ((D + 4) * E32 * (h.abs() @ w.abs().T) / T).amax(1)
    lse = torch.logsumexp(z, 1)
    t = torch.where(live[:, None], t, 0.0)
    logp = torch.log_softmax(t, 1)
    p = logp.exp()
    logp = torch.where(p > 0, logp, 0.0)
    loss = T * T * (lse + (p * (logp - z.gather(1, ids))).sum(1))
    loss_tol = T * T * (2 * dz + 16 * E32 * (1 + lse.abs() + (p * logp.abs()).sum(1) + (p * z.gather(1, ids).abs()).sum(1)))
    loss, loss_tol = torch.where(live, loss, 0.0), torch.where(live, loss_tol, 0.0)
    rows = max(1, int(live.sum()))
    up = torch.ones((), dtype=torch.float64, device="cuda") if grad is None else torch.as_tensor(grad, device="cuda").double()
    up = up.expand(shape).reshape(n) if up.numel() != 1 else up.reshape(1).expand(n)
    if reduction == "mean":
        up = up / rows
    q = (z - lse[:, None]).exp()
    aim = torch.zeros_like(q).scatter_add_(1, ids, p)
    f = torch.where(live, up * T, 0.0)[:, None]
    G = (q - aim) * f
    dG = u * G.abs() + f.abs() * (q + aim) * (2 * dz + 16 * E32 * (1 + lse.abs()))[:, None] * (1 + u) + \
        tiny * f.abs().amax() * live[:, None]
    gh, gw = G @ w, G.T @ h
    gh_tol = dG @ w.abs() + (V + 4) * E32 * (G.abs() @ w.abs())
    gw_tol = (dG + (u + u * u) * G.abs()).T @ h.abs() + (n + 4) * E32 * (G.abs().T @ h.abs())
    out = {"gh": gh.view(*shape, D), "gw": gw,
           "gh_tol": (gh_tol + u * (gh.abs() + gh_tol) + tiny).view(*shape, D),
           "gw_tol": gw_tol + u * (gw.abs() + gw_tol) + tiny}
    if reduction == "none":
        out["loss"], out["loss_tol"] = loss.view(shape), loss_tol.view(shape)
    else:
        by = rows if reduction == "mean" else 1
        out["loss"] = loss.sum() / by
        out["loss_tol"] = (loss_tol.sum() + (n / 32 + 64) * E32 * loss.abs().sum()) / by
    return out


def near(got, want, name):
    x, y, tol = got.double(), want[name], want[name + "_tol"]
    assert x.shape == y.shape
    off = (x - y).abs()
    assert bool((off <= tol).all()), f"{name}: off by {float((off - tol).max()):.3g} more than {float(tol.max()):.3g}"


def check(hidden, weight, *args, valid=None, T=None, reduction="mean", grad=None):
    kd = len(args) == 2
    more = {"temperature": T or 1.0} if kd else {}
    want = formula(hidden, weight, *args, valid=valid, T=T or 1.0, reduction=reduction, grad=grad)
    loss_of, grads_of = (ops.vocab_distillation, ops.vocab_distillation_grads) if kd else \
        (ops.vocab_cross_entropy, ops.vocab_cross_entropy_grads)
    loss, gh, gw = grads_of(hidden, weight, *args, valid, grad, reduction=reduction, **more)
    assert loss.dtype == torch.float32 and gh.dtype == gw.dtype == hidden.dtype
    near(loss, want, "loss"), near(gh, want, "gh"), near(gw, want, "gw")
    near(loss_of(hidden, weight, *args, valid, reduction=reduction, **more), want, "loss")  # (sums about another reference)
    h, w = hidden.detach().requires_grad_(True), weight.detach().requires_grad_(True)
    auto = loss_of(h, w, *args, valid, reduction=reduction, **more)
    up = torch.ones_like(auto) if grad is None else torch.as_tensor(grad, device="cuda", dtype=torch.float32).expand_as(auto)
    ah, aw = torch.autograd.grad(auto, (h, w), up)
    for name in ("gh", "gw"):
        want[name + "_tol"] = want[name + "_tol"] * (1 + 2 ** -8) + torch.finfo(gh.dtype).eps / 2 * want[name].abs()
    near(auto.detach(), want, "loss"), near(ah, want, "gh"), near(aw, want, "gw")
    return loss, gh, gw


SIZES = [(1, 1, 1, 1), (1, 1, 64, 512), (1, 2, 7, 3), (3, 5, 40, 255), (1, 127, 64, 256), (2, 64, 65, 257),
         (1, 129, 128, 1256), (4, 97, 200, 1000), (3, 171, 136, 513), (2, 300, 770, 4099), (8, 64, 1024, 8256)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,L,D,V", SIZES)
def test_cross_entropy(B, L, D, V, dtype):
    hidden, weight, targets = make(B, L, D, V, dtype=dtype, seed=D + V)
    check(hidden, weight, targets, grad=512.0 if dtype == torch.float16 else None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K,T", [(1, 1.0), (2, 3.0), (33, 1.0), (50, 2.0), (256, 0.7)])
@pytest.mark.parametrize("B,L,D,V", [SIZES[0], SIZES[3], SIZES[7], SIZES[9]])
def test_distillation(B, L, D, V, K, T, dtype):
    args = make(B, L, D, V, K, dtype=dtype, seed=K)
    check(*args, T=T, grad=512.0 if dtype == torch.float16 else None)


@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
@pytest.mark.parametrize("K", [0, 20])
def test_reductions_and_what_comes_down_to_the_loss(reduction, K):
    args = make(3, 90, 96, 700, K)
    shape = (3, 90) if reduction == "none" else ()
    grad = torch.randn(shape, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    check(*args, reduction=reduction, grad=grad)
    check(*args, reduction=reduction, grad=-0.125)
    if reduction == "none":  # a gradient that is not contiguous, and the one that sum() sends down
        check(*args, reduction=reduction, grad=torch.randn(90, 3, device="cuda").t())
        h = args[0].requires_grad_(True)
        loss = (ops.vocab_distillation if K else ops.vocab_cross_entropy)(h, *args[1:], reduction="none")
        one, = torch.autograd.grad(loss.sum(), h)
        near(one, formula(*args, reduction="sum"), "gh")


@pytest.mark.parametrize("K", [0, 20])
@pytest.mark.parametrize("kind", ["ragged", "random", "one", "nothing", "negative"])
def test_rows_that_do_not_count(kind, K):
    B, L = 5, 83
    args = list(make(B, L, 72, 611, K))
    g = torch.Generator("cuda").manual_seed(3)
    valid = torch.rand(B, L, device="cuda", generator=g) < 0.6
    if kind == "ragged":
        valid = torch.arange(L, device="cuda") < torch.tensor([L, 0, 1, 40, 82], device="cuda")[:, None]
    elif kind in ("one", "nothing"):
        valid = torch.zeros(B, L, dtype=torch.bool, device="cuda")
        valid[3, 17] = kind == "one"
    if kind == "negative":  # padding shows in the ids alone
        at = valid if not K else valid[..., None]
        args[2] = torch.where(at, args[2], -1)
        want = check(*args)
    else:
        want = check(*args, valid=valid.to(torch.uint8))
    again = check(*args, valid=valid, reduction="none")
    assert bool((again[0][~valid] == 0).all()) and bool((want[1][~valid] == 0).all())
    if kind == "nothing":
        assert float(want[0]) == 0 and not bool(want[2].any())
    # what the other rows hold is not looked at
    args[0] = torch.where(valid[..., None], args[0], float("nan"))
    if K:
        args[3] = torch.where(valid[..., None], args[3], float("nan"))
    args[2] = torch.where(valid if not K else valid[..., None], args[2], 10 ** 9 if kind != "negative" else -7)
    more = {} if kind == "negative" else {"valid": valid}
    for x, y in zip((ops.vocab_distillation_grads if K else ops.vocab_cross_entropy_grads)(*args, **more), want):
        assert torch.equal(x, y)


def test_teachers_entries():
    hidden, weight, ids, logits = make(4, 30, 64, 500, 24)
    ids[0, :, 5:] = -1                       # cut lists
    ids[1, ::3] = -1                         # no list
    logits[2, :, ::2] = -math.inf            # entries without a share
    logits[2, 4] = -math.inf                 # all of them
    logits[3, :, 1] = 300.0                  # one that takes everything
    ids[3, :, 10:20] = ids[3, :, :1]         # the same id again and again
    ids[0, 0, :] = torch.arange(24, device="cuda") % 3 + 497
    logits[0, 1, :] = torch.finfo(torch.float32).min  # the lowest numbers still make a distribution
    for T in (1.0, 2.5):
        check(hidden, weight, ids, logits, T=T)
        check(hidden, weight, ids.long(), logits, T=T, reduction="none")
        wide = make(4, 30, 1040, 500)[:2]  # wide enough for an entry with most of the share to be summed once more
        check(*wide, ids, logits, T=T, reduction="none")
    order = torch.randperm(24, device="cuda")
    a = ops.vocab_distillation(hidden, weight, ids, logits, reduction="none")
    b = ops.vocab_distillation(hidden, weight, ids[..., order].contiguous(), logits[..., order].contiguous(), reduction="none")
    tol = formula(hidden, weight, ids, logits, reduction="none")["loss_tol"]
    assert bool(((a - b).abs() <= 2 * tol).all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_teachers_types(dtype):
    hidden, weight, ids, logits = make(2, 40, 64, 500, 24)
    check(hidden, weight, ids, logits.to(dtype), T=1.5)


def test_ids_outside_the_vocabulary_and_nan_show():
    hidden, weight, targets = make(2, 20, 64, 500)
    for bad in (500, 2 ** 31 - 1):
        targets[1, 3] = bad
        loss = ops.vocab_cross_entropy(hidden, weight, targets, reduction="none")
        assert loss.isnan().nonzero().tolist() == [[1, 3]]
        loss, gh, gw = ops.vocab_cross_entropy_grads(hidden, weight, targets)
        assert bool(loss.isnan()) and bool(gh[1, 3].isnan().all()) and not bool(gh[0].isnan().any()) and bool(gw.isnan().all())
    wide = targets.long()
    wide[1, 3] = 2 ** 32 + 5  # not 5
    assert bool(ops.vocab_cross_entropy(hidden, weight, wide).isnan())
    hidden, weight, ids, logits = make(2, 20, 64, 500, 9)
    ids[0, 2, 4], logits[1, 1, 1], logits[1, 2, 1] = 500, math.nan, math.inf
    loss = ops.vocab_distillation(hidden, weight, ids, logits, reduction="none")
    assert loss.isnan().nonzero().tolist() == [[0, 2], [1, 1], [1, 2]]
    hidden[0, 7, 3] = math.nan
    loss = ops.vocab_distillation(hidden, weight, ids, logits, reduction="none")
    assert loss.isnan().nonzero().tolist() == [[0, 2], [0, 7], [1, 1], [1, 2]]


def test_logits_of_minus_infinity_and_large_ones():
    hidden, weight, targets = make(2, 33, 64, 300)
    hidden[..., 0] = 1.0
    weight[100:, 0] = -math.inf
    targets.clamp_(max=99)
    loss = ops.vocab_cross_entropy(hidden, weight, targets, reduction="none")
    near(loss, formula(hidden, weight[:100], targets, reduction="none"), "loss")
    hidden, weight, targets = make(2, 33, 64, 300, spread=60.0)  # exp(z) overflows 32 bits
    check(hidden, weight, targets)
    assert float((hidden.float() @ weight.float().T).max()) > 100


@pytest.mark.parametrize("K", [0, 12])
def test_strides_and_alignment(K):
    """A batch shifted by one token, columns of a wider state, rows of a larger table that start anywhere, transposed batches."""
    B, L, D, V = 3, 50, 64, 400
    g = torch.Generator("cuda").manual_seed(7)
    state = torch.randn(B, L, D + 24, generator=g, device="cuda").bfloat16()
    table = torch.randn(V + 9, D + 3, generator=g, device="cuda").mul_(0.1).bfloat16()
    tokens = torch.randint(0, V, (B, L), generator=g, device="cuda", dtype=torch.int32)
    valid = (torch.rand(B, L, generator=g, device="cuda") < 0.8).to(torch.uint8)
    ids = torch.randint(0, V, (B, L, 2 * K), generator=g, device="cuda")
    logits = torch.randn(B, L, K + 5, generator=g, device="cuda")
    for h, w in ((state[..., :D], table[9:, :D]), (state[..., 3:D + 3], table[:V, 3:]), (state[..., 8:D], table[5:V + 5, :D - 8]),
                 (state[..., 8:9], table[:V, 1:2])):
        rest = (ids[:, 1:, K:], logits[:, 1:, 2:K + 2]) if K else (tokens[:, 1:],)
        check(h[:, :-1], w, *rest, valid=valid[:, 1:])
    turned = [x.transpose(0, 1) for x in ((state[..., :D], ids[..., :K], logits[..., :K]) if K else (state[..., :D], tokens))]
    check(turned[0], table[:V, :D], *turned[1:], valid=valid.t().bool())
    flat = [x.reshape(B * L, *x.shape[2:]) for x in ((state, ids, logits) if K else (state, tokens))]
    flat = [x[::2] for x in ([flat[0][:, :D], flat[1][:, :K], flat[2][:, :K]] if K else [flat[0][:, :D], flat[1]])]
    check(flat[0], table[:V, :D], *flat[1:])
    rest = (ids[..., :K], logits[..., :K]) if K else (tokens,)
    check(state[..., :D].contiguous(), table[:1, :D].expand(V, D), *rest)       # one row for all ids,
    check(state[..., :D].contiguous(), table[:, :8].as_strided((V, D), (8, 1)), *rest)  # rows that overlap
    one = state[:1, :1, :D].expand(B, L, D)  # one state for all rows
    check(one, table[:V, :D], *((ids[..., :K], logits[..., :K]) if K else (tokens,)))


def test_no_rows():
    for shape in ((0, 64), (0, 5, 64), (5, 0, 64)):
        h, w = torch.empty(shape, device="cuda", dtype=torch.bfloat16), make(1, 1, 64, 100)[1]
        t = torch.empty(shape[:-1], device="cuda", dtype=torch.int64)
        for r in ("none", "sum", "mean"):
            loss, gh, gw = ops.vocab_cross_entropy_grads(h, w, t, reduction=r)
            assert not bool(loss.any()) and gh.shape == h.shape and not bool(gw.any())
            assert loss.shape == ops.vocab_cross_entropy(h, w, t, reduction=r).shape == (shape[:-1] if r == "none" else ())


@pytest.mark.parametrize("K", [0, 16])
def test_gradients_against_differences(K):
    """(loss(h + d) - loss(h - d)) / 2 along one direction: off by a sixth of the third derivative, which a sum of exponents
    bounds by the cube of the logits' range along it."""
    hidden, weight, *rest = make(2, 37, 64, 333, K)
    hidden = hidden.float().clamp(-3.5, 3.5).mul(64).round().div(64).bfloat16()      # h +- d is exact in bf16
    want = formula(hidden, weight, *rest, reduction="sum")
    step = want["gh"].sign().bfloat16() / 64
    loss_of = ops.vocab_distillation if K else ops.vocab_cross_entropy
    grads_of = ops.vocab_distillation_grads if K else ops.vocab_cross_entropy_grads
    assert torch.equal((hidden + step).float(), hidden.float() + step.float())
    assert torch.equal((hidden - step).float(), hidden.float() - step.float())
    hi, lo = (loss_of(x, weight, *rest, reduction="sum").double() for x in (hidden + step, hidden - step))
    _, gh, _ = grads_of(hidden, weight, *rest, reduction="sum")
    along = (gh.double() * step.double()).sum()
    reach = (step.double().reshape(-1, 64) @ weight.double().T)
    cubes = ((reach.amax(1) - reach.amin(1)) ** 3).sum() / 6
    tol = cubes + 2 * want["loss_tol"] + (want["gh_tol"] * step.double().abs()).sum()
    assert abs(float((hi - lo) / 2 - along)) <= float(tol) < 0.1 * abs(float(along))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_backward_twice(dtype):
    """The second pass does not change what the first one gave."""
    hidden, weight, targets = make(2, 150, 72, 700, dtype=dtype)
    h, w = hidden.clone().requires_grad_(True), weight.clone().requires_grad_(True)
    loss = ops.vocab_cross_entropy(h, w, targets)
    want = formula(hidden, weight, targets)
    one = torch.autograd.grad(loss, (h, w), torch.tensor(1.0, device="cuda"), retain_graph=True)
    kept = [x.clone() for x in one]
    two = torch.autograd.grad(loss, (h, w), torch.tensor(4.0, device="cuda"))
    assert all(torch.equal(x, y) for x, y in zip(one, kept))
    for x, y in zip(one, two):
        near(x, want, "gh" if x.dim() == 3 else "gw"), near(y / 4, want, "gh" if x.dim() == 3 else "gw")


def test_only_the_wanted_gradient_is_made():
    hidden, weight, targets = make(2, 40, 64, 500)
    want = formula(hidden, weight, targets)
    for frozen in (0, 1):
        h, w = hidden.clone().requires_grad_(frozen != 0), weight.clone().requires_grad_(frozen != 1)
        ops.vocab_cross_entropy(h, w, targets).backward()
        if frozen:
            near(h.grad, want, "gh")
            assert w.grad is None
        else:
            near(w.grad, want, "gw")
            assert h.grad is None


def test_tied_embedding_takes_both_gradients():
    weight = make(1, 1, 64, 300)[1].requires_grad_(True)
    tokens = torch.randint(0, 300, (2, 21), device="cuda", generator=torch.Generator("cuda").manual_seed(2))
    ops.vocab_cross_entropy(weight[tokens[:, :-1]], weight, tokens[:, 1:]).backward()
    want = formula(weight.detach()[tokens[:, :-1]], weight, tokens[:, 1:])
    full = want["gw"].clone().index_put_((tokens[:, :-1].reshape(-1),), want["gh"].reshape(-1, 64), accumulate=True)
    tol = want["gw_tol"].clone().index_put_((tokens[:, :-1].reshape(-1),), want["gh_tol"].reshape(-1, 64), accumulate=True)
    # torch adds up to 40 rows of the embedding's gradient and the two gradients in 16 bits
    tol += 44 * 2.0 ** -8 * (full.abs() + tol + want["gw"].abs() + want["gh"].abs().sum((0, 1)))
    assert bool(((weight.grad.double() - full).abs() <= tol).all())


@pytest.mark.parametrize("K", [0, 40])
def test_same_inputs_same_bits(K):
    args = make(4, 200, 256, 5000, K)
    grads_of = ops.vocab_distillation_grads if K else ops.vocab_cross_entropy_grads
    first = grads_of(*args)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(grads_of(*args), first))


def test_other_stream_and_other_current_device():
    args = make(2, 100, 128, 3000)
    first = ops.vocab_cross_entropy_grads(*args)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            got.append(ops.vocab_cross_entropy_grads(*args))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, first))


def test_captured_and_replayed():
    """Two graphs, each with both losses, on inputs that change between replays, rows that count among them."""
    a, b = make(3, 70, 128, 2000), make(3, 70, 128, 2000, 30, seed=1)
    valid = torch.ones(3, 70, dtype=torch.uint8, device="cuda")
    scale = torch.ones((), device="cuda")
    h, w = a[0].clone().requires_grad_(True), a[1].clone().requires_grad_(True)
    eager = ops.vocab_cross_entropy(h, w, a[2])  # an eager graph of the same leaves stays alive
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = [*ops.vocab_cross_entropy_grads(h, w, a[2], valid, scale), *ops.vocab_distillation_grads(*b, valid, scale),
                   ops.vocab_cross_entropy(a[0], a[1], a[2], valid, reduction="none")]
        graphs.append((g, out))
    for k in range(3):
        valid.copy_(torch.rand(3, 70, device="cuda") < (0.9, 0.3, 0.0)[k])
        a[2].copy_(torch.randint(0, 2000, (3, 70), device="cuda"))
        b[3].mul_(1.1)
        with torch.no_grad():
            h.add_(0.25)
        scale.fill_(2.0 ** k)
        want = [*ops.vocab_cross_entropy_grads(h, w, a[2], valid, scale), *ops.vocab_distillation_grads(*b, valid, scale),
                ops.vocab_cross_entropy(a[0], a[1], a[2], valid, reduction="none")]
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert all(torch.equal(x, y) for x, y in zip(out, want))
    del eager


def test_autograd_refuses_a_capture():
    hidden, weight, targets = make(2, 20, 64, 500)
    hidden.requires_grad_(True)
    loss = ops.vocab_cross_entropy(hidden, weight, targets)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="vocab_cross_entropy_grads"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.vocab_cross_entropy(hidden, weight, targets)
    torch.cuda.synchronize()
    loss.backward()
    near(hidden.grad, formula(hidden, weight, targets), "gh")


def test_refusals():
    h, w, t = make(2, 8, 16, 50)
    _, _, ids, logits = make(2, 8, 16, 50, 4)
    ce, kd = ops.vocab_cross_entropy, ops.vocab_distillation
    for call, error in [
            (lambda: ce(h.cpu(), w, t), RuntimeError), (lambda: ce(h, w, t.cpu()), RuntimeError),
            (lambda: ce(h.float(), w.float(), t), TypeError), (lambda: ce(h, w.half(), t), TypeError),
            (lambda: ce(h, w, t.short()), TypeError), (lambda: ce(h, w, t, t), TypeError),
            (lambda: ce(h, w, t.float()), TypeError), (lambda: ce(h, w, None), TypeError),
            (lambda: ce(h[0, 0], w, t[0, 0]), ValueError), (lambda: ce(h, w[:, :8], t), ValueError),
            (lambda: ce(h, w[:0], t), ValueError), (lambda: ce(h[..., :0], w[:, :0], t), ValueError),
            (lambda: ce(h, w, t[:, 1:]), ValueError), (lambda: ce(h, w, t, t[:1].bool()), ValueError),
            (lambda: ce(h, w, t, reduction="max"), ValueError), (lambda: ce(h[..., ::2], w[:, ::2], t), ValueError),
            (lambda: ce(h, w.t().contiguous().t(), t), ValueError),
            (lambda: kd(h, w, ids, None), TypeError), (lambda: kd(h, w, ids, logits[..., :3]), ValueError),
            (lambda: kd(h, w, ids, logits.double()), TypeError), (lambda: kd(h, w, ids, logits, temperature=0.0), ValueError),
            (lambda: kd(h, w, ids, logits, temperature=math.nan), ValueError),
            (lambda: kd(h, w, ids, logits, temperature=math.inf), ValueError),
            (lambda: kd(h, w, ids, logits, temperature=-1.0), ValueError),
            (lambda: kd(h, w, ids, logits, temperature=1e-40), ValueError),
            (lambda: kd(h, w, ids[..., :0], logits[..., :0]), ValueError),
            (lambda: kd(h, w, *(x.repeat(1, 1, 65)[..., :257] for x in (ids, logits))), ValueError),
            (lambda: kd(h, w, ids[..., ::2], logits[..., ::2]), ValueError),
            (lambda: ops.vocab_cross_entropy_grads(h, w, t, None, torch.ones(2, device="cuda")), ValueError),
            (lambda: ops.vocab_cross_entropy_grads(h, w, t, None, torch.ones(2, 8, device="cuda")), ValueError),
            (lambda: ops.vocab_cross_entropy_grads(h, w, t, None, torch.ones((), device="cuda").half()), TypeError),
            (lambda: ops.vocab_cross_entropy_grads(h, w, t, None, torch.ones(()), reduction="none"), ValueError)]:
        with pytest.raises(error):
            call()


def test_a_vocabulary_is_trained_and_a_model_over_it():
    """As they are used together: merges are learned and applied to a padded batch by the batch operators, an output layer over
    the ids that result takes a few steps by cross entropy, and a smaller one learns from its top logits."""
    torch.manual_seed(0)
    text = torch.randint(97, 103, (6, 200), dtype=torch.int32)
    lengths = torch.tensor([200, 150, 3, 200, 90, 0], dtype=torch.int32)
    valid = (torch.arange(200) < lengths[:, None]).to(torch.uint8)
    trainer = GPUBPETrainer(base_vocab=256, merges=24, device="cuda:0")
    merges = trainer.fit([(text * valid, valid, lengths)], log_every=0)["merges"]
    tokens, valid, lengths = (text * valid).cuda(), valid.cuda(), lengths.cuda()
    for m, (a, b) in enumerate(merges):
        tokens, valid, lengths, _ = ops.apply_merge_once(tokens, valid, lengths, a, b, 256 + m)
    V = 256 + len(merges)
    state = torch.randn(V, 64, device="cuda").bfloat16()[tokens.long().clamp(0, V - 1)]
    weight = torch.zeros(V, 64, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    here = (state[:, :-1], weight, tokens[:, 1:], valid[:, 1:])
    for _ in range(3):
        loss = ops.vocab_cross_entropy(*here)
        want = formula(here[0], weight, here[2], valid=here[3])
        near(loss.detach(), want, "loss")
        gw, = torch.autograd.grad(loss, weight)
        near(gw, want, "gw")
        with torch.no_grad():
            weight -= gw
    logits, ids = (state[:, :-1].float() @ weight.detach().float().T).topk(16)
    small = torch.randn(64, 24, device="cuda").bfloat16()
    student = torch.zeros(V, 24, device="cuda", dtype=torch.bfloat16).requires_grad_(True)
    for _ in range(3):
        h = state[:, :-1] @ small
        loss = ops.vocab_distillation(h, student, ids, logits, valid[:, 1:], temperature=2.0)
        want = formula(h, student, ids, logits, valid=valid[:, 1:], T=2.0)
        near(loss.detach(), want, "loss")
        gw, = torch.autograd.grad(loss, student)
        near(gw, want, "gw")
        with torch.no_grad():
            student -= gw


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("K", [0, 5])
def test_more_rows_and_ids_than_are_held_at_a_time(K, dtype):
    """2 300 rows over 300 001 ids are two chunks of rows (or two pieces of the vocabulary); fewer rows than a chunk count, too."""
    args = make(1, 2300, 64, 300_001, K, dtype=dtype)
    check(*args, grad=64.0)
    check(*args, grad=64.0, reduction="none")
    valid = torch.arange(2300, device="cuda")[None] % 3 == 0
    check(*args, valid=valid, grad=64.0)


@pytest.mark.parametrize("K", [0, 7])
def test_rows_of_any_height(K):
    """Rows whose logits lie far above or below 0 beside ordinary ones: an offset along one column of hidden."""
    hidden, weight, *rest = make(3, 200, 64, 1000, K)
    weight[:, 0] = 1.0
    hidden[..., 0] = 0.0
    hidden[0, 17, 0], hidden[0, 18, 0], hidden[1, 150:, 0], hidden[2, :2, 0] = 90.0, -90.0, 250.0, -3000.0
    check(hidden, weight, *rest)
    check(hidden, weight, *rest, reduction="none")
    # as much of it as exponentials about a fixed reference are kept of
    hidden, weight, *rest = make(3, 900, 64, 10_000, K)
    weight[:, 0] = 1.0
    hidden[..., 0] = 0.0
    hidden[0, 17, 0], hidden[0, 18, 0], hidden[1, 850:, 0], hidden[2, :2, 0] = 90.0, -90.0, 250.0, -3000.0
    check(hidden, weight, *rest)
    check(hidden, weight, *rest, reduction="sum", grad=0.5)


def test_splits_of_the_depth():
    """Few tiles over a long vocabulary or many rows."""
    check(*make(1, 5, 64, 40_000))
    check(*make(2, 2500, 72, 130))
    check(*make(1, 300, 520, 20_000, 3))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,D,V", [(1, 8, 1), (1, 1024, 8256), (2, 64, 33), (3, 2000, 50_001), (4, 256, 9473), (8, 520, 20_011),
                                      (8, 2048, 700), (8, 2056, 700), (9, 512, 3000), (1, 16_384, 300), (5, 70, 999)])
def test_a_few_rows_are_scored(rows, D, V, dtype):
    hidden, weight, targets = make(1, rows, D, V, dtype=dtype, seed=rows + V)
    for reduction in ("none", "mean", "sum"):
        near(ops.vocab_cross_entropy(hidden, weight, targets, reduction=reduction), formula(hidden, weight, targets, reduction=reduction), "loss")
    valid = torch.arange(rows, device="cuda")[None] % 2 == 1
    hidden = torch.where(valid[..., None], hidden, float("nan"))
    want = formula(hidden, weight, targets, valid=valid)
    near(ops.vocab_cross_entropy(hidden, weight, targets, valid), want, "loss")
    near(ops.vocab_cross_entropy(hidden.transpose(0, 1), weight, targets.t().long(), valid.t()), want, "loss")
    each = ops.vocab_cross_entropy(hidden, weight, torch.where(valid, targets, -1), reduction="none")
    assert bool((each[~valid] == 0).all())
    if rows > 1:
        targets[0, 1] = V
        assert ops.vocab_cross_entropy(hidden, weight, targets, valid, reduction="none").isnan().nonzero().tolist() == [[0, 1]]


@pytest.mark.parametrize("N,V,D", [(300, 530_003, 4096), (2048, 1_100_003, 64)])
def test_offsets_beyond_31_bits(N, V, D):
    """More than 2^31 numbers in the weight and its gradient, or in what is held of the exponentials; checked by columns."""
    hidden, weight, targets = make(1, N, D, V)
    targets[0, -3:] = torch.tensor([V - 1, V - 2, 0], device="cuda")
    loss, gh, gw = ops.vocab_cross_entropy_grads(hidden, weight, targets, grad_loss=float(N))
    h, t = hidden[0].double(), targets[0].long()
    spans = [(v, min(v + 65536, V)) for v in range(0, V, 65536)]
    logits = lambda a, b: h @ weight[a:b].double().T  # noqa: E731
    dz = lambda a, b: (D + 4) * E32 * (h.abs() @ weight[a:b].double().abs().T)  # noqa: E731
    lse = torch.logsumexp(torch.stack([torch.logsumexp(logits(a, b), 1) for a, b in spans]), 0)
    off = torch.stack([dz(a, b).amax(1) for a, b in spans]).amax(0)
    zt = (h * weight[t].double()).sum(1)
    tol = 2 * off + 16 * E32 * (1 + lse.abs() + zt.abs())
    assert abs(float(loss) - float((lse - zt).mean())) <= float(tol.mean()) + (N / 32 + 64) * E32 * float((lse - zt).abs().mean())
    u, full, full_tol = 2.0 ** -8, torch.zeros_like(h), torch.zeros_like(h)
    for a, b in spans:
        w = weight[a:b].double()
        q = (logits(a, b) - lse[:, None]).exp()
        aim = torch.zeros_like(q)
        inside = (t >= a) & (t < b)
        aim[inside, t[inside] - a] = 1.0
        G = q - aim
        dG = u * G.abs() + (q + aim) * (2 * off + 16 * E32 * (1 + lse.abs()))[:, None] * (1 + u)
        full += G @ w
        full_tol += dG @ w.abs() + (V + 4) * E32 * (G.abs() @ w.abs())
        want = G.T @ h
        bound = (dG + (u + u * u) * G.abs()).T @ h.abs() + (N + 4) * E32 * (G.abs().T @ h.abs())
        assert bool(((gw[a:b].double() - want).abs() <= bound + u * (want.abs() + bound) + 2.0 ** -133).all())
    assert bool(((gh[0].double() - full).abs() <= full_tol + u * (full.abs() + full_tol) + 2.0 ** -133).all())
