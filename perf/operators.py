"""Losses over a large vocabulary: cross entropy and distillation from a teacher's top logits, at the output layer.

``hidden[B, L, D]`` times ``weight[V, D]`` are the logits of a padded batch of token ids, over a vocabulary of
``base_vocab + merges`` ids (1 256, 8 256, 32 256 and 50 256 ids are 1 000 to 50 000 merges over bytes; one more where an
end-of-text id is added) or one that fills 16 bits.

Kinds of work
  score     the loss of every token and nothing else: comparing vocabularies or models on held-out text
  grads     loss and both gradients by the explicit call, as a captured training step makes it
  autograd  the same through ``torch.autograd``

``loss`` is "ce" (targets are token ids) or "kd" (the teacher's ids and logits, K a row).
"""
from __future__ import annotations

import math

import torch

own = False
DEVICE = "cuda:0"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def listed():
    return [
        # one generated token is scored: fixed costs
        {"name": "score one token", "loss": "ce", "kind": "score", "rows": 1, "width": 1, "dim": 1024, "vocab": 8256,
         "k": 1, "type": "bf16", "ragged": False, "temperature": 1.0},
        # a padded batch of held-out documents under a 32 000-merge vocabulary
        {"name": "score ragged 16x512", "loss": "ce", "kind": "score", "rows": 16, "width": 512, "dim": 1024,
         "vocab": 32256, "k": 1, "type": "bf16", "ragged": True, "temperature": 1.0},
        # a small model in a test or a notebook: the 1 000-merge vocabulary
        {"name": "step small 8x256", "loss": "ce", "kind": "grads", "rows": 8, "width": 256, "dim": 512, "vocab": 1256,
         "k": 1, "type": "bf16", "ragged": True, "temperature": 1.0},
        # an ordinary step of a 1 to 2 billion parameter model, shifted targets, through autograd
        {"name": "step 4x2047", "loss": "ce", "kind": "autograd", "rows": 4, "width": 2047, "dim": 2048, "vocab": 32256,
         "k": 1, "type": "bf16", "ragged": False, "temperature": 1.0},
        # half precision with a loss scale, ragged documents, 50 000 merges and an end-of-text id
        {"name": "step fp16 16x511", "loss": "ce", "kind": "grads", "rows": 16, "width": 511, "dim": 1024,
         "vocab": 50257, "k": 1, "type": "fp16", "ragged": True, "temperature": 1.0},
        # sizes that no alignment fits
        {"name": "step odd 5x333", "loss": "ce", "kind": "grads", "rows": 5, "width": 333, "dim": 770, "vocab": 10007,
         "k": 1, "type": "bf16", "ragged": True, "temperature": 1.0},
        # the largest output layer: a 7 billion parameter model's width over a vocabulary that fills 16 bits
        {"name": "step 4x2048 largest", "loss": "ce", "kind": "grads", "rows": 4, "width": 2048, "dim": 4096,
         "vocab": 65536, "k": 1, "type": "bf16", "ragged": False, "temperature": 1.0},
        # distillation: two short rows
        {"name": "distil small 2x128", "loss": "kd", "kind": "grads", "rows": 2, "width": 128, "dim": 512, "vocab": 8256,
         "k": 16, "type": "bf16", "ragged": True, "temperature": 2.0},
        # how far a student is from its teacher on held-out text
        {"name": "distil score 4x1024", "loss": "kd", "kind": "score", "rows": 4, "width": 1024, "dim": 2048,
         "vocab": 32256, "k": 32, "type": "bf16", "ragged": False, "temperature": 1.0},
        # an ordinary distillation step through autograd
        {"name": "distil 4x2047", "loss": "kd", "kind": "autograd", "rows": 4, "width": 2047, "dim": 2048,
         "vocab": 32256, "k": 64, "type": "bf16", "ragged": False, "temperature": 1.0},
        # half precision, a teacher cut at 50 entries, odd vocabulary, softened
        {"name": "distil fp16 16x511", "loss": "kd", "kind": "grads", "rows": 16, "width": 511, "dim": 1024,
         "vocab": 50257, "k": 50, "type": "fp16", "ragged": True, "temperature": 2.0},
        # the largest distillation step
        {"name": "distil 4x2048 largest", "loss": "kd", "kind": "grads", "rows": 4, "width": 2048, "dim": 4096,
         "vocab": 65536, "k": 128, "type": "bf16", "ragged": False, "temperature": 1.0},
    ]


def draw(rng):
    def log_int(lo, hi):
        return min(hi, int(round(lo * (hi / lo) ** rng.random())))

    rows = log_int(1, 16)
    dim = log_int(64, 4096)
    if rng.random() < 0.7:  # most models' widths
        dim = max(64, dim // 64 * 64)
    vocab = log_int(512, 65536)
    loss = rng.choice(["ce", "kd"])
    return {"loss": loss, "kind": rng.choice(["score", "grads", "autograd"]), "rows": rows,
            "width": log_int(1, 8192 // rows), "dim": dim, "vocab": vocab,
            "k": 1 if loss == "ce" else log_int(1, 128), "type": rng.choice(["bf16", "bf16", "fp16"]),
            "ragged": rng.random() < 0.5, "temperature": 1.0 if loss == "ce" else rng.choice([1.0, 2.0, 3.5])}


def _lengths(case):
    """Tokens in the rows of a ragged batch, shortest first: evenly spread, the longest fills its row."""
    if not case["ragged"]:
        return [case["width"]] * case["rows"]
    return [max(1, case["width"] * (r + 1) // case["rows"]) for r in range(case["rows"])]


# ------------------------------------------------------------------------------------ inputs
def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    B, L, D, V, K = case["rows"], case["width"], case["dim"], case["vocab"], case["k"]
    n, dtype = B * L, TYPES[case["type"]]
    weight = torch.randn(V, D, generator=g, device=DEVICE).mul_(0.02)
    # token ids by rank: 1 / rank, as of text
    targets = (V ** torch.rand(n, generator=g, device=DEVICE)).long().sub_(1).clamp_(0, V - 1)
    # a normalised state that leans towards the next token's row
    hidden = torch.randn(n, D, generator=g, device=DEVICE).add_(weight[targets], alpha=5.0).to(dtype).view(B, L, D)
    lens = torch.tensor(_lengths(case), device=DEVICE)[torch.randperm(B, generator=g, device=DEVICE)]
    inside = torch.arange(L, device=DEVICE)[None, :] < lens[:, None]
    state = {"case": case, "hidden": hidden, "weight": weight.to(dtype),
             "valid": inside.to(torch.uint8) if case["ragged"] else None,
             # half precision trains with a loss scale
             "grad_loss": torch.tensor(4096.0 if case["type"] == "fp16" else 1.0, device=DEVICE)}
    if case["loss"] == "ce":
        state["targets"] = torch.where(inside, targets.view(B, L), -1).to(torch.int32)
    else:
        ids, logits = [], []
        prior = -torch.log(torch.arange(1, V + 1, device=DEVICE, dtype=torch.float32))
        for part in targets.split(1024):  # the teacher knows the next token, and is otherwise as unsure as text is
            t = prior - torch.empty(len(part), V, device=DEVICE).exponential_(generator=g).clamp_min_(1e-30).log_()
            t[torch.arange(len(part), device=DEVICE), part] += 2.0
            v, i = t.topk(min(K, V), dim=1)
            ids.append(i), logits.append(v)
        ids, logits = torch.cat(ids), torch.cat(logits)
        few = torch.rand(n, generator=g, device=DEVICE) < 0.125  # rows whose list the teacher cut short
        kept = torch.arange(K, device=DEVICE) < torch.where(few, (K + 1) // 2, K)[:, None]
        state["teacher_ids"] = torch.where(kept & inside.reshape(n, 1), ids, -1).to(torch.int32).view(B, L, K)
        state["teacher_logits"] = logits.view(B, L, K).contiguous()
    if case["kind"] == "autograd":
        state["hidden"].requires_grad_(True), state["weight"].requires_grad_(True)
    return state


# ------------------------------------------------------------------------------------ plain forms
def _plain(state):
    case = state["case"]
    shape = state["hidden"].shape[:-1]
    dtype, T = state["hidden"].dtype, case["temperature"]
    with torch.no_grad():
        h, w = state["hidden"].reshape(-1, case["dim"]).float(), state["weight"].float()
        counted = torch.ones(len(h), dtype=torch.bool, device=h.device)
        if state["valid"] is not None:
            counted = state["valid"].reshape(-1) != 0
        z = h @ w.T
        if T != 1.0:
            z = z / T
        top = z.amax(1, keepdim=True)
        lse = top + (z - top).exp().sum(1, keepdim=True).log()
        if case["loss"] == "ce":
            ids = state["targets"].reshape(-1, 1).long()
            counted = counted & (ids[:, 0] >= 0)
            p, there = torch.ones_like(lse), ids >= 0
            loss = (lse - z.gather(1, ids.clamp_min(0)))[:, 0]
        else:
            ids = state["teacher_ids"].reshape(len(h), -1).long()
            there = ids >= 0
            counted = counted & there.any(1)
            t = torch.where(there, state["teacher_logits"].reshape(len(h), -1).float() / T, -torch.inf)
            most = t.amax(1, keepdim=True)
            t = t - torch.where(most > -torch.inf, most, 0.0)
            p = t.exp() / t.exp().sum(1, keepdim=True).clamp_min(1e-30)
            logp = t - t.exp().sum(1, keepdim=True).clamp_min(1e-30).log()
            each = p * (logp - z.gather(1, ids.clamp_min(0)) + lse)
            loss = torch.where(there & (p > 0), each, 0.0).sum(1) * (T * T)
        loss = torch.where(counted, loss, 0.0)
        if case["kind"] == "score":
            return {"loss": loss.view(shape)}
        rows = counted.sum().clamp_min(1)
        g = z.sub_(lse).exp_()
        g.scatter_add_(1, ids.clamp_min(0), torch.where(there, -p, 0.0))
        g.mul_(torch.where(counted, state["grad_loss"] * T / rows, 0.0)[:, None])
        return {"loss": loss.sum() / rows, "grad_hidden": (g @ w).to(dtype).view(state["hidden"].shape),
                "grad_weight": (g.T @ torch.where(counted[:, None], h, 0.0)).to(dtype)}


# ------------------------------------------------------------------------------------ the framework's calls
def _own(state):
    from supertoken_b200 import ops
    case = state["case"]
    if case["loss"] == "ce":
        args, more, loss_of, grads_of = (state["targets"], state["valid"]), {}, ops.vocab_cross_entropy, \
            ops.vocab_cross_entropy_grads
    else:
        args, more = (state["teacher_ids"], state["teacher_logits"], state["valid"]), {"temperature": case["temperature"]}
        loss_of, grads_of = ops.vocab_distillation, ops.vocab_distillation_grads
    hidden, weight = state["hidden"], state["weight"]
    if case["kind"] == "score":
        return {"loss": loss_of(hidden, weight, *args, reduction="none", **more)}
    if case["kind"] == "grads":
        loss, gh, gw = grads_of(hidden, weight, *args, grad_loss=state["grad_loss"], **more)
    else:
        loss = loss_of(hidden, weight, *args, **more)
        gh, gw = torch.autograd.grad(loss, (hidden, weight), grad_outputs=state["grad_loss"])
    return {"loss": loss.detach(), "grad_hidden": gh, "grad_weight": gw}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------------------------ what it takes
def work(case):
    n, D, V, K = sum(_lengths(case)), case["dim"], case["vocab"], case["k"]
    read = 2 * (n + V) * D + n * (4 if case["loss"] == "ce" else 8 * K)
    if case["kind"] == "score":
        return {"bytes": read + 4 * n, "flops": 2 * n * V * D}
    return {"bytes": read + 2 * (case["rows"] * case["width"] + V) * D, "flops": 6 * n * V * D}


# ------------------------------------------------------------------------------------ definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    B, L, D, V, T = case["rows"], case["width"], case["dim"], case["vocab"], case["temperature"]
    x, w = s["hidden"].detach().double().reshape(B * L, D), s["weight"].detach().double()
    loss, gh, gw = torch.zeros(B * L, device=DEVICE, dtype=torch.float64), torch.zeros_like(x), torch.zeros_like(w)
    live = torch.ones(B * L, dtype=torch.bool, device=DEVICE) if s["valid"] is None else s["valid"].reshape(-1).bool()
    if case["loss"] == "ce":
        live &= s["targets"].reshape(-1) >= 0
    else:
        live &= (s["teacher_ids"].reshape(B * L, -1) >= 0).any(dim=1)
    scale = float(s["grad_loss"]) / max(1, int(live.sum()))
    for at in live.nonzero()[:, 0].split(1024):
        logq = torch.log_softmax(x[at] @ w.T / T, dim=1)
        want = torch.zeros_like(logq)  # the distribution that is aimed at
        if case["loss"] == "ce":
            want[torch.arange(len(at), device=DEVICE), s["targets"].reshape(-1)[at].long()] = 1.0
            loss[at] = -(want * logq).sum(dim=1)
        else:
            i, t = s["teacher_ids"].reshape(B * L, -1)[at].long(), s["teacher_logits"].reshape(B * L, -1)[at].double()
            logp = torch.log_softmax(t.div(T).masked_fill(i < 0, -math.inf), dim=1)
            want.scatter_add_(1, i.clamp(min=0), logp.exp())
            share = logp.exp()
            loss[at] = T * T * (torch.xlogy(share, share).sum(dim=1) - (want * logq).sum(dim=1))
        if case["kind"] != "score":
            dz = (logq.exp() - want) * (T * scale)
            gh[at] = dz @ w
            gw += dz.T @ x[at]
    if case["kind"] == "score":
        return {"loss": loss.view(B, L)}
    return {"loss": loss.sum() / max(1, int(live.sum())), "grad_hidden": gh.view(B, L, D), "grad_weight": gw}
