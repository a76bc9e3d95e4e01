"""Arguments that the losses over a large vocabulary refuse before any GPU work, and the size of their workspace."""
import ctypes

import pytest
import torch

from supertoken_b200 import _lib as L
from supertoken_b200 import losses, ops


def _args(**more):
    a = L.VocabLoss()
    a.outer, a.inner, a.vocab, a.dim, a.type, a.k, a.ids_bytes = 4, 512, 32256, 1024, 0, 0, 4
    a.reduction, a.want, a.temperature = 2, 3, 1.0
    a.hidden, a.weight, a.weight_stride, a.hidden_outer, a.hidden_inner = 1 << 20, 2 << 20, 1024, 512 * 1024, 1024
    a.grad_hidden, a.grad_weight = 3 << 20, 4 << 20
    for name, value in more.items():
        setattr(a, name, value)
    return a


def _need(a):
    n, err = ctypes.c_int64(-1), ctypes.create_string_buffer(256)
    st = L.load().stbpe_vocab_loss_workspace(ctypes.byref(a), ctypes.byref(n), err, 256)
    return st, n.value, err.value.decode()


@pytest.mark.parametrize("more", [
    {"outer": -1}, {"inner": -1}, {"vocab": 0}, {"dim": 0}, {"vocab": 1 << 31}, {"dim": 1 << 21}, {"outer": 1 << 22, "inner": 1 << 10},
    {"type": 2}, {"type": -1}, {"k": -1}, {"k": 257}, {"ids_bytes": 2}, {"k": 4, "logits_type": 3}, {"reduction": 3},
    {"reduction": -1}, {"want": 0}, {"temperature": 2.0}, {"k": 4, "temperature": 0.0}, {"k": 4, "temperature": float("nan")},
    {"k": 4, "temperature": float("inf")}, {"k": 4, "temperature": 1e-40}])
def test_bad_arguments_are_refused(more):
    st, n, text = _need(_args(**more))
    assert st == L.E_BADARG and n == -1 and text.startswith("stbpe_vocab_loss: ")


def test_nothing_runs_without_what_it_needs():
    lib, err = L.load(), ctypes.create_string_buffer(256)
    assert lib.stbpe_vocab_loss_run(None, None, err, 256) == L.E_BADARG
    assert lib.stbpe_vocab_loss_workspace(None, None, None, 0) == L.E_BADARG
    a = _args()
    _, need, _ = _need(a)
    for space, size in ((0, need), (1 << 30, need - 1), ((1 << 30) + 512, need)):
        a.workspace, a.workspace_bytes = space, size
        assert lib.stbpe_vocab_loss_run(ctypes.byref(a), None, err, 256) == L.E_CAPACITY
    a.workspace, a.workspace_bytes = 1 << 30, need
    assert lib.stbpe_vocab_loss_run(ctypes.byref(a), None, err, 256) == L.E_BADARG and b"output" in err.value
    a.lse2 = a.loss = 5 << 20
    assert lib.stbpe_vocab_loss_run(ctypes.byref(a), None, err, 256) == L.E_BADARG and b"input" in err.value


def test_workspace_holds_no_logits():
    """Its size follows the rows and a bounded piece of the vocabulary, not their product."""
    logits = 32 * 2048 * 262144 * 2
    for want in (1, 3):
        st, n, _ = _need(_args(outer=32, inner=2048, vocab=262144, want=want))
        assert st == L.OK and n < logits / 8
    assert _need(_args(want=1))[1] < _need(_args(want=3))[1]
    # a weight that starts anywhere is copied
    assert _need(_args(weight=(2 << 20) + 2))[1] - _need(_args())[1] == 32256 * 1024 * 2
    assert _need(_args(dim=1023))[1] > _need(_args())[1]
    assert _need(_args(outer=0))[0] == L.OK


def test_cpu_tensors_are_refused():
    h, w, t = torch.zeros(2, 8, dtype=torch.bfloat16), torch.zeros(5, 8, dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int32)
    for call in (lambda: ops.vocab_cross_entropy(h, w, t), lambda: ops.vocab_cross_entropy_grads(h, w, t),
                 lambda: ops.vocab_distillation(h, w, t[:, None], torch.zeros(2, 1)),
                 lambda: ops.vocab_distillation_grads(h, w, t[:, None], torch.zeros(2, 1))):
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            call()
    with pytest.raises(TypeError):
        losses.vocab_distillation(h, w, t[:, None], None)


def test_temperatures_that_32_bits_do_not_hold():
    for t in (2.0 ** -16, 0.01, 2.0 ** 16):
        assert _need(_args(k=4, logits_type=2, temperature=t))[0] == L.OK
    for t in (1e-20, 1e-10, 1e-5, 65537.0, 1e20, -2.0):
        st, n, text = _need(_args(k=4, logits_type=2, temperature=t))
        assert st == L.E_BADARG and n == -1 and "temperature" in text


def test_no_workspace_for_a_gradient_that_is_not_wanted():
    many = dict(outer=8, inner=2048, vocab=65536, dim=4096, hidden_outer=2048 * 4096, hidden_inner=4096, weight_stride=4096)
    at_once, later = dict(many, want=3), dict(many, want=2, lse2=6 << 20)
    assert _need(_args(**at_once))[1] - _need(_args(**at_once, grad_weight=0))[1] == 65536 * 4096 * 4
    assert _need(_args(**later))[1] - _need(_args(**later, grad_hidden=0))[1] == 8 * 2048 * 4096 * 4


def test_scoring_many_rows_takes_a_bounded_workspace():
    """What follows from rows times vocabulary is held for a chunk of the rows: 2^20 rows of 262 144 ids have 2 GiB of sums and maxima per 131 072 rows."""
    rows = dict(outer=1024, inner=1024, vocab=262144, dim=64, hidden_outer=1024 * 64, hidden_inner=64, weight_stride=64, want=1)
    inputs = (1 << 20) * 64 * 2
    assert _need(_args(**rows))[1] < (1 << 30) + 2 * inputs
    # a teacher's rows have two bytes for every 256 ids, too
    assert _need(_args(**rows, k=16, logits_type=2))[1] < (1 << 30) + 4 * inputs + (1 << 20) * 1024 * 2


def test_calls_run_on_their_tensors_device(monkeypatch):
    """Another device is current: launches, the gradients' scaling and the question for a capture go to the tensors' own, and the current one stays."""
    now, seen = [1], []

    class Switch:
        def __init__(self, device):
            self.index = device if isinstance(device, int) else device.index

        def __enter__(self):
            self.before, now[0] = now[0], self.index

        def __exit__(self, *_):
            now[0] = self.before

    class Library:
        def stbpe_vocab_loss_workspace(self, *_):
            seen.append(("workspace", now[0]))
            return L.E_BADARG

        def stbpe_scale_gradients(self, *args):
            seen.append(("scale", now[0], args[-1]))
            return L.OK

    monkeypatch.setattr(torch.cuda, "current_device", lambda: now[0])
    monkeypatch.setattr(torch.cuda, "device", Switch)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: seen.append(("capture", now[0])) or False)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
    monkeypatch.setattr(L, "load", Library)
    for index in (0, 1, 2):
        device = torch.device("cuda", index)
        with pytest.raises(ValueError):
            losses._run(_args(), device)
        by = type("Up", (), {"device": device, "data_ptr": lambda self: 512})()
        losses._scale(None, None, by)
        losses._refuse_capture(device)
        assert seen == [("workspace", index), ("scale", index, 100 + index), ("capture", index)] and now == [1]
        seen.clear()


def test_the_bounds_in_norms_see_a_loss_of_precision():
    """Mistakes that are planted in the formula: logits in 16 bits, a factor of half a percent, a target's logit that is cut off."""
    from test_vocab_loss_edges_gpu import loss_bound, near_in_norm
    g = torch.Generator().manual_seed(0)
    rows, D, V, u = 256, 1024, 2048, 2.0 ** -8
    hidden = torch.randn(1, rows, D, generator=g).bfloat16()
    weight = (torch.randn(V, D, generator=g) / 32).bfloat16()
    t = torch.randint(0, V, (rows,), generator=g)
    z = hidden[0].double() @ weight.double().T
    bound = loss_bound(hidden, weight, (t[None],))

    def results(z, factor=1.0):
        lse = torch.logsumexp(z, 1)
        G = (z - lse[:, None]).exp()
        G[torch.arange(rows), t] -= 1.0
        G *= factor
        return lse - z[torch.arange(rows), t], (G @ weight.double()).bfloat16(), (G.T @ hidden[0].double()).bfloat16()

    loss, gh, gw = results(z)
    want = [x.double() for x in results(z)[1:]]
    near_in_norm(gh, want[0], u, 0.0, "gh"), near_in_norm(gw, want[1], u, 0.0, "gw")
    for factor in (1.005, 0.995):
        for got, right in zip(results(z, factor)[1:], want):
            with pytest.raises(AssertionError):
                near_in_norm(got, right, u, 0.0, "")
    assert bool(((results(z.bfloat16().double())[0] - loss).abs() > bound).any())
    cut = z.clone()
    cut[torch.arange(rows), t] *= 1 - 2.0 ** -13
    assert bool(((results(cut)[0] - loss).abs() > bound).any())
    assert float((bound / loss).max()) < 2e-5
