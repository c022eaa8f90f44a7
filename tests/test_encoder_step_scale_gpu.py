"""The size of every gradient of an encoder layer's training step (test_encoder_step_gpu.py), which a direction does not
show: a missing factor of dropout, of the softmax's scale or of a mean turns no gradient.

Bounds. Every tensor between two ops is rounded to bf16, by errors that are independent from one element to the next
and from one rounding to the next, even, and at most u = 2^-8 of the value: of a deviation u / sqrt(3) at most. Forward and
back the longest way has K = 24 roundings, of two branches each, and the ops behind one pass a relative change on by a
factor of at most 2. So a gradient's error is of a norm of
  D = 2 sqrt(2 K) u / sqrt(3) = 0.0313
of its own at most, in the mean of the squares; over 64 elements and more a norm is within 3 / sqrt(2 * 64) of that:
  |got - want| <= 1.27 D |want|.
Along the gradient itself the errors of N elements add up as independent ones do: of |want|^2 they make D sqrt(3 / N) at
most (3: the fourth moment of a normal distribution, for elements of unequal size), with three deviations and N >= 64
  |<got, want> / <want, want> - 1| <= 3 D sqrt(3 / 64) = 0.0203.
The loss -log softmax(SCALE y . docs) has the forward's 12 roundings in y: they move a score by
SCALE |docs| 2 sqrt(24) u / sqrt(3) / sqrt(HIDDEN), as a random vector lies to a document; a loss by the difference of two
such, which is below four deviations of sqrt(2) of that."""
import math

import pytest

import step_ref as S
import test_encoder_step_gpu as E

D = 2 * math.sqrt(48) * 2.0 ** -8 / math.sqrt(3)
ALONG = 3 * D * math.sqrt(3 / 64)


def loss_bound(docs):
    longest = docs.double().norm(dim=1).max().item()
    return 4 * math.sqrt(2) * E.SCALE * longest * 2 * math.sqrt(24) * 2.0 ** -8 / math.sqrt(3) / math.sqrt(E.HIDDEN)


def hold(got, want, docs):
    """Names of the results of a step that are off."""
    off = []
    for name, w in want.items():
        g = got[name].double()
        if name == "loss":
            bad = (g - w).abs().max().item() > loss_bound(docs)
        else:
            assert w.numel() >= 64
            along = (g.flatten() @ w.flatten()).item() / (w.flatten() @ w.flatten()).item() - 1
            error = ((g - w).norm() / w.norm()).item()
            print(f"{name}: along {along:.2e} error {error:.2e}", flush=True)
            bad = abs(along) > ALONG or error > 1.27 * D
        if bad or not bool(g.isfinite().all()):
            off.append(name)
    return off


def _inputs(torch, inl, dev):
    cu = [sum(E.LENGTHS[:i]) for i in range(len(E.LENGTHS) + 1)]
    pos = torch.from_numpy(inl.positions(cu)).to(dev)
    cos, sin = (torch.from_numpy(t).to(dev) for t in inl.rope_table(E.HD, E.THETA, max(E.LENGTHS)))
    g = torch.Generator(device=dev).manual_seed(2)
    x = torch.randn(sum(E.LENGTHS), E.HIDDEN, generator=g, device=dev)
    targets = torch.tensor([3, 0, 23, 7, 7], dtype=torch.int32, device=dev)
    return cu, pos, cos, sin, x, E._weights(torch, dev), targets


@pytest.mark.gpu
def test_step_has_the_right_size(cuda, inl):
    import torch
    cu, pos, cos, sin, x, w, targets = _inputs(torch, inl, cuda)
    plan = inl.AttnPlan(inl.make_attn_desc(cu, E.HQ, E.HKV, E.HD, causal=True, q_row_stride=(E.HQ + E.HKV) * E.HD,
                                           k_row_stride=(E.HQ + E.HKV) * E.HD,
                                           v_row_stride=(E.HQ + 2 * E.HKV) * E.HD))
    offs = torch.tensor(cu, dtype=torch.int32, device=cuda)
    got = E._step(inl, torch, x, w, plan, cu, offs, pos, cos, sin, targets, torch.tensor([17, 9], device=cuda))
    torch.cuda.synchronize()
    assert hold(got, E._reference(torch, x, w, pos, cos, sin, targets, 17, 9), w["docs"]) == []


def test_the_bounds_see_a_wrong_size():
    """On the CPU, with mistakes in the float64 step: dropout's factor, a scale, an error beside the gradient."""
    import torch

    import inl_hip
    _, pos, cos, sin, x, w, targets = _inputs(torch, inl_hip, torch.device("cpu"))
    want = E._reference(torch, x, w, pos, cos, sin, targets, 17, 9)
    assert hold(want, want, w["docs"]) == []
    names = [n for n in want if n != "loss"]
    for factor in (1 - E.DROP, 1 / (1 - E.DROP), 0.97, 1.03, -1.0):
        assert hold({**want, **{n: want[n] * factor for n in names}}, want, w["docs"]) == names
    g = torch.Generator().manual_seed(1)
    noise = {n: torch.randn(want[n].shape, generator=g, dtype=torch.float64) for n in names}
    beside = {n: want[n] + 0.1 * want[n].norm() / noise[n].norm() * noise[n] for n in names}
    assert hold({**want, **beside}, want, w["docs"]) == names
    assert hold({**want, "loss": want["loss"] * 1.02}, want, w["docs"]) == ["loss"]
    # the dropout of the last addition without its factor, and of other draws
    kept, factor = S.factor, E.DROP
    try:
        S.factor = lambda *a: kept(*a) * ((1 - factor) if a[5] == 3 else 1)
        off = hold(E._reference(torch, x, w, pos, cos, sin, targets, 17, 9), want, w["docs"])
        assert "down" in off and "gu" in off
        S.factor = lambda *a: kept(*a[:4], a[4] + (a[5] == 3), *a[5:])
        assert len(hold(E._reference(torch, x, w, pos, cos, sin, targets, 17, 9), want, w["docs"])) >= 10
    finally:
        S.factor = kept
