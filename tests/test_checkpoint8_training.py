"""Training the particle transformer with its activations kept in 8 bits (encoder.checkpoint_bits: 8)."""
import copy

import pytest
import torch

from conftest import GOLDEN


def build(golden, name, bits, dropout):
    from pipeline.configs import ExperimentConfigs
    from model.multimodal_bridge_matching import MultiModalBridgeMatching
    g = golden(name)
    cfg = copy.deepcopy(g.cfg)
    cfg["data"]["target_path"] = GOLDEN
    cfg["encoder"]["dropout"] = dropout
    cfg["encoder"]["checkpoint_bits"] = bits
    model = MultiModalBridgeMatching(ExperimentConfigs(cfg))
    model.load_state_dict(g.params, strict=True)
    return g, model


def test_other_encoders_and_widths_are_refused(golden):
    for name, bits in (("tr_tiny", 4), ("mm_tiny", 8), ("toy", 8)):
        with pytest.raises(ValueError, match="checkpoint_bits"):
            build(golden, name, bits, 0.0)
    build(golden, "tr_tiny", 8, 0.0)


def step(g, model, seed=5, backward=True, reps=1):
    from tensorclass import TensorMultiModal
    from datamodules.datasets import DataCoupling
    t = g.t
    c = lambda a: None if a is None else torch.cat([a] * reps).cuda()  # noqa: E731
    model.manual_seed(seed)
    state = TensorMultiModal(c(t["time"]), c(t.get("xt")), c(t["kt"]), c(t["mask"]))
    src = TensorMultiModal(None, c(t.get("x0")), c(t["k0"]), torch.ones_like(c(t["mask"])))
    batch = DataCoupling(src, TensorMultiModal(None, c(t.get("x1")), c(t["k1"]), c(t["mask"])), None)
    out = model.step_from_state(state, batch, "train", True)
    held = torch.cuda.memory_allocated()
    if backward:
        out["loss"].backward()
    return out["loss"].detach().clone(), held


def grads(model):
    return {n: q.grad.detach().clone() for n, q in model.named_parameters() if q.grad is not None}


@pytest.mark.gpu
@pytest.mark.parametrize("name,dropout", [("tr_tiny", 0.0), ("tr_tiny", 0.2), ("tr_odd", 0.0), ("S4", 0.0), ("S4", 0.2)])
def test_gradients_near_those_of_float_activations(golden, name, dropout):
    """The forward is the same; a gradient differs by what a code is off: every activation by at most 1/127 of the largest of
    its 32, some ten of them one after another down to the first layer.  Their roundings are independent, so the relative
    distance of a whole gradient stays well below 10 x 1/127 (the bound, 0.08); its direction therefore within 0.08."""
    res = {}
    for bits in (None, 8):
        g, model = build(golden, name, bits, dropout)
        model = model.cuda().train()
        loss, _ = step(g, model)
        res[bits] = loss, grads(model)
        if bits == 8:
            first = res[8][1]
            model.zero_grad(set_to_none=True)
            loss2, _ = step(g, model)
            assert torch.equal(loss, loss2)
            step(g, model)                                      # a second backward adds to the gradients
            for n, q in model.named_parameters():
                if q.grad is not None:
                    torch.testing.assert_close(q.grad, 2 * first[n], rtol=1e-4, atol=1e-5 * float(first[n].abs().max()) + 1e-9)
    assert torch.equal(res[None][0], res[8][0])
    assert res[None][1].keys() == res[8][1].keys()
    flat = lambda d: torch.cat([v.double().flatten() for v in d.values()])  # noqa: E731
    a, b = flat(res[None][1]), flat(res[8][1])
    assert b.isfinite().all()
    assert float((a - b).norm() / a.norm()) < 10 / 127
    layers = [n for n in res[8][1] if ".transformer.layers." in n]
    assert layers and any(not torch.equal(res[None][1][n], res[8][1][n]) for n in layers)     # (the codes were really used)


class Lossless:
    def __init__(self, x):
        self.x, self.shape = x.clone(), x.shape

    @staticmethod
    def grad_weight(q, dZ, dW=None, db=None, accumulate=False, want_db=True):
        w, b = (dZ.double().t() @ q.x.double()).float(), dZ.double().sum(0).float()
        if dW is None:
            return w, b
        return dW.add_(w), db.add_(b)


@pytest.mark.gpu
@pytest.mark.parametrize("name,dropout", [("tr_tiny", 0.0), ("tr_odd", 0.2), ("S4", 0.2)])
def test_with_a_coder_that_loses_nothing(golden, name, dropout, monkeypatch):
    """Everything but the code: freed and restored tensors, the attention run again, weight gradients from what was kept.
    With a lossless coder in the code's place the gradients are those of float activations up to the order of 32-bit sums
    (a few thousand terms of either sign: some 1e-6 of a gradient's norm, 2e-5 is asked for)."""
    from mmb_hip import ops
    g, model = build(golden, name, None, dropout)
    model = model.cuda().train()
    step(g, model)
    want = grads(model)
    monkeypatch.setattr(ops, "checkpoint_rows", lambda x, keep_nonzero=False: Lossless(x))
    monkeypatch.setattr(ops, "restore_rows", lambda q, dtype=None, out=None: out.copy_(q.x))
    monkeypatch.setattr(ops, "grad_weight_rows_q8", Lossless.grad_weight)
    g, model = build(golden, name, 8, dropout)
    model = model.cuda().train()
    step(g, model)
    got = grads(model)
    assert got.keys() == want.keys()
    for n in want:
        assert float((got[n] - want[n]).norm()) <= 2e-5 * float(want[n].norm()) + 1e-9, n


class PlainCode(Lossless):
    """The code by its definition, in 64 bits: 32 features share the smallest step 2^e with 127 steps >= the largest."""

    def __init__(self, x, keep_nonzero=False):
        M, K = x.shape
        xb = torch.nn.functional.pad(x.double(), (0, -K % 32)).view(M, -1, 32)
        top = xb.abs().amax(-1, keepdim=True)
        e = torch.frexp(top / 127)[1].double()                  # 2^e > top / 127 >= 2^(e - 1)
        step = torch.exp2(torch.where(127 * torch.exp2(e - 1) >= top, e - 1, e).clamp(min=-127))
        c = torch.round(xb / step)
        if keep_nonzero:
            c = torch.where((c == 0) & (xb != 0), xb.sign(), c)
        self.x, self.shape = (c * step).view(M, -1)[:, :K].float().contiguous(), x.shape


@pytest.mark.gpu
@pytest.mark.parametrize("name,dropout", [("tr_tiny", 0.0), ("tr_tiny", 0.2), ("tr_odd", 0.2), ("S4", 0.0), ("S4", 0.2)])
def test_gradients_are_those_of_the_decoded_activations(golden, name, dropout, monkeypatch):
    """The kernels' codes against the code by its definition in their place, weight gradients in 64 bits from the values it
    stands for: what is left is the order of 32-bit sums, as with the lossless coder above."""
    from mmb_hip import ops
    g, model = build(golden, name, 8, dropout)
    model = model.cuda().train()
    step(g, model)
    got = grads(model)
    used = []
    monkeypatch.setattr(ops, "checkpoint_rows", lambda x, keep_nonzero=False: used.append(keep_nonzero) or PlainCode(x, keep_nonzero))
    monkeypatch.setattr(ops, "restore_rows", lambda q, dtype=None, out=None: out.copy_(q.x))
    monkeypatch.setattr(ops, "grad_weight_rows_q8", PlainCode.grad_weight)
    g, model = build(golden, name, 8, dropout)
    model = model.cuda().train()
    step(g, model)
    want = grads(model)
    assert any(used) and not all(used) and got.keys() == want.keys()
    for n in want:
        assert float((got[n] - want[n]).norm()) <= 2e-5 * float(want[n].norm()) + 1e-9, n


@pytest.mark.gpu
def test_memory_held_between_the_passes(golden):
    """What the tape holds when the forward is done: the layers' matrices at 33/128 of their size; the other tensors (both
    branch outputs, heads, embeddings, inputs) stay, so half is asked for."""
    held = {}
    for bits in (None, 8):
        g, model = build(golden, "S4", bits, 0.2)
        model = model.cuda().train()
        step(g, model, reps=16)
        model.zero_grad(set_to_none=True)
        torch.cuda.synchronize()
        base = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        _, h = step(g, model, reps=16)
        held[bits] = h - base, torch.cuda.max_memory_allocated() - base
    assert held[8][0] < 0.5 * held[None][0], held
    assert held[8][1] < held[None][1], held
