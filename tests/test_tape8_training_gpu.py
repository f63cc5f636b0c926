"""MAgNet's chains on the 8-bit tape: where it is written, and training of the models."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_tape_where_no_gradient_is_recorded(monkeypatch):
    """under ``no_grad`` parameters still ask for gradients: nothing is kept, packed or written for them"""
    from magnet_amd import autograd as AG, ops
    from tests.test_tape8_gpu import chain_case
    monkeypatch.setenv("MAGNET_KEEP_TAPE", "1")
    lins, norm, pk, params, x = chain_case(700, 64, 32, 64, 3, True)
    calls = []
    pack, keep = ops.tape8_pack, AG._keep_tape
    monkeypatch.setattr(ops, "tape8_pack", lambda *a, **k: (calls.append("pack"), pack(*a, **k))[1])
    monkeypatch.setattr(AG, "_keep_tape", lambda *a, **k: (calls.append("keep"), keep(*a, **k))[1])
    with AG.tape8():
        y = AG.mlp(700, [ops.Term(x, 64)], pk, params)
        assert "pack" in calls and "keep" in calls
        del calls[:]
        with torch.no_grad():
            z = AG.mlp(700, [ops.Term(x, 64)], pk, params)
    assert not calls and torch.equal(y.detach(), z)


def _model(tag, on, **hparams):
    from magnet_amd.models.factory import FACTORY
    from oracle import models as O
    from oracle.weightgen import fill_state_dict
    from tests.helpers import load_case
    name, hp, salt, batch, d = load_case(tag)
    for k, v in hparams.items():
        setattr(hp, k, v)
    hp.tape8 = on
    oracle = O.build(name, hp)
    fill_state_dict(oracle, salt)
    model = FACTORY[name](hp)
    model.load_state_dict(oracle.state_dict())
    return model.cuda().train(), {k: v.cuda() for k, v in batch.items()}


@pytest.mark.parametrize("teacher_forcing", [False, True])
@pytest.mark.parametrize("tag", ["magnet_cnn_1d", "magnet_cnn_2d"])
def test_magnet_cnn_trains_with_the_tape_in_8_bits(tag, teacher_forcing):
    """the loss has the bits of the fp32 tape's; every parameter's gradient is within the rounding of the activations (0.4 - 1 % a chain, several
    chains behind one another)"""
    got = []
    for on in (False, True):
        model, cb = _model(tag, on, teacher_forcing=teacher_forcing)
        loss = model.training_step(cb, 0)
        loss.backward()
        got.append((loss.detach(), {n: p.grad for n, p in model.named_parameters()}))
    assert torch.equal(got[0][0], got[1][0])
    assert any(not torch.equal(got[1][1][n], g) for n, g in got[0][1].items() if g is not None)
    for n, g in got[0][1].items():
        if g is None:
            assert got[1][1][n] is None
            continue
        off = float((got[1][1][n] - g).norm() / g.norm()) if float(g.norm()) else 0.0
        assert off <= 0.05, (n, off)


@pytest.mark.parametrize("tag", ["magnet_gnn_tiny", "magnet_cnn_2d"])
def test_hooks_on_parameters_see_the_gradients_of_the_tape(tag):
    """parameters with hooks (as a data-parallel wrapper puts them there) get their gradients through autograd, the same ones"""
    model, cb = _model(tag, True)
    params = [(n, p) for n, p in model.named_parameters() if p.requires_grad]
    torch.manual_seed(5)
    model.training_step(cb, 0).backward()
    want = {n: p.grad.clone() for n, p in params if p.grad is not None}
    seen = {}
    for n, p in params:
        p.grad = None
        p.register_post_accumulate_grad_hook(lambda p_, n=n: seen.__setitem__(n, seen.get(n, 0) + 1))
    torch.manual_seed(5)
    model.training_step(cb, 0).backward()
    assert all(seen.get(n, 0) == 1 for n in want)
    for n, p in params:
        if n in want and float(want[n].abs().max()) > 0:
            # (the same sums, added by autograd instead of by the kernels: a few additions in fp32)
            assert float((p.grad - want[n]).norm()) <= 1e-5 * float(want[n].norm()), n
