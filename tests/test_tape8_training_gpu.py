"""MAgNet's chains on the 8-bit tape: where it is written, and training."""
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
