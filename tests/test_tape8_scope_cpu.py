"""The 8-bit tape's operators on any machine: what they refuse at the ends of their ranges, what their workspaces take, and where the
training scopes hold."""
import ctypes as C
import threading

import pytest
import torch

from magnet_amd import _lib, autograd as AG, ops


def test_widths_beyond_32_bits_are_refused():
    """a kernel counts columns in 32 bits"""
    wide = 2 ** 32 + 5
    meta = lambda *s, **k: torch.empty(*s, device="meta", **k)  # noqa: E731
    for W in (2 ** 31, wide):
        with pytest.raises(ValueError, match="columns"):
            ops.tape8_pack(meta(1, W, dtype=torch.bfloat16))
        with pytest.raises(ValueError, match="width"):
            ops.tape8_empty(1, W, device="meta")
        with pytest.raises(ValueError, match="columns"):
            ops.tape8_linear_bwd(meta(1, W), ops.tape8_empty(1, 40, device="meta"), meta(W, 40))
    nb = (wide + 31) // 32
    with pytest.raises(ValueError, match="width"):
        ops.tape8_unpack(ops.Tape8(meta(1, 32 * nb, dtype=torch.uint8), meta(1, nb, dtype=torch.uint8), wide))


def test_the_workspace_of_a_wide_weight():
    n = C.c_long(0)
    entry = _lib.lib().magnet_tape8_linear_bwd_workspace
    for M in (1, 100, 1 << 20):
        for K in (128, 4096, 4097, 200_000, 1 << 24, (1 << 31) - 256):
            assert entry(C.c_long(M), C.c_long(128), C.c_long(K), C.byref(n)) == 0
            assert 0 < 4 * n.value <= 512 << 20, (M, K, n.value)
    assert entry(C.c_long(1), C.c_long(1), C.c_long((1 << 31) - 1), C.byref(n)) == -2
    assert entry(C.c_long(1), C.c_long((1 << 31) - 1), C.c_long(1), C.byref(n)) == -2


@pytest.mark.parametrize("scope,state", [(lambda: AG.tape8(), lambda: AG._TAPE8["on"]), (lambda: AG.accumulate_param_grads(), lambda: AG._ACCUM["on"])])
def test_a_training_scope_belongs_to_its_thread(scope, state, monkeypatch):
    """a thread that trains beside one inside the scope does not see it, and threads that enter and leave overlapping leave it off"""
    monkeypatch.setattr(AG, "ACCUM_PARAM_GRADS", True)
    seen, steps = {}, [threading.Event() for _ in range(3)]

    def first():
        with scope():
            steps[0].set()
            steps[1].wait(10)
            seen["first"] = state()
        steps[2].set()

    def second():
        steps[0].wait(10)
        seen["before"] = state()
        with scope():
            steps[1].set()
            steps[2].wait(10)
            seen["second"] = state()
        seen["after"] = state()
    threads = [threading.Thread(target=f) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(20)
    assert seen == {"first": True, "before": False, "second": True, "after": False}
    assert not state()


def test_one_scope_object_in_two_threads():
    both, inside, leave, after = AG.tape8(), threading.Event(), threading.Event(), []

    def other():
        with AG.tape8(False), both:
            inside.set()
            leave.wait(10)
        after.append(AG._TAPE8["on"])
    t = threading.Thread(target=other)
    with both:
        t.start()
        inside.wait(10)
    assert not AG._TAPE8["on"]
    leave.set()
    t.join(20)
    assert after == [False]


def test_norm_join_keeps_a_tape_only_where_gradients_are_recorded(monkeypatch):
    asked = []

    def fake(x, f, *, tape, **kw):
        asked.append(tape)
        return ops.NormJoin(x + f, None)
    monkeypatch.setattr(ops, "norm_join", fake)
    x, gain = torch.randn(4, 8), torch.nn.Parameter(torch.ones(8))
    with torch.no_grad():
        AG.norm_join(x, x, post=(gain, None))
    assert asked == [False]
    AG.norm_join(x, x, post=(gain, None))
    AG.norm_join(x, x, post=(gain.detach(), None))
    assert asked == [False, True, False]


@pytest.mark.parametrize("side", ["post", "pre"])
def test_norm_join_refuses_a_norm_without_a_gain(side):
    """(as ops.norm_join does: a bias without a gain is no norm of this kind, not an absent one)"""
    x, v = torch.randn(4, 8), torch.ones(8)
    for bad in ((None, v), (None, None), (v,), (v, v, v), v):
        with pytest.raises(ValueError, match=side):
            AG.norm_join(x, x, **{side: bad})
