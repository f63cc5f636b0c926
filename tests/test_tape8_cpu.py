"""What the 8-bit tape's operators refuse, on any machine: nothing here launches a kernel (every wrong call is found before the device is
looked at, and a right one on the CPU ends with "no CPU path")."""
import pytest
import torch

from magnet_amd import _lib, ops


def tape(M, W, kind="signed"):
    return ops.tape8_empty(M, W, kind, "cpu")


def test_right_calls_need_a_device():
    x = torch.randn(4, 40)
    for call in (lambda: ops.tape8_pack(x), lambda: ops.tape8_unpack(tape(4, 40)),
                 lambda: ops.tape8_linear_bwd(torch.randn(4, 8), tape(4, 40), torch.randn(8, 40)),
                 lambda: ops.norm_join(x, x, post=(torch.ones(40), None), norm="rms"),
                 lambda: ops.norm_join_bwd(x, post_tape=tape(4, 40))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()


def test_pack_refusals():
    with pytest.raises(ValueError, match="kind"):
        ops.tape8_pack(torch.randn(4, 4), "unsigned")
    with pytest.raises(TypeError, match="float64"):
        ops.tape8_pack(torch.randn(4, 4, dtype=torch.float64))
    with pytest.raises(TypeError, match="tensor"):
        ops.tape8_pack([[1.0]])
    for shape in ((4,), (2, 3, 4), (4, 0)):
        with pytest.raises(ValueError, match="shape"):
            ops.tape8_pack(torch.randn(*shape))
    with pytest.raises(ValueError, match="kind|tape"):
        ops.tape8_pack(torch.randn(4, 4), "relu", out=tape(4, 4))
    with pytest.raises(ValueError, match="expected 4 of 4"):
        ops.tape8_pack(torch.randn(4, 4), out=tape(5, 4))
    with pytest.raises(ValueError):
        ops.tape8_empty(4, 0)


def test_unpack_refusals():
    with pytest.raises(TypeError, match="Tape8"):
        ops.tape8_unpack(torch.zeros(4, 4))
    with pytest.raises(TypeError, match="float64"):
        ops.tape8_unpack(tape(4, 4), dtype=torch.float64)
    good = tape(4, 40)
    for bad in (ops.Tape8(good.codes[:, :32], good.bytes, 40), ops.Tape8(good.codes, good.bytes[:3], 40), ops.Tape8(good.codes.float(), good.bytes, 40),
                ops.Tape8(good.codes, good.bytes, 70), ops.Tape8(good.codes, good.bytes, 40, "other"),
                ops.Tape8(torch.empty(4 * 64 + 1, dtype=torch.uint8)[1:].view(4, 64), good.bytes, 40)):
        with pytest.raises(ValueError):
            ops.tape8_unpack(bad)


def test_linear_bwd_refusals():
    dz, w = torch.randn(6, 8), torch.randn(8, 40)
    go = ops.tape8_linear_bwd
    with pytest.raises(ValueError, match="act"):
        go(dz, tape(6, 40), w, act="gelu")
    with pytest.raises(ValueError, match="'relu'"):
        go(dz, tape(6, 40), w, act="relu")
    with pytest.raises(ValueError, match="'signed'"):
        go(dz, tape(6, 40, "relu"), w)
    with pytest.raises(ValueError, match="columns"):
        go(dz[:, :7], tape(6, 40), w)
    with pytest.raises(ValueError, match="expected 6 of 40"):
        go(dz, tape(6, 41), w)
    with pytest.raises(ValueError, match="expected 6 of 40"):
        go(dz, tape(5, 40), w)
    with pytest.raises(TypeError, match="bfloat16"):
        go(dz.bfloat16(), tape(6, 40), w)
    with pytest.raises(ValueError, match="accumulate"):
        go(dz, tape(6, 40), w, accumulate=True)
    for kw in (dict(dx=torch.empty(6, 41)), dict(dW=torch.empty(40, 8)), dict(db=torch.empty(9)), dict(dW=torch.empty(40, 8).t()),
               dict(dx=torch.empty(6, 40, dtype=torch.float16))):
        with pytest.raises(ValueError):
            go(dz, tape(6, 40), w, **kw)
    big = torch.randn(6, 80)
    with pytest.raises(ValueError, match="overlap"):
        go(big[:, 20:60], tape(6, 40), torch.randn(40, 40), dx=big[:, :40])
    with pytest.raises(ValueError, match="overlap"):
        go(dz, tape(6, 40), w, dW=w)


def test_norm_join_refusals():
    x = torch.randn(6, 40)
    g, b = torch.ones(40), torch.zeros(40)
    with pytest.raises(ValueError, match="at most"):
        ops.norm_join(torch.randn(2, 4097), torch.randn(2, 4097))
    with pytest.raises(ValueError, match="norm 'batch'"):
        ops.norm_join(x, x, norm="batch")
    with pytest.raises(TypeError, match="float16"):
        ops.norm_join(x.half(), x.half())
    with pytest.raises(TypeError, match="bfloat16"):
        ops.norm_join(x, x.bfloat16())
    with pytest.raises(ValueError, match="expected"):
        ops.norm_join(x, x[:5])
    for bad in (g, (None, b), (g,), (g[:39], b), (g.double(), b), (g, b[:39])):
        with pytest.raises(ValueError):
            ops.norm_join(x, x, post=bad)
    for gate in (torch.ones(4, 40), torch.ones(6, 39), torch.ones(0, 40), torch.ones(12, 40)):
        with pytest.raises(ValueError):
            ops.norm_join(x, x, gate=gate)
    with pytest.raises(TypeError):
        ops.norm_join(x, x, gate=torch.ones(6, 40).bfloat16())
    with pytest.raises(ValueError, match="scale"):
        ops.norm_join(x, x, scale=torch.ones(()))
    t, r = tape(6, 40), torch.ones(6)
    with pytest.raises(ValueError, match="gh"):
        ops.norm_join_bwd(x, x, post_tape=t)
    with pytest.raises(ValueError, match="gh"):
        ops.norm_join_bwd(x, post_tape=t, pre=(g, b))
    with pytest.raises(TypeError, match="pre_tape"):
        ops.norm_join_bwd(x, x, post_tape=t, pre=(g, b))
    with pytest.raises(TypeError, match="post_rstd"):
        ops.norm_join_bwd(x, post_tape=t, post=(g, b))
    with pytest.raises(ValueError, match="post_rstd"):
        ops.norm_join_bwd(x, post_tape=t, post=(g, b), post_rstd=r[:5])
    with pytest.raises(ValueError, match="expected 6 of 40"):
        ops.norm_join_bwd(x, post_tape=tape(6, 72))


def test_c_entries_refuse():
    """the C entries check what they can by themselves: -2, nothing launched (no device here)"""
    import ctypes as C
    L = _lib.lib()
    z, one, n = C.c_void_p(0), C.c_void_p(16), C.c_long(0)
    long = C.c_long
    assert L.magnet_tape8_pack(one, 3, long(4), long(1), 4, 0, one, one, z) == -2          # no such type
    assert L.magnet_tape8_pack(one, 0, long(3), long(1), 4, 0, one, one, z) == -2          # stride under the width
    assert L.magnet_tape8_pack(one, 0, long(4), long(1), 4, 2, one, one, z) == -2          # no such kind
    assert L.magnet_tape8_pack(one, 0, long(4), long(1), 4, 0, C.c_void_p(8), one, z) == -2
    assert L.magnet_tape8_pack(one, 0, long(4), long(0), 4, 0, one, one, z) == 0           # no rows: nothing to do
    assert L.magnet_tape8_unpack(one, one, long(-1), 4, 0, one, 0, long(4), z) == -2
    assert L.magnet_tape8_linear_bwd_workspace(long(100), long(0), long(4), C.byref(n)) == -2
    assert L.magnet_tape8_linear_bwd_workspace(long(100), long(128), long(128), C.byref(n)) == 0 and n.value == 4 * (128 * 128 + 128)
    assert L.magnet_norm_join_bwd_workspace(long(100), long(128), long(3), C.byref(n)) == -2      # 3 gates for 100 rows
    assert L.magnet_norm_join_bwd_workspace(long(100), long(4097), long(0), C.byref(n)) == -2


def test_the_context_nests_and_the_caller_s_stays():
    """one context object entered twice restores what was; a model without ``tape8`` trains as the surrounding context says, one with it
    in 8 bits"""
    import contextlib
    import types
    from magnet_amd import autograd as AG
    from magnet_amd.models.magnet_common import _RolloutScope
    both = AG.tape8()
    with both:
        with both:
            assert AG._TAPE8["on"]
        assert AG._TAPE8["on"]
        with AG.tape8(False):
            assert not AG._TAPE8["on"]
        assert AG._TAPE8["on"]
    assert not AG._TAPE8["on"]
    for outer in (False, True):
        for own in (False, True):
            model = types.SimpleNamespace(training=True, tape8=own, _guard=types.SimpleNamespace(armed=contextlib.nullcontext))
            with AG.tape8(outer):
                with _RolloutScope(model):
                    assert AG._TAPE8["on"] is (outer or own)
                assert AG._TAPE8["on"] is outer
            assert not AG._TAPE8["on"]


def test_a_tape_is_kept_only_where_the_rows_that_become_it_fit(monkeypatch):
    """the chain's launch writes fp32 rows before they are packed: four times the tape, in memory for a moment"""
    from magnet_amd import autograd as AG
    monkeypatch.delenv("MAGNET_KEEP_TAPE", raising=False)
    monkeypatch.setattr(torch.cuda, "mem_get_info", lambda dev: (100 << 30, 288 << 30))
    monkeypatch.setattr(torch.cuda, "memory_reserved", lambda dev: 0)
    monkeypatch.setattr(torch.cuda, "memory_allocated", lambda dev: 0)
    monkeypatch.setenv("MAGNET_TAPE_CAP", "1.0")
    for passing, kept in ((0, True), (40 << 30, True), (60 << 30, False)):
        monkeypatch.setattr(AG, "_MEM", dict(dev=None, t=0.0, total=0, free=0, granted=0))
        assert AG._keep_tape(15 << 30, "a device", passing) is kept


def test_outputs_share_no_memory():
    """an output on top of an input, of the tape or of another output is refused (the rows are walked in no order)"""
    dz, w = torch.randn(6, 8), torch.randn(8, 40)
    both = torch.empty(400)
    for kw, names in ((dict(dW=both[:320].view(8, 40), db=both[319:327]), "db must not overlap dW"),
                      (dict(dx=both[:240].view(6, 40), dW=both[80:].view(8, 40)), "dW must not overlap dx")):
        with pytest.raises(ValueError, match=names):
            ops.tape8_linear_bwd(dz, tape(6, 40), w, **kw)
    mem = torch.zeros(6, 40)
    t = ops.Tape8(mem.view(torch.uint8).view(-1)[:6 * 64].view(6, 64), torch.zeros(6, 2, dtype=torch.uint8), 40)
    with pytest.raises(ValueError, match="dx must not overlap the tape"):
        ops.tape8_linear_bwd(dz, t, w, dx=mem)
    with pytest.raises(ValueError, match="out must not overlap x"):
        ops.tape8_pack(mem, out=t)
    with pytest.raises(ValueError, match="out must not overlap the tape"):
        ops.tape8_unpack(t, out=mem)
    t.codes, t.bytes = torch.zeros(6, 64, dtype=torch.uint8), mem.view(torch.uint8).view(-1)[100:112].view(6, 2)
    with pytest.raises(ValueError, match="out must not overlap x"):
        ops.tape8_pack(mem, out=t)
    t.bytes = t.codes.view(-1)[12:24].view(6, 2)
    with pytest.raises(ValueError, match="out must not overlap itself"):
        ops.tape8_pack(mem, out=t)
