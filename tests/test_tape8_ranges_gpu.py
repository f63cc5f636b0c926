"""A Linear walked back from an 8-bit tape: what each row of dx and each column block of dW owes to its own magnitudes, the launches with
and without conditions at every shape of workgroup."""
import math

import pytest
import torch

from tests.test_tape8_gpu import linear_case, ref_values

pytestmark = pytest.mark.gpu
ACTS = ["relu", "none", "swish"]


def own_ref(dz, t, w, act):
    """(dx, dW, db) in 64 bits and a bound for each value, from the magnitudes that it is made of.

    dz goes as two fp16 pieces of dz 2^s with the row's largest magnitude in [2^14, 2^15): rounding the high piece leaves 2^-11, rounding
    the low one 2^-11 of that, or half of fp16's smallest number, 2^-25 against 2^14: 2^-39 of the row's largest.  w likewise, a column's
    largest from 2^13: 2^-38 of it.  The product of the low pieces is left out: 2^-22.  Together under 2^-20 of |dz| |w|.
    A sum of n terms in fp32 is off by n 2^-24 of the sum of magnitudes, three products a term.
    dW: the tape's values enter times a power of two that puts the largest product of a row's largest dz and its block's step at code 2^5 or up
    to 2^3 below (room for larger ones): codes 2^25 and more below that largest product lose what lies under 2^-25 there: with |dz| of the row
    at 2^15 of its largest, the code's step 2^5 at the top and 2^3 of room, 2^(15 - 25 - 14 - 5 + 3) = 2^-26 |dz| / (the row's largest)
    of that product.  Swish's value takes two pieces: 2^-22 of it, and in every row half of 2^-24, where the largest product of a row's
    largest dz and its block's largest value lies at 2^14 or up to 2^4 below: 2^(15 - 25 - 14 - 14 + 4) = 2^-34 of that product.  Its
    exponential's argument is off by 2^-23 of itself."""
    z, wd = dz.double(), w.double()
    v = ref_values(t.codes, t.bytes, t.width, t.kind).to(dz.device)
    step = torch.where(t.bytes == 0, 0.0, torch.exp2(t.bytes.double() - 127)).repeat_interleave(32, 1)[:, :t.width]
    M, N = z.shape
    if act == "swish":
        p = torch.sigmoid(v)
        one = v * p * torch.sigmoid(-v)
        d, x = p + one, v * p
        ex = 2.0 ** -19 * (1 + v.abs().clamp(max=128) / 8)
        ed = ex * (p + one.abs()) + 2.0 ** -118
    else:
        d, x, ex = (v > 0).double() if act == "relu" else torch.ones_like(v), v, torch.zeros_like(v)
        ed = ex
    tops = z.abs().amax(1, keepdim=True)
    s = z.abs() @ wd.abs()
    dx = d * (z @ wd)
    bx = (d.abs() * ((2.0 ** -20 + 3 * N * 2.0 ** -24) * s + 2.0 ** -39 * tops * wd.abs().sum(0) + 2.0 ** -38 * wd.abs().amax(0) * z.abs().sum(1, keepdim=True))
          + ed * s + 2.0 ** -20 * ed * s + 2.0 ** -126)
    if act == "swish":
        step = torch.stack([x[:, c:c + 32].abs().amax(1) for c in range(0, t.width, 32)], 1).repeat_interleave(32, 1)[:, :t.width]
    prod = tops * step
    top = torch.stack([prod[:, c:c + 32].amax() for c in range(0, t.width, 32)]).repeat_interleave(32)[:t.width]
    low = torch.ones_like(prod) if act == "swish" else (prod < 2.0 ** -24 * top).double()
    share = torch.where(tops > 0, z.abs() / tops, torch.zeros_like(z))
    n = max(64, M / 128 + 512)
    bw = ((2.0 ** -20 + n * 2.0 ** -24) * (z.abs().t() @ x.abs()) + z.abs().t() @ (ex * x.abs()) + 2.0 ** -39 * tops.t() @ x.abs()
          + 2.0 ** (-34 if act == "swish" else -26) * (share.t() @ low) * top + 2.0 ** -126)
    return (dx, z.t() @ x, z.sum(0)), (bx, bw, (2.0 ** -23 + n * 2.0 ** -24) * z.abs().sum(0))


def check_own(dz, t, w, act, got):
    want, bound = own_ref(dz, t, w, act)
    for name, g, r, b in zip(("dx", "dW", "db"), got, want, bound):
        off = (g.double() - r).abs()
        assert bool((off <= b).all()), (name, float((off / b).max()), int((off > b).sum()), float(off.max()))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(64, 64, 64), (65, 64, 64), (4099, 64, 64), (4099, 128, 64), (4099, 64, 128), (333, 128, 128), (1001, 100, 200),
                                   (333, 128, 384), (129, 4, 1152), (97, 60, 36), (70, 99, 128), (63, 128, 128), (300, 256, 256), (9, 129, 65)])
def test_every_shape_of_workgroup(act, M, N, K):
    """widths of 64 and 128 and the blocks of wider ones, a last step that repeats rows, lanes whose columns do not exist; rows and columns of
    different magnitude"""
    from magnet_amd import ops
    dz, t, w = linear_case(M, N, K, act, seed=M + 3 * N + K, spread=2.0)
    dz = dz * torch.exp2(-20.0 * (torch.arange(N, device="cuda") % 3 == 1).float())
    got = ops.tape8_linear_bwd(dz, t, w, act)
    check_own(dz, t, w, act, got)
    again = ops.tape8_linear_bwd(dz, t, w, act)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(300, 96, 128), (5000, 128, 128), (700, 64, 64), (301, 130, 70), (20, 33, 40)])
def test_a_row_of_dx_is_its_own(act, M, N, K):
    """rows whose magnitudes lie 2^60 apart in no order: each row of dx has the bits that it has alone, however large the other rows are, and is
    right for its own size"""
    from magnet_amd import ops
    dz, t, w = linear_case(M, N, K, act, seed=M)
    dz = dz * torch.exp2(torch.randint(-40, 21, (M, 1), device="cuda").float())
    got = ops.tape8_linear_bwd(dz, t, w, act)
    check_own(dz, t, w, act, got)
    loud = dz.clone()
    loud[::7] *= 2.0 ** 50
    dx = ops.tape8_linear_bwd(loud, t, w, act)[0]
    rest = torch.arange(M, device="cuda") % 7 != 0
    assert torch.equal(dx[rest], got[0][rest])
    for r in (1, M // 2, M - 1):
        alone = ops.tape8_linear_bwd(dz[r:r + 1], ops.Tape8(t.codes[r:r + 1].clone(), t.bytes[r:r + 1].clone(), K, t.kind), w, act)[0]
        assert torch.equal(alone[0], got[0][r]), r


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(1500, 128, 128), (700, 64, 64), (515, 100, 200), (40, 20, 77)])
def test_a_block_of_columns_of_dw_is_its_own(act, M, N, K):
    """blocks of 32 columns of the tape that are 2^50 apart: dW of the small ones is as good as of the large ones"""
    from magnet_amd import ops
    dz, _, w = linear_case(M, N, K, act, seed=K)
    far = torch.tensor([0.0, -50.0, 3.0, -31.0, -12.0, -40.0, 2.0], device="cuda").repeat_interleave(32)[:K]
    x = torch.randn(M, K, device="cuda") * torch.exp2(far + torch.randn(M, 1, device="cuda"))
    t = ops.tape8_pack(x, "relu" if act == "relu" else "signed")
    check_own(dz, t, w, act, ops.tape8_linear_bwd(dz, t, w, act))


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N,K", [(300, 128, 128), (300, 64, 64), (200, 96, 200), (31, 33, 40), (70, 200, 100)])
def test_a_column_of_dx_is_its_own(act, M, N, K):
    """columns of the weight 2^60 apart, neighbours among them: each column of dx has the bits that it has beside others of its own size"""
    from magnet_amd import ops
    dz, t, w = linear_case(M, N, K, act, seed=N)
    w = w * torch.exp2(torch.randint(-60, 1, (K,), device="cuda").float())
    got = ops.tape8_linear_bwd(dz, t, w, act)
    check_own(dz, t, w, act, got)
    loud = w.clone()
    loud[:, ::5] *= 2.0 ** 40
    rest = torch.arange(K, device="cuda") % 5 != 0
    assert torch.equal(ops.tape8_linear_bwd(dz, t, loud, act)[0][:, rest], got[0][:, rest])


@pytest.mark.parametrize("act", ["relu", "none"])
@pytest.mark.parametrize("M,N,K", [(1500, 128, 128), (700, 64, 64), (301, 70, 45)])
def test_large_gradients_of_small_rows(act, M, N, K):
    """rows of dz 2^a times, rows of the tape 2^-a times as large: every row's share of dW is of the same order"""
    from magnet_amd import ops
    torch.manual_seed(M)
    a = torch.randint(-30, 31, (M, 1), device="cuda").float()
    t = ops.tape8_pack(torch.randn(M, K, device="cuda") * torch.exp2(-a), "relu" if act == "relu" else "signed")
    dz, w = torch.randn(M, N, device="cuda") * torch.exp2(a - 20), torch.randn(N, K, device="cuda") / K ** 0.5
    got = ops.tape8_linear_bwd(dz, t, w, act)
    check_own(dz, t, w, act, got)
    want = own_ref(dz, t, w, act)[0]
    assert float((got[1].double() - want[1]).norm()) <= 2.0 ** -18 * float(want[1].norm())


@pytest.mark.parametrize("act", ["relu", "none"])
def test_rows_that_lie_far_below_the_largest_add_up(act):
    """one row is 2^28 times as large as 4000 others: their codes lose bits, their sum is still there"""
    from magnet_amd import ops
    torch.manual_seed(2)
    M, N, K = 4000, 64, 64
    dz = torch.randn(M, N, device="cuda")
    x = torch.randn(M, K, device="cuda")
    dz[0] *= 2.0 ** 14
    x[0] = x[0].abs() * 2.0 ** 14
    x[0, 1:] = 0                                          # (column 0 alone has it: the other columns' sums are the small rows')
    t = ops.tape8_pack(x, "relu" if act == "relu" else "signed")
    w = torch.randn(N, K, device="cuda")
    got = ops.tape8_linear_bwd(dz, t, w, act)
    check_own(dz, t, w, act, got)
    z, v = dz.double(), ref_values(t.codes, t.bytes, K, t.kind).cuda()
    want = (z.t() @ v)[:, 1:32]
    assert float((got[1][:, 1:32].double() - want).norm()) <= 2.0 ** -4 * float(want.norm())


def test_zero_rows_and_rows_that_are_not_finite():
    """rows of zeros, and rows without one finite value, beside ordinary and tiny ones"""
    from magnet_amd import ops
    for act in ACTS:
        dz, t, w = linear_case(200, 64, 96, act, seed=4)
        dz = dz * torch.exp2(torch.randint(-30, 1, (200, 1), device="cuda").float())
        dz[5::9] = 0
        got = ops.tape8_linear_bwd(dz, t, w, act)
        check_own(dz, t, w, act, got)
        assert not got[0][5::9].any()
        z = dz.clone()
        z[7] = math.nan
        z[8] = math.inf
        dx = ops.tape8_linear_bwd(z, t, w, act)[0]
        keep = torch.ones(200, dtype=torch.bool, device="cuda")
        keep[7:9] = False
        assert torch.equal(dx[keep], got[0][keep])
        on = t.codes[7, :96] != 0 if act == "relu" else torch.ones(96, dtype=torch.bool, device="cuda")
        assert torch.isnan(dx[7][on]).all()
        everything = ops.tape8_linear_bwd(torch.zeros_like(dz), t, w, act)
        assert not any(o.any() for o in everything)
        tiny = torch.full_like(dz, 1e-44) * torch.randint(-3, 4, dz.shape, device="cuda")       # subnormal: multiples of 2^-149
        check_own(tiny, t, w, act, ops.tape8_linear_bwd(tiny, t, w, act))


def test_far_arguments_of_swish():
    """Swish and its derivative from the most negative argument that a tape holds to the largest: 0, v e^v on the way, v and 1"""
    from magnet_amd import ops
    for v0 in (-1e38, -1e34, -1e6, -1000.0, -200.0, -104.0, -90.0, -88.0, -87.0, -86.0, -60.0, -20.0, -1.25, -1e-3, 0.0, 1e-30, 0.7, 20.0, 90.0, 1e6, 1e34, 1e38):
        x = torch.zeros(2, 32, device="cuda")
        x[:, 3] = v0
        t = ops.tape8_pack(x)
        dz, w = torch.ones(2, 1, device="cuda"), torch.ones(1, 32, device="cuda")
        dx, dW, _ = ops.tape8_linear_bwd(dz, t, w, "swish")
        v = ref_values(t.codes, t.bytes, 32, "signed")[0, 3]
        s, r = torch.sigmoid(v), torch.sigmoid(-v)
        one = float(v * s * r)
        # (the exponential's argument is off by 2^-23 of itself; under -87 the value, under 2^-118, is taken as 0)
        rel = 2.0 ** -19 * (1 + min(abs(float(v)), 128.0) / 8)
        assert abs(float(dx[0, 3]) - float(s + v * s * r)) <= rel * (float(s) + abs(one)) + 2.0 ** -118, v0
        assert abs(float(dW[0, 3]) - 2 * float(v * s)) <= 2 * rel * abs(float(v * s)) + 2.0 ** -117, v0
        assert v0 > -1e3 or (float(dx[0, 3]) == 0.0 and float(dW[0, 3]) == 0.0)


@pytest.mark.parametrize("act", ACTS)
def test_a_very_wide_weight(act):
    """more than 65 536 blocks of columns; and a workspace that does not grow with the width"""
    from magnet_amd import ops
    K = 65536 * 128 + 261
    t = ops.tape8_pack(torch.randn(3, K, device="cuda"), "relu" if act == "relu" else "signed")
    dz, w = torch.randn(3, 2, device="cuda"), torch.randn(2, K, device="cuda")
    dx, dW, db = ops.tape8_linear_bwd(dz, t, w, act)
    for a in (0, 4096 - 32, 65535 * 128, K // 32 * 32 - 4096):     # pieces of it, from blocks of 32 columns
        b = min(a + 4200, K)
        part = ops.Tape8(t.codes[:, a:(b + 31) // 32 * 32].contiguous(), t.bytes[:, a // 32:(b + 31) // 32].contiguous(), b - a, t.kind)
        want = ops.tape8_linear_bwd(dz, part, w[:, a:b], act)
        assert torch.allclose(dx[:, a:b], want[0], rtol=1e-5, atol=1e-5) and torch.allclose(dW[:, a:b], want[1], rtol=1e-5, atol=1e-5) and torch.equal(db, want[2])
        check_own(dz, part, w[:, a:b], act, want)


@pytest.mark.parametrize("act", ACTS)
def test_weights_wider_than_one_launch(act):
    from magnet_amd import ops
    dz, t, w = linear_case(200, 5, 9000, act, seed=1)
    got = ops.tape8_linear_bwd(dz, t, w, act)
    check_own(dz, t, w, act, got)
    dW, db = torch.ones_like(got[1]), torch.ones_like(got[2])
    ops.tape8_linear_bwd(dz, t, w, act, dW=dW, db=db, accumulate=True)
    assert torch.equal(dW, 1 + got[1]) and torch.equal(db, 1 + got[2])
    dz, t, w = linear_case(70, 131, 8300, act, seed=2)
    check_own(dz, t, w, act, ops.tape8_linear_bwd(dz, t, w, act))
