"""The 8-bit tape on the GPU: its quantisation bit for bit, a Linear walked back from it, and the norms around a residual block - each against
its formula in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DT = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# --------------------------------------------------------------------------------------------------------------- the format, in 64 bits
def ref_pack(x, kind):
    """codes and bytes of x (any float type), from the definition, on the CPU in 64 bits"""
    x = x.detach().cpu().double()
    M, W = x.shape
    pad = -W % 32
    x = torch.nn.functional.pad(x, (0, pad)).view(M, -1, 32)
    most = 255.0 if kind == "relu" else 127.0
    seen = torch.where(x <= 0, torch.zeros_like(x), x) if kind == "relu" else x.abs()
    bad = ~torch.isfinite(seen).all(2)
    top = torch.where(torch.isfinite(seen), seen, torch.zeros_like(seen)).amax(2)
    e = torch.full_like(top, -126.0)
    for k in range(-126, 121):                            # the smallest exponent whose largest code reaches the top
        e = torch.where(most * math.ldexp(1.0, k) < top, torch.full_like(e, k + 1.0), e)
    step = torch.pow(2.0, e)[:, :, None]
    q = torch.round(x / step)
    if kind == "relu":
        # (of the largest step codes end at 127: what is finite comes back finite)
        q = torch.where(x > 0, torch.where(e[:, :, None] == 121, q.clamp(1, 127), q.clamp(1, 255)), torch.zeros_like(q))
        q = torch.where(bad[:, :, None], torch.where(x <= 0, 0.0, 255.0).double(), q)
    else:
        q = torch.where(bad[:, :, None], torch.zeros_like(q), q.clamp(-127, 127))
    byte = torch.where(bad, torch.full_like(e, 255.0), torch.where(top > 0, e + 127, torch.zeros_like(e)))
    return (q.long() & 255).to(torch.uint8).view(M, -1), byte.to(torch.uint8)


def ref_values(codes, byte, W, kind):
    c = codes.cpu().double()
    c = torch.where(c > 127, c - 256, c) if kind == "signed" else c
    s = torch.pow(2.0, byte.cpu().double() - 127)
    s = torch.where(byte.cpu() == 255, torch.full_like(s, math.nan), torch.where(byte.cpu() == 0, torch.zeros_like(s), s))
    return (c * s.repeat_interleave(32, 1))[:, :W]


def check_pack(x, kind):
    from magnet_amd import ops
    t = ops.tape8_pack(x, kind)
    codes, byte = ref_pack(x, kind)
    assert torch.equal(t.bytes.cpu(), byte)
    assert torch.equal(t.codes.cpu(), codes)
    want = ref_values(codes, byte, x.shape[1], kind)
    for dt in (torch.float32, torch.bfloat16):            # (both hold every code times every step exactly)
        got = ops.tape8_unpack(t, dtype=dt).cpu().double()
        same = (got == want) | (torch.isnan(got) & torch.isnan(want))
        assert bool(same.all()), (dt, int((~same).sum()))
        assert bool(torch.isfinite(got).all()) or bool((byte == 255).any())
    return t


@pytest.mark.parametrize("kind", ["relu", "signed"])
@pytest.mark.parametrize("dtype", ["fp32", "bf16", "fp16"])
@pytest.mark.parametrize("M,W", [(1, 1), (3, 31), (5, 32), (7, 33), (100, 128), (33, 200), (2, 1152), (4099, 25)])
def test_pack_is_the_definition(kind, dtype, M, W):
    torch.manual_seed(M * 1000 + W)
    x = torch.randn(M, W, device="cuda") * torch.exp2(4 * torch.randn(M, 1, device="cuda"))
    check_pack(x.to(DT[dtype]), kind)


@pytest.mark.parametrize("kind", ["relu", "signed"])
def test_pack_borders(kind):
    """tops at and next to a full code, halves (ties to even), zeros of both signs, subnormals, the largest numbers, what is not finite"""
    f = torch.finfo(torch.float32)
    rows = []
    for k in (-149, -140, -127, -126, -120, -20, 0, 30, 120, 121):
        for m in (255.0, 127.0, 128.0, 254.9999, 127.00001, 0.5, 1.0):
            v = m * 2.0 ** k if m * 2.0 ** k < f.max else f.max
            rows.append([v, -v / 2, v / 3, 0.0, -0.0, v / 255, v / 510, v / 600])
    for q in range(0, 254, 7):                             # exact halves under a step of 1
        rows.append([200.0, q / 2 + 0.5, -q / 2 - 0.5, 1.5, 2.5, -1.5, 0.5, -0.5])
    rows += [[f.max, -f.max, f.tiny, 1.0, 0, 0, 0, 0], [-f.max, f.tiny, -f.tiny, f.tiny / 8, 0, 0, 0, 0], [0.0] * 8, [-1.0] * 8]
    rows += [[math.nan, 1.0, -1.0, 0, 0, 0, 0, 0], [math.inf, 1.0, -1.0, 0, 0, 0, 0, 0], [-math.inf, 1.0, -1.0, 0, 0, 0, 0, 0],
             [1.0, -math.nan, 2.0, 0, 0, 0, 0, 0]]
    x = torch.tensor(rows, dtype=torch.float32, device="cuda")
    check_pack(x, kind)
    # two blocks a row: what is not finite stays in its own
    y = torch.cat([x, torch.zeros(x.shape[0], 24, device="cuda"), torch.ones(x.shape[0], 5, device="cuda")], 1)
    t = check_pack(y, kind)
    assert bool((t.bytes[:, 1] == t.bytes[0, 1]).all())


def test_pack_error_is_half_a_step():
    from magnet_amd import ops
    torch.manual_seed(3)
    x = torch.randn(513, 96, device="cuda")
    for kind in ("signed", "relu"):
        t = ops.tape8_pack(x, kind)
        want = x.clamp(min=0) if kind == "relu" else x
        step = torch.exp2(t.bytes.float() - 127).repeat_interleave(32, 1)
        off = (ops.tape8_unpack(t) - want).abs()
        assert bool((off <= step / 2 + (step / 2 if kind == "relu" else 0) * ((want > 0) & (want < step / 2))).all())
        assert bool(((t.codes != 0) == (want > 0)).all()) or kind == "signed"
        assert bool((step <= want.abs().view(513, 3, 32).amax(2).repeat_interleave(32, 1) * (2 / (127.0 if kind == "signed" else 255.0))).all())


def test_pack_strides_and_out():
    from magnet_amd import ops
    torch.manual_seed(4)
    big = torch.randn(50, 300, device="cuda")
    for x in (big[:, 4:104], big[:, 3:103], big[::2, 8:40], big.t(), big[:1, 1:2], big[:, :1].expand(50, 40)):
        t, c = ops.tape8_pack(x), ops.tape8_pack(x.contiguous())
        assert torch.equal(t.codes, c.codes) and torch.equal(t.bytes, c.bytes)
        out = torch.full((x.shape[0], x.shape[1] + 9), 7.0, device="cuda")
        for o in (1, 4):
            ops.tape8_unpack(t, out=out[:, o:o + x.shape[1]])
            assert torch.equal(out[:, o:o + x.shape[1]], ops.tape8_unpack(t))
            assert bool((out[:, o + x.shape[1]:] == 7.0).all()) and bool((out[:, :1] == 7.0).all())
    t = ops.tape8_empty(50, 300)
    assert ops.tape8_pack(big, out=t) is t and torch.equal(t.codes, ops.tape8_pack(big).codes)
    e = ops.tape8_pack(big[:0])
    assert e.rows == 0 and ops.tape8_unpack(e).shape == (0, 300)


# -------------------------------------------------------------------------------------------------------------- a Linear walked back
def linear_case(M, N, K, act, seed=0, spread=1.0):
    from magnet_amd import ops
    torch.manual_seed(seed)
    kind = "relu" if act == "relu" else "signed"
    t = ops.tape8_pack(torch.randn(M, K, device="cuda") * torch.exp2(spread * torch.randn(M, 1, device="cuda")), kind)
    dz = torch.randn(M, N, device="cuda") * torch.exp2(spread * torch.randn(M, 1, device="cuda") - 20)
    w = torch.randn(N, K, device="cuda") / K ** 0.5
    return dz, t, w


def linear_ref(dz, t, w, act):
    """(dx, dW, db) in 64 bits and, for each, the bound of this arithmetic: |dz|, |w|, |x| carry 2^-21 each (two fp16 pieces: the high one
    towards zero leaves under 2^-10, the low one halves 2^-11 of it), the product of the low pieces left out is under 2^-20, the tape's
    codes are exact; an addition in fp32 is off by 2^-24 of its result, so a sum of n terms by n 2^-24 of the sum of magnitudes; what lies
    2^-38 under the largest magnitude of dz (of w) is lost.  Swish: the exponential's argument is off by 2^-23 of itself."""
    z, wd = dz.double(), w.double()
    v = ref_values(t.codes, t.bytes, t.width, t.kind).to(dz.device)
    M, N, K = z.shape[0], z.shape[1], v.shape[1]
    if act == "swish":
        p = torch.sigmoid(v)
        d, x = p + v * p * torch.sigmoid(-v), v * p
        ex = 2.0 ** -19 * (1 + float(v.abs().max()) / 8)
    else:
        d, x, ex = (v > 0).double() if act == "relu" else torch.ones_like(v), v, 0.0
    top = float(z.abs().max()) if M else 0.0
    dx = d * (z @ wd)
    bx = d.abs() * ((2.0 ** -19 + N * 2.0 ** -24) * (z.abs() @ wd.abs()) + 2.0 ** -36 * top * float(wd.abs().max()) * N) + ex * dx.abs() + ex * (z.abs() @ wd.abs())
    # (at least 32 rows are added one after the other; more rows than 128 workgroups hold, M / 128 of them; then the workgroups)
    n = max(64, M / 128 + 512)
    bw = (2.0 ** -19 + ex + n * 2.0 ** -24) * (z.abs().t() @ x.abs()) + 2.0 ** -36 * top * x.abs().sum(0)
    return (dx, z.t() @ x, z.sum(0)), (bx, bw, (2.0 ** -23 + n * 2.0 ** -24) * z.abs().sum(0))


def check_linear(dz, t, w, act, got):
    want, bound = linear_ref(dz, t, w, act)
    for name, g, r, b in zip(("dx", "dW", "db"), got, want, bound):
        off = (g.double() - r).abs() - b
        assert off.numel() == 0 or float(off.max()) <= 0, (name, float(off.max()), float((g.double() - r).norm() / r.norm()))


@pytest.mark.parametrize("act", ["relu", "none", "swish"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (31, 25, 100), (33, 64, 64), (1000, 128, 128), (70001, 64, 128), (257, 128, 33), (4097, 130, 257),
                                   (5000, 300, 64), (129, 3, 1152)])
def test_linear_bwd(act, M, N, K):
    from magnet_amd import ops
    dz, t, w = linear_case(M, N, K, act, seed=M + N + K)
    got = ops.tape8_linear_bwd(dz, t, w, act)
    check_linear(dz, t, w, act, got)
    if act == "relu":
        assert bool((got[0][t.codes[:, :K] == 0] == 0).all())
    again = ops.tape8_linear_bwd(dz, t, w, act)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("act", ["relu", "none", "swish"])
@pytest.mark.parametrize("direction", [1, -1])
def test_linear_bwd_scales_grow_and_shrink(act, direction):
    """rows whose magnitudes run over 2^60 (of dz) and 2^20 (of the tape), upwards and downwards: every workgroup meets larger ones later"""
    from magnet_amd import ops
    torch.manual_seed(7)
    M, N, K = 33000, 96, 128
    run = torch.arange(M, device="cuda").float()[:, None] / M
    run = run if direction > 0 else 1 - run
    t = ops.tape8_pack(torch.randn(M, K, device="cuda") * torch.exp2(20 * run - 18), "relu" if act == "relu" else "signed")
    dz, w = torch.randn(M, N, device="cuda") * torch.exp2(60 * run - 40), torch.randn(N, K, device="cuda")
    check_linear(dz, t, w, act, ops.tape8_linear_bwd(dz, t, w, act))


@pytest.mark.parametrize("scale", [2.0 ** -120, 2.0 ** -60, 2.0 ** 60, 2.0 ** 100])
def test_linear_bwd_whole_range(scale):
    """the weights, the tape or dz as small or as large as fp32 lets the products be"""
    from magnet_amd import ops
    for which in range(3):
        dz, t, w = linear_case(300, 40, 70, "none", seed=which, spread=0.0)
        if which == 0:
            dz = dz * 2.0 ** 20 * scale
        elif which == 1:
            w = w * scale
        else:
            t = ops.tape8_pack(ops.tape8_unpack(t) * scale)
        got = ops.tape8_linear_bwd(dz, t, w)
        want, _ = linear_ref(dz, t, w, "none")
        for g, r in zip(got, want):
            # (results under 2^-126 are multiples of 2^-149: two roundings of half of it each, per value)
            assert float((g.double() - r).norm()) <= 2.0 ** -18 * float(r.norm()) + g.numel() ** 0.5 * 2.0 ** -149


def test_linear_bwd_not_finite():
    """a gradient that is not finite reaches its row of dx and its column's sums, a block that is not finite its own columns of dW; the rest is as
    it would be without"""
    from magnet_amd import ops
    dz, t, w = linear_case(200, 64, 96, "relu", seed=5)
    clean = ops.tape8_linear_bwd(dz, t, w, "relu")
    for bad in (math.nan, math.inf, -math.inf):
        z = dz.clone()
        z[77, 3] = bad
        dx, dW, db = ops.tape8_linear_bwd(z, t, w, "relu")
        on = t.codes[77] != 0
        assert not torch.isfinite(dx[77][on]).any() and not torch.isfinite(dW[3][(t.codes[77] != 0)]).any() and not torch.isfinite(db[3])
        rows, cols = torch.arange(200, device="cuda") != 77, torch.arange(64, device="cuda") != 3
        assert torch.equal(dx[rows], clean[0][rows]) and torch.equal(dW[cols], clean[1][cols]) and torch.equal(db[cols], clean[2][cols])
    x = ops.tape8_unpack(t)
    x[13, 40] = math.nan
    t2 = ops.tape8_pack(x, "relu")
    dx, dW, db = ops.tape8_linear_bwd(dz, t2, w, "relu")
    assert torch.isnan(dW[:, 32:64]).all() and torch.equal(dW[:, :32], clean[1][:, :32]) and torch.equal(dW[:, 64:], clean[1][:, 64:])
    keep = torch.ones(200, 96, dtype=torch.bool, device="cuda")
    keep[13, 32:64] = False
    assert torch.equal(dx[keep], clean[0][keep]) and torch.equal(db, clean[2]) and torch.isfinite(dx).all()


def test_linear_bwd_outputs_strides_and_accumulate():
    from magnet_amd import ops
    dz, t, w = linear_case(777, 60, 100, "relu", seed=8)
    want = ops.tape8_linear_bwd(dz, t, w, "relu")
    wide_z, wide_x, wide_w = (torch.full((s[0], s[1] + 11), 5.0, device="cuda") for s in (dz.shape, (777, 100), w.shape))
    for o in (4, 3):                                       # 16-byte aligned columns and not
        wide_z[:, o:o + 60], wide_w[:, o:o + 100] = dz, w
        dW, db = torch.ones(60, 100, device="cuda"), torch.ones(60, device="cuda")
        wide_x.fill_(5.0)
        dx, a, b = ops.tape8_linear_bwd(wide_z[:, o:o + 60], t, wide_w[:, o:o + 100], "relu", dx=wide_x[:, o:o + 100], dW=dW, db=db, accumulate=True)
        assert a is dW and b is db
        assert torch.equal(dx, want[0]) and torch.equal(dW, 1 + want[1]) and torch.equal(db, 1 + want[2])
        assert bool((wide_x[:, :o] == 5.0).all()) and bool((wide_x[:, o + 100:] == 5.0).all())
    none, a, b = ops.tape8_linear_bwd(dz, t, w, "relu", need_dx=False)
    assert none is None and torch.equal(a, want[1]) and torch.equal(b, want[2])
    empty = ops.tape8_pack(torch.empty(0, 100, device="cuda"), "relu")
    dx, a, b = ops.tape8_linear_bwd(dz[:0], empty, w, "relu")
    assert dx.shape == (0, 100) and not a.any() and not b.any()
    a.fill_(2.0), b.fill_(3.0)
    ops.tape8_linear_bwd(dz[:0], empty, w, "relu", dW=a, db=b, accumulate=True)
    assert bool((a == 2.0).all()) and bool((b == 3.0).all())


def test_linear_bwd_no_rows_of_a_large_weight():
    """more than 2^31 values of dW to clear"""
    from magnet_amd import ops
    n = 46400
    w = torch.empty(n, n, device="cuda")
    dW = torch.ones(n, n, device="cuda")
    _, a, b = ops.tape8_linear_bwd(torch.empty(0, n, device="cuda"), ops.tape8_empty(0, n), w, dW=dW)
    assert a is dW and not any(bool(rows.any()) for rows in dW.split(4096)) and not b.any()


def test_linear_bwd_one_buffer_for_several_gradients():
    """dW and db inside wider buffers, N in two blocks of 128: neighbours are left alone"""
    from magnet_amd import ops
    dz, t, w = linear_case(500, 150, 70, "none", seed=12)
    want = ops.tape8_linear_bwd(dz, t, w)
    flat = torch.full((150, 90), 4.0, device="cuda")
    tail = torch.full((160,), 4.0, device="cuda")
    dx, dW, db = ops.tape8_linear_bwd(dz, t, w, dW=flat[:, 7:77], db=tail[5:155])
    assert torch.equal(dx, want[0]) and torch.equal(flat[:, 7:77], want[1]) and torch.equal(tail[5:155], want[2])
    assert bool((flat[:, :7] == 4).all()) and bool((flat[:, 77:] == 4).all()) and bool((tail[:5] == 4).all()) and bool((tail[155:] == 4).all())


def test_offsets_beyond_32_bits():
    """17 000 000 rows of 128: the tape's offsets pass 2^31 bytes, the gradients' 2^32; the ends give what they give alone"""
    from magnet_amd import ops
    M, W, tail = 17_000_000, 128, 512
    x = torch.randn(4096, W, device="cuda", dtype=torch.bfloat16).repeat((M + 4095) // 4096, 1)[:M]
    x[-tail:] = torch.randn(tail, W, device="cuda").bfloat16()
    t = ops.tape8_pack(x, "relu")
    end = ops.tape8_pack(x[-tail:].clone(), "relu")
    assert torch.equal(t.codes[-tail:], end.codes) and torch.equal(t.bytes[-tail:], end.bytes)
    assert torch.equal(ops.tape8_unpack(t, torch.bfloat16)[-tail:], ops.tape8_unpack(end, torch.bfloat16))
    del x
    dz = torch.zeros(M, W, device="cuda")
    dz[-tail:] = torch.randn(tail, W, device="cuda") * 1e-6
    w = torch.randn(W, W, device="cuda") / 11
    dx, dW, db = ops.tape8_linear_bwd(dz, t, w, "relu")
    want, bound = linear_ref(dz[-tail:], end, w, "relu")
    for g, r, b in zip((dx[-tail:], dW, db), want, bound):
        assert float(((g.double() - r).abs() - b).max()) <= 0
    assert not dx[:-tail].any()
    del dx, t
    z = torch.zeros(M, W, device="cuda")
    z[-tail:] = torch.randn(tail, W, device="cuda")
    one = (torch.ones(W, device="cuda"), None)
    r = ops.norm_join(dz, z, post=one, tape=True)
    e = ops.norm_join(dz[-tail:].clone(), z[-tail:].clone(), post=one, tape=True)
    assert torch.equal(r.y[-tail:], e.y) and torch.equal(r.post_tape.codes[-tail:], e.post_tape.codes) and torch.equal(r.post_rstd[-tail:], e.post_rstd)
    del r.y
    g = ops.norm_join_bwd(z, post_tape=r.post_tape, post_rstd=r.post_rstd, post=one)
    ge = ops.norm_join_bwd(z[-tail:].clone(), post_tape=e.post_tape, post_rstd=e.post_rstd, post=one)
    assert torch.equal(g.f[-tail:], ge.f) and torch.equal(g.x[-tail:], ge.x)


# ------------------------------------------------------------------------------------------------------ norms around a residual block
EPS = 1e-5


def join_case(M, W, G, norm, post, pre, vec, dt, seed=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    r = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    pair = lambda on: ((1 + 0.2 * r(W), 0.3 * r(W) if norm == "layer" else None) if on else None)  # noqa: E731
    return dict(x=(2 * r(M, W)).to(dt), f=(3 * r(M, W) + 1).to(dt), post=pair(post), pre=pair(pre), gate=torch.sigmoid(r(G, W)).to(dt) if G else None,
                scale=0.7 + 0.2 * r(W) if vec else 0.7, norm=norm)


def ref_norm(v, norm):
    v = v - v.mean(1, keepdim=True) if norm == "layer" else v
    r = ((v * v).mean(1, keepdim=True) + EPS) ** -0.5
    return v * r, r[:, 0]


def ref_affine(v, p):
    if p is None:
        return v
    return v * p[0] + (p[1] if p[1] is not None else 0.0)


def ref_gate(c, M):
    return 1.0 if c["gate"] is None else c["gate"].repeat_interleave(M // c["gate"].shape[0], 0)


def as64(c):
    d = lambda v: v.double() if isinstance(v, torch.Tensor) else tuple(d(u) for u in v) if isinstance(v, tuple) else v  # noqa: E731
    return {k: d(v) for k, v in c.items()}


def ref_join(c):
    """y, h and the two normalised rows with their factors, in 64 bits"""
    c = as64(c)
    M = c["x"].shape[0]
    fh, fr = ref_norm(c["f"], c["norm"]) if c["post"] else (c["f"], None)
    y = c["x"] + c["scale"] * ref_gate(c, M) * ref_affine(fh, c["post"])
    if not c["pre"]:
        return y, None, (fh, fr), (None, None)
    yh, yr = ref_norm(y, c["norm"])
    return y, ref_affine(yh, c["pre"]), (fh, fr), (yh, yr)


# A norm in fp32: the mean and the mean square over W terms are tree sums, off by a few 2^-24 times log2(W) < 13; the factor's root and
# quotient add 2^-23; a value less its mean is off by 2^-24 of the LARGER of the two, here under 4 deviations.  Each normalised value is off
# by at most about (13 + 2 + 8) 2^-24 of the row's deviation, twice that behind the second norm: 64 2^-24 of the array's norm bounds it.
REL32 = 64 * 2.0 ** -24


def near(got, want, dt, rel=REL32):
    if want is None:
        assert got is None
        return
    off = (got.double() - want).abs()
    if dt == torch.bfloat16:                               # ... plus one rounding to bf16, half a step of the value
        off = (off - 2.0 ** -8 * want.abs()).clamp(min=0)
    top = float(want.norm())
    assert float(off.norm()) <= rel * top + 1e-30, (float(off.norm()), top)


CASES = [(1, 1, 0), (5, 16, 0), (100, 128, 0), (100, 128, 2), (37, 100, 37), (64, 64, 1), (33, 33, 3), (2049, 128, 683), (9000, 36, 4500),
         (130, 256, 130), (77, 512, 7), (66, 1000, 66), (12, 1024, 0), (9, 1025, 3), (10, 2048, 10), (5, 4096, 5), (3, 3333, 1)]


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("M,W,G", CASES)
def test_norm_join_forward(dtype, norm, M, W, G):
    from magnet_amd import ops
    for post, pre, vec in ((True, True, True), (True, False, False), (False, True, True), (False, False, False)):
        c = join_case(M, W, G, norm, post, pre, vec, DT[dtype], seed=M + W)
        y, h, (fh, fr), (yh, yr) = ref_join(c)
        r = ops.norm_join(**c, tape=True)
        near(r.y, y, DT[dtype])
        near(r.h, h, DT[dtype])
        near(r.post_rstd, fr, torch.float32)
        near(r.pre_rstd, yr, torch.float32)
        for t, v in ((r.post_tape, fh), (r.pre_tape, yh)):
            if v is None:
                assert t is None
                continue
            step = torch.where(t.bytes == 0, torch.zeros((), device="cuda"), torch.exp2(t.bytes.float() - 127)).double().repeat_interleave(32, 1)[:, :W]
            assert float(((ops.tape8_unpack(t).double() - v).abs() - step / 2).max()) <= REL32 * max(1.0, float(v.abs().max()))
            assert not t.codes[:, W:].any()
        plain = ops.norm_join(**c)
        assert torch.equal(plain.y, r.y) and plain.post_tape is None and (h is None or torch.equal(plain.h, r.h))


def ref_join_bwd(c, gy, gh, fh, fr, yh, yr):
    """gradients from the taped rows, in 64 bits"""
    c, M = as64(c), gy.shape[0]

    def back(u, v, r):
        return r[:, None] * (u - (u.mean(1, keepdim=True) if c["norm"] == "layer" else 0.0) - v * (u * v).mean(1, keepdim=True))
    D, out = gy.double(), {}
    if c["pre"]:
        gh = gh.double()
        D = D + back(gh * c["pre"][0], yh, yr)
        out["pre"] = ((gh * yh).sum(0), gh.sum(0) if c["pre"][1] is not None else None)
    t, gate = ref_affine(fh, c["post"]), ref_gate(c, M)
    out["x"] = D
    if c["gate"] is not None:
        G = c["gate"].shape[0]
        out["gate"] = (D * c["scale"] * t).reshape(G, M // G, -1).sum(1)
    if isinstance(c["scale"], torch.Tensor):
        out["scale"] = (D * gate * t).sum(0)
    v = D * c["scale"] * gate
    if c["post"]:
        out["post"] = ((v * fh).sum(0), v.sum(0) if c["post"][1] is not None else None)
        v = back(v * c["post"][0], fh, fr)
    out["f"] = v
    return out


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("M,W,G", CASES)
def test_norm_join_backward(dtype, norm, M, W, G):
    from magnet_amd import ops
    dt = DT[dtype]
    for post, pre, vec in ((True, True, True), (True, False, False), (False, True, True), (False, False, False)):
        c = join_case(M, W, G, norm, post, pre, vec, dt, seed=M * 3 + W)
        r = ops.norm_join(**c, tape=True)
        gy, gh = (torch.randn(M, W, device="cuda") * 2e-6).to(dt), (torch.randn(M, W, device="cuda") * 1e-6).to(dt)
        args = {k: c[k] for k in ("post", "pre", "gate", "scale", "norm")}
        kept = dict(post_tape=r.post_tape, post_rstd=r.post_rstd, pre_tape=r.pre_tape, pre_rstd=r.pre_rstd)
        g = ops.norm_join_bwd(gy, gh if pre else None, **kept, **args)
        val = lambda t: ref_values(t.codes, t.bytes, t.width, t.kind).cuda() if t is not None else None  # noqa: E731
        f64 = lambda v: v.double() if v is not None else None  # noqa: E731
        want = ref_join_bwd(c, gy, gh, val(r.post_tape), f64(r.post_rstd), val(r.pre_tape), f64(r.pre_rstd))
        # (the gradient at a norm's input is a difference: of rows of a few columns little is left, so it is held against what it is a difference of)
        size = float(gy.double().norm()) + float(gh.double().norm()) * (float(r.pre_rstd.max()) if pre else 0.0) * 2
        sizes = {"x": size, "f": 2 * size * (float(r.post_rstd.max()) if post else 1.0)}
        for k in ("x", "f", "gate", "scale"):
            got, ref = getattr(g, k), want.get(k)
            if ref is None:
                assert got is None
                continue
            off = (got.double() - ref).abs()
            if got.dtype == torch.bfloat16:
                off = (off - 2.0 ** -8 * ref.abs()).clamp(min=0)
            # sums over rows: M terms, each off like D itself
            top = sizes.get(k, size * float(val(r.post_tape).abs().max() + 1) * 2 * (M ** 0.5 if k == "scale" else 1.0))
            assert float(off.norm()) <= REL32 * top, (k, float(off.norm()), top)
        for k in ("post", "pre"):
            for got, ref in zip(getattr(g, k) or (), want.get(k) or ()):
                if ref is None:
                    assert got is None
                else:
                    assert float((got.double() - ref).norm()) <= REL32 * size * 8 * M ** 0.5, k
        again = ops.norm_join_bwd(gy, gh if pre else None, **kept, **args)
        assert torch.equal(again.x, g.x) and torch.equal(again.f, g.f) and (g.gate is None or torch.equal(again.gate, g.gate))
        assert all(torch.equal(a, b) for k in ("post", "pre") for a, b in zip(getattr(g, k) or (), getattr(again, k) or ()) if a is not None)


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("M,W,G", [(4099, 600, 4099), (4098, 700, 2049), (2051, 1000, 0), (1027, 1500, 1027), (4202, 1100, 2101), (603, 2000, 3), (1, 1000, 1),
                                   (515, 2500, 515), (65537, 20, 0)])
def test_norm_join_workgroups_of_several_rows(norm, M, W, G):
    """wide rows two at a time in a workgroup, the last one alone; gate rows one and two at a time"""
    for dtype in ("fp32", "bf16"):
        test_norm_join_forward(dtype, norm, M, W, G)
        test_norm_join_backward(dtype, norm, M, W, G)


def test_norm_join_strides():
    """rows inside wider arrays, aligned to 16 bytes and not, give the same bits"""
    from magnet_amd import ops
    c = join_case(50, 100, 5, "layer", True, True, True, torch.float32)
    want = ops.norm_join(**c, tape=True)
    for o in (4, 1):
        wide = {k: torch.full((c[k].shape[0], 120), 9.0, device="cuda") for k in ("x", "f", "gate")}
        for k, v in wide.items():
            v[:, o:o + 100] = c[k]
        r = ops.norm_join(**{**c, **{k: v[:, o:o + 100] for k, v in wide.items()}}, tape=True)
        assert torch.equal(r.y, want.y) and torch.equal(r.h, want.h) and torch.equal(r.post_tape.codes, want.post_tape.codes)
    one = ops.norm_join(**{**c, "gate": c["gate"][0]})
    assert torch.equal(one.y, ops.norm_join(**{**c, "gate": c["gate"][:1].expand(50, 100).contiguous()}).y)


@pytest.mark.parametrize("M", [0, 50])
def test_norm_join_one_gate_for_all_rows(M):
    """a gate of shape [W] gets a gradient of that shape, the one that [1, W] gets"""
    from magnet_amd import ops
    c = join_case(M, 100, 1, "rms", True, False, False, torch.float32)
    r = ops.norm_join(**c, tape=True)
    args = dict(post_tape=r.post_tape, post_rstd=r.post_rstd, post=c["post"], scale=c["scale"], norm="rms")
    gy = torch.randn(M, 100, device="cuda")
    a, b = (ops.norm_join_bwd(gy, gate=g, **args) for g in (c["gate"], c["gate"][0]))
    assert a.gate.shape == (1, 100) and b.gate.shape == (100,) and torch.equal(a.gate[0], b.gate) and torch.equal(a.f, b.f)


def test_norm_join_no_rows():
    from magnet_amd import ops
    c = join_case(0, 64, 3, "layer", True, True, True, torch.float32)
    r = ops.norm_join(**c, tape=True)
    assert r.y.shape == (0, 64) and r.h.shape == (0, 64)
    g = ops.norm_join_bwd(r.y, r.h, post_tape=r.post_tape, post_rstd=r.post_rstd, pre_tape=r.pre_tape, pre_rstd=r.pre_rstd,
                          **{k: c[k] for k in ("post", "pre", "gate", "scale", "norm")})
    assert not g.gate.any() and not g.scale.any() and not g.post[0].any() and not g.pre[1].any()


def test_norm_join_constant_and_not_finite_rows():
    """a row without variation is its bias; a row that is not finite spoils itself alone"""
    from magnet_amd import ops
    c = join_case(20, 128, 0, "layer", True, True, False, torch.float32)
    c["f"][3] = 5.0
    r = ops.norm_join(**c, tape=True)
    near(r.y, ref_join(c)[0], torch.float32)
    assert not r.post_tape.codes[3].any() and not r.post_tape.bytes[3].any()
    clean = ops.norm_join(**c, tape=True)
    for bad in (math.nan, math.inf):
        d = dict(c, f=c["f"].clone())
        d["f"][7, 70] = bad
        r = ops.norm_join(**d, tape=True)
        assert torch.isnan(r.y[7]).all() and torch.isnan(r.h[7]).all() and bool((r.post_tape.bytes[7] == 255).all())
        keep = torch.arange(20, device="cuda") != 7
        assert torch.equal(r.y[keep], clean.y[keep]) and torch.equal(r.pre_tape.codes[keep], clean.pre_tape.codes[keep])


def test_norm_tape_is_the_tape_of_norm_join():
    from magnet_amd import ops
    for norm in ("layer", "rms"):
        for W, dt in ((64, torch.float32), (100, torch.bfloat16), (1500, torch.float32)):
            c = join_case(77, W, 0, norm, True, False, False, dt)
            want = ops.norm_join(**c, tape=True)
            t, r = ops.norm_tape(c["f"], norm)
            assert torch.equal(t.codes, want.post_tape.codes) and torch.equal(t.bytes, want.post_tape.bytes) and torch.equal(r, want.post_rstd)
            g, gy = (ops.norm_join_bwd(c["x"], post_tape=t, post_rstd=r, post=c["post"], norm=norm, need_x=x) for x in (False, True))
            assert g.x is None and torch.equal(g.f, gy.f) and torch.equal(g.post[0], gy.post[0]) and torch.equal(gy.x, c["x"])


# --------------------------------------------------------------------------------------------------------------------- gradients
def exact_join(c, x, f):
    M = x.shape[0]
    y = x + c["scale"] * ref_gate(c, M) * ref_affine(ref_norm(f, c["norm"])[0] if c["post"] else f, c["post"])
    return y, ref_affine(ref_norm(y, c["norm"])[0], c["pre"]) if c["pre"] else None


@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("uses", ["both", "y", "h"])
@pytest.mark.parametrize("G", [0, 1, 6, 300])
def test_norm_join_gradients(norm, uses, G):
    """autograd.norm_join against the formula's gradients (fp64 autograd) and against differences of the formula along a direction.  What
    the tape rounds: codes of normalised rows (deviation 1, block tops about 2.5) are off by step / sqrt(12) <= 2.5 / 127 / sqrt(12) = 0.6 %
    of the deviation; it enters a gradient through v^ mean(u v^) and the gains' sums: a share below that of the whole.  2 % bounds it."""
    from magnet_amd import autograd as AG
    M, W = 300, 128
    c = join_case(M, W, G, norm, True, True, True, torch.float32, seed=G + 1)
    leaves = {"x": c["x"], "f": c["f"], "gate": c["gate"], "scale": c["scale"], "post_g": c["post"][0], "post_b": c["post"][1], "pre_g": c["pre"][0], "pre_b": c["pre"][1]}
    leaves = {k: v for k, v in leaves.items() if v is not None}
    torch.manual_seed(5)
    wy, wh = torch.randn(M, W, device="cuda"), torch.randn(M, W, device="cuda")

    def case(v):
        return dict(c, x=v["x"], f=v["f"], gate=v.get("gate"), scale=v["scale"], post=(v["post_g"], v.get("post_b")), pre=(v["pre_g"], v.get("pre_b")))

    def loss(y, h, a, b):
        return ((y * a).sum() if uses != "h" else 0.0) + ((h * b).sum() if uses != "y" else 0.0)
    mine = {k: v.clone().requires_grad_() for k, v in leaves.items()}
    d = case(mine)
    y, h = AG.norm_join(d["x"], d["f"], post=d["post"], pre=d["pre"], gate=d["gate"], scale=d["scale"], norm=norm)
    loss(y, h, wy, wh).backward()
    exact = {k: v.double().requires_grad_() for k, v in leaves.items()}
    d = case(exact)
    ye, he = exact_join(d, d["x"], d["f"])
    near(y.detach(), ye.detach(), torch.float32)
    near(h.detach(), he.detach(), torch.float32)
    loss(ye, he, wy.double(), wh.double()).backward()
    for k, v in exact.items():
        if v.grad is None or (uses == "y" and k.startswith("pre")):
            assert mine[k].grad is None or not mine[k].grad.any()
            continue
        assert mine[k].grad.dtype == mine[k].dtype and mine[k].grad.shape == mine[k].shape
        assert float((mine[k].grad - v.grad).norm()) <= 0.02 * float(v.grad.norm()), k
    # differences: the loss along one direction of all leaves, central, 64 bits (error of the second order in 1e-5)
    dirs = {k: torch.randn(v.shape, device="cuda", dtype=torch.float64) for k, v in leaves.items()}
    with torch.no_grad():
        at = [loss(*exact_join(case({k: v + s * dirs[k] for k, v in exact.items()}), exact["x"] + s * dirs["x"], exact["f"] + s * dirs["f"]),
                   wy.double(), wh.double()) for s in (1e-5, -1e-5)]
        slope = float(at[0] - at[1]) / 2e-5
        got = sum(float((mine[k].grad.double() * dirs[k]).sum()) for k in leaves if mine[k].grad is not None)
        size = sum(float((v.grad * dirs[k]).norm()) for k, v in exact.items() if v.grad is not None)
    assert abs(got - slope) <= 0.02 * size + 1e-6 * abs(slope), (got, slope)


def chain_case(M, hidden, D, K, seed, ln):
    """an MLP of five Linears on dense rows, its packed namespace and the torch parameters behind it"""
    import types

    from magnet_amd.packing import pack, pad_to
    torch.manual_seed(seed)
    dims = [K, hidden, hidden, hidden, hidden, D]
    lins = [torch.nn.Linear(a, b).cuda() for a, b in zip(dims, dims[1:])]
    norm = torch.nn.LayerNorm(D).cuda() if ln else None
    if ln:
        torch.nn.init.normal_(norm.weight, 1.0, 0.2)
        torch.nn.init.normal_(norm.bias, 0.0, 0.2)
    Dp = pad_to(D)
    pad = lambda v: torch.nn.functional.pad(v.detach(), (0, Dp - D)).contiguous()  # noqa: E731
    pk = types.SimpleNamespace(layers=[pack(m.weight.detach(), m.bias.detach(), "fp16x3") for m in lins], ln=(pad(norm.weight), pad(norm.bias), norm.eps) if ln else None,
                               ht=pad_to(hidden) // 32, ot=Dp // 32, out_dim=D, col_map=None)
    params = [p for m in lins for p in (m.weight, m.bias)] + ([norm.weight, norm.bias] if ln else [])
    return lins, norm, pk, params, torch.randn(M, K, device="cuda")


@pytest.mark.parametrize("M,hidden,D,K,ln", [(5000, 128, 128, 128, True), (5000, 64, 32, 64, True), (777, 128, 1, 32, False), (4500, 64, 10, 64, False)])
@pytest.mark.parametrize("in_place", [False, True])
def test_mlp_with_the_tape_in_8_bits(M, hidden, D, K, ln, in_place, monkeypatch):
    """the whole chain: the forward's bits are those of the fp32 tape, the saved activations a quarter; the ReLU masks are exact, so the gradients
    are those of the fp32 tape but for the activations' rounding: step / sqrt(12) with step <= 2 top / 255 and block tops of 32 rectified
    normals about 2.3 sigma against 0.7 sigma of root mean square - 0.8 % - in every dW, 1 % with the LayerNorm's tape; 2.5 % bounds it"""
    from magnet_amd import autograd as AG, ops
    monkeypatch.setenv("MAGNET_KEEP_TAPE", "1")
    lins, norm, pk, params, x = chain_case(M, hidden, D, K, 3, ln)
    if ln and not ops.L.query("magnet_mlp_supported", 5, pk.ht, pk.ot, ops.ACT_RELU, 0, 1, ops.EPI_STORE):
        pytest.skip("no such chain")
    gy = torch.randn(M, D, device="cuda")
    runs, kept = {}, {}
    for on in (False, True):
        for p in params:
            p.grad = None
        xi = x.clone().requires_grad_()
        saved = []
        if in_place:
            with AG.tape8(on), AG.accumulate_param_grads():
                y = AG.mlp(M, [ops.Term(xi, K)], pk, params)
        else:
            with torch.autograd.graph.saved_tensors_hooks(lambda t: (saved.append(t.numel() * t.element_size()), t)[1], lambda t: t), AG.tape8(on):
                y = AG.mlp(M, [ops.Term(xi, K)], pk, params)
        y.backward(gy)
        kept[on] = sum(saved) - 2 * M * K * 4 - sum(p.numel() * 4 for p in params)           # (x twice: the source and the assembled input)
        runs[on] = [y.detach(), xi.grad] + [p.grad.clone() for p in params]
        if in_place:                                       # a second backward of the same step adds to what is there
            with AG.tape8(on), AG.accumulate_param_grads():
                y2 = AG.mlp(M, [ops.Term(x.clone().requires_grad_(), K)], pk, params)
            y2.backward(gy)
            for p, g in zip(params, runs[on][2:]):
                assert float((p.grad - 2 * g).norm()) <= 1e-5 * float(g.norm())
    assert torch.equal(runs[False][0], runs[True][0])
    assert in_place or kept[True] <= 0.27 * kept[False] + 4 * M, kept
    for i, (a, b) in enumerate(zip(runs[True][1:], runs[False][1:])):
        assert float((a - b).norm()) <= 0.025 * float(b.norm()), (i, float((a - b).norm() / b.norm()))
    # and against fp64 autograd through the same chain
    net = [m.__class__(m.in_features, m.out_features).cuda().double() for m in lins]
    for a, b in zip(net, lins):
        a.load_state_dict(b.state_dict())
    x64 = x.double().requires_grad_()
    v = x64
    for i, m in enumerate(net):
        v = m(v)
        v = torch.relu(v) if i < 4 else v
    if ln:
        v = torch.nn.functional.layer_norm(v, (D,), norm.weight.detach().double(), norm.bias.detach().double(), norm.eps)
    v.backward(gy.double())
    for a, b in zip(runs[True][2:], [p.grad for m in net for p in (m.weight, m.bias)]):
        assert float((a - b).norm()) <= 0.03 * float(b.norm())


@pytest.mark.parametrize("teacher_forcing", [False, True])
def test_magnet_gnn_trains_with_the_tape_in_8_bits(teacher_forcing):
    """a model's own training step with ``tape8`` in its hparams: the loss has the bits of the fp32 tape's, every parameter a gradient within the
    rounding of the activations (a rollout of several forwards: errors of 1 % a chain, independent from chain to chain)"""
    from magnet_amd.models.factory import FACTORY
    from oracle import models as O
    from oracle.weightgen import fill_state_dict
    from tests.helpers import load_case
    name, hp, salt, batch, d = load_case("magnet_gnn_tiny")
    hp.teacher_forcing = teacher_forcing
    oracle = O.build(name, hp)
    fill_state_dict(oracle, salt)
    cb = {k: v.cuda() for k, v in batch.items()}
    got = []
    for on in (False, True):
        hp.tape8 = on
        model = FACTORY[name](hp)
        model.load_state_dict(oracle.state_dict())
        model = model.cuda().train()
        assert model.tape8 is on
        loss = model.training_step(cb, 0)
        loss.backward()
        got.append((loss.detach(), {n: p.grad for n, p in model.named_parameters()}))
    assert torch.equal(got[0][0], got[1][0])
    for n, g in got[0][1].items():
        if g is None:
            assert got[1][1][n] is None
            continue
        off = float((got[1][1][n] - g).norm() / g.norm()) if float(g.norm()) else 0.0
        assert off <= 0.05, (n, off)


def test_a_captured_training_step_with_the_tape_in_8_bits():
    """graphs.TrainStepGraph over a model that trains with ``tape8``: the replays' losses and parameters are those of the eager steps"""
    from magnet_amd.graphs import TrainStepGraph
    from magnet_amd.models.factory import FACTORY
    from oracle import models as O
    from oracle.weightgen import fill_state_dict
    from tests.helpers import load_case
    name, hp, salt, batch, d = load_case("magnet_gnn_tiny")
    hp.tape8 = True
    hp.teacher_forcing = True
    oracle = O.build(name, hp)
    fill_state_dict(oracle, salt)
    cb = {k: v.cuda() for k, v in batch.items()}
    runs = []
    for captured in (False, True):
        model = FACTORY[name](hp)
        model.load_state_dict(oracle.state_dict())
        model = model.cuda().train()
        opt = model.configure_optimizers()["optimizer"]
        step = TrainStepGraph(model, opt) if captured else None
        torch.manual_seed(3)
        losses = []
        for _ in range(5):
            if captured:
                losses.append(float(step(cb).detach()))
            else:
                opt.zero_grad()
                loss = model.training_step(cb, 0)
                loss.backward()
                opt.step()
                losses.append(float(loss.detach()))
        runs.append((losses, [p.detach().clone() for p in model.parameters()]))
        assert not captured or (step.replays == 5 and step.eager_steps == 0)
    assert runs[0][0] == runs[1][0]
    assert all(torch.equal(a, b) for a, b in zip(runs[0][1], runs[1][1]))


# ------------------------------------------------------------------------------------------------------- together, streams, graphs
def block(x, w1, w2, post, pre, gate, scale, gy, gh):
    """one residual block, forward and backward, through the operators: y = x + scale gate post(relu(h0 w1^T) w2^T), h = pre(y)"""
    from magnet_amd import ops
    a = x @ w1.t()
    t1 = ops.tape8_pack(a, "relu")
    f = a.clamp(min=0) @ w2.t()
    r = ops.norm_join(x, f, post=post, pre=pre, gate=gate, scale=scale, tape=True)
    g = ops.norm_join_bwd(gy, gh, post_tape=r.post_tape, post_rstd=r.post_rstd, pre_tape=r.pre_tape, pre_rstd=r.pre_rstd, post=post, pre=pre, gate=gate, scale=scale)
    da, dw2, db2 = ops.tape8_linear_bwd(g.f, t1, w2, "relu")
    t0 = ops.tape8_pack(x)
    dx, dw1, db1 = ops.tape8_linear_bwd(da, t0, w1)
    return [r.y, r.h, g.x, g.f, g.gate, g.scale, *g.post, *g.pre, da, dw2, db2, dx, dw1, db1, ops.tape8_unpack(r.pre_tape)]


def block_case(M=1500, W=128, H=96, G=3):
    torch.manual_seed(11)
    r = lambda *s: torch.randn(*s, device="cuda")  # noqa: E731
    return dict(x=r(M, W), w1=r(H, W) / W ** 0.5, w2=r(W, H) / H ** 0.5, post=(1 + 0.1 * r(W), 0.1 * r(W)), pre=(1 + 0.1 * r(W), 0.1 * r(W)), gate=torch.sigmoid(r(G, W)),
                scale=0.5 + 0.1 * r(W), gy=r(M, W) * 1e-6, gh=r(M, W) * 1e-6)


def test_block_together_and_on_another_stream():
    c = block_case()
    want = block(**c)
    # the block's gradients against fp64 (1 % of rounding a tape, two tapes behind one another)
    p = {k: v.double() if isinstance(v, torch.Tensor) else tuple(u.double() for u in v) for k, v in c.items()}
    leaves = [p["x"].requires_grad_(), p["w1"].requires_grad_(), p["w2"].requires_grad_()]
    f = torch.relu(p["x"] @ p["w1"].t()) @ p["w2"].t()
    ln = lambda v, q: torch.nn.functional.layer_norm(v, (v.shape[1],), q[0], q[1], EPS)  # noqa: E731
    y = p["x"] + p["scale"] * p["gate"].repeat_interleave(500, 0) * ln(f, p["post"])
    ((y * p["gy"]).sum() + (ln(y, p["pre"]) * p["gh"]).sum()).backward()
    for got, ref in ((want[2] + want[13], leaves[0].grad), (want[14], leaves[1].grad), (want[11], leaves[2].grad)):
        assert float((got - ref).norm()) <= 0.03 * float(ref.norm())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = block(**c)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_block_captured_and_replayed():
    """two graphs of the same calls, replayed in turn with eager work between, on inputs that change: every replay has the eager bits"""
    c, d = block_case(), block_case(M=333, W=64, H=128, G=333)
    graphs = []
    for e in (c, d):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            block(**e)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = block(**e)
        graphs.append((g, out, e))
    for k in range(4):
        for g, out, e in graphs:
            for name in ("x", "gy", "gh"):
                e[name].copy_(torch.randn_like(e[name]) * (1.0 if name == "x" else 10.0 ** (-6 + k)))
            g.replay()
            want = block(**e)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k


def test_a_backward_is_the_same_while_another_runs():
    """two streams at work at the same time on workspaces of their own"""
    from magnet_amd import ops
    dz, t, w = linear_case(60000, 128, 128, "relu", seed=9)
    want = ops.tape8_linear_bwd(dz, t, w, "relu")
    c = join_case(40000, 128, 4, "layer", True, True, True, torch.float32)
    r = ops.norm_join(**c, tape=True)
    args = dict(post_tape=r.post_tape, post_rstd=r.post_rstd, pre_tape=r.pre_tape, pre_rstd=r.pre_rstd, **{k: c[k] for k in ("post", "pre", "gate", "scale", "norm")})
    other = ops.norm_join_bwd(c["x"], c["f"], **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(side):
            g = ops.norm_join_bwd(c["x"], c["f"], **args)
        got = ops.tape8_linear_bwd(dz, t, w, "relu")
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(g.f, other.f) and torch.equal(g.gate, other.gate) and torch.equal(g.scale, other.scale)
