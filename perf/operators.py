"""The training operators around an 8-bit activation tape, as cases that can be measured: the tape's quantisation, a Linear walked back
from it, and the norms before and after a residual block with its gate and residual scale, forward and backward.

``run`` computes a case either from elementary torch operations in 32 bits (``own`` false) or through ``magnet_amd.ops`` (``own`` true).

The tape.  A row of W values is cut into blocks of 32 columns (the last one padded with zeros); a block is 32 codes of 8 bits and one
byte b that stands for the factor 2^(b - 127), the smallest one whose largest code reaches the block's largest magnitude (b in
[1, 248]; 0: every value is zero; 255: the block holds a value that is not finite, and reads as NaN).  ``signed``: code = round(x / 2^e)
in [-127, 127].  ``relu``: code = 0 where x <= 0, else round(x / 2^e) in [1, 255] - never 0, so that the mask x > 0 is kept exactly."""
import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # the hidden activations of one edge chain on the large mesh go onto the tape: the largest array that training keeps
        dict(name="pack relu 2097152x128", op="pack", kind="relu", dtype="fp32", M=2097152, W=128),
        # a bf16 array of odd row count and a width that ends inside a block of 32
        dict(name="pack signed bf16 65521x200", op="pack", kind="signed", dtype="bf16", M=65521, W=200),
        # the smallest mesh of the configurations (2 x 50 nodes): latency
        dict(name="pack relu 100x128", op="pack", kind="relu", dtype="fp32", M=100, W=128),
        # a hidden 128 -> 128 Linear of the edge chain walked back over all edges of the large mesh
        dict(name="linear relu 2097152 128-128", op="linear", act="relu", M=2097152, N=128, K=128),
        # the 64-wide chains at a usual training batch
        dict(name="linear relu 218453 64-64", op="linear", act="relu", M=218453, N=64, K=64),
        # an update net's second Linear over the nodes of four 256 x 256 meshes: Swish, its pre-activation on the tape
        dict(name="linear swish 262144 128-128", op="linear", act="swish", M=262144, N=128, K=128),
        # a small Linear of odd widths (a projection to 25 time steps) over a small batch: latency
        dict(name="linear none 1000 100-25", op="linear", act="none", M=1000, N=25, K=100),
        # the residual join of a rollout step on the smallest mesh: latency
        dict(name="join 100x128", op="join", norm="layer", dtype="fp32", M=100, W=128, G=0, post=True, pre=True, vec=False, tape=False),
        # the same in training on four large meshes, a gate for each mesh, both normalised rows kept on the tape
        dict(name="join tape 262144x128", op="join", norm="layer", dtype="fp32", M=262144, W=128, G=4, post=True, pre=True, vec=True, tape=True),
        # its backward pass
        dict(name="join_bwd 262144x128", op="join_bwd", norm="layer", dtype="fp32", M=262144, W=128, G=4, post=True, pre=True, vec=True),
        # wide rows in bf16, root-mean-square norms, a gate of its own for every element
        dict(name="join bf16 8190x2048", op="join", norm="rms", dtype="bf16", M=8190, W=2048, G=8190, post=True, pre=True, vec=False, tape=False),
        # and backward, a width that ends inside a block
        dict(name="join_bwd bf16 4097x1000", op="join_bwd", norm="rms", dtype="bf16", M=4097, W=1000, G=4097, post=True, pre=True, vec=True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(2.0 ** rng.uniform(torch.tensor(float(lo)).log2().item(), torch.tensor(float(hi)).log2().item())))))


def draw(rng):
    op = rng.choice(["pack", "linear", "linear", "join", "join_bwd"])
    if op == "pack":
        W = rng.choice([32, 64, 128, 256, _spread(rng, 1, 1152), _spread(rng, 1, 1152)])
        return dict(op=op, kind=rng.choice(["relu", "signed"]), dtype=rng.choice(["fp32", "fp32", "bf16", "fp16"]),
                    M=_spread(rng, 1, (1 << 27) // W), W=W)
    if op == "linear":
        N, K = (rng.choice([64, 128, 128, _spread(rng, 1, 256)]) for _ in range(2))
        return dict(op=op, act=rng.choice(["relu", "relu", "swish", "none"]), M=_spread(rng, 1, (1 << 27) // max(N, K, 64)), N=N, K=K)
    # (a norm over a handful of columns has no gradient to speak of: of two, it only keeps which is the larger)
    W = rng.choice([64, 128, 256, _spread(rng, 16, 4096), _spread(rng, 16, 4096)])
    M = _spread(rng, 1, (1 << 25) // W)
    groups = [g for g in (1, 2, 3, 4, 8) if M % g == 0] + [0, M]
    c = dict(op=op, norm=rng.choice(["layer", "rms"]), dtype=rng.choice(["fp32", "bf16"]), M=M, W=W, G=rng.choice(groups), vec=rng.random() < 0.5)
    c["post"], c["pre"] = rng.choice([(True, True), (True, True), (True, False), (False, True)])
    if op == "join":
        c["tape"] = rng.random() < 0.5
    return c


# ----------------------------------------------------------------------------------------------------------------------------- inputs
def _activations(M, W, gen, relu):
    """values as a layer hands them on: normal, the rows of different magnitude; behind a ReLU, half of them zero"""
    x = torch.randn(M, W, device="cuda", generator=gen)
    x *= torch.exp2(torch.randn(M, 1, device="cuda", generator=gen))
    return x.clamp_(min=0.0) if relu else x


def _gradient(M, W, gen):
    """gradients of a mean loss: small, their rows of different magnitude"""
    return torch.randn(M, W, device="cuda", generator=gen) * torch.exp2(torch.randn(M, 1, device="cuda", generator=gen) - 20.0)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    s = dict(case)
    op, M = case["op"], case["M"]
    if op == "pack":
        s["x"] = _activations(M, case["W"], gen, case["kind"] == "relu").to(DTYPES[case["dtype"]])
        return s
    if op == "linear":
        N, K = case["N"], case["K"]
        kind = "relu" if case["act"] == "relu" else "signed"
        s["codes"], s["bytes"] = _quantise(_activations(M, K, gen, kind == "relu"), kind)
        s["dz"] = _gradient(M, N, gen)
        s["w"] = rand(N, K) / K ** 0.5
        return s
    W, G, dt = case["W"], case["G"], DTYPES[case["dtype"]]
    layer = case["norm"] == "layer"
    s["gate"] = torch.sigmoid(rand(G, W)).to(dt) if G else None
    s["scale"] = 0.5 + 0.1 * rand(W) if case["vec"] else 0.5
    for side in ("post", "pre"):
        s[side + "_g"] = 1.0 + 0.1 * rand(W) if case[side] else None
        s[side + "_b"] = 0.1 * rand(W) if case[side] and layer else None
    if op == "join":
        s["x"] = (2.0 * rand(M, W)).to(dt)
        s["f"] = _activations(M, W, gen, False).to(dt)
        return s
    s["gy"] = _gradient(M, W, gen).to(dt)
    s["gh"] = _gradient(M, W, gen).to(dt) if case["pre"] else None
    # what the forward pass kept: the rows of both norms before gain and bias, in 8 bits, and 1 / sqrt(variance + eps)
    for side in ("post", "pre"):
        if side == "pre" and not case["pre"]:
            s["pre_codes"] = s["pre_bytes"] = s["pre_rstd"] = None
            continue
        v = _activations(M, W, gen, False)
        v, r = _normed(v, case["norm"]) if case[side] else (v, None)
        s[side + "_codes"], s[side + "_bytes"] = _quantise(v, "signed")
        s[side + "_rstd"] = r
    return s


# ------------------------------------------------------------------------------------------------------------------ the plain operators
EPS = 1e-5


def _blocks(x):
    W = x.shape[1]
    pad = -W % 32
    x = torch.nn.functional.pad(x, (0, pad)) if pad else x
    return x.reshape(x.shape[0], (W + pad) // 32, 32)


def _two_to(e):
    """2^e in 32 bits, e in [-126, 127], from its bits: a power function may be off by a rounding"""
    return ((e.int() + 127) << 23).view(torch.float32)


def _quantise(x, kind):
    """codes [M, 32 ceil(W / 32)] uint8 (two's complement where signed) and bytes [M, ceil(W / 32)] uint8 of finite values"""
    x = _blocks(x.float())
    top = (x if kind == "relu" else x.abs()).amax(2).clamp(min=0.0)
    frac, e = torch.frexp(top)                                        # top = frac 2^e, frac in [1/2, 1)
    e = e - 7 - (frac <= 255.0 / 256.0).int() if kind == "relu" else e - 6 - (frac <= 127.0 / 128.0).int()
    e = e.clamp(-126, 121)
    q = torch.round(x * _two_to(-e)[:, :, None])
    q = torch.where(x > 0, q.clamp(1, 255), torch.zeros_like(q)) if kind == "relu" else q.clamp(-127, 127)
    codes = q.to(torch.int16).to(torch.uint8) if kind == "relu" else q.to(torch.int8).view(torch.uint8)
    return codes.reshape(x.shape[0], -1), torch.where(top > 0, e + 127, torch.zeros_like(e)).to(torch.uint8)


def _values(codes, bytes_, W, kind):
    q = (codes if kind == "relu" else codes.view(torch.int8)).float().reshape(codes.shape[0], -1, 32)
    return (q * _two_to(bytes_.int() - 127)[:, :, None]).reshape(codes.shape[0], -1)[:, :W]


def _normed(v, norm):
    """(v - mean) / sqrt(variance + eps), or v / sqrt(mean square + eps), and the factor 1 / sqrt(...) of every row"""
    v = v - v.mean(1, keepdim=True) if norm == "layer" else v
    r = 1.0 / torch.sqrt((v * v).mean(1, keepdim=True) + EPS)
    return v * r, r[:, 0]


def _long_product(a, b):
    """a^T b over many rows: blocks of 4096 rows in 32 bits, the blocks' products added in 64"""
    M = a.shape[0] // 4096 * 4096
    out = (a[M:].t() @ b[M:]).double()
    if M:
        blocks = torch.bmm(a[:M].reshape(-1, 4096, a.shape[1]).transpose(1, 2).contiguous(), b[:M].reshape(-1, 4096, b.shape[1]).contiguous())
        out = out + blocks.sum(0, dtype=torch.float64)
    return out.float()


def _linear_bwd(s):
    kind = "relu" if s["act"] == "relu" else "signed"
    x = _values(s["codes"], s["bytes"], s["K"], kind)
    dx = s["dz"] @ s["w"]
    if s["act"] == "relu":
        dx = torch.where(x > 0, dx, torch.zeros_like(dx))
    elif s["act"] == "swish":
        g = 1.0 / (1.0 + torch.exp(-x))
        dx = dx * (g * (1.0 + x * (1.0 - g)))
        x = x * g
    return dx, _long_product(s["dz"], x), s["dz"].sum(0, dtype=torch.float64).float()


def _rows(gate, M):
    """the gate of every row: row r takes gate[r // (M / G)]"""
    return gate.float().repeat_interleave(M // gate.shape[0], 0)


def _join(s):
    x, f = s["x"].float(), s["f"].float()
    fhat, r_post = _normed(f, s["norm"]) if s["post"] else (f, None)
    t = fhat * s["post_g"] if s["post"] else fhat
    t = t + s["post_b"] if s["post_b"] is not None else t
    t = t * _rows(s["gate"], s["M"]) if s["gate"] is not None else t
    y = x + s["scale"] * t
    out = {"y": y.to(s["x"].dtype)}
    if s["pre"]:
        yhat, r_pre = _normed(y, s["norm"])
        h = yhat * s["pre_g"]
        out["h"] = (h + s["pre_b"] if s["pre_b"] is not None else h).to(s["x"].dtype)
    if s["tape"]:
        # (a code has at most seven bits and a sign: bf16 holds what it stands for exactly)
        out["post"], out["post_rstd"] = _values(*_quantise(fhat, "signed"), s["W"], "signed").bfloat16(), r_post
        if s["pre"]:
            out["pre"], out["pre_rstd"] = _values(*_quantise(yhat, "signed"), s["W"], "signed").bfloat16(), r_pre
    return out


def _norm_bwd(d, vhat, r, norm):
    """the gradient at a norm's input from the gradient d at its normalised output"""
    d = d - vhat * (d * vhat).mean(1, keepdim=True) - (d.mean(1, keepdim=True) if norm == "layer" else 0.0)
    return d * r[:, None]


def _sum(v):
    return v.sum(0, dtype=torch.float64).float()


def _join_bwd(s):
    M, W, dt = s["M"], s["W"], s["gy"].dtype
    d = s["gy"].float()
    out = {}
    if s["pre"]:
        yhat, gh = _values(s["pre_codes"], s["pre_bytes"], W, "signed"), s["gh"].float()
        d = d + _norm_bwd(gh * s["pre_g"], yhat, s["pre_rstd"], s["norm"])
        out["pre_g"] = _sum(gh * yhat)
        out["pre_b"] = _sum(gh) if s["pre_b"] is not None else None
    out["x"] = d.to(dt)
    fhat = _values(s["post_codes"], s["post_bytes"], W, "signed")
    t = fhat * s["post_g"] if s["post"] else fhat
    t = t + s["post_b"] if s["post_b"] is not None else t
    gate = _rows(s["gate"], M) if s["gate"] is not None else 1.0
    if s["gate"] is not None:
        dg = d * s["scale"] * t
        out["gate"] = dg.reshape(s["G"], M // s["G"], W).sum(1, dtype=torch.float64).to(dt)
    if s["vec"]:
        out["scale"] = _sum(d * gate * t)
    dt_ = d * s["scale"] * gate
    if s["post"]:
        out["post_g"] = _sum(dt_ * fhat)
        out["post_b"] = _sum(dt_) if s["post_b"] is not None else None
        dt_ = _norm_bwd(dt_ * s["post_g"], fhat, s["post_rstd"], s["norm"])
    out["f"] = dt_.to(dt)
    return out


def run(state):
    s = state
    if own:
        return _run_own(s)
    if s["op"] == "pack":
        return _values(*_quantise(s["x"], s["kind"]), s["W"], s["kind"])
    if s["op"] == "linear":
        dx, dw, db = _linear_bwd(s)
        return {"x": dx, "w": dw, "b": db}
    return _join(s) if s["op"] == "join" else _join_bwd(s)


# ------------------------------------------------------------------------------------------------------------- the framework's operators
def _run_own(s):
    from magnet_amd import ops
    if s["op"] == "pack":
        return ops.tape8_unpack(ops.tape8_pack(s["x"], s["kind"]))
    if s["op"] == "linear":
        tape = ops.Tape8(s["codes"], s["bytes"], s["K"], "relu" if s["act"] == "relu" else "signed")
        dx, dw, db = ops.tape8_linear_bwd(s["dz"], tape, s["w"], act=s["act"])
        return {"x": dx, "w": dw, "b": db}
    post = (s["post_g"], s["post_b"]) if s["post"] else None
    pre = (s["pre_g"], s["pre_b"]) if s["pre"] else None
    kw = dict(post=post, pre=pre, gate=s["gate"], scale=s["scale"], norm=s["norm"])
    if s["op"] == "join":
        r = ops.norm_join(s["x"], s["f"], eps=EPS, tape=s["tape"], **kw)
        out = {"y": r.y}
        if s["pre"]:
            out["h"] = r.h
        if s["tape"]:
            out["post"], out["post_rstd"] = ops.tape8_unpack(r.post_tape, dtype=torch.bfloat16), r.post_rstd
            if s["pre"]:
                out["pre"], out["pre_rstd"] = ops.tape8_unpack(r.pre_tape, dtype=torch.bfloat16), r.pre_rstd
        return out
    tapes = [ops.Tape8(s[k + "_codes"], s[k + "_bytes"], s["W"], "signed") if s[k + "_codes"] is not None else None for k in ("post", "pre")]
    g = ops.norm_join_bwd(s["gy"], s["gh"], post_tape=tapes[0], post_rstd=s["post_rstd"], pre_tape=tapes[1], pre_rstd=s["pre_rstd"], **kw)
    out = {"x": g.x, "f": g.f}
    if s["pre"]:
        out["pre_g"], out["pre_b"] = g.pre
    if s["post"]:
        out["post_g"], out["post_b"] = g.post
    if s["gate"] is not None:
        out["gate"] = g.gate
    if s["vec"]:
        out["scale"] = g.scale
    return out


# ------------------------------------------------------------------------------------------------------------------------------- work
def work(case):
    M, op = case["M"], case["op"]
    tape = lambda w: M * (-(-w // 32) * 33)  # noqa: E731
    if op == "pack":
        W, size = case["W"], DTYPES[case["dtype"]].itemsize
        return {"bytes": M * W * (size + 4) + 2 * tape(W), "flops": 4 * M * W}
    if op == "linear":
        N, K = case["N"], case["K"]
        return {"bytes": 4 * M * (N + K) + tape(K) + 8 * N * K + 4 * N, "flops": 4 * M * N * K + M * N}
    W, size, G = case["W"], DTYPES[case["dtype"]].itemsize, case["G"]
    params = 4 * W * (2 * case["post"] + 2 * case["pre"] + case["vec"])
    if op == "join":
        n = (3 + case["pre"]) * M * W * size + G * W * size + params
        if case["tape"]:
            n += (1 + case["pre"]) * (2 * tape(W) + 2 * M * W + 4 * M)
        return {"bytes": n, "flops": M * W * (4 + 6 * case["post"] + 6 * case["pre"])}
    n = (3 + case["pre"]) * M * W * size + 2 * G * W * size + 2 * params + tape(W) * (1 + case["pre"]) + 4 * M * (case["post"] + case["pre"])
    return {"bytes": n, "flops": M * W * (8 + 10 * case["post"] + 10 * case["pre"])}


# ------------------------------------------------------------------------------------------------------------ the definitions in 64 bits
def _pow2_64(e):
    """2^e, from its bits"""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _tape64(codes, bytes_, W, signed):
    """what a tape stands for: code times 2^(byte - 127)"""
    c = codes.to(torch.float64)
    c = torch.where(c > 127, c - 256, c) if signed else c
    return c[:, :W] * _pow2_64(bytes_.long() - 127).repeat_interleave(32, 1)[:, :W]


def _norm64(v, norm):
    mean = v.sum(1, keepdim=True) / v.shape[1] if norm == "layer" else 0.0
    r = (((v - mean) ** 2).sum(1, keepdim=True) / v.shape[1] + EPS) ** -0.5
    return (v - mean) * r, r


def _rounded64(v, kind):
    """v on the tape: the smallest power of two that the largest code can reach the block's top with, and the nearest code"""
    M, W = v.shape
    most, out = (255.0 if kind == "relu" else 127.0), torch.zeros_like(v)
    for c in range(0, W, 32):
        b = v[:, c:c + 32]
        top = (b.clamp(min=0) if kind == "relu" else b.abs()).max(1, keepdim=True).values
        e = torch.floor(torch.log2(torch.where(top > 0, top, torch.ones_like(top)) / most)) - 2
        for _ in range(4):
            e = torch.where(most * _pow2_64(e) < top, e + 1, e)
        step = _pow2_64(e.clamp(-126, 121))
        q = torch.round(b / step).clamp(-most, most)
        q = torch.where(b > 0, q.clamp(min=1), torch.zeros_like(q)) if kind == "relu" else q
        out[:, c:c + 32] = q * step
    return out


def exact(case, seed):
    s = prepare(case, seed)
    op, M = s["op"], s["M"]
    if op == "pack":
        x, step = s["x"], max(1, (1 << 25) // s["W"])
        return torch.cat([_rounded64(x[i:i + step].double(), s["kind"]).float() for i in range(0, M, step)])
    if op == "linear":
        N, K = s["N"], s["K"]
        w, step = s["w"].double(), 1 << 18
        dx = torch.empty(M, K, device="cuda")
        dw, db = torch.zeros(N, K, device="cuda", dtype=torch.float64), torch.zeros(N, device="cuda", dtype=torch.float64)
        for i in range(0, M, step):
            z = s["dz"][i:i + step].double()
            x = _tape64(s["codes"][i:i + step], s["bytes"][i:i + step], K, s["act"] != "relu")
            g = z @ w
            if s["act"] == "relu":
                g = g * (s["codes"][i:i + step, :K] != 0)
            if s["act"] == "swish":
                p = torch.sigmoid(x)
                g, x = g * (p + x * p * torch.sigmoid(-x)), x * p
            dx[i:i + step] = g.float()
            dw += z.t() @ x
            db += z.sum(0)
        return {"x": dx, "w": dw, "b": db}
    W, G, norm = s["W"], s["G"], s["norm"]
    gate = torch.ones(M, W, device="cuda", dtype=torch.float64)
    if G:
        gate = s["gate"].double()[torch.arange(M, device="cuda") // (M // G)]
    scale = s["scale"].double() if s["vec"] else s["scale"]
    par = {k: s[k].double() if s[k] is not None else (1.0 if k.endswith("g") else 0.0) for k in ("post_g", "post_b", "pre_g", "pre_b")}
    if op == "join":
        fhat, r = _norm64(s["f"].double(), norm) if s["post"] else (s["f"].double(), None)
        y = s["x"].double() + scale * gate * (fhat * par["post_g"] + par["post_b"])
        out = {"y": y}
        if s["pre"]:
            yhat, rp = _norm64(y, norm)
            out["h"] = yhat * par["pre_g"] + par["pre_b"]
        if s["tape"]:
            out["post"], out["post_rstd"] = _rounded64(fhat, "signed"), r[:, 0] if s["post"] else None
            if s["pre"]:
                out["pre"], out["pre_rstd"] = _rounded64(yhat, "signed"), rp[:, 0]
        return out
    # y = x + scale gate t(f), h = norm(y): the chain rule, each norm's gradient through its three terms
    d, out = s["gy"].double(), {}
    if s["pre"]:
        yhat, gh = _tape64(s["pre_codes"], s["pre_bytes"], W, True), s["gh"].double()
        u = gh * par["pre_g"]
        d = d + s["pre_rstd"].double()[:, None] * (u - (u.sum(1, keepdim=True) / W if norm == "layer" else 0.0) - yhat * ((u * yhat).sum(1, keepdim=True) / W))
        out["pre_g"], out["pre_b"] = (gh * yhat).sum(0), gh.sum(0) if s["pre_b"] is not None else None
    fhat = _tape64(s["post_codes"], s["post_bytes"], W, True)
    t = fhat * par["post_g"] + par["post_b"]
    out["x"] = d
    if G:
        out["gate"] = (scale * t * d).reshape(G, M // G, W).sum(1)
    if s["vec"]:
        out["scale"] = (gate * t * d).sum(0)
    v = scale * gate * d
    if s["post"]:
        out["post_g"], out["post_b"] = (v * fhat).sum(0), v.sum(0) if s["post_b"] is not None else None
        u = v * par["post_g"]
        v = s["post_rstd"].double()[:, None] * (u - (u.sum(1, keepdim=True) / W if norm == "layer" else 0.0) - fhat * ((u * fhat).sum(1, keepdim=True) / W))
    out["f"] = v
    return out
