"""The training operators on the GPU (include/ccsm_train_ops.h) against plain implementations in 64 bits.

Tolerances.  h = half a step of the type (fp32 2^-24, fp16 2^-11, bf16 2^-8), relative.
  product    a sum of K products kept in fp32: the k-th addition rounds a partial sum of about sqrt(k) s, s = rms of the products, by 2^-24 at most; the
             roundings add up like a random walk to 2^-24 s K / sqrt(6) = 2^-24 q sqrt(K) / 2.4, q = sqrt(sum (x w)^2).  Eight times that for the largest
             of many, and sqrt(6) for fp32 operands taken as six products of three pieces each: 2^-24 (8 sqrt(K) + 8) q.
  activation slopes are at most 1.13 in magnitude (gelu), the functions within 2^-20 absolute in 16-bit calls and 2^-22 in fp32 ones (times max(1, |z|)).
  rounding   h |y| for what is written, and in a 16-bit backward pass h |d| for each d before its products: errors that are independent of each
             other and of d's sign, so their sum is within 5 h sqrt(sum (d w)^2) (9 standard deviations of a uniform error)."""
import math

import pytest

torch = pytest.importorskip("torch")
from ccsmeth_amd import train_ops as ops  # noqa: E402
from ccsmeth_amd._lib import CcsmError  # noqa: E402

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
H = {F32: 2.0 ** -24, F16: 2.0 ** -11, BF16: 2.0 ** -8}
TINY = {F32: 2.0 ** -149, F16: 2.0 ** -24, BF16: 2.0 ** -133}
ACTS = ["none", "relu", "tanh", "sigmoid", "gelu", "silu"]
DEV = "cuda:0"


def normal(seed, *shape, t=F32, by=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, generator=g) * by).to(t).to(DEV)


def act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp_min(0), "tanh": lambda: z.tanh(), "sigmoid": lambda: torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z), "silu": lambda: z * torch.sigmoid(z)}[act]()


def slope64(z, act):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "tanh": lambda: 1 - z.tanh() ** 2, "sigmoid": lambda: s * (1 - s),
            "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi), "silu": lambda: s * (1 + z * (1 - s))}[act]()


def mm(a, b):
    return torch.mm(a, b)


def sum_tol(n):
    return 2.0 ** -24 * (8 * math.sqrt(n) + 8)


def within(got, ref, tol, t):
    """|got - ref| <= tol + h |ref| (+ the smallest step of the type), everywhere"""
    assert got.dtype is t and got.shape == ref.shape
    d = (got.double().cpu() - ref.cpu()).abs()
    lim = tol.cpu() + H[t] * (ref.cpu().abs() + tol.cpu()) + TINY[t]
    assert torch.isfinite(got.double()).all()
    over = d / lim
    assert float(over.max() if over.numel() else 0) <= 1, (float(over.max()), int(over.argmax()))


def act_tol(z, tz, t):
    return 1.13 * tz + (2.0 ** -22 if t is F32 else 2.0 ** -20) * z.abs().clamp_min(1)


def check_linear(x, w, b, r, act, t, y, z=None):
    x6, w6 = x.double().reshape(-1, x.shape[-1]), w.double()
    ref = mm(x6, w6.t())
    tz = sum_tol(x.shape[-1]) * mm(x6 ** 2, (w6 ** 2).t()).sqrt()
    if b is not None:
        ref = ref + b.double()
        tz = tz + 2.0 ** -23 * (ref.abs() + b.double().abs())
    if z is not None:
        within(z.reshape(ref.shape), ref, tz, t)
    out = act64(ref, act)
    ty = act_tol(ref, tz, t) if act != "none" else tz
    if r is not None:
        r6 = r.double().reshape(ref.shape)
        out, ty = out + r6, ty + 2.0 ** -24 * (out + r6).abs()
    within(y.reshape(ref.shape), out, ty, t)


SIZES = [(1, 1, 1), (1, 512, 768), (2, 11, 9), (3, 64, 5), (7, 129, 33), (16, 768, 256), (17, 40, 520), (33, 8, 130), (64, 256, 64), (65, 72, 128), (127, 31, 257),
         (128, 128, 128), (130, 200, 96), (255, 264, 136), (256, 64, 256), (257, 520, 264), (513, 96, 768), (1000, 11, 768), (1500, 512, 256)]


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear_sizes(t, m, k, n):
    act = ACTS[(m + k + n) % 6]
    x, w, b, r = normal(m, m, k, t=t), normal(k + 1, n, k, t=t, by=k ** -0.5), normal(n + 2, n, t=t, by=0.3), normal(3, m, n, t=t)
    y, z = ops.linear(x, w, b, r, activation=act, keep_preact=True)
    check_linear(x, w, b, r, act, t, y, z)
    check_linear(x, w, None, None, "none", t, ops.linear(x, w))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("m", [1, 5, 96, 300])
def test_linear_activations(t, act, m):
    """pre-activations from -9 to 9: the tails of every activation"""
    k, n = 24, 80
    x, w, b = normal(5, m, k, t=t), normal(6, n, k, t=t, by=0.1), torch.linspace(-9, 9, n).to(t).to(DEV)
    for r in (None, normal(8, m, n, t=t)):
        y, z = ops.linear(x, w, b, r, activation=act, keep_preact=True)
        check_linear(x, w, b, r, act, t, y, z)


def check_backward(dy, x, w, z, act, t, got):
    """x, z: the values that the call reads (of a checkpoint: the ones it stands for), in 64 bits"""
    dx, dw, db = got
    dy6, w6 = dy.double().reshape(-1, dy.shape[-1]), w.double()
    x6 = x.double().reshape(-1, x.shape[-1])
    d = dy6 * (slope64(z.double().reshape(dy6.shape), act) if act != "none" else 1.0)
    off = 0.0 if act == "none" else 2.0 ** -20 if t is not F32 else 2.0 ** -21      # the slope's own error, relative to dy
    hd = 0.0 if t is F32 or act == "none" else 5 * H[t]
    M, N = d.shape
    for out, a, b, ay, n in ((dx, d, w6, dy6, N), (dw, d.t(), x6, dy6.t(), M)):
        if out is None:
            continue
        q = mm(a ** 2, b ** 2).sqrt()
        qy = mm(ay ** 2, b ** 2).sqrt()
        sub = TINY[t] * b.abs().sum(0) if hd else 0.0            # d below the type's normal range
        within(out.reshape(q.shape), mm(a, b), (sum_tol(n) + hd) * q + 5 * off * qy + sub, t)
    if db is not None:
        within(db, d.sum(0), sum_tol(M) * (d ** 2).sum(0).sqrt() + 5 * off * (dy6 ** 2).sum(0).sqrt(), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_backward_sizes(t, m, k, n):
    act = ACTS[(m + k + 2 * n) % 6]
    dy, x, w, z = normal(1, m, n, t=t, by=0.05), normal(2, m, k, t=t), normal(3, n, k, t=t, by=k ** -0.5), normal(4, m, n, t=t)
    check_backward(dy, x, w, z, act, t, ops.linear_backward(dy, x, w, z if act != "none" else None, activation=act))
    check_backward(dy, x, w, z, "none", t, ops.linear_backward(dy, x, w))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
def test_backward_activations(t, act):
    m, k, n = 70, 24, 80
    dy, x, w = normal(1, m, n, t=t), normal(2, m, k, t=t), normal(3, n, k, t=t, by=0.2)
    z = torch.linspace(-9, 9, m * n).reshape(n, m).t().to(t).to(DEV)
    z[0, :3] = 0.0
    check_backward(dy, x, w, z, act, t, ops.linear_backward(dy, x, w, z, activation=act))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("xc,zc", [("int8", None), ("e4m3", None), (None, "int8"), (None, "e4m3"), ("int8", "e4m3"), ("e4m3", "int8")])
@pytest.mark.parametrize("m,k,n", [(1, 8, 8), (5, 33, 31), (64, 64, 96), (130, 40, 264), (257, 520, 72), (1031, 256, 136)])
def test_backward_from_checkpoints(t, xc, zc, m, k, n):
    dy, x, w, z = normal(1, m, n, t=t, by=0.05), normal(2, m, k, t=t), normal(3, n, k, t=t, by=k ** -0.5), normal(4, m, n, t=t, by=2.0)
    cx, cz = ops.checkpoint8(x, xc) if xc else x, ops.checkpoint8(z, zc) if zc else z
    got = ops.linear_backward(dy, cx, w, cz, activation="silu")
    check_backward(dy, in8(x, xc) if xc else x, w, in8(z, zc) if zc else z, "silu", t, got)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(40, 20, 41), (1500, 43, 299)])
def test_codes_behind_the_width_do_not_matter(t, m, k, n):
    """a caller's own checkpoints, the codes behind whose width stand for NaN"""
    dy, w = normal(1, m, n, t=t, by=0.05), normal(3, n, k, t=t, by=0.2)
    x, z = (ops.checkpoint8(normal(4, m, c, t=t), code) for c, code in ((k, "int8"), (n, "e4m3")))
    want = ops.linear_backward(dy, x, w, z, activation="silu")
    for c, nan in ((x, 0x80), (z, 0x7f)):
        c.codes[:, c.shape[-1]:] = nan
    for a, b in zip(want, ops.linear_backward(dy, x, w, z, activation="silu")):
        assert torch.equal(a, b) and torch.isfinite(a.float()).all()
    assert torch.isfinite(x.values().float()).all()


def test_backward_only_what_is_asked_for():
    dy, x, w, z = normal(1, 40, 24), normal(2, 40, 16), normal(3, 24, 16), normal(4, 40, 24)
    full = ops.linear_backward(dy, x, w, z, activation="tanh")
    for k in range(8):
        want = [bool(k & 1), bool(k & 2), bool(k & 4)]
        got = ops.linear_backward(dy, x if want[1] else None, w, z, activation="tanh", need_dx=want[0], need_dw=want[1], need_db=want[2])
        for g, f, on in zip(got, full, want):
            assert (g is None) == (not on) and (g is None or torch.equal(g, f))


@pytest.mark.parametrize("t", TYPES)
def test_no_rows(t):
    w = normal(1, 12, 8, t=t)
    assert ops.linear(normal(2, 0, 8, t=t), w).shape == (0, 12)
    dx, dw, db = ops.linear_backward(normal(2, 0, 12, t=t), normal(2, 0, 8, t=t), w, normal(2, 0, 12, t=t), activation="gelu")
    assert dx.shape == (0, 8) and not dw.any() and not db.any() and dw.shape == (12, 8)
    assert ops.embedding(torch.zeros(0, dtype=torch.int64, device=DEV), w).shape == (0, 8)
    assert not ops.embedding_backward(normal(2, 0, 8, t=t), torch.zeros(0, dtype=torch.int64, device=DEV), 7).any()
    c = ops.checkpoint8(normal(2, 0, 8, t=t))
    assert c.values().shape == (0, 8)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(3, 24, 40), (50, 24, 40), (300, 136, 264)])
def test_strides_and_alignment(t, m, k, n):
    """views into wider matrices, at odd offsets; what lies around the output stays as it was"""
    for off, pad in ((0, 8), (1, 3), (3, 0), (8, 16)):
        big = normal(9, m, k + off + pad, t=t)
        x = big[:, off:off + k]
        w = normal(10, n, k + off + pad, t=t, by=0.2)[:, off:off + k]
        r = normal(11, m, n + off + pad, t=t)[:, off:off + n]
        b = normal(12, n + off, t=t)[off:]
        hold = torch.full((m + 2, n + off + pad), 7.0, dtype=t, device=DEV)
        y = hold[1:m + 1, off:off + n]
        assert ops.linear(x, w, b, r, activation="tanh", out=y) is y
        check_linear(x, w, b, r, "tanh", t, y.clone())
        hold[1:m + 1, off:off + n] = 7.0
        assert (hold == 7).all()
        dy, z = normal(13, m, n + off + pad, t=t)[:, off:off + n], normal(14, m, n + off + pad, t=t)[:, off:off + n]
        check_backward(dy, x, w, z, "gelu", t, ops.linear_backward(dy, x, w, z, activation="gelu"))
        c = ops.checkpoint8(x, "e4m3")
        assert torch.equal(c.values().double(), in8(x, "e4m3"))
    x3 = normal(15, 4, 5, k, t=t)                                    # leading dimensions, and a layout that has to be copied
    w = normal(16, n, k, t=t, by=0.2)
    y3 = ops.linear(x3, w)
    assert y3.shape == (4, 5, n) and torch.equal(y3.reshape(20, n), ops.linear(x3.reshape(20, k), w))
    assert torch.equal(ops.linear(x3.transpose(0, 1), w), ops.linear(x3.transpose(0, 1).contiguous(), w))
    assert torch.equal(ops.linear(x3[0], w.t().contiguous().t()), ops.linear(x3[0], w))
    e = normal(17, 1, n, t=t).expand(20, n)                          # one row for all: a broadcast gradient
    g = ops.linear_backward(e, x3.reshape(20, k), w)
    for a, c in zip(g, ops.linear_backward(e.contiguous(), x3.reshape(20, k), w)):
        assert torch.equal(a, c)


@pytest.mark.parametrize("t", [F32, BF16])
@pytest.mark.parametrize("which", ["dy", "x", "w", "z"])
def test_rows_far_apart(t, which):
    """row strides past the kernels' 32-bit offsets"""
    m, k, n = 20, 24, 40
    dy, x, w, z = normal(1, m, n, t=t, by=0.05), normal(2, m, k, t=t), normal(3, n, k, t=t, by=0.2), normal(4, m, n, t=t)
    given = {"dy": dy, "x": x, "w": w, "z": z}
    far = torch.zeros(given[which].shape[0], (1 << 21) + 8, dtype=t, device=DEV)[:, :given[which].shape[1]]
    far.copy_(given[which])
    given[which] = far
    check_linear(given["x"], given["w"], None, None, "gelu", t, ops.linear(given["x"], given["w"], activation="gelu"))
    check_backward(dy, x, w, z, "silu", t, ops.linear_backward(given["dy"], given["x"], given["w"], given["z"], activation="silu"))


def test_residual_may_be_the_output():
    for t in TYPES:
        for m in (2, 200):
            x, w, r = normal(1, m, 64, t=t), normal(2, 72, 64, t=t, by=0.1), normal(3, m, 72, t=t)
            want = ops.linear(x, w, None, r, activation="relu")
            got = ops.linear(x, w, None, r, activation="relu", out=r)
            assert got is r and torch.equal(want, r)


@pytest.mark.parametrize("t", TYPES)
def test_magnitudes_far_apart(t):
    """rows that differ by 2^40 (fp16: 2^12) each keep their own precision; nothing is scaled by another row's size"""
    k = 96
    x, w = normal(1, 160, k, t=F32), normal(2, 130, k, t=F32, by=k ** -0.5)
    s = torch.exp2(torch.arange(160, device=DEV).float() % (12 if t is F16 else 40) - (6 if t is F16 else 20))
    x = (x * s[:, None]).to(t)
    w = (w * torch.exp2(-(torch.arange(130, device=DEV).float() % (4 if t is F16 else 30)))[:, None]).to(t)
    check_linear(x, w, None, None, "none", t, ops.linear(x, w))
    g = ops.linear_backward(x @ torch.zeros(k, 130, dtype=t, device=DEV) + normal(3, 160, 130, t=t) * s[:, None].to(t), x, w)
    assert all(torch.isfinite(v).all() for v in g)
    if t is F32:
        big = x.clone()
        big[0, 0], big[1, 1] = 3.4e38, -3.4e38                       # finite values at the end of the range
        w0 = torch.zeros_like(w)
        w0[:, 2:] = w[:, 2:]
        assert torch.isfinite(ops.linear(big, w0)).all()


def test_nan_stays_in_its_row():
    for t in TYPES:
        for m in (4, 200):
            x, w = normal(1, m, 64, t=t), normal(2, 48, 64, t=t, by=0.1)
            x[1, 3] = float("nan")
            y = ops.linear(x, w, activation="relu")
            assert y[1].isnan().all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("m,k,n", [(20, 600, 300), (300, 500, 400)])
def test_small_backward_rounds_only_its_results(t, m, k, n):
    """products this small keep what the rounding of d to 16 bits leaves: what is left of the error is the results' own rounding, and a hundredth for the
    sums, the slopes (2^-20 of dy) and the second piece's rounding (2^-11 of half a step in fp16, 2^-8 in bf16)"""
    dy, x, w, z = normal(1, m, n, t=t, by=0.05), normal(2, m, k, t=t), normal(3, n, k, t=t, by=k ** -0.5), normal(4, m, n, t=t)
    d = dy.double() * slope64(z.double(), "gelu")
    dx, dw, _ = ops.linear_backward(dy, x, w, z, activation="gelu")
    for out, ref in ((dx, mm(d, w.double())), (dw, mm(d.t(), x.double()))):
        assert float((out.double() - ref).norm()) <= 1.01 * float((ref.to(t).double() - ref).norm())


@pytest.mark.parametrize("t", [F16, BF16])
@pytest.mark.parametrize("m", [8, 600])
def test_an_infinite_d_stays_infinite(t, m):
    """of both ways: d past the type's range (fp16: 65504 x 1.1), and an infinite dy"""
    dy, x, w = normal(1, m, 40, t=t, by=0.05), normal(2, m, 32, t=t), torch.full((40, 32), 0.5, dtype=t, device=DEV)
    z = torch.full((m, 40), 1.5, dtype=t, device=DEV)             # (gelu's and silu's slope is more than 1 there)
    dy[1, 3], dy[2, 5] = torch.finfo(t).max, float("inf")
    for act in ("gelu", "relu"):
        dx, _, _ = ops.linear_backward(dy, x, w, z, activation=act)
        assert torch.isfinite(dx[0]).all() and torch.isfinite(dx[3:]).all()
        assert bool((dx[2] == float("inf")).all()) and bool((dx[1] > 0).all())


# ---- 8-bit checkpoints ----------------------------------------------------------------------------------------------
def in8(x, code):
    """what the header says, in 64 bits: blocks of 32, the least power of two, nearest code with ties to even, the type's range kept"""
    t = x.dtype
    v = x.detach().double().cpu().reshape(-1, x.shape[-1])                           # on the host, whose pow is exact for whole exponents
    m, n = v.shape
    full = torch.zeros(m, -(-n // 32) * 32, dtype=torch.float64)
    full[:, :n] = v
    full = full.reshape(m, -1, 32)
    fin = torch.isfinite(full)
    most = torch.where(fin, full.abs(), 0.0).amax(2, keepdim=True)
    top = 127.0 if code == "int8" else 448.0
    e = torch.frexp(most).exponent - (7 if code == "int8" else 9)
    p = torch.pow(torch.full_like(most, 2.0), e.clamp_min(-200))
    p = torch.where(most > top * p, 2 * p, p).clamp_min(2.0 ** -126)
    u = full / p
    if code == "int8":
        q = torch.round(u)
    else:
        step = torch.pow(torch.full_like(u, 2.0), torch.frexp(torch.where(fin, u, 0.0)).exponent.clamp_min(-5) - 4)
        q = torch.round(torch.where(fin, u, 0.0) / step) * step
    most_t = float(torch.finfo(t).max)
    below = 63.0 if code == "int8" else 240.0
    q = torch.where((q * p).abs() > most_t, torch.sign(q) * below, q)
    return torch.where(fin, q * p, float("nan")).reshape(m, -1)[:, :n].reshape(x.shape).to(x.device)


def same(a, b):
    a, b = a.double().cpu(), b.double().cpu()
    assert torch.equal(a.isnan(), b.isnan())
    assert torch.equal(torch.nan_to_num(a, 0.0), torch.nan_to_num(b, 0.0))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("m,n", [(1, 1), (1, 31), (2, 32), (3, 33), (5, 64), (7, 500), (65, 512), (130, 96), (1000, 40)])
def test_checkpoint_values(t, code, m, n):
    x = normal(m + n, m, n, t=F32)
    x = (x * torch.exp2(normal(2, m, n) * 3)).to(t)
    c = ops.checkpoint8(x, code)
    assert c.codes.shape == (m, -(-n // 32) * 32) and c.nbytes == c.codes.numel() + c.scales.numel()
    want = in8(x, code)
    same(c.values(), want)
    assert c.values().dtype is t and torch.equal(c.values().double(), want)          # the type holds them exactly
    for o in TYPES:
        same(c.values(o), want.to(o) if o is not F16 else want.float().to(o))
    assert not c.codes[:, n:].any()
    again = ops.checkpoint8(c.values(), code)                                        # a checkpoint of its own values is the same again
    same(again.values(), want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_checkpoint_special_values(t, code):
    inf, nan, mx, tiny = float("inf"), float("nan"), torch.finfo(t).max, torch.finfo(t).tiny
    rows = [[0.0] * 40, [inf] + [1.0] * 39, [nan, -inf, 0.5, -0.25] + [3.0] * 36, [mx, -mx] + [mx / 3] * 38, [tiny] * 40, [tiny / 4, -tiny / 8] + [0.0] * 38,
            [127.0, 63.5, 0.5, 1.5, 2.5, -0.5, -1.5] + [1.0] * 33, [448.0, 17.0, 19.0, 0.001953125, 0.0009765625] + [2.0] * 35, [float(i) for i in range(40)],
            [nan] * 40, [inf, -inf] * 20, [-127.5] + [0.3] * 39, [449.0, 447.0] + [1.0] * 38, [1e-3 * i for i in range(40)]]
    x = torch.tensor(rows, dtype=torch.float64).to(t).to(DEV)
    same(ops.checkpoint8(x, code).values(), in8(x, code))
    x = x[:, :32].contiguous().repeat(1, 2)                                          # whole blocks
    same(ops.checkpoint8(x, code).values(), in8(x, code))


# ---- embedding ------------------------------------------------------------------------------------------------------
IDS = [torch.uint8, torch.int32, torch.int64]


def check_embedding(ids, table, dy, scale, y, dt, t):
    v = table.shape[0]
    i = ids.long().reshape(-1)
    ok = (i >= 0) & (i < v)
    ref = torch.zeros(len(i), table.shape[1], dtype=torch.float64, device=DEV)
    ref[ok] = table.double()[i[ok]] * scale
    within(y.reshape(ref.shape), ref, 2.0 ** -24 * ref.abs(), t)
    d = dy.double().reshape(len(i), -1)[ok].cpu()
    at = i[ok].cpu()
    g = torch.zeros(v, table.shape[1], dtype=torch.float64).index_add_(0, at, d) * scale
    sq = torch.zeros(v, table.shape[1], dtype=torch.float64).index_add_(0, at, d ** 2).sqrt() * abs(scale)
    n = torch.bincount(at, minlength=v).double().sqrt()[:, None]
    within(dt, g, 2.0 ** -24 * (8 * n + 8) * sq, t)
    assert not dt.cpu()[n[:, 0] == 0].any()


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,rows,width", [(1, 1, 1), (1, 300, 8), (2, 5, 8), (31, 5, 8), (33, 4, 12), (64, 70, 9), (1000, 5, 8), (1024, 256, 40), (3000, 200, 264), (4097, 4097, 72),
                                               (5000, 70000, 16), (20000, 33, 3), (9000, 17, 520), (300, 1000, 2056)])
def test_embedding(t, tokens, rows, width):
    for k, it in enumerate(IDS):
        if it is torch.uint8 and rows > 256:
            continue
        g = torch.Generator().manual_seed(tokens + k)
        ids = (torch.rand(tokens, generator=g) ** 3 * rows).long().clamp_max(rows - 1)
        if it is not torch.uint8:
            ids[5::17], ids[6::19] = -1, rows + 3                     # no tokens
        ids = ids.to(it).to(DEV)
        table, dy, scale = normal(1, rows, width, t=t), normal(2, tokens, width, t=t, by=0.1), (1.0, 0.125, width ** 0.5)[k]
        check_embedding(ids, table, dy, scale, ops.embedding(ids, table, scale), ops.embedding_backward(dy, ids, rows, scale), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("tokens,rows,width", [(1, 15, 1), (7, 1, 2048), (300, 15, 4), (5000, 15, 136), (5000, 16, 128), (20000, 2, 1024), (20000, 3, 1024), (300, 15, 137), (40000, 15, 33), (200001, 5, 8)])
def test_embedding_of_few_rows(t, tokens, rows, width):
    """tables that are not sorted for, up to their largest and one more row; a gradient and a table with strides of their own"""
    g = torch.Generator().manual_seed(rows)
    ids = torch.randint(-1, rows + 1, (tokens,), generator=g)
    if rows > 2:
        ids[ids == 1] = 2                                             # a row that no token names
    ids = ids.to(torch.int32).to(DEV)
    table, dy = normal(1, rows, width + 3, t=t)[:, 1:1 + width], normal(2, tokens, width + 5, t=t, by=0.1)[:, 3:3 + width]
    check_embedding(ids, table, dy, 0.5, ops.embedding(ids, table, 0.5), ops.embedding_backward(dy, ids, rows, 0.5), t)
    nan = dy.clone()
    nan[0] = float("nan")
    got = ops.embedding_backward(nan, ids, rows, 0.5)
    at = int(ids[0])
    assert torch.isfinite(got[[r for r in range(rows) if r != at]].float()).all() and (not 0 <= at < rows or got[at].isnan().all())


@pytest.mark.parametrize("t", TYPES)
def test_embedding_extremes(t):
    """every token the same; every token another one; none; the last row only; ids beyond 32 bits; rows that no token names"""
    tokens, width = 9000, 24
    table, dy = normal(1, 9000, width, t=t), normal(2, tokens, width, t=t, by=0.1)
    for ids in (torch.zeros(tokens), torch.full((tokens,), 8999), torch.arange(tokens), torch.arange(tokens).flip(0), torch.full((tokens,), -1),
                torch.arange(tokens) // 32, torch.arange(tokens) // 33 * 7, torch.arange(tokens) * (1 << 33), torch.arange(tokens) - (1 << 40)):
        ids = ids.long().to(DEV)
        check_embedding(ids, table, dy, 2.0, ops.embedding(ids, table, 2.0), ops.embedding_backward(dy, ids, 9000, 2.0), t)
    ids = (torch.arange(tokens) % 7).to(torch.uint8).to(DEV)
    out = torch.full((11, width + 5), 3.0, dtype=t, device=DEV)
    ops.embedding_backward(dy, ids, 9, 1.0, out=out[1:10, 2:2 + width])
    check_embedding(ids, table[:9], dy, 1.0, ops.embedding(ids, table[:9]), out[1:10, 2:2 + width], t)
    out[1:10, 2:2 + width] = 3.0
    assert (out == 3).all()
    i2 = ids.reshape(9, 1000)
    y = ops.embedding(i2, table[:9])
    assert y.shape == (9, 1000, width) and torch.equal(ops.embedding_backward(dy.reshape(9, 1000, width), i2, 9), ops.embedding_backward(dy, ids, 9))
    wide = normal(5, 9, 2 * width + 1, t=t)
    view = wide[:, 1:1 + width]
    assert torch.equal(ops.embedding(ids, view), ops.embedding(ids, view.contiguous()))


@pytest.mark.parametrize("tokens,rows,width", [(131073, 300, 2), (140000, 70000, 1), (524289, 3000, 1), (700001, 5, 3)])
def test_embedding_many_tokens(tokens, rows, width):
    """the sort's larger workgroups, and more of them than add the counts up themselves"""
    for t in (F32, BF16):
        g = torch.Generator().manual_seed(tokens)
        ids = (torch.rand(tokens, generator=g) ** 2 * rows).long().clamp_max(rows - 1)
        ids[::1001] = -7
        ids = ids.to(torch.int32).to(DEV)
        table, dy = normal(1, rows, width, t=t), normal(2, tokens, width, t=t, by=0.1)
        check_embedding(ids, table, dy, 1.5, ops.embedding(ids, table, 1.5), ops.embedding_backward(dy, ids, rows, 1.5), t)


# ---- how the calls are used -----------------------------------------------------------------------------------------
def _step(s, stream=None):
    """tokens -> embedding -> two layers with a residual -> gradients from 8-bit checkpoints -> the table's gradient"""
    h = ops.embedding(s["ids"], s["table"], 4.0, stream=stream)
    a, z = ops.linear(h, s["w1"], s["b1"], activation="gelu", keep_preact=True, stream=stream)
    ch, cz, ca = ops.checkpoint8(h, "e4m3", stream=stream), ops.checkpoint8(z, "e4m3", stream=stream), ops.checkpoint8(a, "int8", stream=stream)
    y = ops.linear(a, s["w2"], s["b2"], h, stream=stream)
    da, dw2, db2 = ops.linear_backward(s["dy"], ca, s["w2"], stream=stream)
    dh, dw1, db1 = ops.linear_backward(da, ch, s["w1"], cz, activation="gelu", stream=stream)
    dh = dh + s["dy"] if stream is None else _add(dh, s["dy"], stream)               # the residual's gradient
    return y, dw2, db2, dw1, db1, ops.embedding_backward(dh, s["ids"], len(s["table"]), 4.0, stream=stream)


def _add(a, b, stream):
    with torch.cuda.stream(stream):
        return a + b


def _state(seed, m=300, v=50, k=64, n=136, t=BF16):
    g = torch.Generator().manual_seed(seed)
    return {"ids": torch.randint(-1, v, (m,), generator=g).to(DEV), "table": normal(seed + 1, v, k, t=t, by=0.25), "w1": normal(seed + 2, n, k, t=t, by=k ** -0.5),
            "b1": normal(seed + 3, n, t=t, by=0.1), "w2": normal(seed + 4, k, n, t=t, by=n ** -0.5), "b2": normal(seed + 5, k, t=t, by=0.1), "dy": normal(seed + 6, m, k, t=t, by=0.1)}


@pytest.mark.parametrize("t", TYPES)
def test_a_step_of_them_together(t):
    """against autograd in 64 bits on the plain formulas: bounded by what 8-bit checkpoints and the types' roundings may do (relative 2-norm: e4m3 keeps a
    factor within 2^-4, on average 2^-5.3; int8 of a block within 2^-7 of its largest; each gradient has two such factors at most)"""
    s = _state(1, t=t)
    got = _step(s)
    p = {k: s[k].double().cpu().requires_grad_() for k in ("table", "w1", "b1", "w2", "b2")}
    ids = s["ids"].cpu()
    h = torch.where((ids >= 0)[:, None], p["table"][ids.clamp_min(0)] * 4.0, 0.0)
    z = h @ p["w1"].t() + p["b1"]
    y = (z * torch.special.ndtr(z)) @ p["w2"].t() + p["b2"] + h
    (y * s["dy"].double().cpu()).sum().backward()
    refs = (y.detach(), p["w2"].grad, p["b2"].grad, p["w1"].grad, p["b1"].grad, p["table"].grad)
    lim = (8 * H[t], 2.0 ** -6 + 8 * H[t], 8 * H[t] + 2.0 ** -22, 2.0 ** -4, 2.0 ** -4, 2.0 ** -4)
    for a, b, m in zip(got, refs, lim):
        assert float((a.double().cpu() - b).norm() / b.norm()) <= m


def test_the_same_bits_every_time_and_on_any_stream():
    s = _state(2, m=5000)
    first = _step(s)
    side = torch.cuda.Stream()
    for k in range(3):
        for a, b in zip(first, _step(s)):
            assert torch.equal(a, b)
    torch.cuda.synchronize()
    got = _step(s, stream=side)
    junk = [torch.full((5000, 136), 9.0, device=DEV, dtype=BF16) for _ in range(8)]      # what the call's scratch was must not be handed out again under it
    side.synchronize()
    for a, b in zip(first, got):
        assert torch.equal(a, b)
    del junk
    with pytest.raises(TypeError):
        ops.linear(s["dy"], s["w1"], stream=7)


def test_captured_and_replayed():
    """two graphs of a step, replayed in turn with eager work between them, on inputs that change in place"""
    sa, sb = _state(3), _state(40, m=777, v=5000, k=72, n=40)
    graphs = []
    for s in (sa, sb):
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            _step(s)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(s)
        graphs.append((g, s, out))
    for k in range(4):
        for j, (g, s, out) in enumerate(graphs):
            new = _state(100 * k + j, m=s["dy"].shape[0], v=s["table"].shape[0], k=s["table"].shape[1], n=s["w1"].shape[0])
            for name in s:
                s[name].copy_(new[name])
            want = [v.clone() for v in _step(s)]
            for v in out:
                v.zero_()
            g.replay()
            if k % 2:
                torch.cuda.synchronize()
            for a, b in zip(want, out):
                assert torch.equal(a, b)


def test_gradient_against_differences():
    """fp32: (L(p + h v) - L(p - h v)) / 2h = <grad, v> for L = sum(y g): the central difference is off by h^2 / 6 times the third derivative
    (|act'''| < 2 over arguments that move by h |v.x| < 4h here: below 2^-12 of the norm at h = 2^-6) and by L's own rounding, 2^-22 |L|-sums / h"""
    m, k, n, h = 96, 48, 80, 2.0 ** -6
    x, w, b, g = normal(1, m, k), normal(2, n, k, by=k ** -0.5), normal(3, n, by=0.2), normal(4, m, n)
    for act in ("tanh", "sigmoid", "gelu", "silu"):
        y, z = ops.linear(x, w, b, activation=act, keep_preact=True)
        grads = ops.linear_backward(g, x, w, z, activation=act)
        for which, grad in enumerate(grads):
            p = (x, w, b)[which]
            v = torch.sign(grad)                                     # along the gradient, so that <grad, v> is not a small difference
            v = v / (8 if which == 1 else 4 if which == 0 else 1)

            def loss(s):
                q = [x, w, b]
                q[which] = p + s * h * v
                return (ops.linear(*q, activation=act).double() * g.double()).sum()
            num = float((loss(1) - loss(-1)) / (2 * h))
            ana = float((grad.double() * v.double()).sum())
            assert abs(num - ana) <= 0.01 * abs(ana), (act, which, num, ana)


def test_refusals_on_the_gpu():
    x, w = normal(1, 4, 8), normal(2, 6, 8)
    for call in (lambda: ops.linear(x, w.half()), lambda: ops.linear(x[:, :7], w), lambda: ops.linear(x, w.cpu()), lambda: ops.linear(x, w, x[0]),
                 lambda: ops.linear(x, w, residual=x), lambda: ops.linear(x, w, out=torch.empty(4, 7, device=DEV)), lambda: ops.linear(x, w, out=torch.empty(6, 4, device=DEV).t()),
                 lambda: ops.linear_backward(x, x, w), lambda: ops.linear_backward(normal(1, 4, 6), x, w, activation="tanh"),
                 lambda: ops.linear_backward(normal(1, 4, 6), ops.checkpoint8(x.half()), w), lambda: ops.linear_backward(normal(1, 4, 6), None, w),
                 lambda: ops.embedding(torch.zeros(3, device=DEV), w), lambda: ops.embedding(torch.zeros(3, dtype=torch.int64), w),
                 lambda: ops.embedding_backward(x, torch.zeros(5, dtype=torch.int64, device=DEV), 3), lambda: ops.embedding_backward(x, torch.zeros(4, dtype=torch.int64, device=DEV), 0),
                 lambda: ops.checkpoint8(x.double()), lambda: ops.checkpoint8(x).values(torch.float64)):
        with pytest.raises(ValueError):
            call()


# ---- the trainer with its gates in 8 bits ---------------------------------------------------------------------------
@pytest.mark.parametrize("n,dropout", [(64, 0.0), (64, 0.5), (512, 0.0), (512, 0.5)])
def test_trainer_with_gates_in_8_bits(n, dropout):
    """64 sites: the stepwise kernels, 512: the fused ones.  The forward pass is the same; each of the 21 backward steps multiplies by four gates that are off
    by 2^-7 at most (half a step of 2^-6: blocks whose largest gate is near 1), with errors that are independent of each other: sqrt(84) 2^-7 /
    sqrt(3) = 0.041 of a gradient's norm at most, below 2^-4."""
    import numpy as np
    from ccsmeth_amd.train import Trainer, PARAM_NAMES
    from ccsmeth_amd.utils import synth
    w, sites = synth.synth_weights(5), synth.synth_sites(n, 6)
    labels = np.random.default_rng(7).integers(0, 2, n)
    h0 = synth.synth_h0(n, 8)
    res = []
    for bits in (32, 8, 8):
        tr = Trainer(w, device=0, max_sites=n + 3, activation_bits=bits)
        loss, logits = tr.forward_backward(sites, labels, h0=h0, dropout_rate=dropout, seed=9, want_logits=True)
        res.append((loss, logits, tr.grads()))
        norm = tr.step(1e-3)
        assert np.isfinite(norm)
        assert np.isfinite(tr.forward_backward(sites, labels, h0=h0, dropout_rate=dropout, seed=9, step=1)[0])
        tr.close()
    (la, ga, a), (lb, gb, b), (lc, gc, c) = res
    assert la == lb == lc and np.array_equal(ga, gb)
    differ = 0
    for k in PARAM_NAMES:
        assert np.array_equal(b[k], c[k])                            # the same bits every time
        off = np.linalg.norm(b[k].astype(np.float64) - a[k]) / np.linalg.norm(a[k].astype(np.float64))
        assert off <= 2.0 ** -4, (k, off)
        differ += off > 0
    assert differ > 20                                               # (the checkpoints are what the gradients are computed from)


def test_trainer_with_gates_in_8_bits_takes_less_memory():
    from ccsmeth_amd.train import Trainer
    from ccsmeth_amd.utils import synth
    w, n, took = synth.synth_weights(5), 2048, []
    for bits in (32, 8):
        torch.cuda.synchronize()
        before = torch.cuda.mem_get_info()[0]
        tr = Trainer(w, device=0, max_sites=n, activation_bits=bits)
        took.append(before - torch.cuda.mem_get_info()[0])
        tr.close()
    rows = 21 * 2 * n * 256                                          # values of one gate array: 24 arrays in fp32 against 8, and 24 of 33 / 32 bytes
    assert abs((took[0] - took[1]) - rows * (16 * 4 - 24 * 33 / 32)) < 64 << 20, took


# ---- gradients over the whole range of dy -----------------------------------------------------------------------------
def check_range(dy, x, w, z, act, t, got, rounds):
    """rounds: the relative error of a d before its products.  In fp16 a d below 2^-28 of dy's largest magnitude A is off by 2^-39 A at most."""
    d = dy.double() * slope64(z.double(), act)
    off = 2.0 ** -20 if t is not F32 else 2.0 ** -21
    step = 2.0 ** -39 * float(dy[torch.isfinite(dy)].abs().max()) if t is F16 else 0.0
    M, N = d.shape
    for out, a, b, ay, n in ((got[0], d, w.double(), dy.double(), N), (got[1], d.t(), x.double(), dy.double().t(), M)):
        q, qy, qb = mm(a ** 2, b ** 2).sqrt(), mm(ay ** 2, b ** 2).sqrt(), (b ** 2).sum(0).sqrt()
        within(out, mm(a, b), (sum_tol(n) + 5 * rounds) * q + 5 * off * qy + 5 * step * qb, t)
    if got[2] is not None:
        within(got[2], d.sum(0), sum_tol(M) * (d ** 2).sum(0).sqrt() + 5 * off * (dy.double() ** 2).sum(0).sqrt(), t)


@pytest.mark.parametrize("act", ["sigmoid", "gelu"])
@pytest.mark.parametrize("by", [2.0 ** -20, 2.0 ** -16, 2.0 ** -12, 1.0, 2.0 ** 8])
@pytest.mark.parametrize("m,k,n", [(600, 40, 72), (3000, 64, 300), (1500, 129, 33)])
def test_fp16_gradients_of_small_and_large_dy(m, k, n, by, act):
    """the tile kernels: more than 512 rows"""
    dy, x, z = normal(1, m, n, t=F16, by=by), normal(2, m, k, t=F16, by=min(1.0, 1 / by)), normal(4, m, n, t=F16)
    w = normal(3, n, k, t=F16, by=k ** -0.5)
    check_range(dy, x, w, z, act, F16, ops.linear_backward(dy, x, w, z, activation=act), H[F16])


def test_fp16_sums_of_many_small_gradients():
    """32768 rows of d = 8.9e-9 (dy: the smallest magnitude that fp16 has): dw = 2.9e-4; and one d past the type's range in a batch of small ones"""
    m = 32768
    dy, x, z = torch.full((m, 8), 2.0 ** -24, dtype=F16, device=DEV), torch.ones(m, 8, dtype=F16, device=DEV), torch.full((m, 8), 1.5, dtype=F16, device=DEV)
    w = normal(3, 8, 8, t=F16)
    check_range(dy, x, w, z, "sigmoid", F16, ops.linear_backward(dy, x, w, z, activation="sigmoid"), H[F16])
    dy = normal(1, 600, 40, t=F16, by=0.05)
    dy[1, 3] = 60000.0                                                # gelu's slope at 1.5 is 1.127
    x, w, z = normal(2, 600, 32, t=F16, by=0.01), normal(3, 40, 32, t=F16, by=0.01), torch.full((600, 40), 1.5, dtype=F16, device=DEV)
    check_range(dy, x, w, z, "gelu", F16, ops.linear_backward(dy, x, w, z, activation="gelu", need_db=False), H[F16])      # (db itself is past the range)


def test_fp16_gradients_of_a_zero_dy():
    dy, x, w, z = torch.zeros(600, 40, dtype=F16, device=DEV), normal(2, 600, 32, t=F16), normal(3, 40, 32, t=F16), normal(4, 600, 40, t=F16)
    assert not any(v.any() for v in ops.linear_backward(dy, x, w, z, activation="gelu"))


# ---- infinities and NaN -----------------------------------------------------------------------------------------------
def check_special(got, ref, tol, t):
    """infinite, of one sign or the other, and NaN where the 64-bit form is; within tolerance elsewhere"""
    got, ref = got.cpu(), ref.cpu()
    fin = torch.isfinite(ref)
    assert 0 < int(fin.sum()) < fin.numel()
    assert torch.equal(got.isnan(), ref.isnan()) and torch.equal(got == float("inf"), ref == float("inf")) and torch.equal(got == -float("inf"), ref == -float("inf"))
    within(got[fin], ref[fin], tol.cpu()[fin], t)


def host_mm(a, b):
    return torch.mm(a.double().cpu(), b.double().cpu())


def with_specials(v, rows, odd=0):
    """v with infinities of both signs, a NaN, and zeros beside them, in the named rows"""
    inf = float("inf")
    v[rows[0], 3 + odd], v[rows[1], 5], v[rows[2], 0], v[rows[2], 7], v[rows[3], 2] = inf, -inf, inf, -inf, float("nan")
    v[rows[4], 3], v[rows[4], 5] = 0.0, 0.0                            # (an infinity of the other operand meets a zero)
    return v


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("m,k,n", [(6, 24, 40), (70, 1100, 40), (90, 1101, 33), (200, 40, 72), (3000, 64, 777)])
def test_infinities_forward(t, m, k, n):
    """the small kernel, the tiles with a split contraction, with staged operands, and without"""
    x, w = with_specials(normal(1, m, k, t=t), (1, 2, 3, 4, 5)), normal(2, n, k, t=t, by=k ** -0.5)
    w[7, 3], w[8, 5] = 0.0, 0.0
    w[9, 1], w[10, 2] = float("inf"), -float("inf")
    ref = host_mm(x, w.t())
    tol = sum_tol(k) * host_mm(x.double() ** 2, w.double().t() ** 2).sqrt()
    check_special(ops.linear(x, w), ref, tol, t)
    y, z = ops.linear(x, w, None, x.new_ones(m, n), activation="relu", keep_preact=True)
    check_special(z, ref, tol, t)
    check_special(y, ref.clamp_min(0) + 1, tol + 2.0 ** -23 * (ref.abs() + 1), t)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ["none", "silu", "relu"])
@pytest.mark.parametrize("m,k,n", [(8, 40, 64), (200, 40, 72), (700, 40, 72), (1500, 65, 77)])
def test_infinities_backward(t, act, m, k, n):
    dy, x, w = with_specials(normal(1, m, n, t=t, by=0.05), (1, 2, 3, 4, 5)), with_specials(normal(2, m, k, t=t), (0, 1, 6, 7, 5), 1), normal(3, n, k, t=t, by=0.2)
    z = normal(4, m, n, t=t)
    w[9, 1], w[10, 2] = float("inf"), -float("inf")
    d = dy.double().cpu() * (slope64(z.double(), act).cpu() if act != "none" else 1.0)
    got = ops.linear_backward(dy, x, w, z if act != "none" else None, activation=act)
    hd, off = (0.0 if t is F32 or act == "none" else 5 * H[t]), (0.0 if act == "none" else 2.0 ** -20)
    for out, a, b, ay, c in ((got[0], d, w, dy.cpu(), n), (got[1], d.t(), x, dy.cpu().t(), m)):
        b = b.double().cpu()
        check_special(out, host_mm(a, b), (sum_tol(c) + hd) * host_mm(a ** 2, b ** 2).sqrt() + 5 * off * host_mm(ay.double() ** 2, b ** 2).sqrt(), t)
    check_special(got[2], d.sum(0), sum_tol(m) * (d ** 2).sum(0).sqrt() + 5 * off * (dy.double().cpu() ** 2).sum(0).sqrt(), t)


@pytest.mark.parametrize("m,k,n", [(6, 24, 40), (70, 1100, 40), (3000, 64, 777)])
def test_products_past_the_range_of_fp32_are_infinite(m, k, n):
    """finite operands; and a NaN whose bits beyond the first sixteen alone say so, values of the smallest kind beside an infinity"""
    x, w = normal(1, m, k), normal(2, n, k, by=k ** -0.5)
    x[1, 3], x[2, 3] = 3.0e38, -3.0e38
    w[:, 3] = 1.7e38
    x[4, 5] = torch.tensor(0x7f800001, dtype=torch.int32).view(torch.float32)
    x[5, 7], w[:, 7] = float("inf"), 2.0 ** -149
    w[3, 7] = -2.0 ** -149
    x[0, 3] = x[3, 3] = 0.0
    x[5:, 3] = 0.0
    y = ops.linear(x, w)
    assert bool((y[1] == float("inf")).all()) and bool((y[2] == -float("inf")).all()) and bool(y[4].isnan().all())
    assert float(y[5, 3]) == -float("inf") and bool((y[5, :3] == float("inf")).all()) and bool((y[5, 4:] == float("inf")).all())
    assert torch.isfinite(y[0]).all() and torch.isfinite(y[3]).all()


@pytest.mark.parametrize("act", ["sigmoid", "gelu"])
@pytest.mark.parametrize("by", [2.0 ** -20, 2.0 ** -16, 2.0 ** -12, 1.0, 2.0 ** 8])
@pytest.mark.parametrize("m,k,n", [(1, 40, 72), (20, 600, 300), (300, 129, 33), (500, 200, 60)])
def test_fp16_gradients_of_small_and_large_dy_small_products(m, k, n, by, act):
    """the small kernel takes d in two pieces of bf16: off by 2^-16 of it (and 2^-133, bf16's smallest step, which is none beside fp16's)"""
    dy, x, z = normal(1, m, n, t=F16, by=by), normal(2, m, k, t=F16, by=min(1.0, 1 / by)), normal(4, m, n, t=F16)
    w = normal(3, n, k, t=F16, by=k ** -0.5)
    check_range(dy, x, w, z, act, F16, ops.linear_backward(dy, x, w, z, activation=act), 2.0 ** -16)


def test_fp16_small_products_of_a_d_past_the_range():
    dy = normal(1, 60, 40, t=F16, by=0.05)
    dy[1, 3], dy[7, 0], dy[8, 0] = 60000.0, 2.0 ** -24, -2.0 ** -20      # gelu's slope at 1.5 is 1.127
    dy[7, 1:], dy[8, 1:] = 0.0, 0.0
    x, w, z = normal(2, 60, 32, t=F16, by=0.01), normal(3, 40, 32, t=F16, by=0.01), torch.full((60, 40), 1.5, dtype=F16, device=DEV)
    w[0] = 60.0
    check_range(dy, x, w, z, "gelu", F16, ops.linear_backward(dy, x, w, z, activation="gelu", need_db=False), 2.0 ** -16)


def test_outputs_that_share_memory_are_refused():
    hold = normal(1, 40, 96)
    x, y, w = hold[:, :32], hold[:, 32:64], normal(2, 32, 32)
    want = ops.linear(x, w, residual=y)
    for call in (lambda: ops.linear(x, w, out=x), lambda: ops.linear(x, w, out=hold[:, 20:52]), lambda: ops.linear(x[:32], w, out=w), lambda: ops.linear(x, w, residual=hold[:, 40:72], out=y),
                 lambda: ops.linear(x, w, bias=hold[3, 33:65], out=y), lambda: ops.embedding(torch.zeros(32, dtype=torch.int64, device=DEV), w, out=w),
                 lambda: ops.embedding_backward(x, torch.zeros(40, dtype=torch.int64, device=DEV), 32, out=hold[:32, 16:48])):
        with pytest.raises(CcsmError, match="shares memory"):
            call()
    got = ops.linear(x, w, residual=y, out=y)                         # beside x in the same rows, and the residual itself
    assert got is y and torch.equal(y, want)
    room = torch.zeros(40 * 32 * 4, dtype=torch.uint8, device=DEV)
    c = ops.checkpoint8(x)
    room[:1280].copy_(c.codes.reshape(-1))
    c = ops.Checkpoint8(room[:1280].view(40, 32), c.scales, c.shape, F32, "int8")
    with pytest.raises(CcsmError, match="shares memory"):
        c.values(out=room.view(F32).view(40, 32))


# ---- sizes past 32 bits -------------------------------------------------------------------------------------------------
def test_products_of_more_than_2_to_32_elements():
    """x of 4.4e9 elements: the last rows are what a call on them alone gives, dw is the sum of its halves'"""
    m, k, n = (1 << 23) + 77, 520, 16
    x = torch.empty(m, k, dtype=BF16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(1))
    w, dy = normal(2, n, k, t=BF16, by=k ** -0.5), normal(3, m, n, t=BF16, by=2.0 ** -6)
    y = ops.linear(x, w)
    for part in (slice(0, 1000), slice(m // 2, m // 2 + 1000), slice(m - 1000, m)):
        check_linear(x[part], w, None, None, "none", BF16, y[part])
    dx, dw, db = ops.linear_backward(dy, x, w)
    ref, q = torch.zeros(n, k, dtype=torch.float64, device=DEV), torch.zeros(n, k, dtype=torch.float64, device=DEV)
    for i in range(0, m, 1 << 20):
        a, b = dy[i:i + (1 << 20)].double().t().contiguous(), x[i:i + (1 << 20)].double()
        ref += mm(a, b)
        q += mm(a ** 2, b ** 2)
    within(dw, ref, sum_tol(m) * q.sqrt(), BF16)
    within(db, dy.double().sum(0), sum_tol(m) * (dy.double() ** 2).sum(0).sqrt(), BF16)
    d, w6 = dy[m - 1000:].double(), w.double()
    within(dx[m - 1000:], mm(d, w6), sum_tol(n) * mm(d ** 2, w6 ** 2).sqrt(), BF16)


def test_lookups_of_more_than_2_to_30_pieces():
    """what a launch covers, and 40 tokens more; dy of more than 2^32 elements"""
    tokens, rows, width = (1 << 27) + 40, 251, 64
    table = normal(1, rows, width, t=BF16)
    ids = (torch.arange(tokens, device=DEV) % rows).to(torch.uint8)
    y = ops.embedding(ids, table)
    for at in (0, (1 << 27) - rows, tokens - rows):
        assert torch.equal(y[at:at + rows], table[ids[at:at + rows].long()])
    y.normal_(generator=torch.Generator(DEV).manual_seed(1))
    d = ops.embedding_backward(y, ids, rows)
    ref, sq = torch.zeros(rows, width, dtype=torch.float64, device=DEV), torch.zeros(rows, width, dtype=torch.float64, device=DEV)
    for i in range(0, tokens, rows << 13):                            # (whole rounds of ids, and the last one's start)
        v = y[i:i + (rows << 13)].double()
        whole = len(v) // rows * rows
        ref += v[:whole].view(-1, rows, width).sum(0)
        sq += (v[:whole] ** 2).view(-1, rows, width).sum(0)
        ref[:len(v) - whole] += v[whole:]
        sq[:len(v) - whole] += v[whole:] ** 2
    n = torch.bincount(ids.long(), minlength=rows).double().sqrt()[:, None]
    within(d, ref, 2.0 ** -24 * (8 * n + 8) * sq.sqrt(), BF16)


def test_checkpoints_of_more_than_2_to_30_pieces():
    rows, width = (1 << 29) + 40, 17
    x = torch.empty(rows, width, dtype=BF16, device=DEV).normal_(generator=torch.Generator(DEV).manual_seed(2))
    c = ops.checkpoint8(x, "int8")
    v = c.values()
    for at in (0, (1 << 29) - 100, rows - 100):
        same(v[at:at + 100], in8(x[at:at + 100], "int8"))
        assert not c.codes[at:at + 100, width:].any()


def test_single_rows_and_tokens():
    """one token without a row of ids, one row without rows, checkpoints of one value, of leading dimensions and into a caller's tensor"""
    for t in TYPES:
        w, x = normal(1, 12, 20, t=t), normal(2, 20, t=t)
        y = ops.linear(x, w, activation="gelu")
        assert y.shape == (12,) and torch.equal(y, ops.linear(x[None], w, activation="gelu")[0])
        a, b = ops.linear_backward(y, x, w), ops.linear_backward(y[None], x[None], w)
        assert a[0].shape == (20,) and torch.equal(a[0], b[0][0]) and torch.equal(a[1], b[1]) and torch.equal(a[2], b[2])
        i = torch.tensor(3, device=DEV)
        e = ops.embedding(i, w, 0.5)
        assert e.shape == (20,) and torch.equal(e, (w[3].float() * 0.5).to(t))
        g = ops.embedding_backward(e, i, 12)
        assert torch.equal(g[3], e) and not g[:3].any() and not g[4:].any()
        one = ops.checkpoint8(x[:1], "e4m3")
        assert one.values().shape == (1,) and one.codes.shape == (1, 32)
        v = normal(3, 2, 3, 20, t=t)
        c = ops.checkpoint8(v)
        hold = torch.full((6, 25), 7.0, dtype=t, device=DEV)
        same(c.values(), in8(v, "int8"))
        c2 = ops.checkpoint8(v.reshape(6, 20))
        assert c2.values(out=hold[:, 2:22]) is not None and torch.equal(hold[:, 2:22], c.values().reshape(6, 20))
        hold[:, 2:22] = 7.0
        assert bool((hold == 7).all())
