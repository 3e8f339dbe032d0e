"""The training operators' tile kernels on the GPU: each tile (128 and 256), with and without a split contraction, with staged operands, ragged in every
direction, with every epilogue; forward, both gradients together and each alone.  Each test says first which kernel it means, and asks the
library (ccsm_train_linear_way) whether that one is taken.  References, tolerances: test_gpu_train_ops.py."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
import test_gpu_train_ops as base  # noqa: E402
from ccsmeth_amd import train_ops as ops  # noqa: E402
from test_gpu_train_ops import ACTS, BF16, DEV, F16, F32, TYPES, check_backward, check_linear, in8, normal  # noqa: E402

pytestmark = pytest.mark.gpu
SMALL16 = [F16, BF16]


def _ld(t):
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def way_forward(x, w, y):
    way = (C.c_int32 * 4)()
    p = ops.Linear(type=TYPES.index(x.dtype), activation=0, rows=x.shape[0], inner=w.shape[1], outer=w.shape[0], x=x.data_ptr(), ldx=_ld(x), w=w.data_ptr(), ldw=_ld(w),
                   y=y.data_ptr(), ldy=_ld(y))
    assert ops.load().ccsm_train_linear_way(C.byref(p), way) == 0
    return way[0], way[1] > 1, way[3]


def way_backward(dy, x, w, z, act, dx=True, dw=True):
    way = (C.c_int32 * 4)()

    def saved(v):
        return ops.Saved() if v is None else ops.Saved(*v._saved()) if isinstance(v, ops.Checkpoint8) else ops.Saved(v.data_ptr(), _ld(v), 0, None, 0)
    out = dy.data_ptr()
    p = ops.LinearGrad(type=TYPES.index(dy.dtype), activation=ops.ACTIVATIONS[act], rows=dy.shape[0], inner=w.shape[1], outer=w.shape[0], dy=dy.data_ptr(), lddy=_ld(dy), x=saved(x),
                       w=w.data_ptr(), ldw=_ld(w), preact=saved(z), dx=out if dx else None, lddx=w.shape[1], dw=out if dw else None, lddw=w.shape[1], dbias=out)
    assert ops.load().ccsm_train_linear_backward_way(C.byref(p), way) == 0
    return way[0], way[1] > 1, way[2] > 1


# rows, inner, outer; tile, split, staged operands; types
FORWARD = [((3001, 67, 777), 128, False, 2, TYPES), ((3001, 520, 777), 128, False, 0, TYPES), ((90, 1101, 33), 128, True, 2, TYPES), ((1025, 1500, 300), 128, True, 0, [F32]),
           ((1025, 1500, 300), 128, True, 2, SMALL16), ((6632, 8, 1800), 256, False, 0, TYPES), ((7016, 88, 1671), 256, False, 0, TYPES), ((6984, 331, 1668), 256, False, 2, TYPES),
           ((136, 1984, 5800), 256, True, 0, [F32]), ((6596, 1990, 146), 256, True, 2, [F32]), ((8994, 5242, 129), 256, True, 2, SMALL16)]


@pytest.mark.parametrize("t,size,tile,split,staged", [(t, s, tile, split, staged) for s, tile, split, staged, types in FORWARD for t in types])
def test_forward(t, size, tile, split, staged):
    m, k, n = size
    x, w, b, r = normal(m, m, k, t=t), normal(k + 1, n, k, t=t, by=k ** -0.5), normal(n + 2, n, t=t, by=0.3), normal(3, m, n, t=t)
    assert way_forward(x, w, r) == (tile, split, staged)
    act = ACTS[(m + k + n + TYPES.index(t)) % 5 + 1]
    y, z = ops.linear(x, w, b, r, activation=act, keep_preact=True)
    check_linear(x, w, b, r, act, t, y, z)
    check_linear(x, w, None, None, "none", t, ops.linear(x, w))
    want = ops.linear(x, w, None, r, activation=act)
    assert ops.linear(x, w, None, r, activation=act, out=r) is r and torch.equal(r, want)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("size,tile,split", [((3001, 67, 777), 128, False), ((90, 1101, 33), 128, True), ((7016, 88, 1671), 256, False)])
def test_forward_epilogues(t, act, size, tile, split):
    """pre-activations from -9 to 9, with and without a residual, of the tiles and of the parts' join"""
    m, k, n = size
    x, w, b, r = normal(5, m, k, t=t), normal(6, n, k, t=t, by=0.5 * k ** -0.5), torch.linspace(-9, 9, n).to(t).to(DEV), normal(8, m, n, t=t)
    assert way_forward(x, w, r)[:2] == (tile, split)
    y, z = ops.linear(x, w, b, r, activation=act, keep_preact=True)
    check_linear(x, w, b, r, act, t, y, z)
    check_linear(x, w, b, None, act, t, ops.linear(x, w, b, activation=act))


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("size,tile,split", [((3001, 67, 777), 128, False), ((90, 1101, 33), 128, True), ((7016, 88, 1671), 256, False)])
def test_strides_and_alignment(t, size, tile, split):
    """views into wider matrices, at odd offsets; what lies around the output stays as it was; NaN stay in their rows"""
    m, k, n = size
    for off, pad in ((1, 3), (0, 8), (8, 16)):
        x, w = normal(9, m, k + off + pad, t=t)[:, off:off + k], normal(10, n, k + off + pad, t=t, by=k ** -0.5)[:, off:off + k]
        r, b = normal(11, m, n + off + pad, t=t)[:, off:off + n], normal(12, n + off, t=t)[off:]
        hold = torch.full((m + 2, n + off + pad), 7.0, dtype=t, device=DEV)
        y = hold[1:m + 1, off:off + n]
        assert way_forward(x, w, y)[:2] == (tile, split)
        assert ops.linear(x, w, b, r, activation="tanh", out=y) is y
        check_linear(x, w, b, r, "tanh", t, y.clone())
        hold[1:m + 1, off:off + n] = 7.0
        assert bool((hold == 7).all())
    x = x.clone()
    x[1, 3] = float("nan")
    y = ops.linear(x, w, activation="relu")
    assert y[1].isnan().all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()


# rows, inner, outer; which of dx, dw; tile, dx's contraction split, dw's; types
BACKWARD = [((600, 40, 72), (1, 1), 128, False, True, [F32]), ((600, 40, 72), (1, 1), 128, False, False, SMALL16), ((1500, 65, 77), (1, 1), 128, False, True, TYPES),
            ((104, 8, 544), (1, 1), 128, True, True, [F32]), ((672, 8, 208), (1, 1), 128, True, True, SMALL16), ((9064, 400, 144), (1, 1), 256, False, True, [F32]),
            ((144, 6424, 584), (1, 1), 256, True, False, [F32]), ((9299, 132, 409), (1, 1), 256, True, True, [F32]),
            ((616, 8144, 552), (1, 1), 256, False, False, SMALL16), ((2410, 2971, 129), (1, 1), 256, False, True, SMALL16),
            ((514, 2851, 2304), (1, 1), 256, True, False, SMALL16), ((6421, 136, 4156), (1, 1), 256, True, True, SMALL16),
            ((600, 40, 72), (1, 0), 128, False, False, TYPES), ((69, 8, 617), (1, 0), 128, True, False, [F32]), ((64, 8, 712), (1, 0), 128, True, False, SMALL16),
            ((2696, 4400, 8), (1, 0), 256, False, False, [F32]), ((7296, 1048, 8), (1, 0), 256, False, False, SMALL16),
            ((9032, 160, 1072), (1, 0), 256, True, False, [F32]), ((8284, 134, 4898), (1, 0), 256, True, False, SMALL16), ((528, 8, 8), (0, 1), 128, False, True, [F32]),
            ((528, 8, 8), (0, 1), 128, False, False, SMALL16), ((1500, 65, 77), (0, 1), 128, False, True, TYPES), ((64, 3224, 3856), (0, 1), 256, False, False, [F32]),
            ((64, 3639, 2316), (0, 1), 256, False, False, SMALL16), ((3344, 131, 4303), (0, 1), 256, False, True, [F32]),
            ((7895, 6570, 132), (0, 1), 256, False, True, SMALL16)]


@pytest.mark.parametrize("t,size,which,tile,split_dx,split_dw", [(t, s, which, tile, a, b) for s, which, tile, a, b, types in BACKWARD for t in types])
def test_backward(t, size, which, tile, split_dx, split_dw):
    m, k, n = size
    act = ACTS[(m + k + 2 * n + TYPES.index(t)) % 5 + 1]
    dy, x, w, z = normal(1, m, n, t=t, by=0.05), normal(2, m, k, t=t), normal(3, n, k, t=t, by=k ** -0.5), normal(4, m, n, t=t)
    assert way_backward(dy, x, w, z, act, *which) == (tile, split_dx, split_dw)
    need = {"need_dx": bool(which[0]), "need_dw": bool(which[1])}
    check_backward(dy, x, w, z, act, t, ops.linear_backward(dy, x, w, z, activation=act, **need))
    check_backward(dy, x, w, z, "none", t, ops.linear_backward(dy, x, w, need_db=False, **need))


@pytest.mark.parametrize("t,size", [(F32, (9064, 400, 144)), (F32, (1500, 65, 77)), (F16, (2410, 2971, 129)), (BF16, (2410, 2971, 129)), (F16, (1500, 65, 77)), (BF16, (1500, 65, 77))])
@pytest.mark.parametrize("codes", [("int8", "e4m3"), ("e4m3", "int8")])
def test_backward_from_checkpoints(t, size, codes):
    m, k, n = size
    dy, x, w, z = normal(1, m, n, t=t, by=0.05), normal(2, m, k, t=t), normal(3, n, k, t=t, by=k ** -0.5), normal(4, m, n, t=t, by=2.0)
    cx, cz = ops.checkpoint8(x, codes[0]), ops.checkpoint8(z, codes[1])
    assert way_backward(dy, cx, w, cz, "silu")[0] == (256 if m > 2000 else 128)
    check_backward(dy, in8(x, codes[0]), w, in8(z, codes[1]), "silu", t, ops.linear_backward(dy, cx, w, cz, activation="silu"))


@pytest.mark.parametrize("t,size", [(F32, (6632, 8, 1800)), (F32, (136, 1984, 5800)), (F16, (6632, 8, 1800)), (BF16, (6632, 8, 1800))])
def test_infinities_forward(t, size):
    assert way_forward(torch.empty(size[0], size[1], dtype=t, device=DEV), torch.empty(size[2], size[1], dtype=t, device=DEV), torch.empty(size[0], size[2], dtype=t, device=DEV))[0] == 256
    base.test_infinities_forward(t, *size)


@pytest.mark.parametrize("t,size", [(F32, (9064, 400, 144)), (F16, (2410, 2971, 129)), (BF16, (2410, 2971, 129))])
def test_infinities_backward(t, size):
    base.test_infinities_backward(t, "silu", *size)


@pytest.mark.parametrize("by", [2.0 ** -20, 2.0 ** 8])
def test_fp16_gradients_of_small_and_large_dy(by):
    """256 tiles, one product's contraction split (its factor is the join's) and the other's not"""
    m, k, n = 2410, 2971, 129
    dy, x, w, z = normal(1, m, n, t=F16, by=by), normal(2, m, k, t=F16, by=min(1.0, 1 / by)), normal(3, n, k, t=F16, by=k ** -0.5), normal(4, m, n, t=F16)
    assert way_backward(dy, x, w, z, "gelu") == (256, False, True)
    base.check_range(dy, x, w, z, "gelu", F16, ops.linear_backward(dy, x, w, z, activation="gelu"), base.H[F16])


@pytest.mark.parametrize("t,k,tile", [(F32, 4210752, 256), (F16, 8421504, 256), (BF16, 8421504 - 3, 256)])
def test_the_longest_contraction(t, k, tile):
    """offsets of the last rows' last pieces end 126 bytes below 2^32; first and last rows differ"""
    m = n = 256
    g = torch.Generator(DEV)
    x, w = (torch.empty(m, k, dtype=t, device=DEV).normal_(generator=g.manual_seed(s)) for s in (1, 2))
    assert way_forward(x, w, torch.empty(m, n, dtype=t, device=DEV))[0] == tile
    w *= 2.0 ** -11
    ref, q = torch.zeros(m, n, dtype=torch.float64, device=DEV), torch.zeros(m, n, dtype=torch.float64, device=DEV)
    for i in range(0, k, 1 << 18):
        a, b = x[:, i:i + (1 << 18)].double(), w[:, i:i + (1 << 18)].double().t()
        ref += torch.mm(a, b.contiguous())
        q += torch.mm(a ** 2, (b ** 2).contiguous())
    base.within(ops.linear(x, w), ref, base.sum_tol(k) * q.sqrt(), t)
    dx, _, db = ops.linear_backward(x, None, w.t().contiguous(), need_dw=False)        # (m, k) by (k, n): the same sums
    base.within(dx, ref, base.sum_tol(k) * q.sqrt(), t)
    base.within(db[:1000], x[:, :1000].double().sum(0), base.sum_tol(m) * (x[:, :1000].double() ** 2).sum(0).sqrt(), t)
    base.within(db[k - 1000:], x[:, k - 1000:].double().sum(0), base.sum_tol(m) * (x[:, k - 1000:].double() ** 2).sum(0).sqrt(), t)
