"""The training operators' interface without a GPU: symbols, refusals before anything is launched, workspace sizes (include/ccsm_train_ops.h)."""
import ctypes as C
import os
import re

import pytest

from conftest import ROOT
from ccsmeth_amd import _lib, train_ops as ops

torch = pytest.importorskip("torch")
INVALID, CAPACITY = _lib.ERR_INVALID_ARG, _lib.ERR_CAPACITY
A = 1 << 20                      # an aligned address that nothing follows


def test_exports_match_header():
    header = open(os.path.join(ROOT, "include", "ccsm_train_ops.h")).read()
    declared = set(re.findall(r"\b(ccsm_train_[a-z0-9_]+)\s*\(", header))
    assert declared == set(ops.EXPORTS)
    lib = ops.load()
    for name in declared:
        assert hasattr(lib, name), name


def _linear(**kw):
    d = dict(type=2, activation=4, rows=64, inner=32, outer=48, x=A, ldx=32, w=A, ldw=32, bias=A, residual=A, ldr=48, y=A, ldy=48, preact=A, ldp=48)
    d.update(kw)
    return ops.Linear(**d)


@pytest.mark.parametrize("kw", [
    dict(type=3), dict(type=-1), dict(activation=6), dict(activation=-1), dict(rows=-1), dict(rows=1 << 40), dict(inner=0), dict(outer=0), dict(inner=-8),
    dict(x=None), dict(w=None), dict(y=None), dict(ldx=31), dict(ldw=0), dict(ldy=47), dict(ldr=40), dict(ldp=-48), dict(x=A + 1), dict(w=A + 1), dict(y=A + 1),
    dict(bias=A + 1), dict(residual=A + 1), dict(preact=A + 1), dict(type=0, x=A + 2),
])
def test_linear_refuses(kw):
    lib = ops.load()
    p = _linear(**kw)
    assert lib.ccsm_train_linear_forward(0, C.byref(p), A, 1 << 40, None) == INVALID
    assert lib.ccsm_train_ops_last_error()
    assert lib.ccsm_train_linear_workspace(C.byref(p)) == 0


def test_linear_null_and_empty():
    lib = ops.load()
    assert lib.ccsm_train_linear_forward(0, None, None, 0, None) == INVALID
    assert lib.ccsm_train_linear_forward(0, C.byref(_linear(rows=0, x=None, y=None)), None, 0, None) == 0       # nothing to do: nothing is launched
    assert lib.ccsm_train_linear_workspace(C.byref(_linear(rows=0))) == 0 and lib.ccsm_train_linear_backward_workspace(C.byref(_grad(rows=0))) == 0
    assert lib.ccsm_train_embedding_backward_workspace(0, 0, 5, 8) == 0


def _grad(**kw):
    s = dict(x=ops.Saved(A, 32, 0, None, 0), preact=ops.Saved(A, 48, 0, None, 0))
    d = dict(type=2, activation=4, rows=64, inner=32, outer=48, dy=A, lddy=48, w=A, ldw=32, dx=A, lddx=32, dw=A, lddw=32, dbias=A, **s)
    d.update(kw)
    return ops.LinearGrad(**d)


@pytest.mark.parametrize("kw", [
    dict(type=7), dict(activation=9), dict(rows=-1), dict(inner=0), dict(outer=0), dict(dy=None), dict(lddy=47), dict(w=None), dict(ldw=31), dict(lddx=31), dict(lddw=31),
    dict(dy=A + 1), dict(dx=A + 1), dict(dw=A + 1), dict(dbias=A + 1),
    dict(x=ops.Saved(None, 32, 0, None, 0)), dict(x=ops.Saved(A, 31, 0, None, 0)), dict(x=ops.Saved(A + 1, 32, 0, None, 0)), dict(preact=ops.Saved(None, 48, 0, None, 0)),
    dict(x=ops.Saved(A, 32, 3, A, 1)), dict(x=ops.Saved(A, 32, 1, None, 1)), dict(x=ops.Saved(A, 33, 1, A, 1)), dict(x=ops.Saved(A, 0, 1, A, 1)),
    dict(x=ops.Saved(A, 32, 2, A, 0)), dict(x=ops.Saved(A + 4, 32, 2, A, 1)), dict(preact=ops.Saved(A, 32, 2, A, 2)), dict(preact=ops.Saved(A, 64, 2, A, 1)),
])
def test_linear_backward_refuses(kw):
    lib = ops.load()
    p = _grad(**kw)
    assert lib.ccsm_train_linear_backward(0, C.byref(p), A, 1 << 40, None) == INVALID
    assert lib.ccsm_train_linear_backward_workspace(C.byref(p)) == 0


def test_too_small_a_workspace_is_refused():
    lib = ops.load()
    p = _grad(rows=1 << 16)
    need = lib.ccsm_train_linear_backward_workspace(C.byref(p))
    assert need > 0
    assert lib.ccsm_train_linear_backward(0, C.byref(p), None, need, None) == CAPACITY
    assert lib.ccsm_train_linear_backward(0, C.byref(p), A, need - 1, None) == CAPACITY
    assert lib.ccsm_train_linear_backward(0, C.byref(p), A + 8, need, None) == INVALID
    need = lib.ccsm_train_embedding_backward_workspace(0, 1000, 5, 8)
    assert need > 0
    args = (0, 0, 1, 1000, A, 5, 8, A, 8, 1.0, A, 8)
    assert lib.ccsm_train_embedding_backward(*args, None, 0, None) == CAPACITY
    assert lib.ccsm_train_embedding_backward(*args, A, need - 1, None) == CAPACITY


def test_embedding_and_act8_refuse():
    lib = ops.load()
    fwd = dict(type=0, id_type=2, tokens=10, ids=A, rows=5, width=8, table=A, ldt=8, scale=1.0, y=A, ldy=8)
    for kw in (dict(type=3), dict(id_type=3), dict(tokens=-1), dict(ids=None), dict(ids=A + 4), dict(rows=0), dict(width=0), dict(table=None), dict(y=None), dict(ldt=7),
               dict(ldy=7), dict(table=A + 2), dict(y=A + 2), dict(rows=1 << 40)):
        d = dict(fwd, **kw)
        assert lib.ccsm_train_embedding_forward(0, *d.values(), None) == INVALID, kw
    bwd = dict(type=0, id_type=2, tokens=10, ids=A, rows=5, width=8, dy=A, lddy=8, scale=1.0, dt=A, ldt=8)
    for kw in (dict(type=3), dict(id_type=-1), dict(tokens=-1), dict(ids=None), dict(rows=0), dict(width=-1), dict(dy=None), dict(dt=None), dict(lddy=7), dict(ldt=7), dict(dy=A + 1)):
        d = dict(bwd, **kw)
        assert lib.ccsm_train_embedding_backward(0, *d.values(), A, 1 << 40, None) == INVALID, kw
    pack = dict(type=0, code=1, rows=4, width=40, x=A, ldx=40, codes=A, ldc=64, scales=A, lds=2)
    for kw in (dict(type=9), dict(code=0), dict(code=3), dict(rows=-1), dict(width=0), dict(x=None), dict(ldx=39), dict(x=A + 2), dict(codes=None), dict(ldc=40), dict(ldc=32),
               dict(ldc=65), dict(scales=None), dict(lds=1), dict(codes=A + 8)):
        d = dict(pack, **kw)
        assert lib.ccsm_train_act8_pack(0, *d.values(), None) == INVALID, kw
    s = ops.Saved(A, 64, 1, A, 2)
    assert lib.ccsm_train_act8_unpack(0, 0, 4, 40, None, A, 40, None) == INVALID
    assert lib.ccsm_train_act8_unpack(0, 0, 4, 40, C.byref(s), A, 39, None) == INVALID
    assert lib.ccsm_train_act8_unpack(0, 0, 4, 40, C.byref(ops.Saved(A, 64, 0, A, 2)), A, 40, None) == INVALID
    assert lib.ccsm_train_act8_unpack(0, 0, 4, 65, C.byref(s), A, 65, None) == INVALID
    assert lib.ccsm_train_act8_pack(0, 0, 1, 0, 40, None, 0, None, 0, None, 0, None) == 0        # no rows


def test_python_refuses_before_the_library_is_called():
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear(x, w)
    with pytest.raises(ValueError, match="GPU"):
        ops.linear_backward(torch.zeros(4, 6), x, w)
    with pytest.raises(ValueError, match="GPU"):
        ops.checkpoint8(x)
    with pytest.raises(ValueError, match="GPU"):
        ops.embedding(torch.zeros(3, dtype=torch.int64), x)
    with pytest.raises(ValueError, match="activation"):
        ops.linear(x, w, activation="softplus")
    with pytest.raises(ValueError, match="code"):
        ops.checkpoint8(x, "int4")
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        ops.linear(x.double(), w)
    with pytest.raises(TypeError):
        ops.linear([[1.0]], w)
    with pytest.raises(ValueError, match="gradient"):
        ops.checkpoint8(torch.zeros(4, 8, requires_grad=True))


def test_checkpoint_tensors_are_checked():
    codes, scales = torch.zeros(4, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.uint8)
    c = ops.Checkpoint8(codes, scales, (2, 2, 40), torch.float16, "e4m3")
    assert c.nbytes == 4 * 66 and tuple(c.shape) == (2, 2, 40)
    for bad in ((codes[:, :40], scales), (codes, scales[:3]), (codes.float(), scales), (codes, scales.int())):
        with pytest.raises(ValueError):
            ops.Checkpoint8(*bad, (2, 2, 40), torch.float16, "e4m3")
    with pytest.raises(ValueError):
        ops.Checkpoint8(codes, scales, (2, 2, 40), torch.float64, "e4m3")
    with pytest.raises(ValueError):
        ops.Checkpoint8(codes, scales, (2, 2, 40), torch.float16, "fp4")


def test_trainm_offers_the_gates_in_8_bits():
    from ccsmeth_amd import trainm
    base = ["--train_file", "t", "--valid_file", "v", "--model_dir", "d"]
    for parser in (trainm.build_parser(), trainm.build_train_parser()):
        assert parser.parse_args(base).activation_bits == 32
        assert parser.parse_args(base + ["--activation_bits", "8"]).activation_bits == 8
        with pytest.raises(SystemExit):
            parser.parse_args(base + ["--activation_bits", "16"])


def test_trainer_refuses_other_widths():
    from ccsmeth_amd import train
    lib = train.load()
    out, w = C.c_void_p(), _lib.Weights()
    for bits in (0, 4, 16, 64):
        assert lib.ccsm_train_create_act(C.byref(w), 0, 16, None, bits, C.byref(out)) == INVALID
        assert b"activation_bits" in lib.ccsm_train_last_error()


@pytest.mark.parametrize("kind,most", [(0, 4210752), (1, 8421504), (2, 8421504)])
def test_contractions_whose_offsets_leave_32_bits_are_refused(kind, most):
    """255 rows of a staged operand and a row's last 128 bytes lie within a buffer's extent of 2^32 - 2 bytes up to `most` columns, and not beyond"""
    lib = ops.load()
    size = 4 if kind == 0 else 2
    assert 255 * most * size + 128 <= 2 ** 32 - 2 < 255 * (most + 8) * size + 128
    for inner, ok in ((most, True), (most - 5, True), (most + 1, False), (9000000, False), (0x00ffff00, False)):
        p = _linear(type=kind, rows=256, inner=inner, outer=256, ldx=inner, ldw=inner, ldy=256, ldr=256, ldp=256)
        assert (lib.ccsm_train_linear_workspace(C.byref(p)) > 0) == ok                  # (both operands are staged: their strides are too long)
        assert lib.ccsm_train_linear_forward(0, C.byref(p), None, 0, None) == (CAPACITY if ok else INVALID)
        g = _grad(type=kind, rows=300, inner=256, outer=inner, lddy=inner, ldw=256, lddx=256, lddw=256, preact=ops.Saved(A, inner, 0, None, 0), x=ops.Saved(A, 256, 0, None, 0))
        assert (lib.ccsm_train_linear_backward_workspace(C.byref(g)) > 0) == ok
        assert lib.ccsm_train_linear_backward(0, C.byref(g), None, 0, None) == (CAPACITY if ok else INVALID)
        g.dx = None                                                                     # dw and dbias run along rows: no limit but that of the columns
        assert lib.ccsm_train_linear_backward(0, C.byref(g), None, 0, None) == CAPACITY


def test_the_way_of_a_call():
    """the query that tests and profiles ask which kernel a call takes"""
    lib, way = ops.load(), (C.c_int32 * 4)()
    for m, k, n, want in ((64, 4096, 4096, (0, 0, 0, 0)), (300, 500, 400, (0, 0, 0, 0)), (3001, 67, 777, (128, 1, 0, 2)), (16384, 4096, 4096, (256, 1, 0, 0))):
        assert lib.ccsm_train_linear_way(C.byref(_linear(rows=m, inner=k, outer=n, ldx=k, ldw=k, ldy=n, ldr=n, ldp=n)), way) == 0 and tuple(way) == want
    for m, k, n, tile in ((20, 60, 40, 0), (600, 40, 72, 128), (16384, 4096, 4096, 256)):
        g = _grad(rows=m, inner=k, outer=n, lddy=n, ldw=k, lddx=k, lddw=k, x=ops.Saved(A, k, 0, None, 0), preact=ops.Saved(A, n, 0, None, 0))
        assert lib.ccsm_train_linear_backward_way(C.byref(g), way) == 0 and way[0] == tile
    assert lib.ccsm_train_linear_way(C.byref(_linear(rows=0)), way) == 0 and tuple(way) == (0, 0, 0, 0)
    assert lib.ccsm_train_linear_way(None, way) == INVALID and lib.ccsm_train_linear_way(C.byref(_linear(inner=0)), way) == INVALID
    assert lib.ccsm_train_linear_way(C.byref(_linear()), None) == INVALID and lib.ccsm_train_linear_backward_way(C.byref(_grad()), None) == INVALID


def test_forward_mode_tangents_are_refused():
    """they would be lost: in every place of a call, and of other tensors' levels nothing is refused"""
    import torch.autograd.forward_ad as fw
    x, w = torch.zeros(4, 8), torch.zeros(6, 8)
    with fw.dual_level():
        dual = fw.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops.linear(dual, w), lambda: ops.linear_backward(dual, x, torch.zeros(8, 8)), lambda: ops.checkpoint8(dual),
                     lambda: ops.embedding(torch.zeros(3, dtype=torch.int64), dual), lambda: ops.embedding_backward(dual, torch.zeros(4, dtype=torch.int64), 5)):
            with pytest.raises(ValueError, match="tangent"):
                call()
        with pytest.raises(ValueError, match="tangent"):
            ops._same(dual, "weight", torch.float32, -1, x)
        with pytest.raises(ValueError, match="GPU"):
            ops.linear(x, w)
        assert ops._same(w, "weight", torch.float32, -1, x) is w


def test_outputs_that_share_memory_are_refused():
    """(on no device: a call that were not refused would end there)"""
    nowhere = 1 << 20
    lib = ops.load()
    apart = dict(x=A, w=A << 1, bias=A << 2, residual=A << 3, y=A << 4, preact=A << 5)
    wide = dict(apart, ldy=112, ldx=112)                             # x beside y in the same rows
    y = A << 4
    for kw in (dict(apart, y=A), dict(apart, y=A << 1), dict(apart, y=(A << 2) + 94), dict(apart, y=A << 5), dict(apart, y=(A << 3) + 2), dict(apart, y=A << 3, ldy=50),
               dict(apart, preact=A << 3), dict(apart, preact=A + 32), dict(apart, x=y + 96, ldx=49), dict(wide, x=y + 94), dict(wide, x=y + 224 - 62), dict(wide, x=y + 224 + 94),
               dict(apart, y=A + 63 * 64 + 62), dict(apart, y=A - 64 * 96 + 2)):
        assert lib.ccsm_train_linear_forward(nowhere, C.byref(_linear(**kw)), None, 0, None) == INVALID, kw
        assert b"shares memory" in lib.ccsm_train_ops_last_error(), kw
    far = dict(dy=A, w=A << 1, dx=A << 2, dw=A << 3, dbias=A << 4, x=ops.Saved(A << 5, 32, 1, A << 6, 1), preact=ops.Saved(A << 7, 64, 2, A << 8, 2))
    for kw in (dict(dx=A), dict(dx=A << 1), dict(dw=(A << 5) + 64), dict(dw=(A << 6) + 2), dict(dbias=A << 7), dict(dbias=(A << 8) + 126), dict(dw=A << 2), dict(dbias=A << 3), dict(dbias=(A << 2) - 2)):
        assert lib.ccsm_train_linear_backward(nowhere, C.byref(_grad(**dict(far, **kw))), A << 9, 1 << 40, None) == INVALID, kw
        assert b"shares memory" in lib.ccsm_train_ops_last_error(), kw
    for ids, table, out in ((A, A << 1, A), (A, A << 1, (A << 1) + 64), (A, A << 1, A - 156), (A, A << 1, A + 76)):
        assert lib.ccsm_train_embedding_forward(nowhere, 0, 2, 10, ids, 5, 8, table, 8, 1.0, out, 8, None) == INVALID
        assert lib.ccsm_train_embedding_backward(nowhere, 0, 2, 10, ids, 5, 8, table, 8, 1.0, out, 8, A << 9, 1 << 40, None) == INVALID
    for x, codes, scales in ((A, A, A << 1), (A, A << 1, A + 48), (A, A << 1, (A << 1) + 255)):
        assert lib.ccsm_train_act8_pack(nowhere, 0, 1, 4, 40, x, 40, codes, 64, scales, 2, None) == INVALID
        assert b"share memory" in lib.ccsm_train_ops_last_error()
    for y, codes, scales in ((A, A, A << 1), (A, A << 1, A + 48)):
        assert lib.ccsm_train_act8_unpack(nowhere, 0, 4, 40, C.byref(ops.Saved(codes, 64, 1, scales, 2)), y, 40, None) == INVALID
    apart = dict(apart, y=A << 4)
    for kw in (apart, dict(wide, x=y + 96), dict(wide, x=y + 224 - 64), dict(apart, y=A << 3), dict(apart, residual=None, preact=None), dict(apart, y=A + 64 * 64), dict(apart, y=A - 64 * 96)):
        assert lib.ccsm_train_linear_forward(nowhere, C.byref(_linear(**kw)), None, 0, None) == _lib.ERR_HIP, kw      # nothing is shared


def test_more_rows_than_a_launch_covers_are_refused():
    """32 rows x 256 columns a workgroup of 256 lanes, 65536 more workgroups for what is staged: less than 2^32 lanes in all"""
    lib, most = ops.load(), 534773728
    assert (most // 32 + 65536) * 256 < 2 ** 32 and most % 32 == 0
    for outer, rows, ok in ((1, most, True), (256, most, True), (256, most + 1, False), (257, most, False), (257, most // 2 // 32 * 32, True), (8, 0x7fffff00, False)):
        g = _grad(rows=rows, inner=1, outer=outer, lddy=outer, ldw=1, lddx=1, lddw=1, x=ops.Saved(A, 1, 0, None, 0), preact=ops.Saved(A, outer, 0, None, 0))
        assert lib.ccsm_train_linear_backward(1 << 20, C.byref(g), None, 0, None) == (CAPACITY if ok else INVALID), (outer, rows)


def test_views_with_their_sign_turned_are_copied():
    ops._init()
    c = torch.tensor([[1 + 2j, 3 - 4j], [5 + 6j, -7 - 8j]], dtype=torch.complex64)
    for v in (c.conj().imag, c.conj().imag[:, :1], c.conj().imag[:1, :1], torch._neg_view(torch.ones(3, 4))):
        assert v.is_neg()
        t, ld = ops._rows(v)
        assert not t.is_neg() and torch.equal(t, v.resolve_neg()) and ld >= t.shape[1]
        with pytest.raises(ValueError):
            ops._out(v, v.shape, torch.float32, v.device, "out")
    assert ops._rows(c.real)[0].data_ptr() != c.data_ptr() and ops._rows(torch.ones(3, 4))[1] == 4
