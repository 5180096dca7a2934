"""CPU: what the row operators refuse, through the C entry points and the Python functions (no GPU call is made)."""
import ctypes as C

import pytest
import torch

INVALID, OVERFLOW = 2, 10
U8, S16, S32, F32, F16, BF16, S64 = 0, 3, 5, 6, 7, 8, 9


def _rows(pkg, dtype=F32, cols=8, count=(4, 1, 1), stride=None, base=4096):
    es = {U8: 1, F16: 2, BF16: 2, S64: 8}.get(dtype, 4)
    r = pkg.rows._Rows(base, dtype, cols)
    stride = stride or (cols * es, 0, 0)
    for k in range(3):
        r.count[k], r.stride[k] = count[k], stride[k]
    return r


def _ln(pkg, src, dst, op=None, ws=None, size=0):
    op = op if op is not None else pkg.rows._LayerNormOp()
    return pkg.rows._lib().b200ppLayerNorm(C.byref(src) if src else None, C.byref(dst) if dst else None, C.byref(op), ws, size, None)


def test_layernorm_refusals(pkg):
    R = lambda **k: _rows(pkg, **k)  # noqa: E731
    assert _ln(pkg, None, R()) == INVALID
    for src, dst in ((S16, F32), (F32, U8), (S32, F32), (F32, S64), (12, F32)):
        assert _ln(pkg, R(dtype=src), R(dtype=dst)) == INVALID, (src, dst)
    assert _ln(pkg, R(), R(cols=9)) == INVALID
    assert _ln(pkg, R(), R(count=(5, 1, 1))) == INVALID
    assert _ln(pkg, R(cols=0), R(cols=0)) == INVALID
    assert _ln(pkg, R(cols=1 << 31), R(cols=1 << 31)) == INVALID
    assert _ln(pkg, R(cols=(1 << 31) - 1), R(cols=(1 << 31) - 1)) == INVALID
    L, size = pkg.rows._lib(), C.c_size_t(0)
    for dtype in (S16, S32, S64, 12):
        assert L.b200ppLayerNormWorkspace(C.byref(R(dtype=dtype)), C.byref(size)) == INVALID
        assert L.b200ppLayerNormBackwardWorkspace(C.byref(R(dtype=dtype)), C.byref(size)) == INVALID
    assert _ln(pkg, R(count=(-1, 1, 1)), R(count=(-1, 1, 1))) == INVALID
    big = dict(count=(1 << 16, 1 << 16, 1), stride=(1 << 40, 32, 0))
    assert _ln(pkg, R(**big), R(**big)) == OVERFLOW
    assert _ln(pkg, R(base=None), R()) == INVALID
    assert _ln(pkg, R(base=4098), R()) == INVALID
    assert _ln(pkg, R(), R(stride=(30, 0, 0))) == INVALID
    assert _ln(pkg, R(), R(stride=(0, 0, 0))) == INVALID  # written rows on top of one another
    assert _ln(pkg, R(), R(stride=(16, 0, 0))) == INVALID
    assert b"overlap" in pkg.rows._lib().b200ppGetLastErrorMessage()
    assert _ln(pkg, R(count=(2, 2, 1), stride=(64, 32, 0)), R(count=(2, 2, 1), stride=(32, 32, 0))) == INVALID
    op = pkg.rows._LayerNormOp()
    for eps in (-1.0, float("nan")):
        op.epsilon = eps
        assert _ln(pkg, R(), R(), op) == INVALID
    for field in ("weight", "bias"):
        op = pkg.rows._LayerNormOp()
        setattr(op, field, 4096)
        setattr(op, field + "Type", U8)
        assert _ln(pkg, R(), R(), op) == INVALID
        setattr(op, field, 4097)
        setattr(op, field + "Type", F16)
        assert _ln(pkg, R(), R(), op) == INVALID
    op = pkg.rows._LayerNormOp()
    op.mean = 4098
    assert _ln(pkg, R(), R(), op) == INVALID
    # nothing to do
    for count in ((0, 1, 1), (1 << 30, 1 << 30, 0), (0, 1 << 40, 1)):
        assert _ln(pkg, R(count=count), R(count=count)) == 0, count


def test_layernorm_backward_refusals(pkg):
    L = pkg.rows._lib()
    R = lambda **k: _rows(pkg, **k)  # noqa: E731

    def call(grad, src, dsrc, ws=65536, size=1 << 30, **fields):
        op = pkg.rows._LayerNormGradOp()
        op.mean = op.rstd = 4096
        for k, v in fields.items():
            setattr(op, k, v)
        return L.b200ppLayerNormBackward(C.byref(grad) if grad else None, C.byref(src), C.byref(dsrc) if dsrc else None, C.byref(op),
                                         ws, size, None)

    assert call(None, R(), R()) == INVALID
    assert call(R(), R(), None) == INVALID
    assert b"No gradient" in L.b200ppGetLastErrorMessage()
    assert call(R(dtype=U8), R(), R()) == INVALID
    assert call(R(), R(dtype=U8), R(dtype=U8)) == INVALID
    assert call(R(cols=9), R(), R()) == INVALID
    assert call(R(), R(), R(count=(3, 1, 1))) == INVALID
    assert call(R(), R(), R(stride=(0, 0, 0))) == INVALID
    assert call(R(), R(), R(), mean=None) == INVALID
    assert call(R(), R(), R(), rstd=None) == INVALID
    assert call(R(), R(), R(), dweight=4096, dweightType=S32) == INVALID
    assert call(R(), R(), R(), dbias=4098, dbiasType=F32) == INVALID
    need = C.c_size_t(0)
    assert L.b200ppLayerNormBackwardWorkspace(C.byref(R()), C.byref(need)) == 0 and need.value == 0  # few short rows
    many = R(count=(400, 1, 1))
    assert L.b200ppLayerNormBackwardWorkspace(C.byref(many), C.byref(need)) == 0 and need.value > 0
    assert call(many, many, many, dweight=4096, dweightType=F32, size=need.value - 1) == INVALID
    assert call(many, many, many, dweight=4096, dweightType=F32, ws=None) == INVALID
    assert call(many, many, many, dweight=4096, dweightType=F32, ws=65544) == INVALID


def test_embedding_refusals(pkg):
    L = pkg.rows._lib()
    R = lambda **k: _rows(pkg, **k)  # noqa: E731
    ids = R(dtype=S32, cols=1)

    def call(i, t, d):
        return L.b200ppEmbedding(C.byref(i) if i else None, C.byref(t), C.byref(d), 1.0, None)

    assert call(None, R(), R()) == INVALID
    assert call(R(dtype=F32, cols=1), R(), R()) == INVALID
    assert call(R(dtype=S32, cols=2), R(), R()) == INVALID
    assert call(ids, R(dtype=U8), R()) == INVALID
    assert call(ids, R(), R(dtype=U8)) == INVALID
    assert call(ids, R(cols=9), R()) == INVALID
    assert call(ids, R(), R(count=(5, 1, 1))) == INVALID
    assert call(ids, R(), R(stride=(0, 0, 0))) == INVALID
    assert call(R(dtype=S32, cols=1, base=4097), R(), R()) == INVALID
    assert call(R(dtype=S32, cols=1, count=(0, 1, 1)), R(), R(count=(0, 1, 1))) == 0


def test_embedding_backward_refusals(pkg):
    L = pkg.rows._lib()
    R = lambda **k: _rows(pkg, **k)  # noqa: E731
    ids = R(dtype=S64, cols=1)
    need = C.c_size_t(0)
    assert L.b200ppEmbeddingBackwardWorkspace(C.byref(R()), C.byref(R()), C.byref(need)) == 0 and need.value == 0
    # many indices are sorted in a workspace
    many, many_ids = R(count=(40000, 1, 1)), R(dtype=S64, cols=1, count=(40000, 1, 1))
    assert L.b200ppEmbeddingBackwardWorkspace(C.byref(many), C.byref(R()), C.byref(need)) == 0 and need.value > 0
    assert L.b200ppEmbeddingBackwardWorkspace(C.byref(many), None, C.byref(need)) == INVALID
    for g, t in ((R(dtype=U8), R()), (R(), R(dtype=S32)), (R(cols=9), R())):
        assert L.b200ppEmbeddingBackwardWorkspace(C.byref(g), C.byref(t), C.byref(C.c_size_t(0))) == INVALID

    def call(g, i, t, ws=65536, size=1 << 30):
        op = pkg.rows._EmbeddingGradOp(1.0, 0, -1)
        return L.b200ppEmbeddingBackward(C.byref(g) if g else None, C.byref(i), C.byref(t), C.byref(op), ws, size, None)

    assert call(None, ids, R()) == INVALID
    assert call(R(dtype=U8), ids, R()) == INVALID
    assert call(R(), ids, R(dtype=S32)) == INVALID
    assert call(R(), R(dtype=F32, cols=1), R()) == INVALID
    assert call(R(cols=4), ids, R()) == INVALID
    assert call(R(count=(3, 1, 1)), ids, R()) == INVALID
    assert call(R(), ids, R(stride=(0, 0, 0))) == INVALID
    assert call(many, many_ids, R(), size=need.value - 1) == INVALID
    assert call(many, many_ids, R(), ws=None) == INVALID
    assert call(many, many_ids, R(), ws=65537) == INVALID
    assert call(R(), ids, R(count=(0, 1, 1))) == 0  # a table without rows


def test_python_functions_refuse_host_tensors_and_wrong_shapes(pkg):
    x = torch.zeros(4, 8)
    if torch.cuda.is_available():
        pytest.skip("the rest of the refusals are GPU tests")
    for call in (lambda: pkg.layernorm(x), lambda: pkg.layernorm_into(x, x), lambda: pkg.layernorm_backward(x, x, x[:, 0], x[:, 0]),
                 lambda: pkg.embedding(torch.zeros(3, dtype=torch.int32), x), lambda: pkg.embedding_backward(x, torch.zeros(4), 5)):
        with pytest.raises((pkg.ops.Error, RuntimeError)):
            call()


def test_rows_of_strided_tensors(pkg):
    """The view of a tensor the C layer gets: dimensions that continue one another are merged, others keep their strides."""
    def f(*args):
        return pkg.rows._Rows.from_buffer_copy(pkg.rows._rows(*args)[0])

    t = torch.zeros(5, 6, 7, 8)
    r = f(t, 1, "t")
    assert (r.cols, list(r.count), r.stride[0]) == (8, [210, 1, 1], 32)
    r = f(t, 3, "t")
    assert (r.cols, list(r.count)) == (336, [5, 1, 1])
    r = f(t[:, ::2], 1, "t")
    assert (list(r.count), list(r.stride)) == ([15, 7, 1], [2 * 7 * 32, 32, 0])
    r = f(t.permute(2, 0, 1, 3), 1, "t")
    assert (list(r.count), list(r.stride)) == ([7, 30, 1], [32, 7 * 32, 0])
    r = f(t[:, :4, :5], 1, "t")
    assert (list(r.count), list(r.stride)) == ([5, 4, 5], [6 * 7 * 32, 7 * 32, 32])
    with pytest.raises(pkg.ops.Error):
        f(t.transpose(2, 3), 1, "t")
    with pytest.raises(pkg.ops.Error):
        f(torch.zeros(3, 4, 5, 6, 7)[:, :3, :4, :5, :6], 1, "t")
    r = f(torch.zeros(3, 0, 8), 1, "t")
    assert r.count[0] * r.count[1] * r.count[2] == 0
