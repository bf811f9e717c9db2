"""Refusals of the training-step operators (embedding, residual norm, gradient clipping): no GPU needed."""
import ctypes
import math

import pytest
import torch

from opus_b200 import _lib, ops
from opus_b200.layers import ResidualNorm, ScaledEmbedding, residual_norm, scaled_embedding
from opus_b200.train import clip_grad_norm_

NULL = ctypes.c_void_p(0)


def rc_of(name, *args):
    rc = getattr(_lib.load(), name)(*args)
    return rc, _lib.last_error()


# ------------------------------------------------------------------ C entry points
@pytest.mark.parametrize("n,vocab,d,bits,dtype,stride,code", [
    (-1, 4, 8, 64, 0, 8, _lib.OPUS_ERR_INVALID), (1, 0, 8, 64, 0, 8, _lib.OPUS_ERR_INVALID),
    (1, 4, 0, 64, 0, 8, _lib.OPUS_ERR_INVALID), (1, 4, 8, 16, 0, 8, _lib.OPUS_ERR_INVALID),
    (1, 4, 8, 64, 7, 8, _lib.OPUS_ERR_UNSUPPORTED), (1, 4, 8, 64, 0, 7, _lib.OPUS_ERR_INVALID),
    (1 << 31, 4, 8, 64, 0, 8, _lib.OPUS_ERR_UNSUPPORTED), (1, 1 << 31, 8, 64, 0, 8, _lib.OPUS_ERR_UNSUPPORTED),
    (1, 4, 65537, 64, 0, 65537, _lib.OPUS_ERR_UNSUPPORTED), (1, 4, 8, 64, 0, 8, _lib.OPUS_ERR_INVALID)])
def test_embedding_entry_point_refuses(n, vocab, d, bits, dtype, stride, code):
    assert rc_of("opus_embedding", NULL, bits, n, NULL, dtype, vocab, stride, d, 1.0, NULL, NULL)[0] == code


def test_embedding_grad_entry_point_refuses():
    one = ctypes.c_void_p(256)  # never followed: every call is refused before the device is touched

    def call(dtype=0, stride=8, bits=64, n=1, vocab=4, d=8, out=one, out_dtype=0, accumulate=1, ws=one, ws_bytes=1 << 20):
        return rc_of("opus_embedding_grad", one, dtype, stride, one, bits, n, vocab, d, 1.0, -1, out, out_dtype, accumulate,
                     ws, ws_bytes, NULL)[0]

    assert call(out=NULL) == _lib.OPUS_ERR_INVALID
    assert call(out_dtype=2) == _lib.OPUS_ERR_UNSUPPORTED
    assert call(stride=7) == _lib.OPUS_ERR_INVALID
    assert call(ws=NULL) == _lib.OPUS_ERR_INVALID
    assert call(ws_bytes=8) == _lib.OPUS_ERR_INVALID and "workspace" in _lib.last_error()
    assert call(ws=ctypes.c_void_p(264)) == _lib.OPUS_ERR_INVALID
    assert call(out=ctypes.c_void_p(257)) == _lib.OPUS_ERR_INVALID
    assert _lib.load().opus_embedding_grad_workspace_bytes(0, 4, 8) == 0
    assert _lib.load().opus_embedding_grad_workspace_bytes(1000, 4, 8) > 0


def norm_args(**kw):
    a = _lib.ResidualNormArgs()
    a.rows, a.d, a.x_dtype, a.y_dtype, a.gate_rows = 4, 8, 0, 0, 1
    a.x = a.h = a.n = a.stats = 256
    a.x_stride = a.y_stride = a.h_stride = a.grad_n_stride = a.grad_h_stride = 8
    a.residual_scale, a.eps = 1.0, 1e-6
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


@pytest.mark.parametrize("kw,code", [
    (dict(rows=-1), _lib.OPUS_ERR_INVALID), (dict(d=0), _lib.OPUS_ERR_INVALID),
    (dict(d=16385), _lib.OPUS_ERR_UNSUPPORTED), (dict(kind=2), _lib.OPUS_ERR_INVALID),
    (dict(x_dtype=5), _lib.OPUS_ERR_UNSUPPORTED), (dict(x_dtype=0, y_dtype=1), _lib.OPUS_ERR_UNSUPPORTED),
    (dict(x_dtype=0, y_dtype=2), _lib.OPUS_ERR_UNSUPPORTED), (dict(post=1), _lib.OPUS_ERR_INVALID),
    (dict(post_weight=256), _lib.OPUS_ERR_INVALID), (dict(gate=256), _lib.OPUS_ERR_INVALID),
    (dict(gate=256, y=256, gate_rows=3), _lib.OPUS_ERR_INVALID), (dict(gate=256, y=256, gate_rows=0), _lib.OPUS_ERR_INVALID),
    (dict(weight=256, weight_dtype=9), _lib.OPUS_ERR_UNSUPPORTED), (dict(weight=257), _lib.OPUS_ERR_INVALID),
    (dict(x=0), _lib.OPUS_ERR_INVALID), (dict(x=257), _lib.OPUS_ERR_INVALID), (dict(stats=260), _lib.OPUS_ERR_INVALID),
    (dict(x_stride=7), _lib.OPUS_ERR_INVALID), (dict(y=256, y_stride=7), _lib.OPUS_ERR_INVALID),
    (dict(h=None, residual_scale=0.5), _lib.OPUS_ERR_INVALID), (dict(h=None, y=256), _lib.OPUS_ERR_INVALID)])
def test_residual_norm_entry_point_refuses(kw, code):
    assert rc_of("opus_residual_norm", norm_args(**kw), NULL)[0] == code


@pytest.mark.parametrize("kw", [
    dict(grad_x=0), dict(grad_n=0, grad_h=0), dict(y=256, grad_y=0), dict(grad_y=256), dict(grad_weight=256),
    dict(weight=256, grad_weight=257), dict(h_stride=7), dict(grad_n_stride=7), dict(grad_n=257), dict(stats=0)])
def test_residual_norm_grad_entry_point_refuses(kw):
    kw = {"grad_x": 256, "grad_n": 256, "grad_h": 256} | kw
    rc, _ = rc_of("opus_residual_norm_grad", norm_args(**kw), ctypes.c_void_p(256), 1 << 30, NULL)
    assert rc == _lib.OPUS_ERR_INVALID


def test_residual_norm_grad_entry_point_refuses_workspaces():
    a = norm_args(grad_x=256, grad_n=256)
    assert rc_of("opus_residual_norm_grad", a, ctypes.c_void_p(256), 16, NULL)[0] == _lib.OPUS_ERR_INVALID
    assert rc_of("opus_residual_norm_grad", a, ctypes.c_void_p(264), 1 << 30, NULL)[0] == _lib.OPUS_ERR_INVALID
    assert rc_of("opus_residual_norm_grad", a, NULL, 0, NULL)[0] == _lib.OPUS_ERR_INVALID
    assert rc_of("opus_residual_norm", None, NULL)[0] == _lib.OPUS_ERR_INVALID


def test_clip_entry_points_refuse():
    lib = _lib.load()
    ptr, n, ty = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(4), (ctypes.c_int * 1)(0)
    ws, bytes_ = ctypes.c_void_p(256), 1 << 24

    def norm(ptr=ptr, n=n, ty=ty, count=1, kind=2, ws=ws, size=bytes_, out=ctypes.c_void_p(256)):
        return lib.opus_grad_norm(ptr, n, ty, count, kind, ws, size, out, NULL)

    assert norm(count=-1) == _lib.OPUS_ERR_INVALID
    assert norm(ptr=None) == _lib.OPUS_ERR_INVALID
    assert norm(n=(ctypes.c_int64 * 1)(-4)) == _lib.OPUS_ERR_INVALID
    assert norm(n=(ctypes.c_int64 * 1)(1 << 62)) == _lib.OPUS_ERR_UNSUPPORTED
    assert norm(ty=(ctypes.c_int * 1)(3)) == _lib.OPUS_ERR_UNSUPPORTED
    assert norm(ptr=(ctypes.c_void_p * 1)(0)) == _lib.OPUS_ERR_INVALID
    assert norm(ptr=(ctypes.c_void_p * 1)(257)) == _lib.OPUS_ERR_INVALID
    assert norm(kind=1) == _lib.OPUS_ERR_INVALID
    assert norm(ws=NULL) == _lib.OPUS_ERR_INVALID
    assert norm(ws=ctypes.c_void_p(260)) == _lib.OPUS_ERR_INVALID
    assert norm(size=8) == _lib.OPUS_ERR_INVALID
    assert norm(out=NULL) == _lib.OPUS_ERR_INVALID
    assert lib.opus_clip_grads(ptr, ty, None, ty, n, 1, 2, 1.0, ws, bytes_, ws, NULL) == _lib.OPUS_ERR_INVALID
    assert lib.opus_scale_grads(ptr, ty, ptr, ty, n, 1, 1.0, NULL, NULL) == _lib.OPUS_ERR_INVALID
    assert lib.opus_grad_norm_workspace_bytes(0) > 0


@pytest.mark.parametrize("grads,outs", [
    ([(1024, 6, 1), (4096, 4, 1), (1024, 6, 1)], None), ([(1024, 4, 1), (1036, 3, 1)], None), ([(1028, 1, 0), (1024, 6, 1)], None),
    ([(1024, 6, 1), (4096, 6, 1)], [(8192, 6, 1), (8204, 6, 1)]), ([(1024, 6, 1), (4096, 6, 1)], [(4096, 6, 1), (1024, 6, 1)]),
    ([(1024, 6, 1)], [(1044, 6, 0)]), ([(1024, 6, 0)], [(1024, 6, 1)]), ([(1024, 600, 0), (5000, 2, 0)], [(9000, 600, 0), (1100, 2, 0)])])
def test_clip_entry_points_refuse_overlaps(grads, outs):
    """Lists of (address, elements, type) that would write an element twice, or write what they read elsewhere."""
    lib, k = _lib.load(), len(grads)

    def arrays(of):
        return (ctypes.c_void_p * k)(*[a for a, _, _ in of]), (ctypes.c_int * k)(*[t for _, _, t in of])

    (ptr, ty), (optr, oty) = arrays(grads), arrays(outs or grads)
    n = (ctypes.c_int64 * k)(*[n for _, n, _ in grads])
    ws = ctypes.c_void_p(256)
    assert lib.opus_clip_grads(ptr, ty, optr, oty, n, k, 2, 1.0, ws, 1 << 24, ws, NULL) == _lib.OPUS_ERR_INVALID
    assert "twice" in _lib.last_error()
    assert lib.opus_scale_grads(ptr, ty, optr, oty, n, k, 1.0, ws, NULL) == _lib.OPUS_ERR_INVALID
    assert "twice" in _lib.last_error()


# ------------------------------------------------------------------ torch front end
def test_embedding_refuses():
    w, t = torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for bad in (dict(tokens=t.float()), dict(tokens=t.to(torch.int16)), dict(weight=w[0]), dict(weight=w.double()),
                dict(weight=w.int()), dict(weight=w[:0]), dict(weight=w[:, :0]), dict(out=torch.zeros(3, 7)),
                dict(out=torch.zeros(3, 8, dtype=torch.float16)), dict(out=torch.zeros(8, 3).t())):
        with pytest.raises(ValueError):
            ops.embedding(**({"tokens": t, "weight": w} | bad))
    with pytest.raises(TypeError):
        ops.embedding([0, 1], w)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.embedding(t, w)
    with pytest.raises(ValueError, match="padding_idx"):
        scaled_embedding(t, w, padding_idx=5)
    assert ScaledEmbedding(5, 8, padding_idx=-1).padding_idx == 4
    with pytest.raises(TypeError):
        ScaledEmbedding(5, 8, max_norm=1.0)


def test_embedding_grad_refuses():
    g, t = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64)
    out = torch.zeros(5, 8)
    for bad in (dict(grad_out=g[:2]), dict(grad_out=g.double()), dict(grad_out=g[:, :0]), dict(num_embeddings=0),
                dict(padding_idx=5), dict(padding_idx=-6), dict(accumulate=True), dict(out=out[:4]), dict(out=out.half()),
                dict(out=out, out_dtype=torch.float16), dict(out_dtype=torch.bfloat16), dict(tokens=t[:, None]),
                dict(out=torch.zeros(8, 5).t()), dict(grad_out=g.half(), out_dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            ops.embedding_grad(**({"grad_out": g, "tokens": t, "num_embeddings": 5} | bad))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.embedding_grad(g, t, 5)


def test_residual_norm_refuses():
    x, d = torch.zeros(2, 3, 8), torch.ones(8)
    for bad in (dict(kind="batch"), dict(y=x[:, :2]), dict(y=x.half(), x=x.bfloat16()), dict(y=x, x=x.half()),
                dict(x=x.double()), dict(x=x[..., :0]), dict(weight=d[:7]), dict(bias=d.double()), dict(gate=d),
                dict(post=True), dict(y=x, post=False, post_weight=d), dict(y=x, gate=torch.ones(3, 8)),
                dict(y=x, gate=torch.ones(2, 3, 8)), dict(y=x, gate=torch.ones(1)), dict(y=x, gate=torch.ones(2, 3, 1)),
                dict(y=x, gate=torch.ones(1, 2, 8)), dict(y=x, out_dtype=torch.float16),
                dict(x=x.half(), out_dtype=torch.float32)):
        with pytest.raises(ValueError):
            ops.residual_norm(**({"x": x} | bad))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.residual_norm(x, x, weight=d, gate=torch.ones(2, 1, 8))
    with pytest.raises(ValueError, match="CUDA tensor"):
        residual_norm(x, x, weight=d, post=True)


def test_residual_norm_grad_refuses():
    x, stats, d = torch.zeros(2, 3, 8), torch.zeros(6, 4), torch.ones(8)
    for bad in (dict(grad_n=None, grad_h=None), dict(grad_n=x[:1]), dict(grad_h=x.half()), dict(stats=stats[:5]),
                dict(stats=stats.double()), dict(wanted=["x"]), dict(grad_n=x.half(), y=x), dict(gate=d)):
        with pytest.raises(ValueError):
            ops.residual_norm_grad(**({"grad_n": x, "grad_h": x, "h": x, "stats": stats, "weight": d} | bad))
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.residual_norm_grad(x, x, x, stats, weight=d)


def test_residual_norm_layer_refuses():
    x = torch.zeros(2, 3, 8)
    with pytest.raises(ValueError):
        ResidualNorm(8, kind="group")
    with pytest.raises(ValueError, match="gate of its own"):
        ResidualNorm(8, gate=True)(x, x, gate=torch.ones(8))
    with pytest.raises(ValueError, match="needs y"):
        ResidualNorm(8)(x, gate=torch.ones(8))


def test_clip_refuses():
    a, b = torch.zeros(6), torch.zeros(4)
    for bad in ([a.double()], [a.int()], [a, torch.zeros(2, device="meta")], [a.to_sparse()]):
        with pytest.raises(ValueError):
            ops.clip_grads(bad, 1.0)
        with pytest.raises(ValueError):
            ops.grad_norm(bad)
    with pytest.raises(ValueError, match="expanded"):
        ops.clip_grads([torch.zeros(1).expand(4)], 1.0)
    for norm_type in (1, 0, 3.0, -math.inf, math.nan):
        with pytest.raises(ValueError, match="norm_type"):
            ops.clip_grads([a], 1.0, norm_type=norm_type)
        with pytest.raises(ValueError, match="norm_type"):
            ops.grad_norm([a], norm_type)
    for out in ([a], [b, b], [torch.zeros(7), b], [torch.zeros(12)[::2], b], [a.double(), b]):
        with pytest.raises(ValueError):
            ops.clip_grads([a, b], 1.0, out=out)
    buf = torch.zeros(12)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.clip_grads([buf[:6]], 1.0, out=[buf[6:]])
    for norm in (torch.zeros(2), torch.zeros((), dtype=torch.float64)):
        with pytest.raises(ValueError, match="norm must be"):
            ops.scale_grads([a], 1.0, norm)
    with pytest.raises(ValueError, match="CUDA tensor"):
        ops.grad_norm([a])


def test_clip_of_nothing():
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(ops.grad_norm([])) == 0.0 and float(ops.clip_grads([], 1.0)) == 0.0
    assert float(clip_grad_norm_([p], 1.0)) == 0.0 and float(clip_grad_norm_(p, 1.0, error_if_nonfinite=True)) == 0.0
    ops.scale_grads([], 1.0, torch.zeros(()))


def test_dense_layouts():
    x = torch.zeros(4, 6, 5)
    for dense in (x, x.permute(2, 0, 1), x[1:3], x.transpose(0, 1), x[:1, :, :], torch.zeros(()), torch.zeros(0, 3)):
        assert ops._dense(dense)
    for gaps in (x[:, :3], x[..., ::2], x.transpose(0, 2)[1:2], torch.zeros(1).expand(4)):
        assert not ops._dense(gaps)
