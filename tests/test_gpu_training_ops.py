"""The training-step operators against plain implementations in 64 bits (GPU).

Tolerances.  With u = 2^-24 (half a step of f32) and e = finfo(t).eps / 2 (half
a step of the output's type), a result that is computed in f32 and rounded
once is off by at most e |v| + K u M: M is the same formula over magnitudes
(every subtraction an addition), K the length of the longest chain of f32
operations behind a value.  Each test states its K.
"""
import subprocess
import sys

import numpy as np
import pytest
import torch

from conftest import ROOT
from opus_b200 import ops
from opus_b200.layers import GCLinear, ResidualNorm, ScaledEmbedding, residual_norm, scaled_embedding
from opus_b200.train import clip_grad_norm_, find_GClayers, get_batch_opus, initialize_projector
from tiny_model import ProxyLoader

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = 2.0 ** -24
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(*shape, device=DEV, generator=g) * scale).to(dtype)


def half_step(t):
    return torch.finfo(t).eps / 2


def within(got, want, bound, what=""):
    """|got - want| <= bound elementwise (bound in float64, a subnormal step of the type added)."""
    t = got.dtype
    bound = bound + torch.finfo(t).smallest_normal * torch.finfo(t).eps
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bool(bad.any()), (f"{what}: {int(bad.sum())} of {bad.numel()} off, worst "
                                 f"{float((off / bound).nan_to_num(nan=float('inf')).max()):.3g} times the bound")


# ============================================================================ embedding
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,V,d", [((1,), 1, 1), ((0,), 5, 8), ((7,), 3, 64), ((2, 33), 50257, 771), ((3, 1, 5), 9, 1600),
                                       ((300,), 151936, 2048), ((1,), 50304, 1600), ((129,), 17, 12)])
def test_embedding_lookup(shape, V, d, dtype):
    g = gen(V + d)
    w = randn(g, V, d, dtype=dtype)
    t = torch.randint(0, V, shape, device=DEV, generator=g)
    for tok in (t, t.to(torch.int32)):
        for scale in (1.0, 27.7128):
            got = ops.embedding(tok, w, scale=scale)
            assert got.shape == (*shape, d) and got.dtype == dtype
            # one f32 product, one rounding: the same two roundings as here, so the same bits
            assert torch.equal(got, (w[t].float() * torch.tensor(scale, device=DEV)).to(dtype))
    ops.check_device_error()


def test_embedding_strides_and_out():
    g = gen(1)
    table = randn(g, 50, 96, dtype=torch.bfloat16)
    t = torch.randint(0, 50, (4, 6), device=DEV, generator=g)
    for w in (table[:, 8:40], table[:, 3:36], table[::2], table.t(), table[5:6]):
        tok = t % w.shape[0]
        assert torch.equal(ops.embedding(tok, w), w[tok])
        assert torch.equal(ops.embedding(tok.t(), w), w[tok.t()])
    out = torch.empty(4, 6, 96, device=DEV, dtype=torch.bfloat16)
    assert ops.embedding(t, table, out=out) is out and torch.equal(out, table[t])


def test_embedding_tokens_out_of_range():
    w = torch.ones(5, 24, device=DEV)
    t = torch.tensor([0, 5, -1, 4, -100, 1 << 40], device=DEV)
    got = ops.embedding(t, w)
    with pytest.raises(IndexError, match="token"):
        ops.check_device_error("embedding")
    assert got.sum(1).tolist() == [24, 0, 0, 24, 0, 0]
    dw = ops.embedding_grad(got + 1, t, 5)
    with pytest.raises(IndexError, match="token"):
        ops.check_device_error("embedding_grad")
    assert dw[:, 0].tolist() == [2, 0, 0, 0, 2]
    ops.embedding(t[:1], w)
    ops.check_device_error()  # cleared


def grad_reference(dy, t, V, scale, padding_idx, out=None):
    """(reference, magnitudes, positions of each token) in 64 bits."""
    rows = dy.reshape(-1, dy.shape[-1]).double()
    flat = t.reshape(-1).long()
    live = (flat >= 0) & (flat < V)
    if padding_idx is not None:
        live &= flat != padding_idx % V  # a negative one counts from the end, as nn.Embedding's
    ref = torch.zeros(V, rows.shape[1], dtype=torch.float64, device=DEV)
    mag, count = ref.clone(), torch.zeros(V, 1, dtype=torch.float64, device=DEV)
    ref.index_add_(0, flat[live], rows[live])
    mag.index_add_(0, flat[live], rows[live].abs())
    count.index_add_(0, flat[live], torch.ones(int(live.sum()), 1, dtype=torch.float64, device=DEV))
    s = float(np.float32(scale))
    ref, mag = ref * s, mag * abs(s)
    if out is not None:
        ref, mag = ref + out.double(), mag + out.double().abs()
    return ref, mag, count


def check_embedding_grad(dy, t, V, scale=1.0, padding_idx=None, out=None, out_dtype=None):
    base = None if out is None else out.clone()
    got = ops.embedding_grad(dy, t, V, scale=scale, padding_idx=padding_idx, out=out, accumulate=out is not None,
                             out_dtype=out_dtype)
    ref, mag, count = grad_reference(dy, t, V, scale, padding_idx, base)
    # K: a sum of `count` terms, the scale, the sum with out
    within(got, ref, half_step(got.dtype) * ref.abs() + (count + 3) * U * mag, "embedding_grad")
    if base is not None:  # rows that no token names keep their bits
        untouched = count[:, 0] == 0
        assert torch.equal(got[untouched], base[untouched])
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,V,d", [(0, 5, 8), (1, 1, 1), (1, 7, 8), (31, 3, 5), (32, 2, 64), (33, 1, 24), (64, 50257, 16),
                                   (2047, 511, 40), (2048, 512, 33), (2049, 513, 8), (5000, 11, 771), (4097, 151936, 64),
                                   (20000, 300, 128), (70000, 50304, 32)])
def test_embedding_grad(n, V, d, dtype):
    g = gen(n + V + d)
    # half of the positions on two tokens, so that runs cross many units; the others over the whole range
    t = torch.where(torch.rand(n, device=DEV, generator=g) < 0.5, torch.randint(0, min(V, 2), (n,), device=DEV, generator=g),
                    torch.randint(0, V, (n,), device=DEV, generator=g))
    dy = randn(g, n, d, dtype=dtype)
    got = check_embedding_grad(dy, t, V, scale=2.5)
    assert torch.equal(got, ops.embedding_grad(dy, t.to(torch.int32), V, scale=2.5))  # the same bits again
    check_embedding_grad(dy, t, V, padding_idx=0)
    check_embedding_grad(dy, t, V, padding_idx=-1, out_dtype=torch.float32)
    check_embedding_grad(dy, t, V, out=randn(g, V, d, dtype=dtype))
    check_embedding_grad(dy, t, V, out=randn(g, V, d), scale=0.5)
    ops.check_device_error()


@pytest.mark.parametrize("n,V,d", [(2048, 50304, 8), (4096, 5, 16), (4097, 70, 8), (16384, 151936, 16), (32768, 262143, 8),
                                   (32769, 262144, 8), (81920, 50257, 64), (188416, 50304, 16), (188417, 50304, 16),
                                   (300_000, 3, 8), (250_000, 300_000, 24)])
def test_embedding_grad_sort_sizes(n, V, d):
    """One to sixteen blocks of the sorting cluster, one to three digits, and lists that are sorted through global memory."""
    g = gen(n)
    t = (V ** torch.rand(n, device=DEV, generator=g, dtype=torch.float64)).long().clamp_(max=V - 1)  # log-uniform: long runs
    dy = randn(g, n, d)
    got = check_embedding_grad(dy, t, V, padding_idx=V - 1)
    assert torch.equal(got, ops.embedding_grad(dy, t, V, padding_idx=V - 1))
    check_embedding_grad(dy, t, V, out=randn(g, V, d))
    check_embedding_grad(dy, torch.arange(n, device=DEV) * 7919 % V, V)
    ops.check_device_error()


@pytest.mark.parametrize("n,V,d,step", [(2, 3, 1601, 1), (32, 50304, 4099, 1), (32, 40, 2048, 1), (33, 9, 1024, 1),
                                        (33, 9, 1032, 1), (64, 1, 4096, 1), (65, 2, 512, 1), (512, 30, 512, 7),
                                        (513, 30, 512, 7), (1000, 2, 64, 1), (2048, 1, 128, 1), (2048, 700, 31, 3),
                                        (2048, 1000003, 8, 977), (256, 19398657, 1, 65537)])
def test_embedding_grad_short_lists(n, V, d, step):
    """Lists at the bounds of the single launch: runs of one to all positions, shares of the table with and without names."""
    g = gen(n + d)
    t = (torch.arange(n, device=DEV) // 3 * step) % V  # runs of three, and of more where the table is short
    t = torch.where(torch.rand(n, device=DEV, generator=g) < 0.3, t[torch.randint(0, n, (n,), device=DEV, generator=g)], t)
    for dtype in (torch.bfloat16, torch.float32):
        dy = randn(g, n, d, dtype=dtype)
        a = check_embedding_grad(dy, t, V, scale=0.5)
        assert torch.equal(a, ops.embedding_grad(dy, t, V, scale=0.5))
        check_embedding_grad(dy, t.int(), V, padding_idx=int(t[0]), out_dtype=torch.float32)
        check_embedding_grad(dy, t, V, padding_idx=-1, out=randn(g, V, d, dtype=dtype))


@pytest.mark.parametrize("pattern", ["one", "each", "pairs", "descending", "padding", "blocks"])
def test_embedding_grad_patterns(pattern):
    n, V, d = 6000, 7000, 72
    i = torch.arange(n, device=DEV)
    t = {"one": i * 0 + 123, "each": (i * 4099) % V, "pairs": i // 2, "descending": n - 1 - i, "padding": i * 0 + 9,
         "blocks": (i // 32) % 5}[pattern]
    dy = randn(gen(3), n, d, dtype=torch.bfloat16)
    got = check_embedding_grad(dy, t, V, padding_idx=9)
    if pattern == "padding":
        assert not bool(got.any())


def test_embedding_grad_strides():
    g = gen(8)
    t = torch.randint(0, 40, (6, 50), device=DEV, generator=g)
    wide = randn(g, 6, 50, 200, dtype=torch.bfloat16)
    for dy in (wide[..., :64], wide[..., 8:72], wide[..., 3:60], wide[..., 1:2], wide[:, :, ::2],
               randn(g, 50, 6, 64, dtype=torch.bfloat16).transpose(0, 1), randn(g, 64, dtype=torch.float32).expand(6, 50, 64),
               randn(g, 1, 1, 1).expand(6, 50, 24)):
        check_embedding_grad(dy, t, 40)
    check_embedding_grad(wide[..., :64].transpose(0, 1), t.t(), 40)


def test_embedding_grad_not_finite():
    t = torch.tensor([0, 1, 2, 1], device=DEV)
    dy = torch.ones(4, 8, device=DEV)
    dy[1, 0], dy[2, 1], dy[3, 2] = float("nan"), float("inf"), float("-inf")
    got = ops.embedding_grad(dy, t, 4)
    want = torch.tensor([[1.0] * 8, [2.0] * 8, [1.0] * 8, [0.0] * 8], device=DEV)
    want[1, 0], want[2, 1], want[1, 2] = float("nan"), float("inf"), float("-inf")
    assert torch.equal(got.nan_to_num(nan=7.0), want.nan_to_num(nan=7.0))


def test_embedding_beyond_32_bit_offsets():
    V, d = 1_100_000, 2048  # 2.25e9 elements: row offsets pass 31 bits
    w = torch.zeros(V, d, dtype=torch.bfloat16, device=DEV)
    w[-1], w[-2, 0] = 3.0, 5.0
    t = torch.tensor([V - 1, V - 2, 0], device=DEV)
    got = ops.embedding(t, w, scale=2.0)
    assert got[0].unique().tolist() == [6.0] and got[1, :2].tolist() == [10.0, 0.0] and not bool(got[2].any())
    dw = ops.embedding_grad(got, t, V, out=w)
    assert dw[-1].unique().tolist() == [6.0] and dw[-2, :2].tolist() == [10.0, 0.0] and float(dw[:-2].abs().max()) == 0.0
    all_rows = torch.arange(V, device=DEV)
    y = ops.embedding(all_rows, w)  # as many outputs
    assert torch.equal(y, w)
    assert torch.equal(ops.embedding_grad(y, all_rows, V), w)


# ============================================================================ residual norm
def norm_case(seed, shape, d, dtype=torch.float32, x_dtype=None, p_dtype=None, y=True, post=False, gate=None, bias=False,
              affine=True):
    g = gen(seed)
    x_dtype, p_dtype = x_dtype or dtype, p_dtype or dtype
    x = randn(g, *shape, d, dtype=x_dtype, scale=2.0) + 0.5
    c = {"x": x.to(x_dtype), "y": randn(g, *shape, d, dtype=dtype) if y else None}
    p = {}
    if affine:
        p["weight"] = randn(g, d, dtype=p_dtype) * 0.1 + 1
        if bias:
            p["bias"] = randn(g, d, dtype=p_dtype)
        if post:
            p["post_weight"] = randn(g, d, dtype=p_dtype) * 0.1 + 1
            if bias:
                p["post_bias"] = randn(g, d, dtype=p_dtype)
    if gate == "channel":
        p["gate"] = randn(g, d, dtype=p_dtype)
    elif gate == "sample":
        p["gate"] = randn(g, shape[0], *([1] * (len(shape) - 1)), d, dtype=p_dtype)
    n_dtype = dtype if y else x_dtype
    return c, p, randn(g, *shape, d, dtype=n_dtype), randn(g, *shape, d, dtype=x_dtype)


def stats64(v, kind, eps):
    mean = v.mean(-1, keepdim=True) if kind == "layer" else torch.zeros_like(v[..., :1])
    return mean, 1.0 / torch.sqrt(((v - mean) ** 2).mean(-1, keepdim=True) + eps)


def wide_mag(v, kind):
    """Magnitudes behind v - mean."""
    return v.abs() + v.abs().mean(-1, keepdim=True) if kind == "layer" else v.abs()


def check_norm(c, p, dn, dh, kind="rms", post=False, r=1.0, eps=1e-5):
    """Forward against 64 bits, backward against the formulas in 64 bits at the stored h.

    K = 192 for the forward: the longest chain is a row's sum (16 elements a
    thread, 5 shuffles, up to 64 warps by fours), twice for a layer norm and twice
    again with a norm of y.  K = 768 + rows for the backward: four such sums
    in a row, and sums over rows.
    """
    x, y = c["x"], c["y"]
    n, h, stats = ops.residual_norm(x, y, **p, kind=kind, post=post, residual_scale=r, eps=eps)
    f = {k: v.double() for k, v in p.items()}
    one = torch.ones((), dtype=torch.float64, device=DEV)
    zero = one * 0
    w, b, pw, pb, gate = (f.get(k, d) for k, d in (("weight", one), ("bias", zero), ("post_weight", one),
                                                   ("post_bias", zero), ("gate", one)))
    if gate.dim() == 2 and gate.shape[0] != 1 and x.dim() > 2:
        gate = gate.view(gate.shape[0], *([1] * (x.dim() - 2)), -1)
    r32, K = float(np.float32(r)), 192
    h_ref, h_mag = r32 * x.double(), (r32 * x.double()).abs()
    if y is not None:
        z = zm = y.double()
        zm = z.abs()
        if post:
            ym, yr = stats64(y.double(), kind, eps)
            yh, yw = (y.double() - ym) * yr, wide_mag(y.double(), kind) * yr
            z, zm = yh * pw + pb, yw * pw.abs() + pb.abs()
        h_ref, h_mag = h_ref + gate * z, h_mag + gate.abs() * zm
    within(h, h_ref, half_step(h.dtype) * h_ref.abs() + K * U * h_mag, "h")
    h64 = h.double()
    hm, hr = stats64(h64, kind, eps)
    hat, hw = (h64 - hm) * hr, wide_mag(h64, kind) * hr
    n_ref, n_mag = hat * w + b, hw * w.abs() + b.abs()
    within(n, n_ref, half_step(n.dtype) * n_ref.abs() + K * U * n_mag, "n")

    got = ops.residual_norm_grad(dn, dh, h, stats, y, **p, kind=kind, post=post, residual_scale=r)
    again = ops.residual_norm_grad(dn, dh, h, stats, y, **p, kind=kind, post=post, residual_scale=r)
    assert set(got) == {"x"} | ({"y"} if y is not None else set()) | set(p)
    assert all(torch.equal(got[k], again[k]) for k in got)
    rows = h.numel() // h.shape[-1]
    K = 768 + rows
    lead = tuple(range(h.dim() - 1))

    def total(v, dims=lead):
        return v.sum(dims) if dims else v  # sum(()) would be the sum of everything

    def back(a, am, hat, hw, rstd):
        """The norm's backward and its magnitudes."""
        v = a - hat * (a * hat).mean(-1, keepdim=True)
        m = am + hw * (am * hw).mean(-1, keepdim=True)
        if kind == "layer":
            v, m = v - a.mean(-1, keepdim=True), m + am.mean(-1, keepdim=True)
        return v * rstd, m * rstd

    dn64 = torch.zeros_like(h64) if dn is None else dn.double()
    a, am = dn64 * w, (dn64 * w).abs()
    v, m = back(a, am, hat, hw, hr)
    if dh is not None:
        v, m = v + dh.double(), m + dh.double().abs()

    def check(name, ref, mag):
        assert got[name].dtype == (x if name == "x" else y if name == "y" else p[name]).dtype
        ref, mag = ref.reshape(got[name].shape), mag.reshape(got[name].shape)
        within(got[name], ref, half_step(got[name].dtype) * ref.abs() + K * U * mag, name)

    check("x", r32 * v, abs(r32) * m)
    if "weight" in p:
        check("weight", total(dn64 * hat), total(dn64.abs() * hw))
    if "bias" in p:
        check("bias", total(dn64), total(dn64.abs()))
    if y is not None:
        dz, dzm = gate * v, gate.abs() * m
        if "gate" in p:
            keep = lead if p["gate"].dim() == 1 else lead[1:]
            check("gate", total(v * z, keep), total(m * zm, keep))
        if post:
            if "post_weight" in p:
                check("post_weight", total(dz * yh), total(dzm * yw))
            if "post_bias" in p:
                check("post_bias", total(dz), total(dzm))
            check("y", *back(dz * pw, dzm * pw.abs(), yh, yw, yr))
        else:
            check("y", dz, dzm)
    return n, h, stats, got


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("post,gate", [(False, None), (True, "channel"), (True, "sample"), (False, "sample")])
@pytest.mark.parametrize("shape,d", [((1, 1), 1), ((2, 3), 7), ((3, 5), 64), ((1, 1), 2048), ((2, 9), 768), ((4, 33), 771),
                                     ((2, 2), 4096), ((3, 1), 4104), ((1, 3), 8192), ((2, 2), 4099), ((1, 2), 16384),
                                     ((2, 130), 128), ((5, 40), 1600)])
def test_residual_norm_f32(shape, d, post, gate, kind):
    check_norm(*norm_case(d, shape, d, post=post, gate=gate, bias=kind == "layer"), kind=kind, post=post, r=0.5)


@pytest.mark.parametrize("dtype,x_dtype,p_dtype", [(torch.bfloat16, None, None), (torch.float16, None, None),
                                                   (torch.bfloat16, torch.float32, torch.float32),
                                                   (torch.float16, torch.float32, None),
                                                   (torch.bfloat16, None, torch.float32)])
@pytest.mark.parametrize("shape,d,post,gate", [((2, 65), 768, True, "sample"), ((1, 1), 2048, False, None),
                                               ((3, 50), 1600, False, "channel"), ((2, 7), 771, True, None),
                                               ((9, 3), 72, True, "channel"), ((1, 4), 8200, True, "sample"),
                                               ((1, 2), 16384, False, None), ((1, 3), 12289, True, "channel")])
def test_residual_norm_types(dtype, x_dtype, p_dtype, shape, d, post, gate):
    for kind in ("rms", "layer"):
        check_norm(*norm_case(d + 1, shape, d, dtype, x_dtype, p_dtype, post=post, gate=gate, bias=True), kind=kind, post=post)


def test_residual_norm_forms():
    for kind in ("rms", "layer"):
        for dtype in (torch.bfloat16, torch.float32):
            c, p, dn, dh = norm_case(5, (3, 20), 96, dtype, y=False, bias=True)
            n, h, stats, _ = check_norm(c, p, dn, dh, kind=kind)
            assert h.data_ptr() == c["x"].data_ptr()  # no second residual stream
            check_norm(c, p, dn, None, kind=kind)
            check_norm(c, p, None, dh, kind=kind)
            check_norm(c, p, dn, dh, kind=kind, r=-1.5)
            c, p, dn, dh = norm_case(6, (3, 20), 96, dtype, affine=False)
            check_norm(c, p, dn, dh, kind=kind)
            check_norm(c, p, dn, None, kind=kind, post=True)
            check_norm(c, p, None, dh, kind=kind, post=True, r=0.0)
            c, p, dn, dh = norm_case(7, (20,), 96, dtype, gate="sample", post=True)  # a gate for each row
            check_norm(c, p, dn, dh, kind=kind, post=True)
            c, p, dn, dh = norm_case(8, (), 96, dtype, gate="channel")  # one vector
            check_norm(c, p, dn, dh, kind=kind)
            c, p, dn, dh = norm_case(9, (2, 3, 4), 40, dtype, gate="sample", post=True)
            check_norm(c, p, dn, dh, kind=kind, post=True)
            p["gate"] = p["gate"].reshape(2, 40)
            check_norm(c, p, dn, dh, kind=kind, post=True)


@pytest.mark.parametrize("rows", [1, 63, 64, 65, 700, 3001])
def test_residual_norm_many_rows(rows):
    check_norm(*norm_case(rows, (rows,), 136, torch.bfloat16, post=True, gate="channel", bias=True), kind="layer", post=True)
    check_norm(*norm_case(rows, (2, rows), 136, post=True, gate="sample"), post=True)
    check_norm(*norm_case(rows, (rows, 2), 24, post=False, gate="sample"))


@pytest.mark.parametrize("dtype,x_dtype", [(torch.bfloat16, None), (torch.float32, None), (torch.float16, torch.float32)])
@pytest.mark.parametrize("d", [2047, 2048, 2049, 2056, 4095, 4096, 4097, 4100, 4104, 8191, 8192, 8193, 8200, 16383])
def test_residual_norm_where_rows_are_split(d, dtype, x_dtype):
    """Widths at which a row passes from one block to a cluster of two, four and eight."""
    for kind, post, gate in (("rms", False, None), ("layer", True, "sample")):
        check_norm(*norm_case(d, (3, 3), d, dtype, x_dtype, post=post, gate=gate, bias=kind == "layer"), kind=kind, post=post)


@pytest.mark.parametrize("shape,d", [((3, 133), 4104), ((2, 200), 8193), ((5, 40), 16384), ((301, 2), 5001)])
def test_residual_norm_many_wide_rows(shape, d):
    """More rows than clusters run at once: several rows a cluster, whose runs cross samples."""
    check_norm(*norm_case(d, shape, d, torch.bfloat16, post=True, gate="sample", bias=True), kind="layer", post=True)
    check_norm(*norm_case(d, shape, d, post=True, gate="channel"), post=True)
    check_norm(*norm_case(d, shape, d, torch.bfloat16))


def test_residual_norm_more_gates_than_one_launch_joins():
    check_norm(*norm_case(3, (70000,), 24, gate="sample"))
    check_norm(*norm_case(4, (140000, 1), 8, torch.bfloat16, gate="sample", post=True, bias=True), kind="layer", post=True)


def test_residual_norm_no_rows():
    for shape, gate in (((0,), "channel"), ((2, 0), "sample"), ((0, 3), None)):
        c, p, dn, dh = norm_case(1, shape, 32, gate=gate, post=True, bias=True)
        n, h, stats = ops.residual_norm(c["x"], c["y"], **p, kind="layer")
        assert n.shape == c["x"].shape and h.shape == c["x"].shape
        got = ops.residual_norm_grad(dn, dh, h, stats, c["y"], **p, kind="layer")
        assert all(not bool(got[k].any()) for k in p) and got["x"].shape == c["x"].shape


def test_residual_norm_strides():
    c, p, dn, dh = norm_case(11, (4, 30), 64, torch.bfloat16, post=True, gate="sample")
    wide = randn(gen(12), 4, 30, 200, dtype=torch.bfloat16)
    for x, y in ((wide[..., :64], wide[..., 64:128]), (wide[..., 1:65], wide[..., 3:67]), (wide[..., :64], c["y"]),
                 (wide.transpose(0, 1)[:4, :, :64].reshape(4, 4, 64).transpose(0, 1), wide[:, :4, 100:164]),
                 (wide[:, :1, :64].expand(4, 30, 64), wide[0, 0, :64].expand(4, 30, 64))):
        shape = x.shape
        g = {**p, "gate": p["gate"][: shape[0]]}
        d1, d2 = randn(gen(1), *shape[:-1], 90, dtype=torch.bfloat16)[..., 8:72], randn(gen(2), 1, 1, 64).to(x.dtype).expand(shape)
        check_norm({"x": x, "y": y}, g, d1, d2, post=True)


def test_residual_norm_not_finite_and_zero_rows():
    """A row of zeros is normed to zeros; NaN and infinities stay in their rows."""
    x, y = torch.ones(5, 40, device=DEV), torch.zeros(5, 40, device=DEV)
    x[0] = 0.0
    x[2, 3], x[3, 4] = float("nan"), float("inf")
    for kind in ("rms", "layer"):
        n, h, stats = ops.residual_norm(x, y, kind=kind)
        assert not bool(n[0].any()) and bool(n[2].isnan().all()) and bool(n[3].isnan().any())
        assert bool(n[[1, 4]].isfinite().all())
        g = ops.residual_norm_grad(torch.ones_like(x), None, h, stats, y, kind=kind)
        assert bool(g["x"][[0, 1, 4]].isfinite().all()) and bool(g["x"][2].isnan().all())


def test_residual_norm_large_offset_layer():
    """A mean far from zero: the variance is summed about it, so it keeps its digits."""
    g = gen(31)
    x = randn(g, 6, 1024) + 1000.0
    n, h, _ = ops.residual_norm(x, torch.zeros_like(x), kind="layer", eps=0.0)
    v = x.double()
    ref = (v - v.mean(-1, keepdim=True)) / v.std(-1, keepdim=True, correction=0)
    # the mean is off by at most 192 u 1000, and everything else by 192 u of values below 6
    within(n, ref, 192 * U * (1000.0 + 6.0) * torch.ones_like(ref))


def test_residual_norm_beyond_32_bit_offsets():
    rows, d = 140_000, 16384  # 2.29e9 elements
    x = torch.zeros(rows, d, dtype=torch.bfloat16, device=DEV)
    x[-1, ::2], x[-1, 1::2] = 3.0, -3.0
    n, h, stats = ops.residual_norm(x, x, eps=0.25)
    assert h[-1, :2].tolist() == [6.0, -6.0] and not bool(h[:5].any())
    # 6 / sqrt(36.25) = 0.996546, between the bf16 neighbours 1 - 2^-8 = 0.99609375 and 1
    assert n[-1, :2].tolist() == [0.99609375, -0.99609375] and not bool(n[-2].any())
    del n
    got = ops.residual_norm_grad(None, h, h, stats, x, residual_scale=0.5)
    assert got["x"][-1, :2].tolist() == [3.0, -3.0] and got["y"][-1, :2].tolist() == [6.0, -6.0]
    assert not bool(got["x"][-2].any())


def numeric(f, values, direction, step=1e-5):
    """Directional derivative of f over a list of float64 tensors by central differences."""
    up = f([v + step * d for v, d in zip(values, direction)])
    down = f([v - step * d for v, d in zip(values, direction)])
    return float((up - down) / (2 * step))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_gradient_against_differences(kind):
    """Autograd through the layer against differences of the formula in 64 bits.

    The gradients are f32 sums of at most 1300 terms: 2^-24 of that many
    magnitudes of order 10 is 1e-3 in absolute terms over all inputs; a
    central difference at 1e-5 is off by about 1e-8 of the function's size.
    """
    c, p, dn, dh = norm_case(77, (3, 6), 24, gate="sample", post=True, bias=True)
    names = ["x", "y", *p]
    leaves = [t.clone().requires_grad_() for t in (c["x"], c["y"], *p.values())]
    kw = dict(zip(names, leaves))
    n, h = residual_norm(**kw, kind=kind, residual_scale=0.5, eps=1e-5)
    grads = torch.autograd.grad((n * dn).sum() + (h * dh).sum(), leaves)

    def f(v):
        v = dict(zip(names, v))
        ym, yr = stats64(v["y"], kind, 1e-5)
        h = 0.5 * v["x"] + v["gate"] * ((v["y"] - ym) * yr * v["post_weight"] + v["post_bias"])
        hm, hr = stats64(h, kind, 1e-5)
        return (((h - hm) * hr * v["weight"] + v["bias"]) * dn.double() + h * dh.double()).sum()

    values = [t.detach().double() for t in leaves]
    for i in range(len(values)):  # each input on its own
        d = [torch.zeros_like(v) for v in values]
        d[i] = torch.randn(values[i].shape, dtype=torch.float64, device=DEV, generator=gen(i))
        want = numeric(f, values, d)
        assert abs(float((grads[i].double() * d[i]).sum()) - want) < 1e-3, names[i]


def test_residual_norm_layer_autograd_forms():
    d = 64
    layer = ResidualNorm(d, device=DEV)
    x = randn(gen(0), 4, d).requires_grad_()
    n, h = layer(x)  # no block yet: h is x, and its gradient joins
    (n.sum() + 2 * h.sum()).backward()
    ref = x.detach().double().requires_grad_()
    (torch.nn.functional.rms_norm(ref, (d,), eps=1e-6).sum() + 2 * ref.sum()).backward()
    # K u of magnitudes below 16 (|dn| = 1 over rows whose 1 / sd is about 1)
    within(x.grad, ref.grad, 1024 * U * 16 * torch.ones_like(ref))
    for used in ("n", "h"):
        layer = ResidualNorm(d, kind="layer", bias=True, post=True, gate=True, residual_scale=0.5, device=DEV)
        x, y = (randn(gen(s), 4, d).requires_grad_() for s in (1, 2))
        out = dict(zip("nh", layer(x, y)))[used]
        out.sum().backward()
        assert x.grad is not None and y.grad is not None and layer.gate.grad is not None
        assert (layer.weight.grad is not None) or used == "h"
    frozen = ResidualNorm(d, device=DEV).requires_grad_(False)
    x = randn(gen(5), 4, d).requires_grad_()
    n, h = frozen(x, randn(gen(6), 4, d))
    n.sum().backward()
    assert frozen.weight.grad is None and x.grad is not None
    with torch.no_grad():
        assert not frozen(x, x)[0].requires_grad
    n16, h32 = residual_norm(x, out_dtype=torch.bfloat16)
    assert n16.dtype == torch.bfloat16 and h32.dtype == torch.float32
    (g,) = torch.autograd.grad(h32.sum(), x)
    assert torch.equal(g, torch.ones_like(x))


# ============================================================================ gradient clip
def norm64(tensors):
    return float(torch.sqrt(sum((t.double() ** 2).sum() for t in tensors)))


# the squares' sum is off by at most 10 u (8 fused additions a lane of four, two to join them; the rest is in
# double), its root by half of that, and the result is rounded once
NORM_TOL = 6.5 * U


def coefficient(norm, max_norm):
    """min(1, max_norm / (norm + 1e-6)) in f32, operation by operation."""
    with np.errstate(all="ignore"):
        c = np.float32(max_norm) / (np.float32(norm) + np.float32(1e-6))
    return torch.tensor(np.float32(1.0) if c > 1 else c, device=DEV)


def check_clip(grads, max_norm, out=None):
    src = [t.clone() for t in grads]
    want = norm64(src)
    got = ops.grad_norm(grads)
    assert got.shape == () and got.dtype == torch.float32
    assert abs(float(got) - want) <= NORM_TOL * want
    norm = ops.clip_grads(grads, max_norm, out=out)
    assert torch.equal(norm, got)
    c = coefficient(float(norm), max_norm)
    for i, s in enumerate(src):
        t = (grads if out is None else out)[i]
        assert torch.equal(t, (s.float() * c).to(t.dtype)), i
        if out is not None:
            assert torch.equal(grads[i], s)
    return norm, c


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sizes", [[1], [7], [8], [16384], [16385, 3], [5, 0, 1000, 1, 40000], [100000] * 3, [33] * 1025,
                                   [1, 2, 3] * 700, [3_000_001]])
def test_clip_grads(sizes, dtype):
    g = gen(len(sizes) + sizes[0])
    for above in (True, False):
        grads = [randn(g, n, dtype=dtype, scale=0.01) for n in sizes]
        bound = norm64(grads) * (0.3 if above else 2.0)
        _, c = check_clip(grads, bound)
        assert (float(c) < 1) == above
        for to in TYPES:
            check_clip([randn(g, n, dtype=dtype, scale=0.01) for n in sizes], bound,
                       out=[torch.full((n,), 9.0, device=DEV, dtype=to) for n in sizes])


def test_clip_grads_mixed_types_views_and_layouts():
    g = gen(9)
    flat = randn(g, 5000, dtype=torch.bfloat16)
    f32 = randn(g, 5000)
    grads = [flat[1:1002], flat[1003:1003], flat[1005:3006], f32[3:], randn(g, 40, 50).t(), randn(g, 40, 50)[:, ::2],
             randn(g, 3, 4, 5, dtype=torch.float16).permute(2, 0, 1), randn(g, 7)[2:3], torch.randn((), device=DEV)]
    rest = flat.clone()
    norm, _ = check_clip(grads, 1.0)
    assert torch.equal(flat[:1], rest[:1]) and torch.equal(flat[1002:1005], rest[1002:1005])  # the gaps keep their bits
    assert torch.equal(flat[3006:], rest[3006:])
    out = [torch.empty(t.shape, device=DEV) for t in grads]
    check_clip(grads, 0.01, out=out)
    buf = torch.empty(5000, device=DEV, dtype=torch.float16)
    check_clip([f32[3:]], 0.01, out=[buf[1:4998]])  # the two sides reach their boundaries apart
    check_clip([f32[3:]], 0.01, out=[buf[3:]])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_grad_norm_extremes(dtype):
    g = gen(2)
    for scale in (1e25, 1e-25, 1e19, 1e-19, 3e38):
        t = (torch.rand(5000, device=DEV, generator=g) + 0.1).to(dtype) * scale if scale < 3e38 else \
            torch.full((1,), 3e38, device=DEV, dtype=dtype)
        t[17 % t.numel()] = 0
        if scale == 3e38:
            t[0] = 3e38
        want = norm64([t])
        assert abs(float(ops.grad_norm([t])) - want) <= NORM_TOL * want
        assert float(ops.grad_norm([t], float("inf"))) == float(t.abs().max())
    assert float(ops.grad_norm([torch.zeros(100, device=DEV, dtype=dtype)])) == 0.0
    z = torch.zeros(100, device=DEV, dtype=dtype)
    assert float(ops.clip_grads([z], 1.0)) == 0.0 and not bool(z.any())


def test_grad_norm_infinity():
    g = gen(4)
    grads = [randn(g, n, dtype=t) for n, t in ((1, torch.float32), (70001, torch.bfloat16), (0, torch.float32), (90, torch.float16))]
    grads[1][-1] = -50.0
    assert float(ops.grad_norm(grads, float("inf"))) == 50.0
    norm = ops.clip_grads(grads, 5.0, norm_type=float("inf"))
    assert float(norm) == 50.0 and float(grads[1][-1]) == -5.0


def test_clip_grads_not_finite():
    def grads():
        return [torch.ones(300, device=DEV), torch.ones(20000, device=DEV, dtype=torch.bfloat16)]

    for kind in (2.0, float("inf")):
        g = grads()
        g[1][777] = float("nan")
        assert bool(ops.grad_norm(g, kind).isnan())
        assert bool(ops.clip_grads(g, 1.0, norm_type=kind).isnan())
        assert all(bool(t.isnan().all()) for t in g)
        g = grads()
        g[0][5] = float("-inf")
        assert float(ops.clip_grads(g, 1.0, norm_type=kind)) == float("inf")
        assert bool(g[0][5].isnan()) and not bool(g[0][:5].any()) and not bool(g[1].any())
    p = [torch.nn.Parameter(t) for t in grads()]
    for q in p:
        q.grad = torch.ones_like(q)
    p[0].grad[0] = float("nan")
    with pytest.raises(RuntimeError, match="not finite"):
        clip_grad_norm_(p, 1.0, error_if_nonfinite=True)
    assert bool((p[1].grad == 1).all())  # left as they are


def test_clip_grad_norm_matches_torch():
    """The same rule as torch's: factors one f32 step apart at most, so values two roundings apart."""
    g = gen(12)
    for norm_type in (2.0, float("inf")):
        a = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((64, 32), (32,), (5, 7, 3), (1,))]
        b = [torch.nn.Parameter(torch.zeros(s, device=DEV)) for s in ((64, 32), (32,), (5, 7, 3), (1,))]
        for p, q in zip(a[:-1], b[:-1]):  # the last has no gradient
            p.grad = randn(g, *p.shape)
            q.grad = p.grad.clone()
        n = clip_grad_norm_(a, 0.7, norm_type=norm_type)
        m = torch.nn.utils.clip_grad_norm_(b, 0.7, norm_type=norm_type)
        assert abs(float(n) - float(m)) <= 16 * U * float(m)
        for p, q in zip(a[:-1], b[:-1]):
            within(p.grad, q.grad.double(), 24 * U * q.grad.double().abs())
        assert float(clip_grad_norm_(a, 0.7, norm_type=norm_type, error_if_nonfinite=True)) <= 0.7 * (1 + 16 * U)


def test_scale_grads_with_a_joined_norm():
    """Two shards: the norm of the whole from the shards' norms, then each shard scaled by it."""
    g = gen(20)
    shards = [[randn(g, 1000), randn(g, 77, dtype=torch.bfloat16)], [randn(g, 5000)]]
    whole = norm64([t for s in shards for t in s])
    norm = torch.linalg.vector_norm(torch.stack([ops.grad_norm(s) for s in shards]))
    for s in shards:
        before = [t.clone() for t in s]
        ops.scale_grads(s, 1.0, norm)
        c = coefficient(float(norm), 1.0)
        assert all(torch.equal(t, (b.float() * c).to(t.dtype)) for t, b in zip(s, before))
    after = norm64([t for s in shards for t in s])
    assert whole > 1 and after <= 1.0 * (1 + 2 * half_step(torch.bfloat16))


def test_clip_grads_refuses_what_it_would_write_twice():
    a, b = torch.ones(600, device=DEV), torch.ones(40, device=DEV)
    p = torch.nn.Parameter(torch.zeros(3, device=DEV))
    p.grad = torch.ones(3, device=DEV)
    for grads, out in (([a, b, a], None), ([a[:4], a[3:]], None), ([a[1:2], a], None), ([a, b], [torch.empty_like(a), b[:]]),
                       ([a[:300]], [a[299:599]])):
        if out is not None and out[-1].data_ptr() == b.data_ptr():
            ops.clip_grads(grads, 1e9, out=out)  # one member in place and another not: allowed
            continue
        with pytest.raises(ValueError, match="twice"):
            ops.clip_grads(grads, 1.0, out=out)
        with pytest.raises(ValueError, match="twice"):
            ops.scale_grads(grads, 1.0, torch.ones((), device=DEV), out=out)
    with pytest.raises(ValueError, match="twice"):
        clip_grad_norm_([p, p], 1.0)
    assert bool((a == 1).all()) and bool((b == 1).all()) and bool((p.grad == 1).all())
    gaps = torch.full((6, 8), 2.0, device=DEV)
    for grads in ([gaps[:, :3], gaps[:, :3]], [a, gaps[:, 1::2], gaps[:, 1::2]]):
        with pytest.raises(ValueError, match="twice"):
            ops.clip_grads(grads, 1.0)
        with pytest.raises(ValueError, match="twice"):
            ops.scale_grads(grads, 1.0, torch.ones((), device=DEV))
    assert bool((gaps == 2).all())
    ops.scale_grads([gaps[:, :3], gaps[:, 2:5], gaps[:0, :3], gaps[:0, :3]], 1.0, torch.full((), 4.0, device=DEV))
    c = np.float32(1.0) / (np.float32(4.0) + np.float32(1e-6))
    assert bool((gaps[:, :5] == float(np.float32(2.0) * c)).all()) and bool((gaps[:, 5:] == 2).all())  # scaled once
    assert float(ops.grad_norm([b, b])) == float(np.float32(80 ** 0.5))  # reading twice is fine
    assert float(ops.clip_grads([a[:300], a[300:]], 1.0)) > 1  # neighbours share no element


def test_clip_grads_beyond_32_bit_offsets():
    n = (1 << 31) + 12345
    t = torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    t[-1], t[0] = 4.0, 3.0
    assert float(ops.grad_norm([t])) == 5.0
    assert float(ops.clip_grads([t], 2.5)) == 5.0
    assert float(t[-1]) == 2.0 and float(t[0]) == 1.5  # the factor 2.5 / 5.000001 rounds to these in bf16


# ============================================================================ streams and graphs
def training_ops(s):
    """One run of every operator on the tensors of s."""
    y = ops.embedding(s["t"], s["w"], scale=3.0)
    dw = ops.embedding_grad(s["dy"], s["t"], s["w"].shape[0], padding_idx=2)
    n, h, st = ops.residual_norm(s["x"], s["y"], weight=s["pw"], post_weight=s["pw"], gate=s["gate"])
    g = ops.residual_norm_grad(s["dn"], s["dh"], h, st, s["y"], weight=s["pw"], post_weight=s["pw"], gate=s["gate"])
    norm = ops.clip_grads(s["grads"], 0.5, out=s["out"])
    return [y, dw, n, h, *g.values(), norm, ops.grad_norm(s["grads"]), *s["out"]]


def training_state(seed):
    g = gen(seed)
    b, T, d, V = 3, 70, 136, 900
    s = {k: randn(g, b, T, d, dtype=torch.bfloat16) for k in ("dy", "x", "y", "dn", "dh")}
    s |= {"t": torch.randint(0, V, (b, T), device=DEV, generator=g), "w": randn(g, V, d, dtype=torch.bfloat16),
          "pw": randn(g, d, dtype=torch.bfloat16), "gate": randn(g, b, 1, d, dtype=torch.bfloat16),
          "grads": [randn(g, n) for n in (30, 70000, 5)]}
    s["out"] = [torch.zeros_like(t) for t in s["grads"]]
    return s


def test_captured_and_replayed():
    """Two captured graphs of the same operators, replayed in turn and on new inputs, give the eager results."""
    a, b = training_state(1), training_state(2)
    want = [[t.clone() for t in training_ops(s)] for s in (a, b)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for s in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(training_ops(s))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
    torch.cuda.synchronize()
    for got, ref in zip(outs, want):
        assert all(torch.equal(x, y) for x, y in zip(got, ref))
    fresh = training_state(3)
    ref = [t.clone() for t in training_ops(fresh)]
    for k, v in fresh.items():
        for dst, src in zip(a[k] if isinstance(v, list) else [a[k]], v if isinstance(v, list) else [v]):
            dst.copy_(src)
    graphs[0].replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(outs[0], ref))
    assert all(torch.equal(x, y) for x, y in zip(outs[1], want[1]))
    ops.check_device_error()


FIRST_CALL_CAPTURED = """
import sys, torch
sys.path.insert(0, sys.argv[1])
from opus_b200 import ops
w, t = torch.randn(100, 64, device="cuda"), torch.arange(50, device="cuda") % 7
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    y = ops.embedding(t, w, scale=2.0)
    dw = ops.embedding_grad(y, t, 100)
    n, h, stats = ops.residual_norm(y, y)
    g = ops.residual_norm_grad(n, h, h, stats, y)
    norm = ops.grad_norm([dw, n])
graph.replay()
torch.cuda.synchronize()
assert torch.equal(y, w[t] * 2) and float(norm) > 0 and bool(g["x"].isfinite().all())
ops.check_device_error()
print("captured")
"""


@pytest.mark.parametrize("d", [5120, 4099])
def test_wide_rows_captured_and_on_streams_at_once(d):
    """Rows split among clusters: replayed in a graph, and from several streams together, with the eager results."""
    c, p, dn, dh = norm_case(d, (3, 100), d, torch.bfloat16, post=True, gate="sample", bias=True)

    def run():
        n, h, stats = ops.residual_norm(c["x"], c["y"], **p, kind="layer")
        got = ops.residual_norm_grad(dn, dh, h, stats, c["y"], **p, kind="layer")
        return [n, h, stats, *(got[k] for k in sorted(got))]

    want = run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(3):
        graph.replay()
        for st in streams:
            with torch.cuda.stream(st):
                got.append(run())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for x in (captured, *got) for a, b in zip(x, want))
    ops.check_device_error()


def test_first_call_may_be_captured():
    """A process whose first use of the library is inside a captured graph (its error word is made there)."""
    out = subprocess.run([sys.executable, "-c", FIRST_CALL_CAPTURED, str(ROOT)], capture_output=True, text=True, timeout=300)
    assert out.returncode == 0 and "captured" in out.stdout, out.stderr[-2000:]


def test_on_other_streams_at_once():
    states = [training_state(s) for s in range(4)]
    want = [[t.clone() for t in training_ops(s)] for s in states]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in states]
    got = [None] * len(states)
    for _ in range(5):
        for i, (st, s) in enumerate(zip(streams, states)):
            with torch.cuda.stream(st):
                got[i] = training_ops(s)
    torch.cuda.synchronize()
    for x, ref in zip(got, want):
        assert all(torch.equal(a, b) for a, b in zip(x, ref))


# ============================================================================ a run of them together
class NormedLM(torch.nn.Module):
    """Embedding, blocks of capture linears joined by residual norms, head: a model as this package's layers build it."""

    def __init__(self, vocab=300, d=64, hidden=128, blocks=2, kind="rms"):
        super().__init__()
        torch.manual_seed(5)
        self.vocab = vocab
        self.embed = ScaledEmbedding(vocab, d, padding_idx=0, scale=d ** 0.5)
        with torch.no_grad():
            self.embed.weight.mul_(d ** -0.5)
        self.fc1 = torch.nn.ModuleList([GCLinear(d, hidden, bias=False) for _ in range(blocks)])
        self.fc2 = torch.nn.ModuleList([GCLinear(hidden, d, bias=False) for _ in range(blocks)])
        self.first = ResidualNorm(d, kind=kind)
        self.joints = torch.nn.ModuleList([ResidualNorm(d, kind=kind, post=True, gate=True) for _ in range(blocks)])
        self.lm_head = torch.nn.Linear(d, vocab, bias=False)

    def forward(self, input_seq, target_seq=None, sliding_window_num_blocks=None):
        if input_seq.ndim == 1:
            input_seq = input_seq[None]
        n, h = self.first(self.embed(input_seq))
        for fc1, fc2, joint in zip(self.fc1, self.fc2, self.joints):
            n, h = joint(h, fc2(torch.nn.functional.gelu(fc1(n))))
        logits = self.lm_head(n)
        if target_seq is not None:
            return torch.nn.functional.cross_entropy(logits.float().view(-1, self.vocab), target_seq.reshape(-1))
        return logits


def plain_logits(model, tokens, params):
    """NormedLM's forward in plain float64 torch, from a dict of its parameters."""
    def norm(v, w, layer):
        v = v - v.mean(-1, keepdim=True) if layer else v
        return v / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-6) * w

    layer = model.first.kind == "layer"
    e = params["embed.weight"]
    h = e[tokens] * float(np.float32(model.embed.scale))
    n = norm(h, params["first.weight"], layer)
    for i in range(len(model.fc1)):
        y = torch.nn.functional.gelu(n @ params[f"fc1.{i}.weight"].T) @ params[f"fc2.{i}.weight"].T
        h = h + params[f"joints.{i}.gate"] * norm(y, params[f"joints.{i}.post_weight"], layer)
        n = norm(h, params[f"joints.{i}.weight"], layer)
    return n @ params["lm_head.weight"].T


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_training_step_of_the_layers(kind):
    """Forward, backward and clip of a whole model against the same in float64.

    The f32 products of torch's linears (f32 sums of up to 128 terms through
    six matrices) dominate: 1e-4 of a gradient's largest value covers them.
    """
    model = NormedLM(kind=kind).to(DEV)
    tokens = torch.randint(1, 300, (6, 33), device=DEV, generator=gen(1))
    tokens[4:, 20:] = 0  # padded rows
    loss = model(tokens[:, :-1], tokens[:, 1:])
    loss.backward()
    params = {k: p.detach().double().requires_grad_() for k, p in model.named_parameters()}
    ref = torch.nn.functional.cross_entropy(plain_logits(model, tokens[:, :-1], params).view(-1, 300), tokens[:, 1:].reshape(-1))
    grads = dict(zip(params, torch.autograd.grad(ref, list(params.values()))))
    grads["embed.weight"][0] = 0.0  # the padding row
    assert abs(float(loss.detach()) - float(ref.detach())) < 1e-4 * float(ref.detach())
    for k, p in model.named_parameters():
        assert float((p.grad.double() - grads[k]).abs().max()) <= 1e-4 * float(grads[k].abs().max()), k
    before = {k: p.grad.clone() for k, p in model.named_parameters()}
    norm = clip_grad_norm_(model.parameters(), 0.05)
    want = norm64(before.values())
    assert abs(float(norm) - want) <= NORM_TOL * want
    c = coefficient(float(norm), 0.05)
    assert float(c) < 1 and all(torch.equal(p.grad, before[k] * c) for k, p in model.named_parameters())
    torch.optim.AdamW(model.parameters(), lr=1e-3).step()
    ops.check_device_error()


def test_selection_round_over_the_layers():
    """A selection round on a model of these layers: capture sees through them, and picks a subset."""
    model = NormedLM(vocab=256).to(DEV)
    opt = torch.optim.AdamW(model.parameters(), lr=6e-4, betas=(0.9, 0.95))
    g = gen(3)
    buf = torch.randint(1, 256, (8, 128), device=DEV, generator=g)
    model(buf[:, :-1], buf[:, 1:]).backward()
    clip_grad_norm_(model.parameters(), 1.0)
    opt.step()
    opt.zero_grad()
    prox = torch.randint(1, 256, (4, 128), device=DEV, generator=g)
    loader = ProxyLoader({"input_ids": prox, "attention_mask": torch.ones_like(prox), "labels": prox.clone()})
    initialize_projector(sketch_dim=1024, seed=42, device=DEV)
    layers = find_GClayers(model)
    scores, sim = get_batch_opus(model, buf, buf.clone(), None, None, opt, layers, loader, 0.25, 128, score_len=128,
                                 return_scores_only=True)
    assert bool(torch.isfinite(scores).all()) and bool((sim.diagonal() > 0).all())
    picks = get_batch_opus(model, buf, buf.clone(), None, None, opt, layers, loader, 0.25, 128, score_len=128,
                           selection_method="greedy")
    assert len(set(picks.tolist())) == 2


def test_layers_backward_captured():
    """A whole training step of the layers in a captured graph, replayed, against the eager one."""
    model = NormedLM().to(DEV)
    tokens = torch.randint(1, 300, (4, 17), device=DEV, generator=gen(9))
    names = [k for k, _ in model.named_parameters()]
    params = list(model.parameters())

    def step():
        loss = model(tokens[:, :-1], tokens[:, 1:])
        grads = list(torch.autograd.grad(loss, params))
        return grads, ops.clip_grads(grads, 0.05)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            want, norm = step()
    torch.cuda.current_stream().wait_stream(side)
    want, norm = [w.clone() for w in want], norm.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got, got_norm = step()
    graph.replay()
    torch.cuda.synchronize()
    # torch's own products may take other kernels under capture: compare to their rounding (as above)
    assert abs(float(got_norm) - float(norm)) <= 1e-4 * float(norm)
    for k, x, y in zip(names, got, want):
        assert float((x - y).abs().max()) <= 1e-4 * float(y.abs().max()), k
