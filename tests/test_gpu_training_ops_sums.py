"""Sums over many rows and tokens of the training-step operators, on values whose sums are exact in f32 (GPU).

Terms are whole numbers, and every partial sum stays below 2^24: whatever the
order, the only rounding is that of the result to its type, so outputs have to
be equal to the formula's in 64 bits, rounded once.  A lost or repeated row, run
or slice shows however long the sum is.  Outputs lie in memory that was filled
with NaN, between guards.
"""
import pytest
import torch

from opus_b200 import ops
from test_gpu_training_ops import U, check_norm, gen, half_step, norm_case, stats64, wide_mag, within

pytestmark = pytest.mark.gpu
DEV = "cuda"


def whole(g, *shape, most, dtype=torch.float32):
    """Whole numbers of [-most, most]."""
    return torch.randint(-most, most + 1, shape, device=DEV, generator=g).to(dtype)


def rounded(v, dtype):
    """v (exact in f32) in a type, rounded once."""
    assert bool((v.float().double() == v).all())
    return v.float().to(dtype)


# ============================================================================ embedding
class Guarded:
    """[V, d] of a type at an offset in elements of a larger buffer, filled with NaN, and the memory around it."""

    def __init__(self, V, d, dtype, offset):
        self.buf = torch.full((V * d + 64,), 77.0, dtype=dtype, device=DEV)
        self.start, self.end = 16 + offset, 16 + offset + V * d
        self.table = self.buf[self.start:self.end].view(V, d)
        self.table.fill_(float("nan"))

    def check(self):
        assert bool((self.buf[: self.start] == 77).all()) and bool((self.buf[self.end:] == 77).all())


def exact_grad(dy, t, V, padding=None):
    keep = t != padding if padding is not None else torch.ones_like(t, dtype=torch.bool)
    return torch.zeros(V, dy.shape[1], dtype=torch.float64, device=DEV).index_add_(0, t[keep], dy[keep].double())


# short lists (one launch); the cluster's sort, up to 188416; the sort through global memory
SIZES = [(1, 9, 8), (300, 70, 40), (2048, 700, 31), (2048, 3, 64), (2049, 50304, 8), (40000, 3, 24), (100000, 7, 8),
         (188416, 2, 8), (188417, 50304, 8), (300000, 3, 8), (700000, 1, 16), (1200000, 5, 4)]


@pytest.mark.parametrize("dtype,out_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                             (torch.bfloat16, torch.float32), (torch.float16, torch.float32)])
@pytest.mark.parametrize("n,V,d", SIZES)
def test_embedding_grad_sums_are_exact(n, V, d, dtype, out_dtype):
    """Runs of up to all positions: 700000 terms of at most 8 stay below 2^24, and so do 1.2 million of five tokens."""
    g = gen(n + V)
    hot = torch.rand(n, device=DEV, generator=g) < 0.5  # half of the positions on one token
    t = torch.where(hot, torch.zeros(n, dtype=torch.int64, device=DEV), torch.randint(0, V, (n,), device=DEV, generator=g))
    dy = whole(g, n, d, most=8, dtype=dtype) + 1  # a mean of one: the long sums are far from zero
    want = exact_grad(dy, t, V)
    assert float(want.abs().max()) < 2 ** 24 and (n < 10000 or float(want[0].abs().min()) > n / 4)
    assert n < 188418 or V > 10 or n / 2 / 32 > 1024  # runs of more units than one turn of the join counts
    for offset in (0, 1, 4):
        out = Guarded(V, d, out_dtype, offset)
        ops.embedding_grad(dy, t, V, out=out.table)
        assert torch.equal(out.table, rounded(want, out_dtype))
        out.check()
    out = Guarded(V, d, out_dtype, 0)
    ops.embedding_grad(dy, t.int(), V, out=out.table, padding_idx=0)
    assert torch.equal(out.table, rounded(exact_grad(dy, t, V, 0), out_dtype)) and not bool(out.table[0].any())
    out.check()
    if out_dtype == torch.float32:  # into what is there: rows that no token names keep it, NaN and all
        out = Guarded(V, d, out_dtype, 3)
        named = torch.zeros(V, dtype=torch.bool, device=DEV).index_fill_(0, t, True)
        out.table[named] = 5.0
        ops.embedding_grad(dy, t, V, out=out.table, accumulate=True, scale=2.0)
        assert torch.equal(out.table[named], rounded(2 * want + 5, out_dtype)[named])
        assert bool(out.table[~named].isnan().all())
        out.check()


@pytest.mark.parametrize("n,V,d,dtype", [(1, 3, 5, torch.bfloat16), (20, 40001, 7, torch.float32), (500, 3001, 3, torch.bfloat16),
                                         (5000, 40001, 7, torch.bfloat16), (5000, 30001, 5, torch.float32),
                                         (190000, 40001, 3, torch.float32), (190000, 30001, 5, torch.bfloat16)])
def test_embedding_grad_zeroes_every_row_that_no_token_names(n, V, d, dtype):
    """Tables whose bytes are no multiple of 16, from every offset of an element in 16 bytes, and nothing beside them."""
    g = gen(n)
    t = torch.randint(0, V // 2, (n,), device=DEV, generator=g) * 2  # even rows at most
    dy = whole(g, n, d, most=3, dtype=dtype)
    want = rounded(exact_grad(dy, t, V), dtype)
    for offset in range(16 // dtype.itemsize):
        out = Guarded(V, d, dtype, offset)
        ops.embedding_grad(dy, t, V, out=out.table)
        assert torch.equal(out.table, want)
        out.check()


def test_embedding_grad_of_no_tokens_zeroes_the_table():
    out = Guarded(50, 3, torch.bfloat16, 1)
    ops.embedding_grad(torch.empty(0, 3, dtype=torch.bfloat16, device=DEV), torch.empty(0, dtype=torch.int64, device=DEV), 50,
                       out=out.table)
    assert not bool(out.table.any())
    out.check()


# ============================================================================ residual norm
@pytest.mark.parametrize("gate", [None, "channel", "sample"])
@pytest.mark.parametrize("kind,bias", [("rms", False), ("rms", True), ("layer", False), ("layer", True)])
@pytest.mark.parametrize("d", [512, 516, 764, 768, 896, 1024, 1532, 1600, 1792, 2044, 2048, 2560, 3712, 4096, 4100])
def test_residual_norm_where_a_gate_is_kept_apart(d, kind, bias, gate):
    """f32 rows on both sides of the rule that folds a gate into the norm's weight, and more rows than run at once."""
    for dtype, x_dtype in ((torch.float32, None), (torch.bfloat16, None), (torch.bfloat16, torch.float32),
                           (torch.float16, torch.float32)):
        check_norm(*norm_case(d, (3, 5), d, dtype, x_dtype, post=True, gate=gate, bias=bias), kind=kind, post=True, r=0.5)
    c, p, _, _ = norm_case(d, (4, 500), d, post=True, gate=gate, bias=bias)
    n, h, stats = ops.residual_norm(c["x"], c["y"], **p, kind=kind)
    for rows in (slice(0, 3), slice(497, 500)):  # a row's values do not depend on the rows beside it
        part = ops.residual_norm(c["x"][:, rows], c["y"][:, rows], **p, kind=kind)
        assert torch.equal(part[0], n[:, rows]) and torch.equal(part[1], h[:, rows])


# ---------------------------------------------------------------------------- backward
EXACT = [((140000, 1), 8), ((70000,), 24), ((8, 16384), 64), ((1, 100000), 136), ((3, 8192), 1600), ((20, 700), 771),
         ((4, 4096), 4096), ((50, 60), 8192), ((7, 300), 5001), ((2, 600), 16384)]


@pytest.mark.parametrize("kind,post,bias", [("rms", False, False), ("rms", True, False), ("layer", True, True)])
@pytest.mark.parametrize("gate", [None, "channel", "sample"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape,d", EXACT)
def test_residual_norm_sums_are_exact(shape, d, dtype, gate, kind, post, bias):
    """Rows whose normed values are +1 and -1 under the statistics given: every column's sum is one of whole numbers.

    First the gradients through the norm (weight, bias) with no gradient of h;
    then those behind it (gate, post_weight, post_bias), with a gradient of h
    alone.  dx and dy of the second are whole numbers too, but for the mean over
    a row, which is exact where d is a power of two.
    """
    g = gen(d + shape[0])
    layer = kind == "layer"
    sign = torch.randint(0, 2, (*shape, d), device=DEV, generator=g) * 2.0 - 1.0
    ysign = torch.randint(0, 2, (*shape, d), device=DEV, generator=g) * 2.0 - 1.0
    h = (0.5 * sign + (3.0 if layer else 0.0)).to(dtype)
    y = (2.0 * ysign + (1.0 if layer else 0.0)).to(dtype)
    rows = h.numel() // d
    stats = torch.tensor([3.0 if layer else 0.0, 2.0, 1.0 if layer else 0.0, 0.5], device=DEV).repeat(rows, 1)
    p = {"weight": whole(g, d, most=2)}
    if bias:
        p["bias"] = whole(g, d, most=2)
    if post:
        p["post_weight"] = whole(g, d, most=2)
        if bias:
            p["post_bias"] = whole(g, d, most=2)
    if gate:
        p["gate"] = whole(g, *((shape[0], *[1] * (len(shape) - 1)) if gate == "sample" else ()), d, most=2)
    kw = dict(p, kind=kind, post=post, residual_scale=-2.0)
    lead = tuple(range(len(shape)))
    hat, z = sign.double(), y.double()

    dn = whole(g, *shape, d, most=4, dtype=dtype) + 1
    got = ops.residual_norm_grad(dn, None, h, stats, y, **kw)
    assert torch.equal(got["weight"], rounded((dn.double() * hat).sum(lead), torch.float32))
    if bias:
        assert torch.equal(got["bias"], rounded(dn.double().sum(lead), torch.float32))
    # the whole of dh by the formula; d a power of two: every step is exact in f32 (whole numbers over d)
    if d & (d - 1) == 0 and dtype == torch.float32:
        a = dn.double() * p["weight"].double()
        dh = 2.0 * (a - hat * (a * hat).mean(-1, keepdim=True) - (a.mean(-1, keepdim=True) if layer else 0.0))
        assert torch.equal(got["x"], rounded(-2.0 * dh, dtype))

    dh = whole(g, *shape, d, most=3, dtype=dtype) + 1
    got = ops.residual_norm_grad(None, dh, h, stats, y, **kw)
    assert torch.equal(got["x"], rounded(-2.0 * dh.double(), dtype))
    assert not bool(got["weight"].any())
    g64 = p["gate"].double() if gate else torch.ones((), dtype=torch.float64, device=DEV)
    dz = g64 * dh.double()
    if post:
        yh = ysign.double()
        z = yh * p["post_weight"].double() + (p["post_bias"].double() if bias else 0.0)
        assert torch.equal(got["post_weight"], rounded((dz * yh).sum(lead), torch.float32))
        if bias:
            assert torch.equal(got["post_bias"], rounded(dz.sum(lead), torch.float32))
        if d & (d - 1) == 0:
            c = dz * p["post_weight"].double()
            dy = 0.5 * (c - yh * (c * yh).mean(-1, keepdim=True) - (c.mean(-1, keepdim=True) if layer else 0.0))
            assert torch.equal(got["y"], rounded(dy, dtype))
    else:
        assert torch.equal(got["y"], rounded(dz, dtype))
    if gate == "channel":
        assert torch.equal(got["gate"], rounded((dh.double() * z).sum(lead), torch.float32))
    elif gate == "sample":
        want = dh.double() * z
        want = want.sum(tuple(range(1, len(shape))), keepdim=True) if len(shape) > 1 else want
        assert torch.equal(got["gate"], rounded(want.reshape(p["gate"].shape), torch.float32))


@pytest.mark.parametrize("kind", ["rms", "layer"])
def test_residual_norm_sums_over_many_rows(kind):
    """Ordinary values over 100000 rows, bounded by the chain that the sums really have.

    K = 768 for a row's own arithmetic (four sums over the row behind one
    another) and, for the columns, a worker's rows (a 148th of them at most),
    the groups of a block (384 at most), 24 for the join of at most 592 blocks in
    32 slices.  The values have means, so that the sums are far larger than
    their bounds: asserted, so that no bound passes anything.
    """
    rows, d = 100_000, 64
    c, p, dn, dh = norm_case(9, (rows,), d, post=True, gate="channel", bias=True)
    ramp = torch.linspace(-3.0, 3.0, d, device=DEV)  # columns' means
    x, y, dn, dh = c["x"] + ramp, c["y"] + ramp.flip(0), dn + 1.0, dh + 1.0
    n, h, stats = ops.residual_norm(x, y, **p, kind=kind, post=True, eps=1e-5)
    got = ops.residual_norm_grad(dn, dh, h, stats, y, **p, kind=kind, post=True)
    K = 768 + (rows + 147) // 148 + 384 + 24
    w, pw, pb, gate = (p[k].double() for k in ("weight", "post_weight", "post_bias", "gate"))
    hm, hr = stats64(h.double(), kind, 1e-5)
    hat, hw = (h.double() - hm) * hr, wide_mag(h.double(), kind) * hr
    ym, yr = stats64(y.double(), kind, 1e-5)
    yh, yw = (y.double() - ym) * yr, wide_mag(y.double(), kind) * yr
    a, am = dn.double() * w, (dn.double() * w).abs()
    v, m = a - hat * (a * hat).mean(-1, keepdim=True), am + hw * (am * hw).mean(-1, keepdim=True)
    if kind == "layer":
        v, m = v - a.mean(-1, keepdim=True), m + am.mean(-1, keepdim=True)
    v, m = v * hr + dh.double(), m * hr + dh.double().abs()
    for name, terms, mags in (("weight", dn.double() * hat, dn.double().abs() * hw), ("bias", dn.double(), dn.double().abs()),
                              ("gate", v * (yh * pw + pb), m * (yw * pw.abs() + pb.abs())),
                              ("post_weight", gate * v * yh, gate.abs() * m * yw), ("post_bias", gate * v, gate.abs() * m)):
        ref, bound = terms.sum(0), half_step(torch.float32) * terms.sum(0).abs() + K * U * mags.sum(0)
        within(got[name], ref, bound, name)
        spread = float(ref.square().mean().sqrt())
        assert float(bound.square().mean().sqrt()) < 0.01 * spread, (name, float(bound.max()), spread)
    # of a row: no sum over rows is behind it
    within(got["x"], v, half_step(torch.float32) * v.abs() + 768 * U * m, "x")
