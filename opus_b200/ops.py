"""Torch-tensor front end of the C ABI (include/opus_b200.h).

Every function here takes CUDA tensors, launches on the current CUDA stream of
the tensors' device and returns CUDA tensors.  There is no CPU path: a CPU
tensor or a missing libopus_b200.so raises.
"""
from __future__ import annotations

import ctypes
import math
from collections.abc import Iterable, Sequence

import torch

from . import _lib

_ERR_BAD_PROBS = 0x301
_ERR_BAD_TOKEN = 0x202

_devices: set[int] = set()  # that training-step operators ran on


def _stream(t: torch.Tensor) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(t.device).cuda_stream)


def _ptr(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(0 if t is None else t.data_ptr())


def _cuda(t: torch.Tensor, name: str) -> torch.Tensor:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (the OPUS B200 path runs on the GPU only)")
    return t


def _contig(t: torch.Tensor) -> torch.Tensor:
    return t if t.is_contiguous() else t.contiguous()


def check_device_error(what: str = "opus kernel", tokens: bool = True) -> None:
    """Synchronise and raise if a kernel recorded a device-side error.

    Looks at the current device, and at those that training-step operators
    ran on.  tokens=False looks past tokens outside an embedding's rows, which stay
    recorded: the selection path checks its own kernels that way, behind
    those of the model that it scores.
    """
    code = _lib.device_error(tokens)
    if not code and _devices - {torch.cuda.current_device()}:
        for index in sorted(_devices):
            with torch.cuda.device(index):
                code = _lib.device_error(tokens)
            if code:
                break  # the others keep theirs for the next check
    if code == _ERR_BAD_PROBS:
        raise ValueError(f"{what}: probabilities do not sum to 1")
    if code == _ERR_BAD_TOKEN:
        raise IndexError(f"{what}: token outside the embedding's rows")
    if code:
        raise RuntimeError(f"{what}: device error 0x{code:x}")


# --------------------------------------------------------------------- tables
def pack_hash_sign(hash_: torch.Tensor, sign: torch.Tensor, k: int, validate: bool = True) -> torch.Tensor:
    """int64 buckets + float32 +-1 signs -> uint32 (stored as int32) packed table."""
    _cuda(hash_, "hash")
    _cuda(sign, "sign")
    if hash_.dtype != torch.int64 or sign.dtype != torch.float32:
        raise ValueError("hash must be int64 and sign float32")
    if hash_.numel() != sign.numel():
        raise ValueError("hash and sign must have the same number of elements")
    h, s = _contig(hash_.reshape(-1)), _contig(sign.reshape(-1))
    out = torch.empty(h.numel(), dtype=torch.int32, device=h.device)
    _lib.check(_lib.load().opus_pack_hash_sign(_ptr(h), _ptr(s), h.numel(), int(k), _ptr(out), _stream(h)),
               "opus_pack_hash_sign")
    if validate:
        check_device_error("opus_pack_hash_sign (bucket outside [0,k) or sign not +-1)", tokens=False)
    return out


def bucket_counts(packed: torch.Tensor, k: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Per-bucket element counts [k] int32 and their max [1] int64, on the device."""
    _cuda(packed, "packed")
    packed = _contig(packed.reshape(-1))
    if packed.dtype not in (torch.int32, torch.uint32):
        raise ValueError("packed table must be 32-bit")
    counts = torch.empty(int(k), dtype=torch.int32, device=packed.device)
    out = torch.empty(1, dtype=torch.int64, device=packed.device)
    _lib.check(_lib.load().opus_bucket_max_load(_ptr(packed), packed.numel(), int(k), _ptr(counts), counts.numel(),
                                               _ptr(out), _stream(packed)), "opus_bucket_max_load")
    return counts, out


def bucket_max_load(packed: torch.Tensor, k: int) -> int:
    """Largest number of elements sharing one bucket (bounds the fixed-point sketch)."""
    return int(bucket_counts(packed, k)[1].item())


def sketch_table_entries(d_out: int, d_in: int) -> int:
    return int(_lib.load().opus_sketch_table_entries(int(d_out), int(d_in)))


def build_sketch_table(packed: torch.Tensor, d_out: int, d_in: int, diag: torch.Tensor | None = None,
                       exp_avg_sq: torch.Tensor | None = None, eps: float = 1e-8,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """Tiled (bucket, sign*D) epilogue table for sketch_gemm; 16 bytes per entry."""
    _cuda(packed, "packed")
    n = sketch_table_entries(d_out, d_in)
    if packed.numel() != d_out * d_in:
        raise ValueError(f"packed table has {packed.numel()} elements, layer has {d_out * d_in}")
    for name, t in (("diag", diag), ("exp_avg_sq", exp_avg_sq)):
        if t is not None:
            _cuda(t, name)
            if t.numel() != d_out * d_in:
                raise ValueError(f"{name} has {t.numel()} elements, layer has {d_out * d_in}")
    diag = None if diag is None else _contig(diag.to(torch.float32))
    exp_avg_sq = None if exp_avg_sq is None else _contig(exp_avg_sq.to(torch.float32))
    if out is None or out.numel() * out.element_size() < n * 16:
        out = torch.empty(n * 4, dtype=torch.int32, device=packed.device)
    _lib.check(_lib.load().opus_build_sketch_table(_ptr(packed), _ptr(diag), _ptr(exp_avg_sq), float(eps), int(d_out),
                                                  int(d_in), _ptr(out), n, _stream(packed)),
               "opus_build_sketch_table")
    return out


def adam_diag(exp_avg_sq: torch.Tensor, eps: float = 1e-8) -> torch.Tensor:
    """The AdamW diagonal 1 / (sqrt(v) + eps) in f32, elementwise, same shape as v."""
    _cuda(exp_avg_sq, "exp_avg_sq")
    v = _contig(exp_avg_sq.to(torch.float32))
    out = torch.empty_like(v)
    _lib.check(_lib.load().opus_adam_diag(_ptr(v), float(eps), v.numel(), _ptr(out), _stream(v)), "opus_adam_diag")
    return out


# --------------------------------------------------------------------- stage 3
def split_bf16(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    _cuda(x, "x")
    x = _contig(x.to(torch.float32))
    hi = torch.empty(x.shape, dtype=torch.bfloat16, device=x.device)
    lo = torch.empty_like(hi)
    _lib.check(_lib.load().opus_split_bf16(_ptr(x), x.numel(), _ptr(hi), _ptr(lo), _stream(x)), "opus_split_bf16")
    return hi, lo


def _as3d(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() == 2:
        return t.unsqueeze(0)
    if t.dim() != 3:
        raise ValueError(f"Unexpected {name} shape: {tuple(t.shape)}")
    return t


# Longest row (in tokens) that sketch_gemm forms by merging samples that share an output row.
MERGE_TOKENS = 16384


def sketch_gemm(dLdZ: torch.Tensor, a: torch.Tensor, table: torch.Tensor, k: int, rows_div: int = 1,
                out: torch.Tensor | None = None, accumulate: bool = False,
                max_bucket_load: int = 0, alpha: float = 1.0) -> torch.Tensor:
    """phi[b // rows_div] (+)= alpha * CountSketch(w o (dLdZ_b^T a_b)) for every candidate b.

    dLdZ [B, T, d_out] and a [B, T, d_in] in bf16 (tensor cores directly) or
    f32 (split into bf16 hi/lo; hi*hi + hi*lo + lo*hi accumulated).
    max_bucket_load (see bucket_max_load) enables the fixed-point
    shared-memory sketch; 0 adds every update with f32 global atomics.
    alpha multiplies every update in f32 (the per-sample scaling of dL/dZ).
    """
    _cuda(dLdZ, "dLdZ")
    _cuda(a, "a")
    if dLdZ.dim() != 3 or a.dim() != 3 or dLdZ.shape[:2] != a.shape[:2]:
        raise ValueError(f"Unexpected dLdZ/a shapes: {tuple(dLdZ.shape)}, {tuple(a.shape)}")
    B, T, d_out = dLdZ.shape
    d_in = a.shape[2]
    rows = 0 if B == 0 else (B + rows_div - 1) // rows_div
    # The sketch is linear, and the G of a row of r*T tokens is the sum of its
    # r rows' G: samples that share an output row are merged into one long row
    # (a view), which scatters into the sketch once instead of r times.  The
    # merged row is kept to MERGE_TOKENS tokens: its G is one f32 accumulation
    # over all of them, whose rounding error grows with the length.
    g = math.gcd(rows_div, B)
    r = max([d for d in range(1, g + 1) if g % d == 0 and d * T <= MERGE_TOKENS] or [1])
    if r > 1:
        dLdZ = _contig(dLdZ).view(B // r, r * T, d_out)
        a = _contig(a).view(B // r, r * T, d_in)
        B, T, rows_div = B // r, r * T, rows_div // r
    if out is None:
        out = torch.empty(rows, k, dtype=torch.float32, device=dLdZ.device)
        accumulate = False
    if out.dtype != torch.float32 or not out.is_contiguous() or out.numel() < rows * k:
        raise ValueError("out must be a contiguous float32 tensor of at least [rows, k]")
    n_entries = table.numel() * table.element_size() // 16
    lib = _lib.load()

    def launch(g: torch.Tensor, x: torch.Tensor, acc: bool) -> None:
        _lib.check(lib.opus_sketch_gemm(_ptr(g), _ptr(x), _lib.DTYPE_BF16, B, T, d_out, d_in, _ptr(table), n_entries,
                                        int(k), int(max_bucket_load), int(rows_div), _ptr(out), int(acc),
                                        float(alpha), _stream(g)),
                   "opus_sketch_gemm")

    if dLdZ.dtype == torch.bfloat16 and a.dtype == torch.bfloat16:
        launch(_contig(dLdZ), _contig(a), accumulate)
    else:
        g_hi, g_lo = split_bf16(dLdZ)
        a_hi, a_lo = split_bf16(a)
        launch(g_hi, a_hi, accumulate)
        launch(g_hi, a_lo, True)
        launch(g_lo, a_hi, True)
    return out


def ghost_gram(a: torch.Tensor, dLdZ: torch.Tensor, alpha: float = 1.0, out: torch.Tensor | None = None,
               accumulate: bool = False) -> torch.Tensor:
    """S[i, j] (+)= alpha * <G_i, G_j>, G_b = dLdZ_b^T a_b, for every candidate pair, without forming any G_b.

    a [B, T, d_in], dLdZ [B, T, d_out] in bf16 (tensor cores directly) or f32
    (split into bf16 hi/lo; hi*hi + hi*lo + lo*hi per product).  Widths that
    are not multiples of 8 are zero-padded (zero features add nothing).
    """
    _cuda(a, "a")
    _cuda(dLdZ, "dLdZ")
    if dLdZ.dim() != 3 or a.dim() != 3 or dLdZ.shape[:2] != a.shape[:2]:
        raise ValueError(f"Unexpected dLdZ/a shapes: {tuple(dLdZ.shape)}, {tuple(a.shape)}")
    B, T, d_out = dLdZ.shape
    d_in = a.shape[2]
    if out is None:
        out = torch.empty(B, B, dtype=torch.float32, device=a.device)
        accumulate = False
    if out.dtype != torch.float32 or not out.is_contiguous() or out.numel() < B * B:
        raise ValueError("out must be a contiguous float32 tensor of at least [B, B]")
    a, dLdZ = _pad8(a), _pad8(dLdZ)
    lib = _lib.load()
    if a.dtype == torch.bfloat16 and dLdZ.dtype == torch.bfloat16:
        parts = (_contig(a), None, _contig(dLdZ), None)
    else:
        a_hi, a_lo = split_bf16(a)
        g_hi, g_lo = split_bf16(dLdZ)
        parts = (a_hi, a_lo, g_hi, g_lo)
    _lib.check(lib.opus_ghost_gram(_ptr(parts[0]), _ptr(parts[1]), _ptr(parts[2]), _ptr(parts[3]), _lib.DTYPE_BF16,
                                   B, T, a.shape[2], dLdZ.shape[2], float(alpha), _ptr(out), int(accumulate),
                                   _stream(a)), "opus_ghost_gram")
    return out


def _pad8(x: torch.Tensor) -> torch.Tensor:
    d = x.shape[-1]
    p = (d + 7) // 8 * 8
    return x if p == d else torch.nn.functional.pad(x, (0, p - d))


def per_sample_grad(dLdZ: torch.Tensor, a: torch.Tensor, diag: torch.Tensor | None = None,
                    out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """out[b] (+)= (diag o dLdZ_b^T a_b) flattened: exact per-sample gradients [B, d_out*d_in] in f32.

    dLdZ [B, T, d_out] and a [B, T, d_in] in bf16 (tensor cores directly) or
    f32 (split into bf16 hi/lo; hi*hi + hi*lo + lo*hi accumulated).  Widths
    that are not multiples of 8 are zero-padded for the kernel and the result
    is cut back to [B, d_out*d_in].
    """
    _cuda(dLdZ, "dLdZ")
    _cuda(a, "a")
    if dLdZ.dim() != 3 or a.dim() != 3 or dLdZ.shape[:2] != a.shape[:2]:
        raise ValueError(f"Unexpected dLdZ/a shapes: {tuple(dLdZ.shape)}, {tuple(a.shape)}")
    B, T, d_out = dLdZ.shape
    d_in = a.shape[2]
    if diag is not None:
        if tuple(diag.shape) != (d_out, d_in):
            raise ValueError(f"diag must be [{d_out}, {d_in}], got {tuple(diag.shape)}")
        diag = _contig(_cuda(diag, "diag").to(torch.float32))
    if out is None:
        out = torch.empty(B, d_out * d_in, dtype=torch.float32, device=dLdZ.device)
        accumulate = False
    if out.dtype != torch.float32 or not out.is_contiguous() or out.numel() < B * d_out * d_in:
        raise ValueError("out must be a contiguous float32 tensor of at least [B, d_out * d_in]")
    do_p, di_p = (d_out + 7) // 8 * 8, (d_in + 7) // 8 * 8
    padded = (do_p, di_p) != (d_out, d_in)
    if padded:
        dLdZ = torch.nn.functional.pad(dLdZ, (0, do_p - d_out))
        a = torch.nn.functional.pad(a, (0, di_p - d_in))
        if diag is not None:
            diag = torch.nn.functional.pad(diag, (0, di_p - d_in, 0, do_p - d_out))
        target = torch.empty(B, do_p * di_p, dtype=torch.float32, device=dLdZ.device)
    else:
        target = out
    lib = _lib.load()

    def launch(g: torch.Tensor, x: torch.Tensor, acc: bool) -> None:
        _lib.check(lib.opus_per_sample_grad(_ptr(g), _ptr(x), _lib.DTYPE_BF16, B, T, do_p, di_p, _ptr(diag),
                                            _ptr(target), int(acc), _stream(g)), "opus_per_sample_grad")

    first_acc = accumulate and not padded
    if dLdZ.dtype == torch.bfloat16 and a.dtype == torch.bfloat16:
        launch(_contig(dLdZ), _contig(a), first_acc)
    else:
        g_hi, g_lo = split_bf16(dLdZ)
        a_hi, a_lo = split_bf16(a)
        launch(g_hi, a_hi, first_acc)
        launch(g_hi, a_lo, True)
        launch(g_lo, a_hi, True)
    if padded:
        view = target.view(B, do_p, di_p)[:, :d_out, :d_in].reshape(B, d_out * d_in)
        dst = out.view(-1)[:B * d_out * d_in].view(B, d_out * d_in)
        if accumulate:
            dst += view
        else:
            dst.copy_(view)
    return out


def sketch_dense(w: torch.Tensor, packed: torch.Tensor, d_out: int, d_in: int, k: int, transposed: bool = False,
                 diag: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 accumulate: bool = False, rows: tuple[int, int] | None = None,
                 max_bucket_load: int = 0) -> torch.Tensor:
    """sketch[h] += s * diag * W for a dense [d_out, d_in] (or [d_in, d_out] if transposed) matrix.

    rows=(lo, hi) adds only the rows lo <= o < hi of the [d_out, d_in] layout.
    max_bucket_load (bucket_max_load of the table) tightens the fixed-point
    scale of the shared-memory sketch; 0 falls back to the element count.
    """
    _cuda(w, "w")
    _cuda(packed, "packed")
    if w.numel() != d_out * d_in:
        raise ValueError(f"w has {w.numel()} elements, expected {d_out * d_in}")
    w = _contig(w.to(torch.float32))
    diag = None if diag is None else _contig(diag.to(torch.float32))
    lo, hi = (0, d_out) if rows is None else (int(rows[0]), int(rows[1]))
    if out is None:
        out = torch.empty(k, dtype=torch.float32, device=w.device)
        accumulate = False
    _lib.check(_lib.load().opus_sketch_dense(_ptr(w), int(bool(transposed)), _ptr(packed), _ptr(diag), int(d_out),
                                            int(d_in), lo, hi, int(k), int(max_bucket_load), _ptr(out),
                                            int(accumulate), _stream(w)), "opus_sketch_dense")
    return out


def sketch_dense_rows(w: torch.Tensor, packed: torch.Tensor, k: int, out: torch.Tensor | None = None,
                      accumulate: bool = False, max_bucket_load: int = 0) -> torch.Tensor:
    """CountSketch of every row of a [n, numel] matrix with one table of numel elements, [n, k] f32."""
    _cuda(w, "w")
    _cuda(packed, "packed")
    if w.dim() != 2 or w.shape[1] != packed.numel():
        raise ValueError(f"w must be [n, {packed.numel()}], got {tuple(w.shape)}")
    w = _contig(w.to(torch.float32))
    n = w.shape[0]
    if out is None:
        out = torch.empty(n, k, dtype=torch.float32, device=w.device)
        accumulate = False
    if out.dtype != torch.float32 or not out.is_contiguous() or out.numel() < n * k:
        raise ValueError("out must be a contiguous float32 tensor of at least [n, k]")
    _lib.check(_lib.load().opus_sketch_dense_rows(_ptr(w), n, w.shape[1], _ptr(_contig(packed)), int(k),
                                                 int(max_bucket_load), _ptr(out), int(accumulate), _stream(w)),
               "opus_sketch_dense_rows")
    return out


# --------------------------------------------------------------------- stage 2
def desketch(tau: torch.Tensor, packed: torch.Tensor, d_out: int, d_in: int, scale: float = 1.0,
             diag: torch.Tensor | None = None, exp_avg_sq: torch.Tensor | None = None,
             eps: float = 1e-8) -> torch.Tensor:
    """Dense target v = scale * D * s * tau[h] as a bf16 (hi, lo) pair [2, d_out, d_in]."""
    _cuda(tau, "tau")
    tau = _contig(tau.to(torch.float32))
    diag = None if diag is None else _contig(diag.to(torch.float32))
    exp_avg_sq = None if exp_avg_sq is None else _contig(exp_avg_sq.to(torch.float32))
    out = torch.empty(2, d_out, d_in, dtype=torch.bfloat16, device=tau.device)
    _lib.check(_lib.load().opus_desketch(_ptr(tau), _ptr(packed), _ptr(diag), _ptr(exp_avg_sq), float(eps), int(d_out),
                                        int(d_in), tau.numel(), float(scale), _ptr(out), _stream(tau)),
               "opus_desketch")
    return out


def dense_target_pair(v: torch.Tensor) -> torch.Tensor:
    """f32 [d_out, d_in] target -> bf16 (hi, lo) pair [2, d_out, d_in] for ghost_score."""
    hi, lo = split_bf16(v)
    return torch.stack([hi, lo])


def ghost_score(a: torch.Tensor, dLdZ: torch.Tensor, v_pair: torch.Tensor, alpha: float = 1.0,
                out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """score[b] (+)= alpha * <dLdZ_b^T a_b, v> without forming per-sample gradients."""
    _cuda(a, "a")
    _cuda(dLdZ, "dLdZ")
    if a.dim() != 3 or dLdZ.dim() != 3 or a.shape[:2] != dLdZ.shape[:2]:
        raise ValueError(f"Unexpected a/dLdZ shapes: {tuple(a.shape)}, {tuple(dLdZ.shape)}")
    B, T, d_in = a.shape
    d_out = dLdZ.shape[2]
    if v_pair.shape != (2, d_out, d_in) or v_pair.dtype != torch.bfloat16:
        raise ValueError(f"v_pair must be bf16 [2, {d_out}, {d_in}], got {v_pair.dtype} {tuple(v_pair.shape)}")
    if out is None:
        out = torch.empty(B, dtype=torch.float32, device=a.device)
        accumulate = False
    lib = _lib.load()
    v_pair = _contig(v_pair)

    def launch(x: torch.Tensor, g: torch.Tensor, acc: bool) -> None:
        _lib.check(lib.opus_ghost_score(_ptr(x), _ptr(g), _lib.DTYPE_BF16, B, T, d_in, d_out, _ptr(v_pair),
                                        float(alpha), _ptr(out), int(acc), _stream(x)), "opus_ghost_score")

    if a.dtype == torch.bfloat16 and dLdZ.dtype == torch.bfloat16:
        launch(_contig(a), _contig(dLdZ), accumulate)
    else:
        a_hi, a_lo = split_bf16(a)
        g_hi, g_lo = split_bf16(dLdZ)
        launch(a_hi, g_hi, accumulate)
        launch(a_lo, g_hi, True)
        launch(a_hi, g_lo, True)
    return out


# --------------------------------------------------------------------- dots
def sketch_dot(phi: torch.Tensor, tau: torch.Tensor, alpha: float = 1.0, out: torch.Tensor | None = None,
               accumulate: bool = False) -> torch.Tensor:
    _cuda(phi, "phi")
    phi, tau = _contig(phi), _contig(tau)
    B, k = phi.shape
    if tau.numel() != k:
        raise ValueError("tau length must equal the sketch dimension")
    if out is None:
        out = torch.empty(B, dtype=torch.float32, device=phi.device)
        accumulate = False
    _lib.check(_lib.load().opus_sketch_dot(_ptr(phi), _ptr(tau), B, k, float(alpha), _ptr(out), int(accumulate),
                                          _stream(phi)), "opus_sketch_dot")
    return out


def sketch_dot_layers(phis: torch.Tensor, taus: torch.Tensor, alphas: torch.Tensor,
                      out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    """out[b] (+)= sum_l alphas[l] * phis[l, b] . taus[l], every layer in one launch.

    phis [L, B, k] (each layer's [B, k] block contiguous; the layer stride may be
    larger, as for rows [lo, hi) of a longer buffer), taus [L, k], alphas [L] f32.
    """
    _cuda(phis, "phis")
    if phis.dim() != 3 or phis.stride(2) != 1 or phis.stride(1) != phis.shape[2]:
        raise ValueError("phis must be [L, B, k] with contiguous [B, k] blocks")
    L, B, k = phis.shape
    taus = _contig(taus.to(torch.float32))
    alphas = _contig(alphas.to(device=phis.device, dtype=torch.float32))
    if taus.shape != (L, k) or alphas.numel() != L:
        raise ValueError(f"taus must be [{L}, {k}] and alphas [{L}]")
    if out is None:
        out = torch.empty(B, dtype=torch.float32, device=phis.device)
        accumulate = False
    _lib.check(_lib.load().opus_sketch_dot_layers(_ptr(phis), int(phis.stride(0)), _ptr(taus), _ptr(alphas), L, B,
                                                 k, _ptr(out), int(accumulate), _stream(phis)),
               "opus_sketch_dot_layers")
    return out


def sketch_gram(phi_a: torch.Tensor, phi_b: torch.Tensor | None = None, alpha: float = 1.0,
                out: torch.Tensor | None = None, accumulate: bool = False) -> torch.Tensor:
    _cuda(phi_a, "phi_a")
    phi_a = _contig(phi_a)
    phi_b = phi_a if phi_b is None else _contig(phi_b)
    ra, k = phi_a.shape
    rb = phi_b.shape[0]
    if phi_b.shape[1] != k:
        raise ValueError("sketch dimensions differ")
    if out is None:
        out = torch.empty(ra, rb, dtype=torch.float32, device=phi_a.device)
        accumulate = False
    _lib.check(_lib.load().opus_sketch_gram(_ptr(phi_a), ra, _ptr(phi_b), rb, k, float(alpha), _ptr(out),
                                           int(accumulate), _stream(phi_a)), "opus_sketch_gram")
    return out


# --------------------------------------------------------------------- stage 4 (Muon)
def gemm_bf16(a: torch.Tensor, b: torch.Tensor, out_dtype: torch.dtype = torch.bfloat16, alpha: float = 1.0,
              a_lo: torch.Tensor | None = None, out: torch.Tensor | None = None,
              accumulate: bool = False) -> torch.Tensor:
    """C = alpha * (a (+ a_lo)) @ b^T on the tensor cores: a [M, K], b [N, K] bf16, f32 accumulation.

    out_dtype bfloat16 rounds every f32 sum once (torch's .to(bfloat16));
    float32 keeps it (accumulate adds into out).  K and N multiples of 8.
    """
    _cuda(a, "a")
    _cuda(b, "b")
    if a.dim() != 2 or b.dim() != 2 or a.shape[1] != b.shape[1]:
        raise ValueError(f"gemm_bf16: a [M, K] and b [N, K] expected, got {tuple(a.shape)}, {tuple(b.shape)}")
    if a.dtype != torch.bfloat16 or b.dtype != torch.bfloat16 or (a_lo is not None and a_lo.dtype != torch.bfloat16):
        raise ValueError("gemm_bf16: operands must be bf16")
    if a_lo is not None and a_lo.shape != a.shape:
        raise ValueError("gemm_bf16: a_lo must have a's shape")
    if out_dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("gemm_bf16: out_dtype must be bfloat16 or float32")
    M, K = a.shape
    N = b.shape[0]
    if out is None:
        out = torch.empty(M, N, dtype=out_dtype, device=a.device)
        accumulate = False
    if out.dtype != out_dtype or not out.is_contiguous() or out.numel() < M * N:
        raise ValueError(f"out must be a contiguous {out_dtype} tensor of at least [M, N]")
    if M == 0:
        return out
    dt = _lib.DTYPE_BF16 if out_dtype == torch.bfloat16 else _lib.DTYPE_F32
    a, b = _contig(a), _contig(b)
    a_lo = None if a_lo is None else _contig(a_lo)
    _lib.check(_lib.load().opus_gemm_bf16(_ptr(a), _ptr(a_lo), _ptr(b), M, N, K, float(alpha), _ptr(out), dt,
                                         int(accumulate), _stream(a)), "opus_gemm_bf16")
    return out


def muon_S(m: torch.Tensor) -> torch.Tensor:
    """Muon preconditioner S = a I + b A + c A^2, A = m~ m~^T, m~ = m / ||m||, as bf16 [d_out, d_out].

    m: the momentum buffer [d_out, d_in] (f32 or bf16; other dtypes are cast
    to bf16 first, as the reference does).  Every step rounds to bf16 where
    the reference's bf16 torch arithmetic does; the identity when
    ||m|| < 1e-7.  Widths that are not multiples of 8 are zero-padded (zero
    rows and columns change neither the norm nor the valid block of S).
    """
    _cuda(m, "m")
    if m.dim() != 2:
        raise ValueError(f"muon_S: momentum buffer must be 2-D, got {tuple(m.shape)}")
    if m.dtype not in (torch.float32, torch.bfloat16):
        m = m.to(torch.bfloat16)
    d_out, d_in = m.shape
    do_p, di_p = (d_out + 7) // 8 * 8, (d_in + 7) // 8 * 8
    if (do_p, di_p) != (d_out, d_in):
        m = torch.nn.functional.pad(m, (0, di_p - d_in, 0, do_p - d_out))
    m = _contig(m)
    lib = _lib.load()
    ws_bytes = int(lib.opus_muon_S_workspace_bytes(do_p, di_p))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=m.device)
    S = torch.empty(do_p, do_p, dtype=torch.bfloat16, device=m.device)
    dt = _lib.DTYPE_F32 if m.dtype == torch.float32 else _lib.DTYPE_BF16
    _lib.check(lib.opus_muon_S(_ptr(m), dt, do_p, di_p, _ptr(ws), ws_bytes, _ptr(S), _stream(m)), "opus_muon_S")
    return S if do_p == d_out else S[:d_out, :d_out].contiguous()


def muon_transform(dLdZ: torch.Tensor, S: torch.Tensor, symmetric: bool = False) -> torch.Tensor:
    """einsum('...o,po->...p', dLdZ.float(), S.float().T).to(dLdZ.dtype) on the tensor cores.

    The Muon candidate transform (data_selection.py:495-500): out[..., p] =
    sum_o dLdZ[..., o] S[o, p].  bf16 dLdZ with a bf16 S is one GEMM with a
    bf16 output; f32 dLdZ is split into bf16 hi/lo (two products, f32
    output); an f32 S that bf16 does not hold exactly is split as well.
    symmetric=True skips the transpose of S (the S of muon_S is symmetric).
    """
    _cuda(dLdZ, "dLdZ")
    _cuda(S, "S")
    d_out = dLdZ.shape[-1]
    if S.shape != (d_out, d_out):
        raise ValueError(f"S must be [{d_out}, {d_out}], got {tuple(S.shape)}")
    lead = dLdZ.shape[:-1]
    g = dLdZ.reshape(-1, d_out)
    Bm = S if symmetric else S.t()
    p = (d_out + 7) // 8 * 8
    if p != d_out:
        g = torch.nn.functional.pad(g, (0, p - d_out))
        Bm = torch.nn.functional.pad(Bm, (0, p - d_out, 0, p - d_out))
    Bm = _contig(Bm)
    if Bm.dtype == torch.bfloat16:
        b_hi, b_lo = Bm, None
    else:
        b_hi, b_lo = split_bf16(Bm)
        if not bool(torch.any(b_lo != 0)):
            b_lo = None
    if g.dtype == torch.bfloat16 and b_lo is None:
        out = gemm_bf16(g, b_hi, out_dtype=torch.bfloat16)
    else:
        if g.dtype == torch.bfloat16:
            g_hi, g_lo = _contig(g), None
        else:
            g_hi, g_lo = split_bf16(g)
        out = gemm_bf16(g_hi, b_hi, out_dtype=torch.float32, a_lo=g_lo)
        if b_lo is not None:
            gemm_bf16(g_hi, b_lo, out_dtype=torch.float32, out=out, accumulate=True)
        out = out.to(dLdZ.dtype)
    if p != d_out:
        out = out[:, :d_out]
    return out.reshape(*lead, d_out)


def kernel_launches() -> int:
    """Kernels the library has launched in this process so far."""
    return int(_lib.load().opus_kernel_launches())


# --------------------------------------------------------------------- stage 5
def _sim_operand(sim: torch.Tensor, n: int) -> tuple[torch.Tensor, int]:
    """Dense [n, n] interaction matrix (block 0) or block-diagonal blocks [q, b, b] (block b, q*b == n)."""
    sim = _contig(sim.to(torch.float32))
    if sim.dim() == 3:
        q, b, b2 = sim.shape
        if b != b2 or q * b != n:
            raise ValueError(f"interaction blocks must be [q, b, b] with q*b == {n}, got {tuple(sim.shape)}")
        return sim, b
    if sim.shape != (n, n):
        raise ValueError(f"interaction matrix must be [{n}, {n}]")
    return sim, 0


def boltzmann_select(scores: torch.Tensor, sim: torch.Tensor, n_select: int, temperature: float,
                     uniforms: torch.Tensor) -> torch.Tensor:
    """Stochastic greedy selection on the device; uniforms: float64 [n_select] (one per draw).

    sim is the dense [n, n] interaction matrix, or [q, b, b] blocks of a
    block-diagonal one (candidates sharded over q ranks of b each).
    """
    _cuda(scores, "scores")
    scores = _contig(scores.to(torch.float32).reshape(-1))
    n = scores.numel()
    sim, block = _sim_operand(sim, n)
    if n_select > n:
        raise ValueError(f"cannot select {n_select} of {n} candidates")
    uniforms = _contig(uniforms.to(device=scores.device, dtype=torch.float64).reshape(-1))
    if uniforms.numel() < n_select:
        raise ValueError("need one uniform per draw")
    out = torch.empty(n_select, dtype=torch.int64, device=scores.device)
    lib = _lib.load()
    if block:
        rc = lib.opus_boltzmann_select_blocks(_ptr(scores), _ptr(sim), n, block, int(n_select), float(temperature),
                                              _ptr(uniforms), _ptr(out), _stream(scores))
    else:
        rc = lib.opus_boltzmann_select(_ptr(scores), _ptr(sim), n, int(n_select), float(temperature),
                                       _ptr(uniforms), _ptr(out), _stream(scores))
    _lib.check(rc, "opus_boltzmann_select")
    return out


def greedy_select(scores: torch.Tensor, sim: torch.Tensor, n_select: int) -> torch.Tensor:
    """Greedy selection on the device; sim dense [n, n] or block-diagonal blocks [q, b, b]."""
    _cuda(scores, "scores")
    scores = _contig(scores.to(torch.float32).reshape(-1))
    n = scores.numel()
    sim, block = _sim_operand(sim, n)
    out = torch.empty(n_select, dtype=torch.int64, device=scores.device)
    lib = _lib.load()
    if block:
        rc = lib.opus_greedy_select_blocks(_ptr(scores), _ptr(sim), n, block, int(n_select), _ptr(out),
                                           _stream(scores))
    else:
        rc = lib.opus_greedy_select(_ptr(scores), _ptr(sim), n, int(n_select), _ptr(out), _stream(scores))
    _lib.check(rc, "opus_greedy_select")
    return out


# ------------------------------------------------------- training step: shared
_TYPE_CODES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float32: _lib.DTYPE_F32, torch.float16: _lib.DTYPE_F16}


def _tensor(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor, got {type(t).__name__}")


def _type_code(t: torch.Tensor, name: str) -> int:
    code = _TYPE_CODES.get(getattr(t, "dtype", None))
    if code is None:
        _tensor(t, name)
        raise ValueError(f"{name} must be bfloat16, float16 or float32, got {t.dtype}")
    return code


def _device_index(ref: torch.Tensor, name: str, *others: torch.Tensor | None) -> int:
    """The CUDA device of ref and of every other tensor (looked at after shapes and types, which need no GPU)."""
    index = ref.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            raise ValueError(f"{name} is on {ref.device}, another argument on {t.device}")
    if index < 0:
        _cuda(ref, name)
    return index


def _call(name: str, index: int, *args) -> None:
    """Call an entry point on device `index`, made current, and its current stream; addresses are plain integers."""
    fn = getattr(_lib.load(), name)
    _devices.add(index)
    if index == torch._C._cuda_getDevice():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _lib.check(rc, name)


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """The tensor as rows of its last dimension, and their stride in elements; copied if rows are not evenly spaced."""
    d = t.shape[-1]
    if t.is_contiguous():
        return t, d
    if t.stride(-1) == 1 and t.numel() > 0:
        try:
            v = t.view(-1, d)
        except RuntimeError:
            return t.contiguous(), d
        if v.shape[0] == 1:
            return v, d
        if v.stride(0) >= d:
            return v, v.stride(0)
    return t.contiguous(), d


# ---------------------------------------------------- training step: embedding
def _tokens(tokens: torch.Tensor) -> tuple[torch.Tensor, int]:
    _tensor(tokens, "tokens")
    if tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"tokens must be int32 or int64, got {tokens.dtype}")
    return _contig(tokens), 64 if tokens.dtype == torch.int64 else 32


def embedding(tokens: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """scale * weight[tokens]: [*tokens.shape, d] of weight's type, the product rounded once.

    weight [V, d] in bf16, f16 or f32 (rows may be apart: a column slice of a
    wider table is read in place).  A token outside [0, V) gives a row of
    zeros, and the next check_device_error() raises IndexError.  An out that
    shares memory with weight's rows or the tokens is refused.
    """
    tokens, bits = _tokens(tokens)
    code = _type_code(weight, "weight")
    if weight.dim() != 2 or weight.shape[0] < 1 or weight.shape[1] < 1:
        raise ValueError(f"weight must be [V, d], got {tuple(weight.shape)}")
    V, d = weight.shape
    shape = (*tokens.shape, d)
    if out is not None:
        _tensor(out, "out")
    if out is not None and (out.shape != shape or out.dtype != weight.dtype or not out.is_contiguous()):
        raise ValueError(f"out must be a contiguous {weight.dtype} tensor of shape {shape}")
    index = _device_index(weight, "weight", tokens, out)
    rows, stride = _rows(weight)
    if out is None:
        out = weight.new_empty(shape)
    _call("opus_embedding", index, tokens.data_ptr(), bits, tokens.numel(), rows.data_ptr(), code, V, stride, d,
          float(scale), out.data_ptr())
    return out


def embedding_grad(grad_out: torch.Tensor, tokens: torch.Tensor, num_embeddings: int, scale: float = 1.0,
                   padding_idx: int | None = None, out: torch.Tensor | None = None, accumulate: bool = False,
                   out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """Gradient of embedding() for the weight: out[v] (+)= scale * sum of grad_out over the positions of token v.

    grad_out [*tokens.shape, d] in bf16, f16 or f32; out [num_embeddings, d]
    of its type or float32 (out_dtype, or the type of out).  The sums run in
    f32 over the positions in order: every call gives the same bits.  Rows of
    padding_idx get nothing.  accumulate=True adds into out and touches only
    rows that a token names; without it the rows of other tokens are zeros.
    Tokens out of range add nothing and are reported as by embedding().  An
    out that shares memory with grad_out or the tokens is refused.
    """
    tokens, bits = _tokens(tokens)
    V = int(num_embeddings)
    if V < 1:
        raise ValueError("num_embeddings must be positive")
    code = _type_code(grad_out, "grad_out")
    if grad_out.dim() < 1 or grad_out.shape[:-1] != tokens.shape or grad_out.shape[-1] < 1:
        raise ValueError(f"grad_out must be [*{tuple(tokens.shape)}, d], got {tuple(grad_out.shape)}")
    d = grad_out.shape[-1]
    if padding_idx is not None:
        if not -V <= padding_idx < V:
            raise ValueError(f"padding_idx must be within [-{V}, {V}), got {padding_idx}")
        padding_idx = padding_idx % V
    if accumulate and out is None:
        raise ValueError("accumulate needs out")
    if out is not None:
        _tensor(out, "out")
        if out_dtype is not None and out_dtype != out.dtype:
            raise ValueError(f"out is {out.dtype}, out_dtype {out_dtype}")
        if out.shape != (V, d) or not out.is_contiguous():
            raise ValueError(f"out must be a contiguous tensor of shape {(V, d)}")
    dtype = out.dtype if out is not None else out_dtype or grad_out.dtype
    if dtype not in (grad_out.dtype, torch.float32):
        raise ValueError(f"the gradient is {grad_out.dtype} or float32, not {dtype}")
    index = _device_index(grad_out, "grad_out", tokens, out)
    rows, stride = _rows(grad_out)
    if out is None:
        out = grad_out.new_empty((V, d), dtype=dtype)
    n = tokens.numel()
    ws_bytes = int(_lib.load().opus_embedding_grad_workspace_bytes(n, V, d))
    ws = tokens.new_empty(ws_bytes, dtype=torch.uint8)
    _call("opus_embedding_grad", index, rows.data_ptr(), code, stride, tokens.data_ptr(), bits, n, V, d, float(scale),
          -1 if padding_idx is None else int(padding_idx), out.data_ptr(), _TYPE_CODES[dtype], int(accumulate),
          ws.data_ptr(), ws_bytes)
    return out


# ------------------------------------------------ training step: residual norm
_NORM_KINDS = {"rms": 0, "layer": 1}
_NORM_PARAMS = ("weight", "bias", "post_weight", "post_bias", "gate")


def _norm_args(like: torch.Tensor, y: torch.Tensor | None, y_dtype: torch.dtype, params: Sequence[torch.Tensor | None],
               post: bool, kind: str, eps: float, residual_scale: float) -> tuple[_lib.ResidualNormArgs, list]:
    """The C arguments that forward and backward share, and the contiguous parameters that they point to."""
    if kind not in _NORM_KINDS:
        raise ValueError(f"kind must be 'rms' or 'layer', got {kind!r}")
    shape = like.shape
    if not shape or shape[-1] < 1:
        raise ValueError(f"rows of at least one element expected, got {tuple(shape)}")
    d = shape[-1]
    x_code, y_code = _type_code(like, "x"), _TYPE_CODES.get(y_dtype)
    if y_code is None or (y_code != x_code and x_code != _lib.DTYPE_F32):
        raise ValueError(f"x must be of y's type (bfloat16, float16 or float32) or float32, got {like.dtype} with "
                         f"{y_dtype}")
    if y is None:
        if post or params[4] is not None:
            raise ValueError("a gate or a norm after the block needs y")
    elif y.shape != shape:
        raise ValueError(f"y must have x's shape {tuple(shape)}, got {tuple(y.shape)}")
    if not post and (params[2] is not None or params[3] is not None):
        raise ValueError("post_weight and post_bias belong to post=True")
    kept, ptrs, codes, gate_rows = [], [None] * 5, [0] * 5, 0
    for i, p in enumerate(params):
        if p is None:
            continue
        codes[i] = _type_code(p, _NORM_PARAMS[i])
        if i == 4:
            gate_rows = _gate_rows(p, like)
        elif p.dim() != 1 or p.shape[0] != d:
            raise ValueError(f"{_NORM_PARAMS[i]} must be [{d}], got {tuple(p.shape)}")
        p = _contig(p)
        kept.append(p)
        ptrs[i] = p.data_ptr()
    return _lib.ResidualNormArgs(like.numel() // d, d, _NORM_KINDS[kind], int(post), x_code, y_code, eps, residual_scale,
                                 None, None, 0, 0, *ptrs, *codes, gate_rows), kept


def _gate_rows(gate: torch.Tensor, x: torch.Tensor) -> int:
    """1 for a gate of [d]; the number of samples for one of [B, d] or [B, 1, ..., d] against x [B, ..., d]."""
    d = x.shape[-1]
    if gate.shape == (d,):
        return 1
    if x.dim() >= 2 and gate.dim() >= 2 and gate.shape[-1] == d and gate.shape[0] == x.shape[0] \
            and gate.numel() == x.shape[0] * d and gate.dim() in (2, x.dim()):
        return max(1, x.shape[0])
    raise ValueError(f"gate must be [{d}] or one row for each of x's first dimension, got {tuple(gate.shape)} "
                     f"for x {tuple(x.shape)}")


def residual_norm(x: torch.Tensor, y: torch.Tensor | None = None, *, weight: torch.Tensor | None = None,
                  bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                  post_bias: torch.Tensor | None = None, post: bool | None = None, gate: torch.Tensor | None = None,
                  residual_scale: float = 1.0, kind: str = "rms", eps: float = 1e-6,
                  out_dtype: torch.dtype | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The joint between two blocks of a residual network in one kernel: (n, h, stats).

        z = y, or with post its norm N(y) * post_weight + post_bias
        h = residual_scale * x + gate * z            of x's type: the residual stream
        n = N(h) * weight + bias                     of y's type: what the next block reads

    x and y [..., d], d up to 16384, in bf16, f16 or f32 (x may be float32 with
    a 16-bit y); N is an RMS norm (kind "rms") or a layer norm ("layer") over d.
    Every parameter may be absent (ones, zeros) and has a type of its own.
    gate is [d], or one row for each of x's first dimension ([B, d] or
    [B, 1, d] against x [B, T, d]).  post defaults to whether post_weight or
    post_bias is given.  Without y, h is residual_scale * x (x itself at 1) and
    n of out_dtype (default x's type).  n is the norm of h as it is stored.
    stats is what residual_norm_grad needs of the forward.
    """
    post = (post_weight is not None or post_bias is not None) if post is None else bool(post)
    if not isinstance(x, torch.Tensor) or not (y is None or isinstance(y, torch.Tensor)):
        _tensor(x, "x")
        _tensor(y, "y")
    n_dtype = x.dtype if y is None else y.dtype
    if out_dtype is not None and out_dtype != n_dtype:
        if y is not None:
            raise ValueError(f"out_dtype is y's type where y is given ({y.dtype}), got {out_dtype}")
        n_dtype = out_dtype
    a, kept = _norm_args(x, y, n_dtype, (weight, bias, post_weight, post_bias, gate), post, kind, float(eps),
                         float(residual_scale))
    index = _device_index(x, "x", y, *kept)
    xr, a.x_stride = _rows(x)
    a.x = xr.data_ptr()
    if y is not None:
        yr, a.y_stride = _rows(y)
        a.y = yr.data_ptr()
    plain = y is None and a.residual_scale == 1.0
    h = x if plain else x.new_empty(x.shape)
    n = x.new_empty(x.shape, dtype=n_dtype)
    stats = x.new_empty((a.rows, 4), dtype=torch.float32)
    a.h, a.h_stride, a.n, a.stats = None if plain else h.data_ptr(), a.d, n.data_ptr(), stats.data_ptr()
    _call("opus_residual_norm", index, ctypes.byref(a))
    return n, h, stats


def residual_norm_grad(grad_n: torch.Tensor | None, grad_h: torch.Tensor | None, h: torch.Tensor, stats: torch.Tensor,
                       y: torch.Tensor | None = None, *, weight: torch.Tensor | None = None,
                       bias: torch.Tensor | None = None, post_weight: torch.Tensor | None = None,
                       post_bias: torch.Tensor | None = None, post: bool | None = None,
                       gate: torch.Tensor | None = None, residual_scale: float = 1.0, kind: str = "rms",
                       wanted: Iterable[str] | None = None) -> dict[str, torch.Tensor]:
    """Gradients of residual_norm from those of its outputs n and h (one of them may be None: zeros).

    h and stats are the forward's outputs, the other arguments those it was
    given.  Returns {"x", "y" (if y), and one entry for each parameter given};
    wanted restricts the parameters' gradients to the named ones.  Each is of
    its tensor's type and shape.  Sums over rows run in f32 in a fixed order:
    every call gives the same bits.
    """
    post = (post_weight is not None or post_bias is not None) if post is None else bool(post)
    if grad_n is None and grad_h is None:
        raise ValueError("grad_n or grad_h must be given")
    T = torch.Tensor
    if not (isinstance(h, T) and isinstance(stats, T) and (y is None or isinstance(y, T))
            and (grad_n is None or isinstance(grad_n, T)) and (grad_h is None or isinstance(grad_h, T))):
        for name, t in (("h", h), ("stats", stats), ("y", y), ("grad_n", grad_n), ("grad_h", grad_h)):
            if t is not None or name in ("h", "stats"):
                _tensor(t, name)
    n_dtype = y.dtype if y is not None else grad_n.dtype if grad_n is not None else h.dtype
    params = (weight, bias, post_weight, post_bias, gate)
    a, kept = _norm_args(h, y, n_dtype, params, post, kind, 0.0, float(residual_scale))
    for name, t, dtype in (("grad_n", grad_n, n_dtype), ("grad_h", grad_h, h.dtype)):
        if t is not None and (t.shape != h.shape or t.dtype != dtype):
            raise ValueError(f"{name} must be {dtype} {tuple(h.shape)}, got {t.dtype} {tuple(t.shape)}")
    if stats.shape != (a.rows, 4) or stats.dtype != torch.float32 or not stats.is_contiguous():
        raise ValueError(f"stats must be the forward's, a contiguous float32 [{a.rows}, 4]")
    if wanted is not None:
        wanted = set(wanted)
        if not wanted <= set(_NORM_PARAMS):
            raise ValueError(f"wanted names {sorted(wanted - set(_NORM_PARAMS))}, parameters are {_NORM_PARAMS}")
    index = _device_index(h, "h", stats, y, grad_n, grad_h, *kept)
    hr, a.h_stride = _rows(h)
    grad_x = h.new_empty(h.shape)
    a.h, a.grad_x, a.stats = hr.data_ptr(), grad_x.data_ptr(), stats.data_ptr()
    out = {"x": grad_x}
    if y is not None:
        yr, a.y_stride = _rows(y)
        out["y"] = grad_y = y.new_empty(y.shape)
        a.y, a.grad_y = yr.data_ptr(), grad_y.data_ptr()
    if grad_n is not None:
        nr, a.grad_n_stride = _rows(grad_n)
        a.grad_n = nr.data_ptr()
    if grad_h is not None:
        dr, a.grad_h_stride = _rows(grad_h)
        a.grad_h = dr.data_ptr()
    for name, p in zip(_NORM_PARAMS, params):
        if p is not None and (wanted is None or name in wanted):
            out[name] = g = p.new_empty(p.shape)
            setattr(a, "grad_" + name, g.data_ptr())
    ws_bytes = int(_lib.load().opus_residual_norm_grad_workspace_bytes(ctypes.byref(a)))
    ws = stats.new_empty(ws_bytes, dtype=torch.uint8)
    _call("opus_residual_norm_grad", index, ctypes.byref(a), ws.data_ptr(), ws_bytes)
    return out


# ------------------------------------------------ training step: gradient clip
def _norm_kind(norm_type: float) -> int:
    if norm_type == 2:
        return 2
    if norm_type == math.inf:
        return 0
    raise ValueError(f"norm_type must be 2 or inf, got {norm_type}")


def _dense(t: torch.Tensor) -> bool:
    """Whether the elements fill one run of memory without gaps, in whatever order of dimensions."""
    if t.is_contiguous():
        return True
    run = 1
    for stride, size in sorted(zip(t.stride(), t.shape)):
        if size == 1:
            continue
        if stride != run:
            return False
        run *= size
    return True


class _TensorList:
    """Strided tensors of the three types on one device, and their addresses, lengths and types as the host arrays
    of the C ABI.  A tensor whose elements do not fill one run of memory is copied (tensors), and named in copied."""

    def __init__(self, tensors: torch.Tensor | Iterable[torch.Tensor], name: str, contiguous: bool = False):
        tensors = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
        self.count, self.tensors, self.copied = len(tensors), tensors, []
        scan = _lib.tensor_list().scan
        self.ptrs, self.numels, self.types, self.index, odd = scan(tensors, name)
        for i in odd:
            t = tensors[i]
            if contiguous or not _dense(t):
                self.copied.append(t)
                tensors[i] = t.contiguous()
        if self.copied:
            self.ptrs = scan(tensors, name)[0]

    def cuda(self, name: str) -> int:
        if self.index < 0:
            _cuda(self.tensors[0], name)
        return self.index


def grad_norm(grads: torch.Tensor | Iterable[torch.Tensor], norm_type: float = 2.0) -> torch.Tensor:
    """Norm of all elements of a list of tensors as one vector: a float32 scalar on their device.

    norm_type 2 (square root of the sum of squares) or inf (largest
    magnitude).  bf16, f16 and f32 tensors of any layout, mixed; an empty list
    gives 0 (on the CPU, as torch does).  Nothing waits for the host.
    """
    kind = _norm_kind(norm_type)
    g = _TensorList(grads, "grads")
    if not g.count:
        return torch.tensor(0.0)
    index = g.cuda("grads")
    norm = g.tensors[0].new_empty((), dtype=torch.float32)
    ws_bytes = int(_lib.load().opus_grad_norm_workspace_bytes(g.count))
    ws = norm.new_empty(ws_bytes, dtype=torch.uint8)
    _call("opus_grad_norm", index, g.ptrs, g.numels, g.types, g.count, kind, ws.data_ptr(), ws_bytes,
          norm.data_ptr())
    return norm


def _clip_targets(grads, out, name: str) -> tuple[_TensorList, _TensorList, list]:
    """(sources, targets, [(gradient, its dense copy)] to write back): in place without out."""
    if out is None:
        grads = [grads] if isinstance(grads, torch.Tensor) else list(grads)
        g = _TensorList(grads, "grads")
        if not g.copied:
            return g, g, []
        for t in g.copied:
            if any(stride == 0 and size > 1 for stride, size in zip(t.stride(), t.shape)):
                raise ValueError(f"{name}: a gradient's elements overlap in memory (an expanded tensor)")
        if len({(t.data_ptr(), t.shape, t.stride()) for t in g.copied if t.numel()}) < sum(t.numel() > 0 for t in g.copied):
            raise ValueError(f"{name}: an element would be written twice (a tensor listed twice)")
        return g, g, [(t, c) for t, c in zip(grads, g.tensors) if t is not c]
    g, o = _TensorList(grads, "grads", contiguous=True), _TensorList(out, "out", contiguous=True)
    if o.copied:
        raise ValueError(f"{name}: out must be contiguous tensors")
    if g.numels != o.numels:
        raise ValueError(f"{name}: out must have a tensor of as many elements for each gradient")
    if g.count and g.index != o.index:
        raise ValueError(f"{name}: out and grads are on different devices")
    return g, o, []


def clip_grads(grads: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm_type: float = 2.0,
               out: Sequence[torch.Tensor] | None = None) -> torch.Tensor:
    """Scale gradients so that their joint norm is at most max_norm; returns the norm they had.

    The rule of torch.nn.utils.clip_grad_norm_: each gradient times
    min(1, max_norm / (norm + 1e-6)), in place, or written to out (contiguous
    tensors of the gradients' sizes and any of the types: 16-bit gradients
    into an optimizer's float32 ones).  The factor is held in f32 and each
    product rounded once.  Gradients whose norm is within the bound are not
    written in place.  A list that would write an element twice (a gradient
    listed twice, overlapping views, an out that overlaps the gradients) is
    refused; of views with gaps between their elements only equal ones are,
    and elements that several share are scaled once.  A NaN norm makes every gradient NaN.  The norm is a
    float32 scalar on the device, and nothing waits for the host.
    """
    kind = _norm_kind(norm_type)
    g, o, back = _clip_targets(grads, out, "clip_grads")
    if not g.count:
        return torch.tensor(0.0)
    index = g.cuda("grads")
    norm = g.tensors[0].new_empty((), dtype=torch.float32)
    ws_bytes = int(_lib.load().opus_grad_norm_workspace_bytes(g.count))
    ws = norm.new_empty(ws_bytes, dtype=torch.uint8)
    _call("opus_clip_grads", index, g.ptrs, g.types, o.ptrs, o.types, g.numels, g.count, kind,
          float(max_norm), ws.data_ptr(), ws_bytes, norm.data_ptr())
    for t, c in back:
        t.copy_(c)
    return norm


def scale_grads(grads: torch.Tensor | Iterable[torch.Tensor], max_norm: float, norm: torch.Tensor,
                out: Sequence[torch.Tensor] | None = None) -> None:
    """The second half of clip_grads, for a norm that is known: joined over ranks that hold shards, say.

    norm: a float32 scalar on the gradients' device, in none of the tensors
    that are written.
    """
    g, o, back = _clip_targets(grads, out, "scale_grads")
    _tensor(norm, "norm")
    if norm.numel() != 1 or norm.dtype != torch.float32:
        raise ValueError(f"norm must be a float32 scalar, got {norm.dtype} {tuple(norm.shape)}")
    if not g.count:
        return
    index = _device_index(g.tensors[0], "grads", norm)
    _call("opus_scale_grads", index, g.ptrs, g.types, o.ptrs, o.types, g.numels,
          g.count, float(max_norm), norm.data_ptr())
    for t, c in back:
        t.copy_(c)
