"""What the training-step operators promise beyond their values, as far as it shows without a GPU."""
import contextlib
import ctypes
import importlib.util
import shutil
import subprocess
import sysconfig
import types

import pytest
import torch

from opus_b200 import _lib, ops
from opus_b200.csrc import build as nvbuild
from opus_b200.layers import ScaledEmbedding, scaled_embedding


# ============================================================================ errors recorded on the device
class Devices:
    """Two devices with an error word each, in the place of torch's and the library's."""

    def __init__(self, monkeypatch):
        self.current, self.words, self.launched = 0, {0: 0, 1: 0}, []
        monkeypatch.setattr(torch.cuda, "device", self.device)
        monkeypatch.setattr(torch.cuda, "current_device", lambda: self.current)
        monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: self.current, raising=False)
        monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda index: 100 + index, raising=False)
        monkeypatch.setattr(_lib, "load", lambda: types.SimpleNamespace(opus_fake=self.launch))
        monkeypatch.setattr(_lib, "device_error", self.take)
        monkeypatch.setattr(ops, "_devices", set())

    @contextlib.contextmanager
    def device(self, index):
        before, self.current = self.current, index
        yield
        self.current = before

    def launch(self, code, stream):
        self.launched.append((self.current, stream))
        self.words[self.current] = code
        return 0

    def take(self, tokens=True):
        code, self.words[self.current] = self.words[self.current], 0
        return code


def test_errors_of_another_device_are_reported(monkeypatch):
    d = Devices(monkeypatch)
    ops._call("opus_fake", 1, 0x202)
    assert d.launched == [(1, 101)] and d.current == 0
    with pytest.raises(IndexError, match="token"):
        ops.check_device_error()
    ops.check_device_error()
    with d.device(1):  # a backward's thread, say
        ops._call("opus_fake", 1, 0x202)
    with pytest.raises(IndexError, match="token"):
        ops.check_device_error()
    ops._call("opus_fake", 0, 0x107)
    ops._call("opus_fake", 1, 0x202)
    with pytest.raises(RuntimeError, match="0x107"):
        ops.check_device_error()
    with pytest.raises(IndexError):  # not lost to the other's
        ops.check_device_error()
    assert d.words == {0: 0, 1: 0} and d.current == 0


# ============================================================================ build
@pytest.fixture
def nvcc_alone(tmp_path, monkeypatch):
    """The build in a folder of its own, with a compiler that only makes its output file."""
    fake = tmp_path / "nvcc"
    fake.write_text('#!/bin/sh\nwhile [ $# -gt 0 ]; do [ "$1" = -o ] && : > "$2"; shift; done\n')
    fake.chmod(0o755)
    monkeypatch.setenv("NVCC", str(fake))
    monkeypatch.setattr(nvbuild, "BUILD", tmp_path / "_build")
    monkeypatch.setattr(nvbuild, "LIB", tmp_path / "libopus_b200.so")
    monkeypatch.setattr(nvbuild, "MODULE", tmp_path / nvbuild.MODULE.name)
    return tmp_path


@pytest.mark.parametrize("missing", ["torch", "compiler", "headers"])
def test_library_is_built_where_the_module_cannot_be(nvcc_alone, monkeypatch, missing):
    if missing == "torch":
        find = importlib.util.find_spec
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: None if name == "torch" else find(name, *a))
    elif missing == "compiler":
        monkeypatch.setenv("CXX", str(nvcc_alone / "no-such-compiler"))
    else:
        monkeypatch.setenv("CXX", "false")  # ends with an error, as a compiler without Python.h does
    with pytest.warns(RuntimeWarning, match="_tensor_list"):
        assert nvbuild.build() == nvcc_alone / "libopus_b200.so"
    assert (nvcc_alone / "libopus_b200.so").exists() and not nvbuild.MODULE.exists()


def test_module_is_named_by_interpreter():
    assert nvbuild.MODULE.name == "_tensor_list" + sysconfig.get_config_var("EXT_SUFFIX")
    assert _lib.tensor_list().__file__ == str(nvbuild.MODULE)


# ============================================================================ layers
def test_scaled_embedding_from_pretrained():
    w = torch.randn(6, 4, dtype=torch.bfloat16)
    layer = ScaledEmbedding.from_pretrained(w, padding_idx=-1, scale=2.0)
    assert type(layer) is ScaledEmbedding and layer.scale == 2.0 and layer.padding_idx == 5
    assert layer.weight.data_ptr() == w.data_ptr() and layer.weight.dtype == w.dtype and not layer.weight.requires_grad
    assert (layer.num_embeddings, layer.embedding_dim) == (6, 4) and list(layer.state_dict()) == ["weight"]
    assert ScaledEmbedding.from_pretrained(w, freeze=False).weight.requires_grad
    for like in (dict(max_norm=1.0), dict(sparse=True), dict(scale_grad_by_freq=True)):
        with pytest.raises(TypeError, match=next(iter(like))):  # not offered, as by the constructor
            ScaledEmbedding.from_pretrained(w, **like)
    with pytest.raises(ValueError, match="embeddings"):
        ScaledEmbedding.from_pretrained(w[0])
    with pytest.raises(AssertionError):  # nn.Embedding's check
        ScaledEmbedding.from_pretrained(w, padding_idx=6)


# ============================================================================ answers kept by device
PER_DEVICE = r"""
#include <cstdio>
#include "per_device.h"
int main() {
  static opus::PerDevice<5> known;
  int asked = 0;
  auto answer = [&asked](int n) { return [&asked, n] { ++asked; return n; }; };
  int got[] = {known.get(0, 4, 1, answer(9)), known.get(1, 4, 1, answer(7)), known.get(0, 4, 1, answer(3)),
               known.get(1, 4, 1, answer(3)), known.get(0, 3, 1, answer(0)), known.get(0, 3, 1, answer(6)),
               known.get(0, 3, 1, answer(2)), known.get(-1, 0, 1, answer(5)), known.get(64, 0, 1, answer(4))};
  for (int v : got) std::printf("%d ", v);
  std::printf("%d", asked);
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_answers_are_kept_by_device_and_failures_are_not(tmp_path):
    (tmp_path / "t.cpp").write_text(PER_DEVICE)
    subprocess.run(["g++", "-std=c++17", f"-I{nvbuild.CSRC}", str(tmp_path / "t.cpp"), "-o", str(tmp_path / "t")], check=True)
    out = subprocess.run([str(tmp_path / "t")], capture_output=True, text=True, check=True).stdout
    assert out.split() == ["9", "7", "9", "7", "1", "6", "6", "5", "4", "6"]


# ============================================================================ outputs that overlap inputs
def embedding_rc(tokens, n, weight, vocab, stride, out, d=8, dtype=_lib.DTYPE_F32, bits=64):
    """opus_embedding at addresses that are never followed: every call is refused before the device is touched."""
    rc = _lib.load().opus_embedding(tokens, bits, n, weight, dtype, vocab, stride, d, 1.0, out, None)
    return rc, _lib.last_error()


@pytest.mark.parametrize("n,vocab,stride,out", [
    (4, 10, 8, 4096), (4, 10, 8, 4096 + 9 * 32), (4, 10, 8, 4096 + 9 * 32 + 28), (4, 10, 8, 4096 - 100),
    (1, 10, 16, 4096 + 3 * 64), (1, 10, 16, 4096 + 3 * 64 + 28), (1, 10, 16, 4096 + 2 * 64 + 36), (2, 10, 16, 4096 + 32),
    (1, 1, 1 << 62, 4096 + 28), (1, 2, 1 << 62, 4096), (4, 10, 8, 65536 + 28), (4, 10, 8, 65536 - 124)])
def test_embedding_refuses_an_out_that_overlaps(n, vocab, stride, out):
    """weight of f32 rows of 32 bytes at 4096, tokens of 8 bytes at 65536."""
    rc, message = embedding_rc(65536, n, 4096, vocab, stride, out)
    assert rc == _lib.OPUS_ERR_INVALID and "overlaps" in message


@pytest.mark.parametrize("n,vocab,stride,out,dtype", [
    (10, 4, 8, 4096, 1), (10, 4, 8, 4096 + 9 * 32 + 28, 1), (10, 4, 8, 4096 - 124, 1), (3, 1, 16, 4096 + 2 * 64, 1),
    (3, 1, 16, 4096 + 36, 1), (4, 10, 8, 65536 + 28, 1), (4, 10, 8, 65536 - 316, 1), (10, 4, 8, 4096 + 9 * 16 + 12, 0)])
def test_embedding_grad_refuses_an_out_that_overlaps(n, vocab, stride, out, dtype):
    """grad_out at 4096, tokens at 65536, an f32 grad_weight."""
    rc = _lib.load().opus_embedding_grad(4096, dtype, stride, 65536, 64, n, vocab, 8, 1.0, -1, out, _lib.DTYPE_F32, 1,
                                         1 << 20, 1 << 30, None)
    assert rc == _lib.OPUS_ERR_INVALID and "overlaps" in _lib.last_error()


def test_clip_refuses_a_norm_among_the_gradients():
    """scale_grads: every block reads the norm, and one might scale it first.  Addresses are never followed."""
    lib = _lib.load()
    grads, out, n, ty = (ctypes.c_void_p * 1)(4096), (ctypes.c_void_p * 1)(8192), (ctypes.c_int64 * 1)(6), (ctypes.c_int * 1)(1)
    ws = ctypes.c_void_p(256)
    for to, norm in ((grads, 4096), (grads, 4116), (out, 8192 + 20)):
        assert lib.opus_scale_grads(grads, ty, to, ty, n, 1, 1.0, norm, None) == _lib.OPUS_ERR_INVALID
        assert "norm" in _lib.last_error()
    for to, norm in ((grads, 4096), (out, 4116), (out, 8192)):
        assert lib.opus_clip_grads(grads, ty, to, ty, n, 1, 2, 1.0, ws, 1 << 24, norm, None) == _lib.OPUS_ERR_INVALID
        assert "norm" in _lib.last_error()


# ============================================================================ arguments that are no tensors
def test_arguments_that_are_no_tensors_are_named():
    x, t, stats = torch.zeros(3, 8), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 4)
    for name, call in (("weight", lambda: ops.embedding(t, [[1.0]])), ("out", lambda: ops.embedding(t, x, out=[x])),
                       ("weight", lambda: scaled_embedding(t, [[1.0]])),
                       ("grad_out", lambda: ops.embedding_grad([1.0], t, 3)), ("out", lambda: ops.embedding_grad(x, t, 3, out=[x])),
                       ("x", lambda: ops.residual_norm([1.0])), ("y", lambda: ops.residual_norm(x, [1.0])),
                       ("weight", lambda: ops.residual_norm(x, weight=[1.0] * 8)), ("gate", lambda: ops.residual_norm(x, x, gate=1.0)),
                       ("grad_n", lambda: ops.residual_norm_grad([1.0], None, x, stats)),
                       ("grad_h", lambda: ops.residual_norm_grad(None, 1.0, x, stats)),
                       ("h", lambda: ops.residual_norm_grad(x, None, None, stats)),
                       ("stats", lambda: ops.residual_norm_grad(x, None, x, None)),
                       ("y", lambda: ops.residual_norm_grad(x, None, x, stats, 1.0)),
                       ("norm", lambda: ops.scale_grads([x], 1.0, 3.0))):
        with pytest.raises(TypeError, match=rf"^{name} must be a torch.Tensor"):
            call()
