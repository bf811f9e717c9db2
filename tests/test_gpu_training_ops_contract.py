"""What the training-step operators promise beyond their values: errors, outputs and memory around them (GPU)."""
import numpy as np
import pytest
import torch

from opus_b200 import ops
from opus_b200.train import stochastic_greedy_selection

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ============================================================================ errors recorded on the device
def bad_token():
    ops.embedding(torch.tensor([0, 9], device=DEV), torch.ones(5, 8, device=DEV))


def tables(bucket):
    return torch.tensor([1, bucket, 3], device=DEV), torch.tensor([1.0, -1.0, 1.0], device=DEV)


def test_bad_token_is_not_an_error_of_the_selection_path():
    ops.check_device_error()
    bad_token()
    ops.pack_hash_sign(*tables(2), 8)  # checks its own kernel
    np.random.seed(0)
    assert len(stochastic_greedy_selection(torch.rand(6, device=DEV), torch.eye(6, device=DEV), 2, 1.0)) == 2
    ops.check_device_error("selection", tokens=False)
    with pytest.raises(IndexError, match="token"):
        ops.check_device_error("embedding")
    ops.check_device_error()


def test_bad_token_does_not_hide_an_error_of_the_selection_path():
    for before in (True, False):
        if before:
            bad_token()
        with pytest.raises(RuntimeError, match="bucket"):
            ops.pack_hash_sign(*tables(8), 8)
        if not before:
            ops.pack_hash_sign(*tables(-1), 8, validate=False)
            bad_token()
            with pytest.raises(RuntimeError, match="0x201"):
                ops.check_device_error()  # the kernel's first
        with pytest.raises(IndexError, match="token"):
            ops.check_device_error()
        ops.check_device_error()


# ============================================================================ outputs that overlap inputs
def test_embedding_out_may_lie_between_what_is_read_but_not_in_it():
    table = torch.randint(-9, 10, (12, 16), device=DEV).float()  # sums are exact
    before = table.clone()
    t = torch.tensor([3, 0, 11], device=DEV)
    for bad in (dict(weight=table, out=table[:3]), dict(weight=table[:, :8], out=table.view(-1)[8:32].view(3, 8)),
                dict(weight=table[4:], out=table[2:5])):
        with pytest.raises(ValueError, match="overlaps"):
            ops.embedding(t % bad["weight"].shape[0], **bad)
    with pytest.raises(ValueError, match="overlaps"):
        ops.embedding_grad(table, torch.arange(12, device=DEV), 3, out=table[9:])
    assert torch.equal(table, before)
    # in the gap of one row of weight, and behind its rows
    assert torch.equal(ops.embedding(t[:1], table[:, :8], out=table[5:6, 8:]), before[3:4, :8])
    assert torch.equal(ops.embedding(t[:1], table[:11], out=table[11:]), table[3:4])
    assert torch.equal(table[:5], before[:5]) and torch.equal(table[6:11], before[6:11])
    got = ops.embedding_grad(table[:4], t[:1].expand(4), 8, out=table[4:])
    assert torch.equal(got[3], table[:4].sum(0)) and not bool(got[:3].any()) and not bool(got[4:].any())


def test_scale_grads_with_a_norm_among_the_gradients():
    flat = torch.full((9,), 2.0, device=DEV)
    for bad in ([flat], [flat[:5], flat[5:]]):
        with pytest.raises(ValueError, match="norm"):
            ops.scale_grads(bad, 1.0, flat[5])
    assert bool((flat == 2).all())
    ops.scale_grads([flat[:5], flat[6:]], 1.0, flat[5])  # beside them
    c = float(np.float32(1.0) / (np.float32(2.0) + np.float32(1e-6)))
    assert flat.tolist() == [float(np.float32(2.0) * np.float32(c))] * 5 + [2.0] + [float(np.float32(2.0) * np.float32(c))] * 3
    out = torch.zeros(9, device=DEV)
    ops.scale_grads([flat], 1.0, flat[5], out=[out])  # nothing that is read is written
    assert float(out[5]) == float(np.float32(2.0) * np.float32(c))
