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
