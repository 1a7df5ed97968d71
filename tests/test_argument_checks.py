"""What the Python methods refuse before a device, a kernel or the C ABI's narrower integers see it.  No GPU is needed: the
tensors here take no memory (expanded, or without elements) or the call is refused before it allocates."""
import pytest
import torch

import l2_torch_alloc_b200 as pkg
from l2_torch_alloc_b200 import build


@pytest.fixture(scope="module")
def sa():
    build.build()
    return pkg.SideAware()


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu", 0), "meta"])
def test_rope_precompute_freqs_refuses_devices_that_are_not_cuda(sa, device):
    """torch.device("cpu", 0) has an index: it would have passed for GPU 0."""
    with pytest.raises(AssertionError, match="CUDA"):
        sa.rope_precompute_freqs(64, 16, device=device)
