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


BIG = 2 ** 32 + 3  # 3 in a 32-bit integer


@pytest.mark.parametrize("change", [
    dict(shape=(BIG, 2, 8, 16)), dict(shape=(2, BIG, 8, 16)), dict(shape=(2, 3, 8, BIG)), dict(shape=(2, 3, 2 ** 32 + 8, 16), q=2 ** 32 + 4),
    dict(pairs=2 ** 32 + 8), dict(axes=2 ** 32 + 2), dict(q=2 ** 33 + 4, kv=2 - 2 ** 32),
])
@pytest.mark.parametrize("name", ["rope_axes_forward", "rope_axes_backward"])
def test_rope_axes_refuses_sizes_past_31_bits(sa, name, change):
    v = dict(shape=(2, 3, 8, 16), pairs=8, axes=2, q=4, kv=2)
    v.update(change)
    qkv, one = torch.zeros(1).expand(v["shape"]), torch.zeros(1, dtype=torch.int64)
    positions = one.expand(v["axes"], *v["shape"][:2])
    with pytest.raises(AssertionError, match="2.31"):
        getattr(sa, name)(qkv, positions, one.expand(v["pairs"]), v["q"], v["kv"])


@pytest.mark.parametrize("shape, groups", [((BIG, 0, 8), 4), ((2, 0, 2 ** 32 + 8), 4), ((2, 0, 8), 2 ** 32 + 4), ((2, 0, 8), -4)])
def test_group_norm_refuses_sizes_past_31_bits(sa, shape, groups):
    x, stats = torch.empty(shape), torch.empty(0)
    with pytest.raises(AssertionError, match="2.31"):
        sa.group_norm_forward(x, stats, stats, x, None, None, groups)
    with pytest.raises(AssertionError, match="2.31"):
        sa.group_norm_backward(x, None, None, x, x, stats, stats, None, None, groups)


P = 1 << 20  # an address that is never read: every call here is refused on the host


@pytest.mark.parametrize("place", range(5))
@pytest.mark.parametrize("name", ["rope_forward_ptr", "rope_backward_ptr"])
def test_rope_refuses_sizes_past_31_bits(sa, name, place):
    sizes = [2, 3, 4, 2, 16]
    sizes[place] += 2 ** 32
    with pytest.raises(AssertionError, match="2.31"):
        getattr(sa, name)(P, P, *sizes, True)


@pytest.mark.parametrize("sizes", [(2 ** 32 + 64, 16), (64, 2 ** 32 + 16)])
def test_rope_precompute_freqs_refuses_sizes_past_31_bits(sa, sizes):
    with pytest.raises(AssertionError, match="2.31"):
        sa.rope_precompute_freqs_ptr(P, *sizes, 10000.0, False)


@pytest.mark.parametrize("made, axes", [(3, 2), (2, 3), (1, 2)])
@pytest.mark.parametrize("name", ["rope_axes_forward", "rope_axes_backward"])
def test_rope_axes_refuses_positions_of_other_axes(sa, name, made, axes):
    """A spectrum knows how many axes it was made with (rope_axes_spectrum sets that)."""
    spectrum = torch.zeros(8, dtype=torch.int64)
    spectrum.rope_axes = made
    with pytest.raises(AssertionError, match="axes"):
        getattr(sa, name)(torch.zeros(2, 3, 8, 16), torch.zeros(axes, 2, 3, dtype=torch.int32), spectrum, 4, 2)
