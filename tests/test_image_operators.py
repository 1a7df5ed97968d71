"""Operators of image and video models without a GPU: the C ABI's refusals (they come before any device is touched), the
workspace's size, and the oracle in image_operator_reference.py against published values and 64-bit differentiation."""
import ctypes

import numpy as np
import pytest
import torch

import l2_torch_alloc_b200 as pkg
from l2_torch_alloc_b200 import _binding, build
from tests import image_operator_reference as ref

P = 1 << 20  # an address that is aligned and never read: every call here is refused on the host


@pytest.fixture(scope="module")
def sa():
    build.build()
    return pkg.SideAware()


def refused(sa, rc, text):
    assert rc == 1 and text in sa.last_error(), (rc, sa.last_error())


def rope_shape(**change):
    v = dict(B=2, T=3, Nq=4, Nkv=2, HS=16, pairs=8, axes=2, layout=0, dtype=1, position_dtype=0, stride_b=3 * 128, stride_t=128,
             pos_stride_axis=6, pos_stride_b=3, pos_stride_t=1)
    v.update(change)
    return _binding.RopeAxes(**v)


@pytest.mark.parametrize("change, text", [
    ({"B": -1}, "negative"), ({"HS": 0}, "negative"), ({"axes": 0}, "axes"), ({"axes": 9}, "axes"), ({"pairs": 0}, "pairs"),
    ({"pairs": 9}, "pairs"), ({"layout": 2}, "layout"), ({"dtype": 3}, "dtype"), ({"position_dtype": 2}, "position_dtype"),
    ({"stride_t": 127}, "shorter than a row"), ({"stride_t": -128}, "shorter than a row"), ({"stride_b": 0}, "shorter than a row"),
    ({"stride_b": 200}, "overlap"), ({"B": 1 << 20, "T": 1 << 20}, "tokens"),
])
@pytest.mark.parametrize("name", ["sideaware_rope_axes_forward", "sideaware_rope_axes_backward"])
def test_rope_axes_refuses(sa, name, change, text):
    refused(sa, getattr(sa.lib, name)(P, P, P, ctypes.byref(rope_shape(**change)), 0, None), text)


def test_rope_axes_overlap_is_found_past_64_bits(sa):
    """(T - 1) * stride_t is 2^64 - 2^40 here: rows of the second sample lie among those of the first."""
    s = rope_shape(B=2, T=1 << 24, stride_t=1 << 40, stride_b=1 << 41)
    refused(sa, sa.lib.sideaware_rope_axes_forward(P, P, P, ctypes.byref(s), 0, None), "overlap")


def test_rope_axes_refuses_pointers(sa):
    call, s = sa.lib.sideaware_rope_axes_forward, rope_shape()
    for args in ((None, P, P), (P, None, P), (P, P, None)):
        refused(sa, call(*args, ctypes.byref(s), 0, None), "null pointer")
    for args in ((P + 1, P, P), (P, P + 2, P), (P, P, P + 4)):
        refused(sa, call(*args, ctypes.byref(s), 0, None), "not aligned")
    refused(sa, call(P, P, P, None, 0, None), "no shape")
    for empty in ({"B": 0}, {"T": 0}, {"Nq": 0, "Nkv": 0}):
        assert call(None, None, None, ctypes.byref(rope_shape(**empty)), 0, None) == 0


@pytest.mark.parametrize("pairs, theta, arrangement, text", [
    ([], 1e4, 0, "axes"), ([1] * 9, 1e4, 0, "axes"), ([0, 0], 1e4, 0, "pairs"), ([200, 57], 1e4, 0, "pairs"), ([-1, 4], 1e4, 0, "negative"),
    ([4], 0.0, 0, "theta"), ([4], float("nan"), 0, "theta"), ([4], float("inf"), 0, "theta"), ([4], 1e4, 3, "arrangement"),
])
def test_rope_axes_spectrum_refuses(sa, pairs, theta, arrangement, text):
    array = (ctypes.c_int * max(1, len(pairs)))(*pairs)
    refused(sa, sa.lib.sideaware_rope_axes_spectrum(P, array, len(pairs), theta, arrangement, 0, None), text)


def norm_shape(**change):
    v = dict(S=10, N=2, C=12, G=4, eps=1e-5, silu=1, dtype=1, param_dtype=0)
    v.update(change)
    return _binding.GroupNorm(**v)


def norm_forward(sa, s, out=P, mean=P, rstd=P, x=P, w=P, b=P, workspace=P, size=1 << 30):
    return sa.lib.sideaware_group_norm_forward(out, mean, rstd, x, w, b, ctypes.byref(s), workspace, size, 0, None)


def norm_backward(sa, s, dx=P, dw=P, db=P, dy=P, x=P, mean=P, rstd=P, w=P, b=P, workspace=P, size=1 << 30):
    return sa.lib.sideaware_group_norm_backward(dx, dw, db, dy, x, mean, rstd, w, b, ctypes.byref(s), workspace, size, 0, None)


@pytest.mark.parametrize("change, text", [
    ({"C": 13}, "evenly"), ({"G": 0}, "positive"), ({"N": -1}, "negative"), ({"C": 1 << 21}, "2^20"), ({"dtype": 3}, "dtypes"),
    ({"param_dtype": -1}, "dtypes"), ({"eps": -1.0}, "eps"), ({"eps": float("nan")}, "eps"), ({"silu": 2}, "silu"),
    ({"N": 1 << 24}, "2^24"), ({"S": 1 << 50}, "10^13"), ({"S": 0}, "elements"),
])
def test_group_norm_refuses(sa, change, text):
    refused(sa, norm_forward(sa, norm_shape(**change)), text)
    refused(sa, norm_backward(sa, norm_shape(**change)), text)


def test_group_norm_refuses_pointers_and_workspaces(sa):
    s = norm_shape()
    for name in ("out", "mean", "rstd", "x"):
        refused(sa, norm_forward(sa, s, **{name: None}), "null pointer")
        refused(sa, norm_forward(sa, s, **{name: P + 1}), "not aligned")
    for name in ("dx", "dy", "x", "mean", "rstd"):
        refused(sa, norm_backward(sa, s, **{name: None}), "null pointer")
        refused(sa, norm_backward(sa, s, **{name: P + 1}), "not aligned")
    for name in ("w", "b", "dw", "db"):
        refused(sa, norm_backward(sa, s, **{name: P + 2}), "not aligned")
    refused(sa, norm_forward(sa, s, out=P + 32), "overlaps")
    refused(sa, norm_backward(sa, s, dx=P + 32), "overlaps")
    # a shape that needs a workspace whatever path it takes
    s = norm_shape(S=1 << 20, C=64, N=1)
    for backward, call in ((0, norm_forward), (1, norm_backward)):
        need = sa.lib.sideaware_group_norm_workspace(ctypes.byref(s), backward)
        assert 0 < need < 1 << 30
        refused(sa, call(sa, s, size=need - 1), "workspace")
        refused(sa, call(sa, s, workspace=None), "workspace")
        refused(sa, call(sa, s, workspace=P + 8), "workspace")


def test_dropout_refuses(sa):
    call = sa.lib.sideaware_dropout_forward
    for p in (-0.1, 1.1, float("nan")):
        refused(sa, call(P, P, None, P, p, 8, 1, 0, None), "[0, 1]")
    refused(sa, call(P, P, None, P, 0.1, 8, 3, 0, None), "dtype")
    refused(sa, call(P, P, None, P, 0.1, 1 << 44, 1, 0, None), "2^43")
    for args in ((None, P, None, P), (P, None, None, P), (P, P, None, None)):
        refused(sa, call(*args, 0.1, 8, 1, 0, None), "null pointer")
    for args in ((P + 1, P, None, P), (P, P + 1, None, P), (P, P, P + 1, P), (P, P, None, P + 8)):
        refused(sa, call(*args, 0.1, 8, 1, 0, None), "not aligned")
    refused(sa, call(P + 2, P, None, P, 0.1, 8, 1, 0, None), "overlaps")
    refused(sa, call(P, P + 512, P - 2, P, 0.1, 8, 1, 0, None), "overlaps")
    refused(sa, sa.lib.sideaware_dropout_backward(P + 2, P, P, 0.1, 8, 1, 0, None), "overlaps")
    assert call(None, None, None, None, 0.1, 0, 1, 0, None) == 0  # nothing to do


def test_philox_of_the_oracle_gives_the_published_blocks():
    assert ref.philox([0] * 4, [0] * 2) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    assert ref.philox([0xFFFFFFFF] * 4, [0xFFFFFFFF] * 2) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    assert ref.philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], [0xA4093822, 0x299F31D0]) == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]
    # the numpy form agrees with the integer form, element by element
    seed, call, n, p = 0x0123456789ABCDEF, 0x1122334455667788, 43, 0.37
    want = []
    for i in range(n):
        c = [i // 8, 0, call & 0xFFFFFFFF, call >> 32]
        k = [seed & 0xFFFFFFFF, seed >> 32]
        upper, lower = ref.philox(c, k)[i % 8 // 2], ref.philox([c[0], 0x80000000, c[2], c[3]], k)[i % 8 // 2]
        shift = 16 * (i % 2)
        want.append((((upper >> shift) & 0xFFFF) << 16 | (lower >> shift) & 0xFFFF) >= round(p * 2 ** 32))
    assert np.array_equal(ref.keep_mask(n, seed, call, p), want)


@pytest.mark.parametrize("silu", [False, True])
def test_backward_formula_of_the_oracle_against_differentiation(silu):
    g = torch.Generator().manual_seed(3)
    N, S, C, G = 2, 5, 6, 3
    x, dy = (torch.randn(N, S, C, generator=g, dtype=torch.float64) for _ in range(2))
    w, b = (torch.randn(C, generator=g, dtype=torch.float64) for _ in range(2))

    def f(x, w, b):
        return ref.group_norm(x, w, b, G, 1e-5, silu, torch.float64)[0][0]

    leaves = [v.clone().requires_grad_() for v in (x, w, b)]
    want = torch.autograd.grad(f(*leaves), leaves, dy)
    mean, rstd, _ = ref.statistics(x, G, 1e-5)
    got = ref.group_norm_backward(dy, x, mean, rstd, w, b, silu, torch.float64)
    for (value, _), other in zip(got, want):
        assert torch.allclose(value, other, rtol=1e-10, atol=1e-10)
    # and against central differences along a random direction
    step, way = 1e-6, [torch.randn(v.shape, generator=g, dtype=torch.float64) for v in (x, w, b)]
    ahead = (f(*(v + step * d for v, d in zip((x, w, b), way))) * dy).sum()
    behind = (f(*(v - step * d for v, d in zip((x, w, b), way))) * dy).sum()
    along = sum((value * d).sum() for (value, _), d in zip(got, way))
    assert abs((ahead - behind) / (2 * step) - along) < 1e-6 * (1 + abs(along))


def test_python_wrappers_refuse_cpu_tensors(sa):
    x = torch.zeros(2, 3, 8)
    with pytest.raises(AssertionError, match="CUDA"):
        sa.dropout_forward(x, x, torch.zeros(2, dtype=torch.int64), 0.1)
    with pytest.raises(AssertionError, match="CUDA"):
        sa.group_norm_forward(x, x, x, x, None, None, 2)
    with pytest.raises(AssertionError, match="CUDA"):
        sa.rope_axes_forward(torch.zeros(1, 2, 3, 8), torch.zeros(1, 1, 2, dtype=torch.int32), torch.zeros(4, dtype=torch.int64), 1, 1)


@pytest.mark.parametrize("device", ["cpu", torch.device("cpu", 0), "meta"])
def test_rope_axes_spectrum_refuses_devices_that_are_not_cuda(sa, device):
    """Refused before anything is allocated or launched: the kernel would write through a host address."""
    with pytest.raises(AssertionError, match="CUDA"):
        sa.rope_axes_spectrum((4, 4), device=device)
