"""Group norm of data whose mean is far from zero, in every way the operator has: the statistics are held to roundings of the mean,
not to sums of values of its size."""
import pytest
import torch

from tests import image_operator_reference as ref
from tests.test_gpu_image_operators import BF16, F16, F32, close, norm_forward, randn, sa  # noqa: F401 (sa: the fixture)

pytestmark = pytest.mark.gpu

U = ref.U
SHAPES = [  # N, S, C, G: short samples, samples of a cluster's shared memory, long samples (several slabs, folded rows, single elements)
    (300, 1, 96, 4), (2, 64, 64, 8), (300, 9, 30, 5), (2, 4096, 320, 32), (3, 1000, 96, 2), (1, 2048, 1280, 1), (1, 60000, 64, 4),
    (2, 100000, 330, 2), (1, 100000, 6, 2), (1, 30000, 2056, 8), (1, 200001, 5, 1),
]


@pytest.mark.parametrize("shape", SHAPES)
def test_constant_input(sa, shape):
    """Every deviation from one of the data is exactly 0, so the mean is that value, the variance 0 and the output the bias."""
    N, S, C, G = shape
    w, b = 1 + 0.3 * randn(C, seed=2), 0.3 * randn(C, seed=3)
    for dtype, value in ((F32, 1000.1), (F32, -12345.678), (F32, 1e6 + 0.3), (BF16, 777.7), (F16, -4321.0)):
        x = torch.full((N, S, C), value, dtype=dtype, device="cuda")
        out, mean, rstd = norm_forward(sa, x, w, b, G, silu=False)
        assert torch.equal(mean, x[:, 0, :1].float().expand(N, G)), (value, mean.flatten()[:4])
        close(rstd, torch.full_like(rstd.double(), 1e-5).rsqrt(), 2 * U * rstd.double())  # eps in fp32, its root
        assert torch.equal(out, b.to(dtype).expand(N, S, C)), value


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("offset", [1e3, -3e5])
def test_mean_far_from_zero(sa, shape, offset):
    """Roundings of values of the mean's size, one after the other: those of a thread's rows, the channel's, the group's; 3 joins of
    a cluster's blocks or, of a long sample, a join for every 32 rows of a thread (a row lane has at most S / 444 + 8) and 10 of runs.
    Beside them the spread about the mean, to CHAIN."""
    N, S, C, G = shape
    x = randn(N, S, C, seed=7) * 2 + offset
    out, mean, rstd = norm_forward(sa, x, None, None, G, silu=False)
    g = x.double().view(N, S, G, C // G)
    exact = g.mean(dim=(1, 3))
    spread = (g - exact[:, None, :, None]).abs().amax(dim=(1, 3))
    steps = 3 + (3 if S < 5000 else 10 + (S / 444 + 8) / 32)
    close(mean, exact, steps * U * exact.abs() + ref.CHAIN * spread)


@pytest.mark.parametrize("shape", SHAPES)
def test_large_numbers(sa, shape):
    """The square of a value is past fp32's range, that of a deviation is not."""
    N, S, C, G = shape
    x = torch.full((N, S, C), 1e30, device="cuda")
    out, mean, rstd = norm_forward(sa, x, None, None, G, silu=False)
    assert torch.equal(mean, x[:, 0, :1].expand(N, G)) and not out.any()
    close(rstd, torch.full_like(rstd.double(), 1e-5).rsqrt(), 2 * U * rstd.double())
    x = randn(N, S, C, seed=7) * 1e15 + 1e20
    out, mean, rstd = norm_forward(sa, x, None, None, G, silu=False)
    g = x.double().view(N, S, G, C // G)
    exact = g.mean(dim=(1, 3))
    deviation = g - exact[:, None, :, None]
    error = (3 + (3 if S < 5000 else 10 + (S / 444 + 8) / 32)) * U * exact.abs() + ref.CHAIN * deviation.abs().amax(dim=(1, 3))
    close(mean, exact, error)
    if S * C // G > 1:  # every deviation is off by the error of what it is taken about, twice at most: the square by 2 e |d| + e^2
        var = deviation.square().mean(dim=(1, 3))
        off = 2 * error * deviation.abs().mean(dim=(1, 3)) + error.square() + ref.CHAIN * var
        limit = (var - 2 * off).clamp(min=1e-30).rsqrt() - var.rsqrt()
        close(rstd, var.rsqrt(), limit)
