"""Group norm with SiLU where the activation's argument is far from zero: channels that a bias switches off (down to the type's
lowest value) or drives far up, beside ordinary ones of the same groups, in every way the operator has."""
import pytest
import torch

from tests import image_operator_reference as ref
from tests.test_gpu_image_operators import BF16, F16, F32, close, norm_forward, norm_inputs, randn, sa  # noqa: F401 (sa: the fixture)

pytestmark = pytest.mark.gpu

U = ref.U
DOWN = [-20.0, -30.0, -41.0, -42.0, -50.0, -60.0, -80.0, -87.0, -88.0, -95.0, -200.0, -1e4, -6e4]
FAR = [-1e18, -1e30, -3.3e38]
UP = [20.0, 300.0, 2000.0, 3e4]

SHAPES = [  # N, S, C, G: short samples, samples of a cluster's shared memory, long samples, folded rows, groups that end inside a word
    (2, 64, 64, 8), (400, 1, 96, 4), (300, 9, 30, 5), (2, 4096, 320, 32), (1, 60000, 64, 4), (1, 100000, 6, 2), (2, 3000, 42, 3),
]


def biases(C, dtype, extreme):
    """Every other channel ordinary, the others through the list in turn."""
    b = 0.3 * randn(C, seed=5)
    far = DOWN + UP + (FAR if extreme else []) + ([float(torch.finfo(dtype).min)] if extreme or dtype == F16 else [])
    for i, c in enumerate(range(1, C, 2)):
        b[c] = far[(i * 7) % len(far)]
    return b


def slope(z):
    s = torch.sigmoid(z)
    return s * (1 + z * torch.sigmoid(-z))


def sigmoid_error(z):
    """Relative error of sigmoid: two roundings of the exponent, four steps of 2^-24 for the exponential, two for the reciprocal,
    and the products and sums around them."""
    return 2 * U * z.abs() + 16 * U


# Below -87.3 sigmoid is under 2^-126 and may count as 0 (16-bit storage: numbers below that are dropped; fp32 storage: exp(-z) is
# infinite from -88.7 on).  SiLU and its slope are under 90 * 2^-126 < 2^-119 there.
def lost(z):
    return (z < -87.0) * 2.0 ** -119


def expected(x, mean, rstd, w, b, dm, dr):
    """z, and how far fp32 may be from it when mean and rstd are off by dm and dr."""
    C = x.shape[2]
    m, r, dm, dr = (ref.per_channel(v, C) for v in (mean, rstd, dm, dr))
    u = (x - m) * r
    z = u * w + b
    dz = w.abs() * (r * dm + u.abs() * (dr / r + 4 * U)) + 2 * U * (z.abs() + b.abs())
    return u, z, dz


def check(sa, shape, dtype, params, extreme, shift):
    N, S, C, G = shape
    x, w, _ = norm_inputs(N, S, C, dtype, F32, 3, shift=shift)
    b = biases(C, dtype, extreme).to(params)
    w = w.to(params)
    out, mean, rstd = norm_forward(sa, x, w, b, G)
    xd, wd, bd = x.double(), w.double(), b.double()
    exact_mean, exact_rstd, dm = ref.statistics(xd, G, 1e-5)
    dr = exact_rstd * (ref.CHAIN + (dm * exact_rstd) ** 2)
    u, z, dz = expected(xd, exact_mean, exact_rstd, wd, bd, dm, dr)
    y = z * torch.sigmoid(z)
    # y moves by at most act' times dz, and |act'| <= exp(z) (1 + |z|) below zero, 1.1 anywhere
    steep = torch.minimum(torch.exp((z + dz).clamp(max=1.0)) * (1 + z.abs() + dz), torch.full_like(z, 1.1))
    close(out, y, steep * dz + sigmoid_error(z) * y.abs() + lost(z))

    dout = randn(N, S, C, seed=6, dtype=dtype)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, w, b, G)
    zero = torch.zeros_like(dm)
    u, z, dz = expected(xd, mean.double(), rstd.double(), wd, bd, zero, zero)
    dy, s, off = dout.double(), torch.sigmoid(z), torch.sigmoid(-z)
    d = dy * slope(z)
    # |act''| <= exp(-|z|) (2 + |z|); sigmoid to its error, two roundings; 1 - sigmoid is a difference, off by a rounding of 1 + exp(-z)
    # and two steps of the reciprocal until exp(-z) is under half a rounding of 1
    bend = torch.minimum(torch.exp(-(z.abs() - dz).clamp(min=-1.0)) * (2 + z.abs() + dz), torch.full_like(z, 0.5))
    rel = sigmoid_error(z)
    d_error = dy.abs() * (bend * dz + 2 * rel * s * (1 + z.abs() * off) + 4 * U * s * (1 + z.abs() * off)
                          + 3 * U * s * z.abs() * (off > U / 4) + lost(z))
    m, r = ref.per_channel(mean.double(), C), ref.per_channel(rstd.double(), C)
    u_error = 2 * U * (xd.abs() + m.abs()) * r + U * u.abs()
    close(db, d.sum(dim=(0, 1)), ref.CHAIN * d.abs().sum(dim=(0, 1)) + d_error.sum(dim=(0, 1)))
    close(dw, (d * u).sum(dim=(0, 1)), ref.CHAIN * (d * u).abs().sum(dim=(0, 1)) + (d_error * u.abs() + d.abs() * u_error).sum(dim=(0, 1)))

    def mean_of(v):
        return ref.per_channel(v.view(N, S, G, C // G).mean(dim=(1, 3)), C)

    wz, wz_error = wd * d, wd.abs() * d_error
    m1, m2 = mean_of(wz), mean_of(wz * u)
    m1_error = ref.CHAIN * mean_of(wz.abs()) + mean_of(wz_error)
    m2_error = ref.CHAIN * mean_of((wz * u).abs()) + mean_of(wz_error * u.abs() + wz.abs() * u_error)
    close(dx, r * (wz - m1 - u * m2),
          r * (wz_error + m1_error + u.abs() * m2_error + u_error * m2.abs() + 4 * U * (wz.abs() + m1.abs() + (u * m2).abs())))


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES)
def test_channels_far_from_zero(sa, shape, dtype):
    for shift in (0, 1):  # on and off a 16-byte boundary
        check(sa, shape, dtype, F32, True, shift)
        check(sa, shape, dtype, dtype, dtype != F16, shift)
