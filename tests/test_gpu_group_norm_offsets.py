"""Group norm over more than 2^31 elements, forward and backward, against the definition in 64 bits taken piece by piece."""
import pytest
import torch

from tests import image_operator_reference as ref
from tests.test_gpu_image_operators import BF16, close, norm_forward, randn, sa  # noqa: F401 (sa: the fixture)

pytestmark = pytest.mark.gpu

U = ref.U


def test_backward_offsets_past_31_bits(sa):
    N, S, C, G = 3, (1 << 23) - 5, 96, 32
    piece = 1 << 19
    x = torch.empty(N, S, C, dtype=BF16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(1))
    x += 0.5 * torch.arange(1, N + 1, device="cuda", dtype=BF16).view(N, 1, 1)  # samples differ: one for another would show
    dout = torch.empty_like(x).normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    assert x.numel() > 2 ** 31
    w, b = 1 + 0.3 * randn(C, seed=3), 0.3 * randn(C, seed=4)
    out, mean, rstd = norm_forward(sa, x, w, b, G)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, w, b, G)
    # a row lane adds up S / (148 * 21) = 2,700 rows one after the other, then lanes, runs and shares: under 4,096 roundings
    chain = 4096 * U
    wd, bd = w.double(), b.double()
    sums = torch.zeros(4, C, dtype=torch.float64, device="cuda")  # of dz, dz u and their errors over all samples
    for n in range(N):
        m, r = ref.per_channel(mean[n:n + 1].double(), C)[0], ref.per_channel(rstd[n:n + 1].double(), C)[0]

        def of(rows):
            """u and dz of some rows, and how far fp32 may be off."""
            v, dy = x[n, rows].double(), dout[n, rows].double()
            u = (v - m) * r
            z = u * wd + bd
            s = torch.sigmoid(z)
            dz = dy * s * (1 + z * (1 - s))
            dz_error = dy.abs() * ((ref.sigmoid_error(BF16) + 8 * U) * (1 + z.abs()) * s + 0.5 * 4 * U * ((u * wd).abs() + bd.abs()))
            return u, z, dz, dz_error, 2 * U * (v.abs() + m.abs()) * r + U * u.abs()

        totals, value_sums = torch.zeros(4, C, dtype=torch.float64, device="cuda"), torch.zeros(2, C, dtype=torch.float64, device="cuda")
        for r0 in range(0, S, piece):
            u, _, dz, dz_error, u_error = of(slice(r0, min(S, r0 + piece)))
            v = x[n, r0:r0 + piece].double()
            value_sums += torch.stack((v.sum(0), v.square().sum(0)))
            totals += torch.stack((dz.sum(0), (dz * u).sum(0), (chain * dz.abs() + dz_error).sum(0),
                                   (chain * (dz * u).abs() + dz_error * u.abs() + dz.abs() * u_error).sum(0)))
        sums += totals
        # the forward pass's statistics (data of variance 1 and means up to 1.5)
        first, second = (t.view(G, -1).mean(1) / S for t in value_sums)
        close(mean[n], first, chain * 8)
        close(rstd[n], (second - first.square() + 1e-5).rsqrt(), torch.full_like(first, 2 * chain))

        def of_group(t):
            return (t.view(G, -1).mean(1) / S).repeat_interleave(C // G)

        m1, m2 = of_group(wd * totals[0]), of_group(wd * totals[1])
        m1_error, m2_error = of_group(wd.abs() * totals[2]), of_group(wd.abs() * totals[3])
        for rows in (slice(0, 500), slice(S // 2, S // 2 + 500), slice(S - 500, S)):
            u, z, dz, dz_error, u_error = of(rows)
            d = wd * dz
            close(dx[n, rows], r * (d - m1 - u * m2),
                  r * (wd.abs() * dz_error + m1_error + u.abs() * m2_error + u_error * m2.abs() + 4 * U * (d.abs() + m1.abs() + (u * m2).abs())))
            close(out[n, rows], z * torch.sigmoid(z), 1.1 * (wd.abs() * u_error + 4 * U * (z.abs() + bd.abs())) + ref.sigmoid_error(BF16) * z.abs())
    close(db, sums[0], sums[2])
    close(dw, sums[1], sums[3])
