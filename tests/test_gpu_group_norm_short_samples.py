"""Group norm over many short samples (single tokens, small images): several samples share a block there.  The oracle and its
bounds are those of image_operator_reference.py; a thread adds up at most CHAIN elements of a sample or of a block's samples."""
import pytest
import torch

from tests import image_operator_reference as ref
from tests.test_gpu_image_operators import (BF16, F16, F32, check_backward, check_forward, close, framed, norm_forward, norm_inputs,
                                            randn, sa)  # noqa: F401 (sa: the fixture)

pytestmark = pytest.mark.gpu

SHAPES = [  # N, S, C, G
    (3000, 1, 128, 32), (1, 1, 64, 4), (701, 4, 64, 8), (300, 9, 6, 2), (1000, 1, 8, 2), (40, 3, 2056, 8), (513, 16, 320, 32), (64, 64, 64, 1),
    (2000, 2, 30, 30), (900, 5, 33, 3), (601, 1, 8, 8), (33, 5, 4104, 8), (9, 1, 16384, 4), (7, 1, 65536, 32), (50, 16, 4480, 70), (1200, 7, 24, 2),
    (2500, 1, 1, 1), (640, 64, 16, 16),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("shape", SHAPES)
def test_short_samples(sa, shape, silu, dtype):
    N, S, C, G = shape
    params = F32 if silu else dtype
    for shift in (0, 1):  # on and off a 16-byte boundary
        x, w, b = norm_inputs(N, S, C, dtype, params, 10 * shift, shift=shift)
        _, out, untouched = framed((N, S, C), dtype, 99, offset=shift)
        out, mean, rstd = norm_forward(sa, x, w, b, G, silu=silu, out=out)
        check_forward(x, w, b, G, silu, out, mean, rstd)
        assert untouched()
        dout = randn(N, S, C, seed=5, dtype=dtype)
        _, dx, untouched = framed((N, S, C), dtype, 98, offset=shift)
        dw, db = torch.full_like(w, 9.0), torch.full_like(b, 9.0)
        sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, w, b, G, silu=silu)
        check_backward(dout, x, mean, rstd, w, b, silu, dx, dw, db)
        assert untouched()


@pytest.mark.parametrize("shape", [(800, 1, 96, 4), (500, 8, 30, 5)])
def test_short_samples_far_from_zero_without_parameters_and_in_place(sa, shape):
    N, S, C, G = shape
    x, w, b = norm_inputs(N, S, C, F32, F32, 1, offset=1000.0)
    out, mean, rstd = norm_forward(sa, x, w, b, G)
    check_forward(x, w, b, G, True, out, mean, rstd)
    x.copy_(randn(N, S, C, seed=8))
    x[:, 0, 0] = 3e4  # an outlier that is the first element of its group
    dout = randn(N, S, C, seed=4)
    for ww, bb in ((None, None), (w, None), (None, b)):
        out, mean, rstd = norm_forward(sa, x, ww, bb, G)
        check_forward(x, ww, bb, G, True, out, mean, rstd)
        same = x.clone()
        norm_forward(sa, same, ww, bb, G, out=same)
        assert torch.equal(same, out)
        dx, dw, db = torch.empty_like(x), torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, ww, bb, G)
        check_backward(dout, x, mean, rstd, ww, bb, True, dx, dw, db)
        for over in ("dout", "x"):
            d, v = dout.clone(), x.clone()
            only = torch.empty_like(db)
            sa.group_norm_backward(d if over == "dout" else v, None, only, d, v, mean, rstd, ww, bb, G)
            assert torch.equal(d if over == "dout" else v, dx) and torch.equal(only, db)
        bare = torch.empty_like(dx)
        sa.group_norm_backward(bare, None, None, dout, x, mean, rstd, ww, bb, G)
        assert torch.equal(bare, dx)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(800, 3, 64, 8), (800, 1, 72, 24), (500, 9, 6, 2)])
def test_infinities_stay_in_their_group_of_a_short_sample(sa, shape, dtype):
    N, S, C, G = shape
    D = C // G
    x, w, b = norm_inputs(N, S, C, dtype, F32, 3)
    dout = randn(N, S, C, seed=4, dtype=dtype)

    def both(x):
        out, mean, rstd = norm_forward(sa, x, w, b, G)
        dx = torch.empty_like(x)
        sa.group_norm_backward(dx, None, None, dout, x, mean, rstd, w, b, G)
        return out, dx

    clean = both(x)
    mean, rstd, _ = ref.statistics(x.double(), G, 1e-5)
    oracle = (ref.group_norm(x.double(), w.double(), b.double(), G, 1e-5, True, dtype)[0],
              ref.group_norm_backward(dout.double(), x.double(), mean, rstd, w.double(), b.double(), True, dtype)[0])
    x[1, 0, D] = float("inf")
    x[7, S - 1, C - 1] = float("nan")
    touched = torch.zeros(N, S, C, dtype=torch.bool, device="cuda")
    touched[1, :, D:2 * D] = True
    touched[7, :, C - D:] = True
    for got, was, (value, bound) in zip(both(x), clean, oracle):
        assert torch.isnan(got[touched]).all()
        if dtype == F32:
            assert torch.equal(got[~touched], was[~touched])
        else:  # neighbouring 16-bit sigmoids share a reciprocal: the bound, not the bits
            close(got[~touched], value[~touched], bound[~touched])


def test_short_samples_same_bits_and_recorded(sa):
    N, S, C, G = 3000, 2, 160, 32
    x, w, b = norm_inputs(N, S, C, BF16, F32, 3)
    dout = randn(N, S, C, seed=4, dtype=BF16)
    out, dx, dw, db = torch.empty_like(x), torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    mean, rstd = torch.empty(N, G, device="cuda"), torch.empty(N, G, device="cuda")

    def run():
        sa.group_norm_forward(out, mean, rstd, x, w, b, G)
        sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, w, b, G)

    run()
    torch.cuda.synchronize()
    results = (out, mean, rstd, dx, dw, db)
    want = [t.clone() for t in results]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    for t in results:
        t.fill_(7)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(t, v) for t, v in zip(results, want))
