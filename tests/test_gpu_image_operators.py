"""Operators of image and video models on a B200 against their definitions in 64 bits: rotary positions with several axes,
group norm with SiLU (channels last), dropout with a redrawn mask; forward and backward, at the sizes where they can go wrong,
on other streams, in recorded graphs, and together as the blocks of a model."""

import os
import subprocess
import sys

import numpy as np
import pytest
import torch

from tests import image_operator_reference as ref

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def sa():
    assert torch.cuda.is_available(), "GPU tests need a CUDA device"
    import l2_torch_alloc_b200 as pkg
    return pkg.SideAware()


def randn(*shape, seed, dtype=F32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=g).to(dtype)


def close(got, want, bound, dtype=None):
    """got within bound of want after a rounding to dtype; NaN and infinities in the same places."""
    dtype = dtype or got.dtype
    got, limit = got.double(), ref.rounded(bound, want, dtype)
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    over = ((got - want).abs() > limit) & fine
    assert not over.any(), f"{int(over.sum())} of {over.numel()} off, worst {float(((got - want).abs() / limit)[fine].max()):.3g} of the bound"


def framed(shape, dtype, seed, front=64, back=64, offset=0):
    """A dense tensor inside a larger buffer whose ends show stray writes; offset: elements away from a 16-byte boundary."""
    n = int(np.prod(shape))
    buffer = torch.full((front + offset + n + back,), 123.0, dtype=dtype, device="cuda")
    view = buffer[front + offset:front + offset + n].view(shape)
    if n:
        view.copy_(randn(*shape, seed=seed, dtype=dtype))
    return buffer, view, lambda: bool((buffer[:front + offset] == 123).all() and (buffer[front + offset + n:] == 123).all())


# ---------------------------------------------------------------------------
# rotary positions with several axes
# ---------------------------------------------------------------------------
ROPE_SHAPES = [  # B, T, q, kv, head, pairs of the axes
    (1, 1, 1, 0, 2, (1,)), (2, 3, 1, 1, 8, (2, 2)), (1, 1, 32, 8, 128, (16, 24, 24)), (3, 17, 5, 2, 72, (18, 18)),
    (2, 33, 4, 4, 64, (10, 11, 11)), (1, 5, 7, 1, 6, (1, 2)), (2, 9, 3, 3, 96, (5, 7, 12)), (1, 1000, 2, 1, 80, (40,)),
    (1, 2, 64, 8, 512, (64, 64, 64, 64)), (5, 1, 6, 6, 36, (9, 9)), (1, 130, 12, 0, 32, (3, 0, 13)), (2, 2, 1, 1, 256, (16,) * 8),
    (1, 3, 300, 100, 64, (32,)),
]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("shape", ROPE_SHAPES)
def test_rope_axes(sa, shape, layout, dtype):
    B, T, q, kv, head, pairs = shape
    for seed, (arrangement, inverse, wide, offset) in enumerate([("own", False, False, 0), ("shared", True, True, 0), ("interleaved", False, True, 1)]):
        buffer, x, untouched = framed((B, T, q + 2 * kv, head), dtype, seed, offset=offset)
        before = x.clone()
        g = torch.Generator(device="cuda").manual_seed(seed)
        far = [100, 2 ** 31 - 1, 10 ** 6][seed]
        positions = torch.randint(-far, far, (len(pairs), B, T), device="cuda", generator=g)
        positions = positions if wide else positions.int()
        theta = [10000.0, 500000.0, 100.0][seed]
        spectrum = sa.rope_axes_spectrum(pairs, theta, arrangement)
        (sa.rope_axes_backward if inverse else sa.rope_axes_forward)(x, positions, spectrum, q, kv, layout)
        want, bound = ref.rope(before.double(), positions, pairs, theta, arrangement, q, kv, layout, inverse)
        close(x, want, bound)
        assert untouched()
        # value heads and the part of a head without pairs: the same bits
        assert torch.equal(x[:, :, q + kv:], before[:, :, q + kv:]) and torch.equal(x[..., 2 * sum(pairs):], before[..., 2 * sum(pairs):])


@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_rope_axes_strides(sa, layout):
    """Rows with room between them, time-major memory, positions shared by all sequences or all axes."""
    B, T, q, kv, head, pairs = 3, 7, 4, 2, 64, (8, 12, 12)
    H = q + 2 * kv
    spectrum = sa.rope_axes_spectrum(pairs)
    padded = randn(B, T + 2, H * head + 40, seed=1, dtype=BF16)
    time_major = randn(T, B, H, head, seed=2, dtype=BF16)
    cases = [padded[:, :T, 8:8 + H * head].unflatten(-1, (H, head)),
             padded[:, 1:T + 1, 3:3 + H * head].unflatten(-1, (H, head)), time_major.transpose(0, 1)]
    g = torch.Generator(device="cuda").manual_seed(5)
    full = torch.randint(0, 5000, (3, B, T), device="cuda", generator=g)
    places = [full, full[:, :1].expand(3, B, T), full[:1].expand(3, B, T), full.permute(2, 1, 0).contiguous().permute(2, 1, 0),
              torch.randint(0, 99, (3, B, 2 * T), device="cuda", generator=g, dtype=torch.int32)[..., ::2]]
    for x in cases:
        for positions in places:
            whole, before = (x._base if x._base is not None else x).clone(), x.clone()
            sa.rope_axes_forward(x, positions, spectrum, q, kv, layout)
            want, bound = ref.rope(before.double(), positions, pairs, 10000.0, "own", q, kv, layout)
            close(x, want, bound)
            x.copy_(before)
            assert torch.equal(whole, x._base if x._base is not None else x), "nothing outside the view was written"


@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_rope_axes_offsets_past_31_bits(sa, layout):
    """More than 2^31 elements: the last tokens against the oracle, a middle one untouched by its neighbours' turns."""
    T, q, kv, head = 360_000, 40, 4, 128
    x = torch.zeros(1, T, q + 2 * kv, head, dtype=BF16, device="cuda")
    assert x.numel() > 2 ** 31
    x[:, -50:] = randn(1, 50, q + 2 * kv, head, seed=3, dtype=BF16)
    before = x[:, -50:].clone()
    positions = torch.arange(T, device="cuda").expand(2, 1, T)
    sa.rope_axes_forward(x, positions, sa.rope_axes_spectrum((32, 32)), q, kv, layout)
    want, bound = ref.rope(before.double(), positions[:, :, -50:], (32, 32), 10000.0, "own", q, kv, layout)
    close(x[:, -50:], want, bound)
    assert not x[:, :-50].any()


def test_rope_axes_text_positions_equal_one_axis(sa):
    """Equal positions on all axes with the shared spectrum are the ordinary rotary embedding: the same as one axis, bit for bit."""
    q, kv, head = 4, 2, 64
    a = randn(2, 50, q + 2 * kv, head, seed=1)
    b = a.clone()
    t = torch.arange(50, device="cuda").expand(1, 2, 50)
    sa.rope_axes_forward(a, t.expand(3, 2, 50), sa.rope_axes_spectrum((8, 12, 12), 10000.0, "shared"), q, kv)
    sa.rope_axes_forward(b, t, sa.rope_axes_spectrum((32,), 10000.0, "shared"), q, kv)
    assert torch.equal(a, b)
    # and the table-driven kernel gives the same to fp32 rounding of its angles (|angle| < 50: 3 roundings of it)
    c = randn(2, 50, q + 2 * kv, head, seed=1)
    sa.rope_forward(c, sa.rope_precompute_freqs(head, 50), q, kv)
    assert ((a - c).abs() <= (10 + 3 * 50) * ref.U * 2 * c.abs().max()).all()


def test_rope_axes_backward_is_the_gradient(sa):
    """The backward pass against central differences of the 64-bit definition and against its transpose."""
    B, T, q, kv, head, pairs = 2, 5, 2, 1, 16, (3, 5)
    positions = torch.randint(0, 300, (2, B, T), device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
    x, dy, way = (randn(B, T, q + 2 * kv, head, seed=s).double() for s in (1, 2, 3))

    def f(v):
        return ref.rope(v, positions, pairs, 10000.0, "own", q, kv, "halves")[0]

    along = ((f(x + 1e-5 * way) - f(x - 1e-5 * way)) / 2e-5 * dy).sum()
    dx = dy.float()
    sa.rope_axes_backward(dx, positions, sa.rope_axes_spectrum(pairs), q, kv, "halves")
    assert abs(float((dx.double() * way).sum() - along)) < 1e-5 * float((dy.abs() * way.abs()).sum())


def test_rope_axes_refusals(sa):
    x, places = randn(2, 3, 8, 16, seed=1), torch.zeros(2, 2, 3, dtype=torch.int32, device="cuda")
    spectrum = sa.rope_axes_spectrum((4, 4))
    for bad in (dict(qkv=x[..., :8]), dict(qkv=x.transpose(2, 3)), dict(positions=places[:, :1]), dict(positions=places.float()),
                dict(spectrum=spectrum.int()), dict(qkv=x.double()), dict(n_q_heads=5), dict(layout="other"), dict(positions=places.cpu())):
        args = dict(qkv=x, positions=places, spectrum=spectrum, n_q_heads=4, n_kv_heads=2)
        args.update(bad)
        with pytest.raises(AssertionError):
            sa.rope_axes_forward(**args)
    with pytest.raises(RuntimeError, match="pairs"):
        sa.rope_axes_forward(x, places, sa.rope_axes_spectrum((8, 8)), 4, 2)
    with pytest.raises(RuntimeError, match="stride"):
        sa.rope_axes_forward(x[:, :1].expand(2, 3, 8, 16), places, spectrum, 4, 2)
    sa.rope_axes_forward(x[:, :0], places[:, :, :0], spectrum, 4, 2)  # nothing to do
    sa.rope_axes_forward(x[:0], places[:, :0], spectrum, 4, 2)


# ---------------------------------------------------------------------------
# group norm
# ---------------------------------------------------------------------------
NORM_SHAPES = [  # N, S, C, G
    (1, 1, 1, 1), (2, 7, 6, 3), (1, 64, 1280, 32), (3, 33, 96, 32), (2, 1000, 320, 32), (1, 5, 2048, 1), (2, 300, 40, 40),
    (1, 4099, 48, 16), (4, 257, 64, 2), (1, 1, 512, 32), (2, 9, 30, 2), (1, 70001, 8, 4), (17, 16, 160, 32), (1, 3000, 4104, 8),
    (2, 16384, 128, 32), (1, 40000, 256, 32),
    # long samples: whole words, rows folded to whole words (2, 4 and 8 pixels), rows that cannot be
    (2, 150000, 24, 3), (1, 300000, 64, 4), (2, 100000, 330, 2), (1, 600000, 6, 2), (2, 262144, 1, 1), (1, 400004, 10, 1), (3, 80001, 12, 3),
    (1, 200001, 5, 5), (1, 30000, 2056, 8),
]


def norm_inputs(N, S, C, dtype, params, seed, offset=0.0, shift=0):
    _, x, _ = framed((N, S, C), dtype, seed, offset=shift)
    x.copy_((x.float() * (0.5 + torch.rand(C, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
             + 0.3 * randn(N, 1, C, seed=seed + 1) + offset).to(dtype))
    w, b = (1 + 0.3 * randn(C, seed=seed + 2)).to(params), (0.3 * randn(C, seed=seed + 3)).to(params)
    return x, w, b


def norm_forward(sa, x, w, b, G, eps=1e-5, silu=True, out=None):
    N = x.shape[0]
    out = torch.empty_like(x) if out is None else out
    mean, rstd = (torch.full((N, G), 7.0, device="cuda") for _ in range(2))
    sa.group_norm_forward(out, mean, rstd, x, w, b, G, eps, silu)
    return out, mean, rstd


def check_forward(x, w, b, G, silu, out, mean, rstd, eps=1e-5):
    C = x.shape[-1]
    wd = torch.ones(C, dtype=torch.float64, device="cuda") if w is None else w.double()
    bd = torch.zeros(C, dtype=torch.float64, device="cuda") if b is None else b.double()
    (y, dy), (m, dm), (r, dr) = ref.group_norm(x.double().reshape(x.shape[0], -1, C), wd, bd, G, eps, silu, out.dtype)
    close(mean, m, dm)
    close(rstd, r, dr)
    close(out.reshape(y.shape), y, dy)


def check_backward(dout, x, mean, rstd, w, b, silu, dx, dw, db):
    C = x.shape[-1]
    wd = torch.ones(C, dtype=torch.float64, device="cuda") if w is None else w.double()
    bd = torch.zeros(C, dtype=torch.float64, device="cuda") if b is None else b.double()
    want = ref.group_norm_backward(dout.double(), x.double(), mean.double(), rstd.double(), wd, bd, silu, x.dtype)
    for got, (value, bound) in zip((dx, dw, db), want):
        if got is not None:
            close(got, value, bound)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("silu", [True, False])
@pytest.mark.parametrize("shape", NORM_SHAPES)
def test_group_norm(sa, shape, silu, dtype):
    N, S, C, G = shape
    params = F32 if silu else dtype
    for shift in (0, 1):  # on and off a 16-byte boundary
        x, w, b = norm_inputs(N, S, C, dtype, params, 10 * shift, shift=shift)
        buffer, out, untouched = framed((N, S, C), dtype, 99, offset=shift)
        out, mean, rstd = norm_forward(sa, x, w, b, G, silu=silu, out=out)
        check_forward(x, w, b, G, silu, out, mean, rstd)
        assert untouched()
        dout = randn(N, S, C, seed=5, dtype=dtype)
        buffer, dx, untouched = framed((N, S, C), dtype, 98, offset=shift)
        dw, db = torch.full_like(w, 9.0), torch.full_like(b, 9.0)
        sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, w, b, G, silu=silu)
        check_backward(dout, x, mean, rstd, w, b, silu, dx, dw, db)
        assert untouched()


@pytest.mark.parametrize("shape", [(2, 1000, 320, 32), (1, 64, 64, 8), (2, 300, 30, 3), (1, 60000, 64, 4)])
def test_group_norm_far_from_zero_and_constant(sa, shape):
    N, S, C, G = shape
    x, w, b = norm_inputs(N, S, C, F32, F32, 1, offset=1000.0)
    out, mean, rstd = norm_forward(sa, x, w, b, G)
    check_forward(x, w, b, G, True, out, mean, rstd)
    x.fill_(3.25)  # no variance: rstd = 1 / sqrt(eps), z = b
    out, mean, rstd = norm_forward(sa, x, w, b, G)
    check_forward(x, w, b, G, True, out, mean, rstd)
    dout = randn(N, S, C, seed=5)
    dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, w, b, G)
    check_backward(dout, x, mean, rstd, w, b, True, dx, dw, db)
    # one far outlier in an otherwise ordinary group
    x.copy_(randn(N, S, C, seed=8))
    x[0, 0, 0] = 3e4
    out, mean, rstd = norm_forward(sa, x, w, b, G, silu=False)
    check_forward(x, w, b, G, False, out, mean, rstd)


@pytest.mark.parametrize("shape", [(2, 100, 64, 4), (1, 9, 30, 5), (1, 50000, 32, 4)])
def test_group_norm_without_parameters_and_in_place(sa, shape):
    N, S, C, G = shape
    x, w, b = norm_inputs(N, S, C, BF16, F32, 3)
    for ww, bb in ((None, None), (w, None), (None, b)):
        out, mean, rstd = norm_forward(sa, x, ww, bb, G)
        check_forward(x, ww, bb, G, True, out, mean, rstd)
        same = x.clone()
        norm_forward(sa, same, ww, bb, G, out=same)
        assert torch.equal(same, out)
        dout = randn(N, S, C, seed=4, dtype=BF16)
        dx, dw, db = torch.empty_like(x), torch.empty(C, device="cuda"), torch.empty(C, device="cuda")
        sa.group_norm_backward(dx, dw, db, dout, x, mean, rstd, ww, bb, G)
        check_backward(dout, x, mean, rstd, ww, bb, True, dx, dw, db)
        for over in ("dout", "x"):
            d, v = dout.clone(), x.clone()
            only = torch.empty_like(db)
            sa.group_norm_backward(d if over == "dout" else v, None, only, d, v, mean, rstd, ww, bb, G)
            assert torch.equal(d if over == "dout" else v, dx) and torch.equal(only, db)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(2, 500, 64, 8), (2, 500, 72, 24), (2, 120000, 48, 16), (2, 200000, 6, 2)])
def test_group_norm_infinities_stay_in_their_group(sa, shape, dtype):
    """Groups of odd sizes share words and f32x2 pairs with their neighbours: nothing passes over, forward or backward."""
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
    x[1, 7, D] = float("inf")       # sample 1, group 1
    x[0, 3, C - 1] = float("nan")   # sample 0, the last group
    touched = torch.zeros(N, S, C, dtype=torch.bool, device="cuda")
    touched[1, :, D:2 * D] = True
    touched[0, :, C - D:] = True
    for got, was, (value, bound) in zip(both(x), clean, oracle):
        assert torch.isnan(got[touched]).all()
        if dtype == F32:
            assert torch.equal(got[~touched], was[~touched])
        else:
            # two 16-bit sigmoids share a reciprocal, r = 1 / (a b), so a's last bits do depend on b: r b and its three
            # roundings stay within the oracle's bound whatever b is, equality of bits is not to be had
            close(got[~touched], value[~touched], bound[~touched])


def test_group_norm_spatial_shapes_and_refusals(sa):
    image = randn(2, 8, 6, 5, seed=1).to(memory_format=torch.channels_last)  # [N, C, H, W] in channels-last memory
    view = image.permute(0, 2, 3, 1)
    out, mean, rstd = norm_forward(sa, view, None, None, 4)
    check_forward(view.reshape(2, 30, 8), None, None, 4, True, out.reshape(2, 30, 8), mean, rstd)
    x = randn(2, 12, 8, seed=2)
    ok = dict(out=torch.empty_like(x), mean=torch.empty(2, 4, device="cuda"), rstd=torch.empty(2, 4, device="cuda"), x=x, weight=None, bias=None, groups=4)
    for bad in (dict(x=image), dict(groups=3), dict(out=torch.empty(2, 12, 9, device="cuda")), dict(out=torch.empty_like(x).half()),
                dict(mean=torch.empty(2, 5, device="cuda")), dict(rstd=torch.empty(2, 4, device="cuda", dtype=F16)),
                dict(weight=torch.ones(9, device="cuda")), dict(weight=torch.ones(8, device="cuda"), bias=torch.ones(8, device="cuda").half()),
                dict(x=x.double(), out=torch.empty_like(x).double()), dict(mean=torch.empty(2, 4)), dict(weight=torch.ones(8))):
        with pytest.raises(AssertionError):
            sa.group_norm_forward(**{**ok, **bad})
    with pytest.raises(RuntimeError, match="elements"):
        sa.group_norm_forward(**{**ok, "x": x[:, :0], "out": x[:, :0]})
    sa.group_norm_forward(**{**ok, "x": x[:0], "out": x[:0], "mean": ok["mean"][:0], "rstd": ok["rstd"][:0]})  # nothing to do
    flat = torch.zeros(400, device="cuda")
    with pytest.raises(RuntimeError, match="overlaps"):
        sa.group_norm_forward(**{**ok, "x": flat[:192].view(2, 12, 8), "out": flat[4:196].view(2, 12, 8)})


def test_group_norm_offsets_past_31_bits(sa):
    """More than 2^31 elements: the last sample against the same sample alone."""
    N, S, C, G = 3, 1 << 23, 96, 32
    x = torch.empty(N, S, C, dtype=BF16, device="cuda")
    x[:2].normal_()
    x[2].copy_(randn(S, C, seed=3, dtype=BF16))
    out, mean, rstd = norm_forward(sa, x, None, None, G)
    (y, dy), (m, dm), (r, dr) = ref.group_norm(x[2:, :1000].double(), torch.ones(C, device="cuda").double(), torch.zeros(C, device="cuda").double(), G, 1e-5, True, BF16)
    g = x[2].float().view(S, G, 3)
    assert torch.allclose(mean[2], g.mean(dim=(0, 2)), atol=1e-5) and torch.allclose(rstd[2], (g.double().var(dim=(0, 2), correction=0) + 1e-5).rsqrt().float(), rtol=1e-4)
    tail = x[2, -1000:].float().view(1000, G, 3)
    z = ((tail - mean[2][None, :, None]) * rstd[2][None, :, None]).view(1000, C)
    assert torch.allclose(out[2, -1000:].float(), z * torch.sigmoid(z), rtol=2 ** -7, atol=1e-5)


# ---------------------------------------------------------------------------
# dropout
# ---------------------------------------------------------------------------
def pair(seed, call):
    return torch.tensor([seed, call], dtype=torch.int64, device="cuda")


def kept(n, seed, call, p):
    return torch.from_numpy(ref.keep_mask(n, seed % 2 ** 64, call % 2 ** 64, p)).cuda()


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n", [1, 7, 8, 9, 255, 2047, 2048, 100003])
def test_dropout(sa, n, dtype):
    for k, (p, residual, shift) in enumerate([(0.1, False, 0), (0.5, True, 0), (0.9, True, 1), (1 / 3, False, 3), (0.0, True, 0), (1.0, True, 0), (2.0 ** -32, False, 0)]):
        seed, call = (0x0123456789ABCDEF * (k + 1)) % 2 ** 63, 2 ** 40 + k if k % 2 else -k - 1
        _, x, _ = framed((n,), dtype, k, offset=shift)
        r = randn(n, seed=77, dtype=dtype) if residual else None
        _, out, untouched = framed((n,), dtype, 50, offset=shift)
        sa.dropout_forward(out, x, pair(seed, call), p, residual=r)
        keep = kept(n, seed, call, p)
        scaled = torch.where(keep, x.double() / (1 - p) if p < 1 else torch.zeros_like(x.double()), 0.0)
        want = scaled if r is None else scaled + r.double()
        # the scale's rounding, the product's and the sum's
        close(out, want, 2 * ref.U * scaled.abs() + ref.U * want.abs())
        assert untouched()
        if p == 0.0:
            assert torch.equal(out, (x.float() + r.float()).to(dtype))
        dx = torch.full_like(x, 5.0)
        sa.dropout_backward(dx, x, pair(seed, call), p)
        assert ((dx == 0) | keep).all()
        close(dx, scaled, 2 * ref.U * scaled.abs())


def test_dropout_mask_bit_for_bit(sa):
    """Eight million decisions, about 120 of which need the second block."""
    n, p, seed, call = 8_000_005, 0.3, 987654321012345, 42
    x = torch.ones(n, device="cuda")
    out = torch.empty_like(x)
    sa.dropout_forward(out, x, pair(seed, call), p)
    keep = kept(n, seed, call, p)
    assert torch.equal(out != 0, keep)
    share = float(keep.double().mean())
    assert abs(share - 0.7) < 5 * (0.3 * 0.7 / n) ** 0.5
    # other calls, other seeds: other masks, and independent ones
    for s, c in ((seed, call + 1), (seed + 1, call), (seed, call + 2 ** 33)):
        sa.dropout_forward(out, x, pair(s, c), p)
        both = float(((out != 0) & keep).double().mean())
        assert abs(both - 0.49) < 5 * (0.49 * 0.51 / n) ** 0.5


def test_dropout_offsets_past_32_bits(sa):
    """More than 2^32 elements: the last ones' mask, and a tail that is no whole group."""
    n, p, rng = 2 ** 32 + 4099, 0.3, pair(11, 12)
    x = torch.ones(n, dtype=BF16, device="cuda")
    sa.dropout_forward(x, x, rng, p)
    first = 2 ** 32 - 4096
    keep = torch.from_numpy(ref.keep_mask(n - first, 11, 12, p, first)).cuda()
    assert torch.equal(x[first:] != 0, keep)


def test_dropout_drops_whatever_stands_there_and_works_in_place(sa):
    n, p, rng = 4096, 0.5, pair(3, 4)
    keep = kept(n, 3, 4, p)
    x, r = randn(n, seed=1), randn(n, seed=2)
    x[~keep] = float("nan")
    x[torch.nonzero(~keep)[::2, 0]] = float("inf")
    out = torch.empty_like(x)
    sa.dropout_forward(out, x, rng, p, residual=r)
    assert torch.isfinite(out).all() and torch.equal(out[~keep], r[~keep])
    for where in (0, 1):
        a, b = x.clone(), r.clone()
        sa.dropout_forward((a, b)[where], a, rng, p, residual=b)
        assert torch.equal((a, b)[where], out)
    x[keep] = float("nan")
    sa.dropout_forward(out, x, rng, p)
    assert torch.equal(torch.isnan(out), keep)


def test_dropout_shapes_and_refusals(sa):
    x, rng = randn(4, 6, 10, seed=1, dtype=BF16), pair(1, 2)
    out = torch.empty_like(x)
    sa.dropout_forward(out, x, rng, 0.25, residual=x)
    flat = torch.empty(240, dtype=BF16, device="cuda")
    sa.dropout_forward(flat, x.view(-1), rng, 0.25, residual=x.view(-1))
    assert torch.equal(out.view(-1), flat)
    for bad in (dict(out=out.view(-1)), dict(x=x.transpose(0, 1)), dict(rng=rng.int()), dict(rng=torch.zeros(3, dtype=torch.int64, device="cuda")),
                dict(rng=rng.cpu()), dict(residual=x.float()), dict(residual=x[:1].expand(4, 6, 10)), dict(out=out.half())):
        with pytest.raises(AssertionError):
            sa.dropout_forward(**{**dict(out=out, x=x, rng=rng, p=0.1), **bad})
    for p in (-0.1, 1.5, float("nan")):
        with pytest.raises(RuntimeError, match="0, 1"):
            sa.dropout_forward(out, x, rng, p)
    with pytest.raises(RuntimeError, match="overlaps"):
        sa.dropout_forward(flat[8:], flat[:-8], rng, 0.1)
    with pytest.raises(RuntimeError, match="not aligned"):
        sa.dropout_forward(out, x, torch.zeros(3, dtype=torch.int64, device="cuda")[1:], 0.1)
    sa.dropout_forward(out[:0], x[:0], rng, 0.1)  # nothing to do


# ---------------------------------------------------------------------------
# streams, graphs, ops
# ---------------------------------------------------------------------------
def everything(sa, seed=0):
    """One call of every operator on buffers of its own: a function that runs them, the buffers and what they start as."""
    N, S, C, G = 2, 1500, 64, 8
    x, w, b = norm_inputs(N, S, C, BF16, F32, seed)
    t = dict(x=x, w=w, b=b, y=torch.empty_like(x), mean=torch.empty(N, G, device="cuda"), rstd=torch.empty(N, G, device="cuda"),
             dropped=torch.empty_like(x), rng=pair(seed + 5, 0), qkv=x.view(N, S, 4, 16).clone(), dx=torch.empty_like(x),
             dw=torch.empty_like(w), db=torch.empty_like(b), positions=torch.arange(S, device="cuda").expand(2, N, S), big=torch.empty(1, 60000, 32, device="cuda"),
             bm=torch.empty(1, 4, device="cuda"), br=torch.empty(1, 4, device="cuda"), image=randn(1, 60000, 32, seed=seed))
    spectrum = sa.rope_axes_spectrum((4, 4))

    def run():
        sa.group_norm_forward(t["y"], t["mean"], t["rstd"], t["x"], t["w"], t["b"], G)
        sa.dropout_forward(t["dropped"], t["y"], t["rng"], 0.2, residual=t["x"])
        t["qkv"].copy_(t["dropped"].view(N, S, 4, 16))
        sa.rope_axes_forward(t["qkv"], t["positions"], spectrum, 2, 1)
        sa.rope_axes_backward(t["qkv"], t["positions"], spectrum, 4, 0)
        sa.dropout_backward(t["dropped"], t["qkv"].view(N, S, C), t["rng"], 0.2)
        sa.group_norm_backward(t["dx"], t["dw"], t["db"], t["dropped"], t["x"], t["mean"], t["rstd"], t["w"], t["b"], G)
        sa.group_norm_forward(t["big"], t["bm"], t["br"], t["image"], None, None, 4)
        t["rng"][1] += 1

    return run, t


RESULTS = ("y", "mean", "rstd", "dropped", "qkv", "dx", "dw", "db", "big", "bm", "br")


def test_same_inputs_same_bits_on_any_stream(sa):
    run, t = everything(sa)
    run()
    torch.cuda.synchronize()
    want = {k: t[k].clone() for k in RESULTS}
    for stream in (torch.cuda.Stream(), torch.cuda.Stream(priority=-1)):
        t["rng"][1] = 0
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            run()
        stream.synchronize()
        for k in RESULTS:
            assert torch.equal(t[k], want[k]), k


def test_two_streams_at_once(sa):
    runs = [everything(sa, s) for s in (0, 1)]
    want = []
    for run, t in runs:
        run()
        torch.cuda.synchronize()
        want.append({k: t[k].clone() for k in RESULTS})
    streams = [torch.cuda.Stream() for _ in runs]
    for _ in range(5):
        for _, t in runs:
            t["rng"][1] = 0
        torch.cuda.synchronize()
        for stream, (run, t) in zip(streams, runs):
            with torch.cuda.stream(stream):
                run()
        torch.cuda.synchronize()
        for (_, t), w in zip(runs, want):
            for k in RESULTS:
                assert torch.equal(t[k], w[k]), k


def test_recorded_graphs_replay_and_run_beside_each_other(sa):
    """Two graphs recorded on the same stream, replayed on two: every replay gives the eager bits of its call number."""
    runs = [everything(sa, s) for s in (0, 1)]
    want = []
    for run, t in runs:
        t["rng"][1] = 0
        calls = []
        for _ in range(3):
            run()
            torch.cuda.synchronize()
            calls.append({k: t[k].clone() for k in RESULTS})
        want.append(calls)
        assert not torch.equal(calls[0]["dropped"], calls[1]["dropped"]), "the next call draws another mask"
    graphs = []
    for run, _ in runs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            run()
        graphs.append(g)
    for _, t in runs:
        t["rng"][1] = 0
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in runs]
    for call in range(3):
        for stream, g in zip(streams, graphs):
            with torch.cuda.stream(stream):
                g.replay()
        torch.cuda.synchronize()
        for (_, t), w in zip(runs, want):
            for k in RESULTS:
                assert torch.equal(t[k], w[call][k]), (call, k)


def run_alone(code):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=600, cwd=root,
                       env=dict(os.environ, PYTHONPATH=root + os.pathsep + os.environ.get("PYTHONPATH", "")))
    assert "ALONE-OK" in r.stdout, r.stdout[-2000:] + r.stderr[-3000:]


def test_first_calls_of_a_process_may_be_recorded():
    """Nothing of the library has run before the capture: no operator needs its per-device set-up."""
    run_alone("""
import torch, l2_torch_alloc_b200 as pkg
from tests.test_gpu_image_operators import everything, RESULTS
sa = pkg.SideAware()
run, t = everything(sa)  # makes the spectrum only
t["rng"][1] = 0
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    run()
g.replay()
torch.cuda.synchronize()
got = {k: t[k].clone() for k in RESULTS}
t["rng"][1] = 0
run()
torch.cuda.synchronize()
assert all(torch.equal(t[k], got[k]) for k in RESULTS)
assert sa.error_count() == 0, sa.last_error()
print("ALONE-OK")
""")


def test_operators_under_torch_compile():
    run_alone("""
import torch, l2_torch_alloc_b200 as pkg
sa = pkg.sideaware_init(install_allocator=False)
ops = torch.ops.sideaware
def f(x, w, b, rng):
    out, mean, rstd = torch.empty_like(x), torch.empty(2, 4, device="cuda"), torch.empty(2, 4, device="cuda")
    ops.group_norm_forward(out, mean, rstd, x, w, b, 4, 1e-5, True)
    y = torch.empty_like(x)
    ops.dropout_forward(y, out * 2.0, rng, 0.25, x)
    return y + 1.0
x = torch.randn(2, 60, 32, device="cuda"); w = torch.randn(32, device="cuda"); b = torch.randn(32, device="cuda")
rng = torch.tensor([3, 4], device="cuda")
assert torch.equal(torch.compile(f, fullgraph=True)(x, w, b, rng), f(x, w, b, rng))
print("ALONE-OK")
""")


def test_registered_operators_give_the_same(sa):
    sa.register_ops()
    ops = torch.ops.sideaware
    run, t = everything(sa)
    run()
    want = {k: t[k].clone() for k in RESULTS}
    spectrum = sa.rope_axes_spectrum((4, 4))
    rng = pair(5, 0)
    for k in RESULTS:
        t[k].zero_()
    ops.group_norm_forward(t["y"], t["mean"], t["rstd"], t["x"], t["w"], t["b"], 8)
    ops.dropout_forward(t["dropped"], t["y"], rng, 0.2, t["x"])
    t["qkv"].copy_(t["dropped"].view(t["qkv"].shape))
    ops.rope_axes_forward(t["qkv"], t["positions"], spectrum, 2, 1)
    ops.rope_axes_backward(t["qkv"], t["positions"], spectrum, 4, 0)
    ops.dropout_backward(t["dropped"], t["qkv"].view(t["x"].shape), rng, 0.2)
    ops.group_norm_backward(t["dx"], t["dw"], t["db"], t["dropped"], t["x"], t["mean"], t["rstd"], t["w"], t["b"], 8)
    ops.group_norm_forward(t["big"], t["bm"], t["br"], t["image"], None, None, 4, 1e-5, True)
    for k in RESULTS:
        assert torch.equal(t[k], want[k]), k


def test_side_aware_memory(sa):
    """Buffers from the library's own allocator, between canary pages."""
    from tests import cuda_helpers as ch
    n = 3 * (1 << 20) + 24
    host = np.random.default_rng(3).standard_normal(n).astype(np.float32)
    a, b = ch.Guarded(sa, 4 * n), ch.Guarded(sa, 4 * n)
    ch.h2d(a.ptr, host)
    rng = pair(8, 9)
    torch.cuda.synchronize()
    assert sa.lib.sideaware_dropout_forward(b.ptr, a.ptr, None, rng.data_ptr(), 0.25, n, 0, 0, None) == 0
    ch.sync()
    got = ch.d2h(b.ptr, 4 * n, np.float32)
    keep = ref.keep_mask(n, 8, 9, 0.25)
    assert np.array_equal(got != 0, keep & (host != 0)) and a.canaries_intact() and b.canaries_intact()
    assert np.abs(got - np.where(keep, host / 0.75, 0)).max() <= 4 * ref.U * np.abs(got).max()
    a.free()
    b.free()


# ---------------------------------------------------------------------------
# together: the residual block and the attention block of an image model, trained for one step
# ---------------------------------------------------------------------------
class Norm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, w, b, sa, G):
        out, mean, rstd = torch.empty_like(x), torch.empty(x.shape[0], G, device="cuda"), torch.empty(x.shape[0], G, device="cuda")
        sa.group_norm_forward(out, mean, rstd, x, w, b, G)
        ctx.save_for_backward(x, w, b, mean, rstd)
        ctx.sa, ctx.G = sa, G
        return out

    @staticmethod
    def backward(ctx, dout):
        x, w, b, mean, rstd = ctx.saved_tensors
        dx, dw, db = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
        ctx.sa.group_norm_backward(dx, dw, db, dout.contiguous(), x, mean, rstd, w, b, ctx.G)
        return dx, dw, db, None, None


class Drop(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, rng, sa, p):
        out = torch.empty_like(x)
        sa.dropout_forward(out, x, rng, p, residual=residual)
        ctx.save_for_backward(rng)
        ctx.sa, ctx.p = sa, p
        return out

    @staticmethod
    def backward(ctx, dout):
        dout = dout.contiguous()
        dx = torch.empty_like(dout)
        ctx.sa.dropout_backward(dx, dout, ctx.saved_tensors[0], ctx.p)
        return dx, dout, None, None, None


class Rope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, qkv, positions, spectrum, sa, q, kv):
        out = qkv.clone()
        sa.rope_axes_forward(out, positions, spectrum, q, kv, "halves")
        ctx.save_for_backward(positions, spectrum)
        ctx.sa, ctx.heads = sa, (q, kv)
        return out

    @staticmethod
    def backward(ctx, dout):
        d = dout.clone(memory_format=torch.contiguous_format)
        ctx.sa.rope_axes_backward(d, *ctx.saved_tensors, *ctx.heads, "halves")
        return d, None, None, None, None, None


def test_blocks_of_an_image_model_train(sa):
    """norm + SiLU, a product, dropout onto the residual, then packed q, k, v with two-axis positions, shared key heads and
    attention: the loss's gradients in fp32 against reverse differentiation of the 64-bit definitions."""
    N, side, C, G, q, kv, head, p = 2, 6, 48, 8, 4, 2, 16, 0.25
    S, H = side * side, q + 2 * kv
    x, w, b = norm_inputs(N, S, C, F32, F32, 21)
    m1, m2 = randn(C, C, seed=31) / C ** 0.5, randn(C, H * head, seed=32) / C ** 0.5
    target = randn(N, S, q * head, seed=33)
    grid = torch.stack((torch.arange(S, device="cuda") // side, torch.arange(S, device="cuda") % side)).unsqueeze(1).expand(2, N, S)
    pairs, rng = (4, 4), pair(77, 3)
    spectrum = sa.rope_axes_spectrum(pairs, 100.0)
    keep = kept(N * S * C, 77, 3, p).view(N, S, C)

    def attend(t):
        qh, k, v = t[:, :, :q], t[:, :, q:q + kv].repeat_interleave(q // kv, dim=2), t[:, :, q + kv:].repeat_interleave(q // kv, dim=2)
        a = torch.softmax(torch.einsum("nshd,nthd->nhst", qh, k) / head ** 0.5, dim=-1)
        return torch.einsum("nhst,nthd->nshd", a, v).reshape(N, S, q * head)

    def step(x, w, b, m1, m2, norm, drop, rope):
        h = drop(norm(x, w, b) @ m1, x)
        t = rope((h @ m2).view(N, S, H, head))
        return ((attend(t) - target.to(x.dtype)) ** 2).mean()

    mine = [v.clone().requires_grad_() for v in (x, w, b, m1, m2)]
    loss = step(*mine, lambda x, w, b: Norm.apply(x, w, b, sa, G), lambda y, r: Drop.apply(y, r, rng, sa, p),
                lambda t: Rope.apply(t, grid, spectrum, sa, q, kv))
    theirs = [v.double().requires_grad_() for v in (x, w, b, m1, m2)]
    want = step(*theirs, lambda x, w, b: ref.group_norm(x, w, b, G, 1e-5, True, F32)[0][0], lambda y, r: r + torch.where(keep, y / (1 - p), 0.0),
                lambda t: Definition.apply(t, grid, pairs, q, kv))
    assert abs(float(loss) - float(want)) < 1e-5 * float(want)
    for got, exact in zip(torch.autograd.grad(loss, mine), torch.autograd.grad(want, theirs)):
        assert float((got.double() - exact).norm()) < 2e-5 * float(exact.norm())


class Definition(torch.autograd.Function):
    """The 64-bit rotary definition and its transpose (the test above this file's oracle checks it by differences)."""
    @staticmethod
    def forward(ctx, t, positions, pairs, q, kv):
        ctx.rest = positions, pairs, q, kv
        return ref.rope(t, positions, pairs, 100.0, "own", q, kv, "halves")[0]

    @staticmethod
    def backward(ctx, d):
        positions, pairs, q, kv = ctx.rest
        return ref.rope(d, positions, pairs, 100.0, "own", q, kv, "halves", inverse=True)[0], None, None, None, None


def test_launches_are_counted_as_they_are_made(sa):
    """Two samples: the resident form has one kernel forward, two backward; the streamed one three and four."""

    def count(call):
        before = sa.stats()["kernel_launches"]
        call()
        return sa.stats()["kernel_launches"] - before

    x = randn(1, 4, 6, 16, seed=1)
    spectrum = sa.rope_axes_spectrum((4,))
    positions = torch.zeros(1, 1, 4, dtype=torch.int32, device="cuda")
    assert count(lambda: sa.rope_axes_forward(x, positions, spectrum, 2, 2)) == 1
    assert count(lambda: sa.dropout_forward(torch.empty_like(x), x, pair(1, 2), 0.5)) == 1
    for rows, forward, backward in ((64, 1, 2), (300000, 3, 4)):
        x = randn(2, rows, 64, seed=2, dtype=BF16)
        w, b = torch.ones(64, device="cuda"), torch.zeros(64, device="cuda")
        mean, rstd = torch.empty(2, 8, device="cuda"), torch.empty(2, 8, device="cuda")
        assert count(lambda: sa.group_norm_forward(torch.empty_like(x), mean, rstd, x, w, b, 8)) == forward
        assert count(lambda: sa.group_norm_backward(torch.empty_like(x), torch.empty_like(w), torch.empty_like(b), x, x, mean, rstd, w, b, 8)) == backward
