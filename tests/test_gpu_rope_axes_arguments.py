"""Rotary positions with several axes: calls whose arguments do not fit one another, and the largest rows."""
import pytest
import torch

from tests import image_operator_reference as ref
from tests.test_gpu_image_operators import BF16, F16, F32, close, randn, sa  # noqa: F401 (sa: the fixture)

pytestmark = pytest.mark.gpu


def test_positions_of_other_axes_are_refused(sa):
    x, spectrum = randn(2, 3, 8, 16, seed=1), sa.rope_axes_spectrum((2, 3, 3))
    before = x.clone()
    for axes in (1, 2, 4):
        places = torch.ones(axes, 2, 3, dtype=torch.int32, device="cuda")
        for call in (sa.rope_axes_forward, sa.rope_axes_backward):
            with pytest.raises(AssertionError, match="axes"):
                call(x, places, spectrum, 4, 2)
    assert torch.equal(x, before)
    sa.rope_axes_forward(x, torch.ones(3, 2, 3, dtype=torch.int32, device="cuda"), spectrum, 4, 2)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("layout", ["interleaved", "halves"])
def test_axes_that_the_positions_lack_become_nan(sa, layout, dtype):
    """A copy of the spectrum no longer knows its axes: the kernel sees them in its entries.  Every other element is NaN with them
    (a thread has several pairs) or right; what is not turned stays."""
    B, T, q, kv, pairs = 2, 5, 3, 2, (3, 6, 7)
    for head, arrangement in ((32, "own"), (40, "interleaved")):
        x = randn(B, T, q + 2 * kv, head, seed=3, dtype=dtype)
        before = x.clone()
        places = torch.randint(0, 500, (3, B, T), device="cuda", generator=torch.Generator(device="cuda").manual_seed(2))
        sa.rope_axes_forward(x, places[:2], sa.rope_axes_spectrum(pairs, arrangement=arrangement).clone(), q, kv, layout)
        want, bound = ref.rope(before.double(), places, pairs, 10000.0, arrangement, q, kv, layout)
        lacking = torch.tensor([i for i, (_, a) in enumerate(ref.frequencies(pairs, 10000.0, arrangement)) if a == 2], device="cuda")
        elements = torch.cat((2 * lacking, 2 * lacking + 1) if layout == "interleaved" else (lacking, lacking + sum(pairs)))
        assert torch.isnan(x[:, :, :q + kv, elements]).all()
        assert not torch.isnan(x[:, :, q + kv:]).any() and not torch.isnan(x[..., 2 * sum(pairs):]).any()
        want[torch.isnan(x)] = float("nan")
        close(x, want, bound)


@pytest.mark.parametrize("layout", ["interleaved", "halves"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_heads_in_narrow_words(sa, layout, dtype):
    """2.6 million places and groups of heads of a token (65536 heads of 256 pairs are 4.2 million): more blocks for a token than
    1 << 20 threads fill."""
    q, kv, head, pairs = 40000, 1000, 511, (100, 155)
    x = randn(1, 2, q + 2 * kv, head, seed=4, dtype=dtype)
    before = x.clone()
    places = torch.tensor([[[3, 4000]], [[-7, 99999]]], device="cuda")
    sa.rope_axes_forward(x, places, sa.rope_axes_spectrum(pairs), q, kv, layout)
    for heads in (slice(0, 700), slice(20000, 20500), slice(q + kv - 500, q + kv)):
        part = before[:, :, heads].double()
        want, bound = ref.rope(part, places, pairs, 10000.0, "own", part.shape[2], 0, layout)
        close(x[:, :, heads], want, bound)
    assert torch.equal(x[:, :, q + kv:], before[:, :, q + kv:]) and torch.equal(x[..., 510:], before[..., 510:])


@pytest.mark.parametrize("theta", [1.0, 10000.0, 0.25])
@pytest.mark.parametrize("name", ["rope_axes_forward", "rope_axes_backward"])
def test_angles_of_near_and_far_positions(sa, name, theta):
    """Pairs (1, 0) turn to (cos, sin), the angle to |position| 2^-62 max(1, 1 / theta) + 2^-26 turns as documented.  Beside it an
    evaluation of cos and sin: a rounding of the result, 2^-24 for the polynomial's own roundings, 2e-9 for its truncation.  The
    angle itself is worked out in 60 digits."""
    from decimal import Decimal, getcontext
    getcontext().prec = 60
    two_pi = 2 * Decimal("3.14159265358979323846264338327950288419716939937510582097494")
    pairs, places = 8, [0, 1, -1, 17, 1000, 54321, -123457, 10 ** 6 + 1, 2 ** 31 - 1, -2 ** 31, 2 ** 36 + 5, -2 ** 40 - 1, 3 * 10 ** 13]
    x = torch.zeros(1, len(places), 1, 2 * pairs, device="cuda")
    x[..., :pairs] = 1.0
    positions = torch.tensor(places, device="cuda").view(1, 1, -1)
    getattr(sa, name)(x, positions, sa.rope_axes_spectrum((pairs,), theta), 1, 0, "halves")
    for t, place in enumerate(places):
        for i in range(pairs):
            turns = place * Decimal(theta) ** (Decimal(-i) / pairs) / two_pi
            angle = float((turns - turns.to_integral_value()) * two_pi) * (1 if name == "rope_axes_forward" else -1)
            limit = float(two_pi) * (abs(place) * 2.0 ** -62 * max(1.0, 1.0 / theta) + 2.0 ** -26) + 2 * 2.0 ** -24 + 2e-9
            want = torch.tensor([angle], dtype=torch.float64)
            assert abs(float(x[0, t, 0, i]) - float(want.cos())) <= limit, (place, i)
            assert abs(float(x[0, t, 0, pairs + i]) - float(want.sin())) <= limit, (place, i)
