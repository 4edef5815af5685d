"""The 64-bit statements of the operators around the paged cache (``oracle/rotary.py``, ``oracle/paged_cache.py``)."""
import math

import pytest
import torch

from oracle import paged_cache, rotary


@pytest.mark.parametrize("interleaved", [False, True])
def test_a_turn_is_a_complex_product_and_keeps_what_is_behind_it(interleaved):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 24, dtype=torch.float64, generator=g)
    angle = torch.randn(5, 8, dtype=torch.float64, generator=g)
    y = rotary.turn(x, angle.cos(), angle.sin(), interleaved)
    a, b = (x[:, 0:16:2], x[:, 1:16:2]) if interleaved else (x[:, :8], x[:, 8:16])
    z = torch.complex(a, b) * torch.polar(torch.ones_like(angle), angle)
    p, q = (y[:, 0:16:2], y[:, 1:16:2]) if interleaved else (y[:, :8], y[:, 8:16])
    assert torch.allclose(torch.complex(p, q), z, rtol=0, atol=1e-14) and torch.equal(y[:, 16:], x[:, 16:])


@pytest.mark.parametrize("interleaved,weighted", [(False, True), (True, True), (False, False)])
def test_gradients_agree_with_differences(interleaved, weighted):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(1, 2, 3, 16, dtype=torch.float64, generator=g, requires_grad=True)
    w = torch.randn(16, dtype=torch.float64, generator=g, requires_grad=True) if weighted else None
    angle = torch.randn(4, 8, dtype=torch.float64, generator=g)
    positions = torch.tensor([[2, 0, 3]])
    f = lambda *t: rotary.norm_rotary(t[0], angle.cos(), angle.sin(), positions, t[1] if weighted else None, 1e-6, interleaved)  # noqa: E731
    assert torch.autograd.gradcheck(f, (x, w) if weighted else (x,))


def test_positions_outside_the_tables_turn_by_nan():
    x, t = torch.ones(1, 1, 3, 16, dtype=torch.float64), torch.ones(4, 4, dtype=torch.float64)
    y = rotary.norm_rotary(x, t, t, torch.tensor([[-1, 4, 3]]), None, 1e-6, False)
    assert y[0, 0, :2, :8].isnan().all() and y[0, 0, 2].isfinite().all() and torch.equal(y[..., 8:], x[..., 8:])


def test_e4m3_rounding_is_that_of_the_type():
    exact = torch.arange(256, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    exact = exact[exact.isfinite()].sort()[0]
    between = (exact[1:] + exact[:-1]) / 2          # ties, which have fewer bits than float32
    g = torch.Generator().manual_seed(3)
    some = torch.randn(4000, generator=g).float().double() * torch.exp2(torch.randint(-12, 8, (4000,), generator=g).double())
    for x in (exact, between, some.clamp(-448, 448)):
        assert torch.equal(paged_cache.round_e4m3(x), x.float().to(torch.float8_e4m3fn).double())


def test_least_scale_is_the_least():
    for peak in (448.0, 448.0000001, 447.9, 1.0, 1.75, 1.7500001, 0.875, 2.0 ** -40, 3e38):
        s = paged_cache.least_scale(peak)
        assert peak / s <= 448 < peak / (s / 2) and math.frexp(s)[0] == 0.5
    assert paged_cache.least_scale(0.0) == 2.0 ** -118 == paged_cache.least_scale(1e-40)


def test_appending_token_by_token_gives_the_scales_of_appending_at_once():
    """The scale of a block is that of the largest magnitude in it however the tokens come, as long as it only grows."""
    g = torch.Generator().manual_seed(4)
    x = torch.randn(12, 2, 16, generator=g) * torch.exp2(torch.arange(12) / 2.0)[:, None, None]
    table = torch.tensor([[3, 1]])
    cache, scales = torch.zeros(4, 2, 8, 16), torch.full((4, 2), 2.0 ** 30)
    at_once = paged_cache.append(x, cache, scales, paged_cache.places(torch.tensor([12]), torch.tensor([0, 12]), 12, table, 8, 4))
    step = (cache, scales)
    for i in range(12):
        step = paged_cache.append(x[i:i + 1], *step, paged_cache.places(torch.tensor([i + 1]), None, 1, table, 8, 4))
    assert torch.equal(at_once[1], step[1])
    error = (at_once[0] - step[0]).abs() * step[1][:, :, None, None]
    assert (error <= 2 ** -3 * (step[0].abs() * step[1][:, :, None, None]) + 2 ** -9 * step[1][:, :, None, None]).all()


def test_attention_over_codes_is_dense_attention_over_what_they_stand_for():
    g = torch.Generator().manual_seed(5)
    codes = [torch.randn(6, 2, 4, 16, generator=g).to(torch.float8_e4m3fn) for _ in range(2)]
    scales = [torch.rand(6, 2, generator=g) + 0.1 for _ in range(2)]
    q, lens, table = torch.randn(2, 4, 16, generator=g), torch.tensor([9, 0]), torch.tensor([[5, 0, 2], [1, 1, 1]])
    out, _, _ = paged_cache.attention_fp8(q, *codes, *scales, lens, table, 0.25)
    k, v = ((c.double() * s.double()[:, :, None, None])[table[0]].permute(1, 0, 2, 3).reshape(2, 12, 16)[:, :9].repeat_interleave(2, 0)
            for c, s in zip(codes, scales))
    want = torch.nn.functional.scaled_dot_product_attention(q[0].double()[:, None], k, v, scale=0.25)[:, 0]
    assert torch.allclose(out[0], want, rtol=0, atol=1e-12) and (out[1] == 0).all()
    table[0, 1] = 6
    assert paged_cache.attention_fp8(q, *codes, *scales, lens, table, 0.25)[0][0].isnan().all()
