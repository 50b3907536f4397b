"""bf16 rows behind a norm whose squares, or whose products with the weight, leave fp32's range: finite rows have finite
scales and their codes.  Tolerances as for any row behind a norm: a scale within 64 fp32 half steps, the argument of a
code within 127 of them (tests/test_gpu_int8.py derives both; powers of two that keep sums in range are exact)."""

from __future__ import annotations

import pytest
import torch

from pi05_fast.w4a4 import int8 as i8

pytestmark = pytest.mark.gpu
H = 2.0**-24


def _check(h, w, eps, unit, q, s):
    hd = h.double()
    y = hd / (hd.square().mean(-1, keepdim=True) + eps).sqrt() * (w.double() + (1 if unit else 0))
    amax = y.abs().amax(-1)
    assert torch.isfinite(s).all()
    assert ((s.double() - (amax / 127 + 1e-12)).abs() <= 64 * H * (amax / 127) + H * 1e-12).all()
    assert (q.double() - y / s.double()[:, None]).abs().max().item() <= 0.5 + 127 * 64 * H


@pytest.mark.parametrize("m,k", [(3, 8), (5, 1000), (4, 2048), (1100, 2048), (1100, 512), (7, 8192), (3, 32768)])
@pytest.mark.parametrize("size,eps", [(3e38, 1e-6), (1e30, 1e-6), (2e19, 1e-6), (1e18, 1e-6), (1e-17, 0.0), (1e-20, 0.0),
                                      (1e-36, 0.0), (1e-30, 1e-6), (1e-21, 1e-42)])
def test_sums_of_squares_out_of_range(cuda, m, k, size, eps):
    gen = torch.Generator(device="cuda").manual_seed(m + k)
    x = (torch.rand((m, k), device="cuda", generator=gen) * 2 - 1).bfloat16()
    x[:, 0] = 1  # no row without its largest size
    x[::2] *= size  # ordinary rows between them
    w = (torch.randn((k,), device="cuda", generator=gen) * 0.2).bfloat16()
    eps = torch.tensor(eps).item()  # as the kernel has it
    _check(x, w, eps, True, *i8.rms_norm_int8(x, w, eps))
    r = (x * 0.25).bfloat16() * -1
    q, s, h = i8.add_rms_norm_int8(x, r, w, eps)
    assert torch.equal(h, x + r)
    _check(h, w, eps, True, q, s)


def test_products_with_the_weight_out_of_range(cuda):
    """The weight of one channel is near fp32's largest number; the normalised row is not."""
    x = torch.full((5, 2048), 100.0, dtype=torch.bfloat16, device="cuda")
    x[:, 7] = 30.0
    w = torch.ones(2048, dtype=torch.bfloat16, device="cuda")
    w[7] = 2e38
    _check(x, w, 1e-6, False, *i8.rms_norm_int8(x, w, 1e-6, unit_offset=False))


def test_rows_past_the_range_are_nan(cuda):
    """A normalised row that fp32 does not hold, a NaN and an infinity: scale NaN, codes 0; a row of zeros without an
    eps is 0 / 0."""
    x = torch.full((6, 512), 1e30, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(512, dtype=torch.bfloat16, device="cuda")
    x[1, 100], x[2, 511], x[3] = float("nan"), float("inf"), 0
    w[5] = 3e38
    x[4, :] = 0
    x[4, 5] = 1e30  # 22.6 * 3e38
    x[5, 5] = 0
    q, s = i8.rms_norm_int8(x, w, 0.0, unit_offset=False)
    assert torch.isnan(s[1:5]).all() and not q[1:5].any()
    assert torch.isfinite(s[5]) and (q[5, 6:] == 127).all() and q[5, 5] == 0
