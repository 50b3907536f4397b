"""Adapters of more workgroups than one launch holds: the parts meet without a gap."""

from __future__ import annotations

import pytest
import torch

from pi05_fast import w4a4

pytestmark = pytest.mark.gpu


def test_many_windows_of_many_adapters(cuda):
    """Each row of a window can have its own of 64 adapters: 4095 windows of 64 rows a launch at this width and rank."""
    gen = torch.Generator(device="cuda").manual_seed(31)
    m, n, r, k = 4100 * 64 + 7, 1 << 14, 72, 8
    y = torch.randint(-64, 65, (1, n), device="cuda", generator=gen).bfloat16().expand(m, n)
    x = torch.randint(-2, 3, (m, k), device="cuda", generator=gen).bfloat16()
    a = torch.randint(-1, 2, (64, r, k), device="cuda", generator=gen).bfloat16()
    b = torch.randint(-1, 2, (64, n, r), device="cuda", generator=gen).bfloat16()
    ids = torch.randint(-1, 64, (m,), device="cuda", generator=gen).to(torch.int32)
    got = w4a4.lora_add(y, x, a, b, ids)
    for at in (0, 1000 * 64, 4094 * 64, 4095 * 64, 4098 * 64):
        rows = slice(at, min(at + 128, m))
        assert torch.equal(got[rows], w4a4.lora_add(y[rows], x[rows], a, b, ids[rows]))
        h = torch.bmm(a[ids[rows].clamp(min=0).long()].float(), x[rows].float()[..., None])
        want = y[rows].float() + torch.where(ids[rows, None] >= 0, torch.bmm(b[ids[rows].clamp(min=0).long()].float(), h)[..., 0], 0.0)
        assert torch.equal(got[rows], want.bfloat16())
