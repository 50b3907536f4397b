"""Calls that write into an argument count as changes of it on the direct route too (the launches are left out here)."""

from __future__ import annotations

import pytest
import torch

from pi05_fast import w4a4
from pi05_fast.w4a4 import kv, kv_int8, lora


def _calls(monkeypatch):
    """Each call and the tensors that it writes."""
    for module, name in ((kv, "_append_impl"), (kv, "_rope_append_impl"), (kv_int8, "_append_impl"), (lora, "_lora_impl")):
        monkeypatch.setattr(module, name, lambda *a: a[0])
    q, i, freq = torch.ones(1, 1, 1, 64, dtype=torch.float16), torch.zeros(1, 1, dtype=torch.int32), torch.ones(32)
    cache = w4a4.kv_cache(1, 1, 64, torch.float16, "cpu")
    cache8 = w4a4.int8_kv_cache(1, 1, 64, "cpu")
    x, a, b = torch.ones(1, 64, dtype=torch.float16), torch.ones(1, 8, 64, dtype=torch.float16), torch.ones(1, 64, 8, dtype=torch.float16)
    y = x.clone()
    return {
        "kv_append": (lambda: w4a4.kv_append(q, q, *cache, i, i[0]), cache),
        "qk_norm_rope_append": (lambda: w4a4.qk_norm_rope_append(q, q, q, None, None, 0.0, i, freq, *cache, i, i[0]), cache),
        "int8_kv_append": (lambda: w4a4.int8_kv_append(q, q, *cache8, i, i[0]), cache8),
        "lora_add_": (lambda: w4a4.lora_add_(y[:, :], x, a, b, i[0]), (y,)),
    }


@pytest.mark.parametrize("name", ["kv_append", "qk_norm_rope_append", "int8_kv_append", "lora_add_"])
def test_versions_grow(monkeypatch, name):
    call, written = _calls(monkeypatch)[name]
    for mode in (torch.enable_grad, torch.no_grad, torch.inference_mode):
        before = [t._version for t in written]
        with mode():
            call()
        assert all(t._version > v for t, v in zip(written, before))
    with torch.inference_mode():
        _calls(monkeypatch)[name][0]()  # tensors made here have no version


def test_a_saved_input_is_not_overwritten_unnoticed(monkeypatch):
    call, (y,) = _calls(monkeypatch)["lora_add_"]
    p = torch.ones_like(y, requires_grad=True)
    z = (y * p).sum()
    call()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
