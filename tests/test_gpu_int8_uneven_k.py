"""int8 products whose K ends inside a step of their kernel, whole and in K slices: every form that a K of any multiple of 16
reaches.  Operand rows go on behind K with codes that would show in every sum."""

from __future__ import annotations

import pytest
import torch
from test_gpu_int8 import _check_product, _gen, _product

from pi05_fast.w4a4 import int8 as i8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("m,k,n,sliced", [
    (4, 4112, 67, True), (4, 4112, 2048, True), (13, 16400, 33, True),  # streamed weights, in K slices
    (64, 4112, 2048, True), (500, 8016, 1001, True), (64, 16432, 2049, True),  # 64 x 64 tiles
    (40, 2064, 129, False), (2000, 4112, 300, False),
    (776, 2064, 2561, False), (1071, 2096, 5001, False),  # 128 x 64 tiles
    (700, 12304, 600, True), (2048, 12400, 301, True),
    (3000, 1040, 8001, False),  # 256 x 256 tiles
])
def test_product(cuda, m, k, n, sliced, dtype):
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert (i8.load_int4_gemm().pi05w4a4_int8_gemm_workspace_bytes(m, n, k) > 0) == sliced
    q, sq, w, sw, bias, res = _product(_gen(m + k + n), m, k, n, dtype, True, True)
    wide_q, wide_w = (torch.full((t.size(0), k + 112), 127, dtype=torch.int8, device="cuda") for t in (q, w))
    wide_q[:, :k], wide_w[:, :k] = q, w
    for a, b in ((q, w), (wide_q[:, :k], wide_w[:, :k])):
        _check_product(i8.int8_gemm(a, sq, b, sw, out_dtype=dtype), q, sq, w, sw, None, None)
        _check_product(i8.int8_gemm(a, sq, b, sw, bias, res, out_dtype=dtype), q, sq, w, sw, bias, res)
