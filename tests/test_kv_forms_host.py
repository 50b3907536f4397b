"""The shapes of ``kv_forms`` still reach the forms that they stand for, and all that the rules choose are among them."""

from __future__ import annotations

import ctypes

import pytest
from kv_forms import FORMS

from pi05_fast.w4a4 import extension as ext

CUS = 256


class Plan(ctypes.Structure):
    _fields_ = [("runs", ctypes.c_int), ("waves", ctypes.c_int), ("wide", ctypes.c_bool)]


@pytest.fixture(scope="module")
def plan():
    fn = ext.load_int4_gemm()["_ZN4w4a414kv_attn16_planElliiili"]  # w4a4::kv_attn16_plan
    fn.restype, i32, i64 = Plan, ctypes.c_int32, ctypes.c_int64
    fn.argtypes = [i64, i64, i32, i32, i32, i64, ctypes.c_int]

    def call(b, t, h, kvh, d, pages):
        p = fn(b, t, h, kvh, d, pages, CUS)
        return "wide" if p.wide else "one" if t == 1 else "some", p.waves, p.runs

    return call


def _ahead(runs):
    return 1 if runs == 1 else 4 if runs <= 4 else 16 if runs <= 16 else 64


@pytest.mark.parametrize("kernel,waves,runs,shape", FORMS)
def test_plans(plan, kernel, waves, runs, shape):
    assert plan(*shape) == (kernel, waves, runs)


@pytest.mark.parametrize("d", [64, 128, 256])
def test_no_other_form(plan, d):
    known = {(kernel, 0 if kernel == "wide" else waves, _ahead(runs)) for kernel, waves, runs, shape in FORMS if shape[4] == d}
    for h, kvh in ((8, 1), (32, 8), (5, 5), (40, 2)):
        for b in (1, 3, 8, 64, 300):
            for t in (1, 2, 5, 16, 50, 200, 776):
                for pages in (1, 2, 3, 7, 13, 33, 100, 500):
                    kernel, waves, runs = plan(b, t, h, kvh, d, pages)
                    assert (kernel, 0 if kernel == "wide" else waves, _ahead(runs)) in known, (b, t, h, kvh, pages)
