"""Paged attention with bfloat16 q: every token's weights hold 16 bits, in prompts and in
calls of any sizes as for single tokens (oracle/paged.py, "bf16": 2^-17 a weight)."""

import pytest

import test_gpu_paged
import test_gpu_paged_use
from test_gpu_paged import DEEP, prepared, run

pytestmark = pytest.mark.gpu

BF = ("bf16", "bf16")


def exact_form(c, dt, *_, **__):
    return "f32" if dt == "f32" else "bf16"


@pytest.fixture
def tight(monkeypatch):
    """The other tests' checks, with the bound of 16 bits a weight in place of 8."""
    attend = test_gpu_paged_use.attend
    monkeypatch.setattr(test_gpu_paged, "form_of", exact_form)
    monkeypatch.setattr(test_gpu_paged_use, "attend",
                        lambda q, k, v, see, scale, form: attend(q, k, v, see, scale, form.replace(" prompt", "")))


@pytest.mark.parametrize("H,KH,counts,start,page", [(8, 1, [64], [1500], 16), (6, 2, [300], [97], 32), (4, 2, [130, 0, 90], [900, 5, 1800], 128),
                                                    (7, 1, [201], [0], 16), (32, 8, [700], [260], 64), (28, 4, [90, 1, 260], [0, 700, 31], 32)])
@pytest.mark.parametrize("maxT", [None, DEEP])
def test_prompts_hold_16_bits(H, KH, counts, start, page, maxT, tight):
    run(H, KH, counts, start, *BF, page, maxT=maxT)


@pytest.mark.parametrize("dt,cached", test_gpu_paged.TYPES)
def test_a_servers_run_holds_16_bits(dt, cached, tight):
    """Prompts, single tokens and drafts after one another."""
    s = test_gpu_paged_use.Server(8, 2, 3, 200, 16, dt, cached)
    s.call([300, 0, 77])
    for _ in range(2):
        s.call([1, 0, 1])
    s.call([5, 0, 4], draft=3)
    s.call([700, 900, 1])
    s.call([1, 1, 1])


def test_weights_far_apart_hold_16_bits(tight):
    for maxT in (1500, DEEP):
        c, q = prepared(8, 2, [150, 70], [77, 600], "bf16", maxT)
        for x in (30.0, 1e-4):
            test_gpu_paged.check(c, q * x, [77, 600], [150, 70], "bf16")
