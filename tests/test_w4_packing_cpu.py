"""What ``pack_w4`` would lose is refused: codes of more than four bits, which would run into their neighbours, and scales that are no bf16 numbers."""
from __future__ import annotations

import math

import pytest
import torch

from aginfer_b200.recipes.layout import pack_w4, quantize_w4, unpack_w4

CODES = torch.randint(0, 16, (20, 128), generator=torch.Generator().manual_seed(0)).to(torch.uint8)
SCALES = torch.rand(20, 2, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)


@pytest.mark.parametrize("code", [16, 255, -1])
def test_codes_of_more_than_four_bits_are_refused(code):
    codes = CODES.to(torch.int32)
    codes[7, 100] = code
    with pytest.raises(ValueError, match="four bits"):
        pack_w4(codes, SCALES)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_scales_that_bf16_does_not_hold_are_refused(dtype):
    scales = SCALES.to(dtype)
    words, units = pack_w4(CODES, scales)       # bf16 numbers of another type are fine
    assert torch.equal(units.view(torch.int16), pack_w4(CODES, SCALES)[1].view(torch.int16)) and torch.equal(unpack_w4(words, units, 20), unpack_w4(*pack_w4(CODES, SCALES), 20))
    scales[3, 1] = 1 + 2.0 ** -9
    with pytest.raises(ValueError, match="bf16"):
        pack_w4(CODES, scales)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
def test_a_group_that_is_not_finite_is_nan(value):
    w = torch.randn(20, 128, generator=torch.Generator().manual_seed(2))
    clean = unpack_w4(*pack_w4(*quantize_w4(w, 64)), 20)
    w[4, 70] = value
    codes, scales = quantize_w4(w, 64)
    back = unpack_w4(*pack_w4(codes, scales), 20)
    assert int(codes.max()) <= 15 and bool(scales[4, 1].isnan()) and bool(back[4, 64:].isnan().all())
    back[4, 64:] = clean[4, 64:]
    assert torch.equal(back, clean)
