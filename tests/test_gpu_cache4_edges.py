"""The 4-bit cache and its attention on a B200 where they go wrong most easily:
precision, ranges, shared and full pages. The helpers, and what each
tolerance is made of, are test_gpu_cache4's."""
import numpy as np
import pytest
import torch

import libpktito_b200 as P
from tests import cache4_ref as R
from tests import test_gpu_cache4 as T

pytestmark = [pytest.mark.gpu, pytest.mark.usefixtures("cuda_device")]


@pytest.mark.parametrize("dk,G,rows", [(32, 1, 1), (64, 4, 1), (128, 4, 1), (128, 1, 5), (96, 4, 4), (256, 2, 1), (256, 1, 200)])
def test_weights_of_bf16_rows_have_sixteen_bits(dk, G, rows, monkeypatch):
    # two bf16 parts: each leaves at most 2^-8 of what it is taken from
    monkeypatch.setitem(T.PARTS, "bf16", 2.0 ** -16)
    lens = [3000, 700, 260]
    c = T.filled(lens, 32, 2, dk, seed=dk + rows)
    T.check_attention(c, lens, [rows] * 3, [1, 0, 2], G, "bf16", True, 0)
    T.check_attention(c, lens, [rows] * 3, [0, 2, 1], G, "bf16", False, 0, scale=0.05)
