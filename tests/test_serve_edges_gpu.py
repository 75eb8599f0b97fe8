"""Serving operators on the GPU at the edges of their contract: what a batch may hold that its tensors do not, page
tables with entries that are none, the device status, far arguments of the activations, tensors that overlap, mixed
batches.  Tolerances count roundings as in test_serve_gpu.py."""
import copy
import math

import numpy as np
import pytest
import torch

from test_serve_gpu import BF16, Batch, check_attention, check_linear, gen, packed, values64

pytestmark = pytest.mark.gpu

L = pytest.importorskip("hif4x._lib")
from hif4x import codec, linalg, serve  # noqa: E402


# ------------------------------------------------------------------ values that are none
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_of_values_that_are_none(dtype):
    """NaN, infinities, the type's largest and smallest values: the bits are hif4x_convert's, and other rows' too."""
    T, kvh, dh = 40, 2, 128
    b = Batch([T], [T], kvh, dh, 16, 56, fill=False)
    x = torch.randn(2, T, kvh, dh, generator=gen(57), device="cuda")
    nan, inf, fi = float("nan"), float("inf"), torch.finfo(dtype)
    specials = (nan, inf, -inf, fi.max, -fi.max, fi.tiny, -fi.tiny, fi.smallest_normal / 8, 0.0, -0.0)
    for i, value in enumerate(specials):
        x[0, i, 0, 5] = value                                    # one in a group
        x[0, 10 + i, 1, 64:] = value                             # a group of them
        x[1, 20 + i, 0, ::3] = value                             # many among others
        x[1, 20 + i, 0, 1] = specials[i - 1]
    for i, size in enumerate((0.0, 2.0 ** -60, 2.0 ** 30)):      # NaN among values whose scales meet the E6M2 limits
        x[0, 30 + i] *= size
        x[0, 30 + i, :, 3:40:9] = nan
    x = x.to(dtype)
    serve.kv_append(b.cache, x[0], x[1], *b.args)
    for src, meta, codes in ((x[0], b.cache.k_meta, b.cache.k_codes), (x[1], b.cache.v_meta, b.cache.v_codes)):
        want = codec.convert(src.float().reshape(T * kvh, dh).contiguous(), kind=L.SRC_VALUES, dict5=False, packed=True)
        at = torch.arange(T, device="cuda")
        ids = b.pages[0].long()[at // 16]
        assert torch.equal(meta[ids, :, at % 16].reshape(T * kvh, -1), want["meta"])
        assert torch.equal(codes[ids, :, at % 16].reshape(T * kvh, -1), want["codes"])
    linalg.check_device_status()


