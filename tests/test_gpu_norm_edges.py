"""rms_norm_backward beyond the longest row"""
import pytest
import torch

import spanqr_amd as sp
from spanqr_amd._lib import SpanqrError

pytestmark = pytest.mark.gpu


def test_rows_that_are_too_long(cuda):
    """2^24 elements are the most: the library's own message, forward and backward"""
    x = torch.ones(1, (1 << 24) + 1, dtype=torch.bfloat16, device=cuda)
    for call in (lambda: sp.rms_norm(x, x[0]), lambda: sp.rms_norm_backward(x, x, x[0]), lambda: sp.rms_norm_backward(x, x)):
        with pytest.raises(SpanqrError, match="D = 16777217"):
            call()
