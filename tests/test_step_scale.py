"""Scales that the attention's exponents cannot take are refused before a launch; no GPU is needed."""
import pytest

from mlora import _ext
from test_step_refusals import attention


@pytest.mark.parametrize("scale, code", [
    (2.0 ** -127, _ext.MLORA_ERANGE), (-2.0 ** -149, _ext.MLORA_ERANGE), (2.0 ** 127 * 1.25, _ext.MLORA_ERANGE), (-3.4e38, _ext.MLORA_ERANGE),
    (float("inf"), _ext.MLORA_EINVAL), (float("nan"), _ext.MLORA_EINVAL),
    # within the range: the next check's answer
    (0.0, _ext.MLORA_EINVAL), (-0.0, _ext.MLORA_EINVAL), (2.0 ** -126, _ext.MLORA_EINVAL), (-2.0 ** 127, _ext.MLORA_EINVAL)])
def test_scales(scale, code):
    assert attention(scale=scale, q=None) == code
