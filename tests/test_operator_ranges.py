"""Ranges of the operators' scalar arguments whose ends are not the type's (no GPU needed: they are looked at before any address)."""
import pytest

from katago_b200 import capi


@pytest.mark.parametrize("scale,taken", [(2.0e38, True), (2.3e38, True), (2.4e38, False), (2.9e38, False), (3.4e38, False), (1e-45, True)])
def test_attention_scales_whose_exponents_leave_fp32_are_refused(scale, taken):
    """Exponents are scores times scale / ln 2, which has to be a number: 3.4e38 * ln 2 is 2.36e38."""
    with pytest.raises(capi.KBError) as e:  # a taken one is refused for its views, which come next
        capi.cross_attention(capi.PRECISION_FP32, 1, 2, 2, 2, 1, 8, 8, scale, None, None, None, None)
    assert ("q is NULL" if taken else "the scale") in str(e.value)
