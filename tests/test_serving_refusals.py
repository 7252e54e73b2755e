"""Refusals of the serving calls that depend on a value's range."""
import numpy as np
import pytest

from test_attn_decode import fake


@pytest.mark.parametrize("scale,ok", [(3e38, False), (-2.4e38, False), (np.finfo(np.float32).max, False), (2.3e38, True), (-2.3e38, True), (0.0, True), (1e-45, True)])
def test_attn_scale_has_to_be_finite_in_base_two(scale, ok):
    """The exponentials are taken to base 2: a scale whose product with log2(e) overflows would make NaN of a score of 0."""
    import vvb200
    assert vvb200.vvb_attn_decode_dev(fake(vvb200, scale=scale, n_seqs=0), stream=0) == (vvb200.VV_OK if ok else vvb200.VV_ERR_INVALID_ARG)
