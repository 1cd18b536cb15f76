"""Refusals of the serving operators at the ends of their arguments: no GPU needed."""

import pytest

from test_serving_host import c_cache, c_heads
from tinygrad_mi355x.runtime import kernels as K


@pytest.mark.parametrize("batch,tokens,cols", [(1 << 32, 1 << 32, 2), (4, 1 << 62, 2), (1 << 62, 4, 2), (1, 1, 1 << 58)])
def test_sizes_whose_products_pass_64_bits(batch, tokens, cols):
    """They are refused before anything is computed from the products, which wrap to 0."""
    c, x = c_cache(), c_heads()
    with pytest.raises(ValueError):
        K.call("tgm_kv_append", c, None, None, None, None, None, x, 4096, x, 4096, None, None, None, 4096, cols, cols, 4096, batch,
               tokens, None)
    with pytest.raises(ValueError):
        K.call("tgm_kv_attend", c, x, 4096, 4096, cols, cols, 4096, batch, tokens, 0, 1.0, 4096, 1 << 30, 4096, None)
    with pytest.raises(ValueError):
        K.call("tgm_kv_read", c, 4096, cols, cols, 4096, batch, tokens, 4096, 4096, 13, None)
    assert K.load_library().tgm_kv_attend_workspace(c, 13, 2, batch, tokens, cols, 0) == 0
