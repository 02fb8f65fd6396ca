"""What TokenStream refuses before it touches a GPU."""
from types import SimpleNamespace

import pytest

from h3vae_b200.streaming import TokenStream


@pytest.mark.parametrize("page_size", [0, -64, 24, 256])
def test_page_sizes_that_no_cache_has(page_size):
    decoder = SimpleNamespace(int8=True, cfg=SimpleNamespace(heads=4), device="cuda", blocks=[])
    with pytest.raises(ValueError, match="page_size"):
        TokenStream(decoder, 1, (8, 12), 4, page_size=page_size)
