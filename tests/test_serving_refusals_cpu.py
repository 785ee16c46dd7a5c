"""Refusals of kore_b200.serving that need no GPU."""
import pytest

from kore_b200 import KoreError, serving


@pytest.mark.parametrize("head_dim", [-4, 0, 2, 30, 132, 1 << 28])
def test_a_cache_of_an_unsupported_head_dim_is_refused_before_it_is_allocated(head_dim):
    with pytest.raises(KoreError) as e:
        serving.KV4Cache(1, 1, 1 << 20, head_dim)
    assert "head_dim" in e.value.message
