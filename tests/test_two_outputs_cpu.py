"""Calls with two outputs refuse one place for both (rows of either would be written over the other's)."""
import pytest

ONE = 16        # a pointer that is aligned and never read: the calls are refused, or have nothing to do, before anything is launched


@pytest.mark.parametrize("n_tok,n_head,n_head_kv", [(1, 1, 1), (2, 24, 4), (300, 4, 4)])
def test_queries_and_keys(n_tok, n_head, n_head_kv):
    import bonsai_b200
    L = bonsai_b200.lib()
    strides = (n_head * 256, 256, n_head_kv * 256, 256)
    assert L.bonsai_b200_rope(ONE, 32, ONE, ONE, 64, 64, n_tok, n_head, n_head_kv, 256, 64, 0, 1.0, *strides, None) == 1
    assert L.bonsai_b200_qk_norm_rope(ONE, 32, ONE, ONE, ONE, ONE, 64, 64, n_tok, n_head, n_head_kv, 256, 64, *strides, 1e-6, None) == 1
    # nothing to write: nothing in the way
    assert L.bonsai_b200_rope(ONE, 32, ONE, ONE, 64, 64, 0, n_head, n_head_kv, 256, 64, 0, 1.0, *strides, None) == 0
    assert L.bonsai_b200_qk_norm_rope(ONE, 32, ONE, ONE, ONE, ONE, 64, 64, 0, n_head, n_head_kv, 256, 64, *strides, 1e-6, None) == 0
