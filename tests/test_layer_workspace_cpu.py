"""Scratch memory that the layer operators ask for, by the C ABI's queries (148 SMs where there is no device)."""

import pytest

from test_layer_capi_cpu import F16, lib  # noqa: F401

SMS = 148


@pytest.mark.parametrize("width,blocks", [(8, 8), (1024, 8), (4096, 8), (4104, 4), (8192, 4), (8200, 2), (16384, 2),
                                          (33000, 2)])
def test_norm_backward_follows_the_width(lib, width, blocks):  # noqa: F811
    """A partial row of both sums for each block that can be resident (2048 threads an SM, a block as wide as the
    row's lanes), not for 16 blocks an SM."""
    ask = lib.spmm_layer_norm_backward_workspace_bytes
    assert ask(1 << 20, width) == blocks * SMS * 2 * width * 4
    assert ask(5, width) == 5 * 2 * width * 4


def test_weight_gradient_parts(lib):  # noqa: F811
    """Parts of at most 16384 rows: as many slots as the groups can need, none beyond."""
    ask, K = lib.spmm_grouped_weight_grad_workspace_bytes, 2048
    slot = K * K * 4
    assert ask(1 << 20, 1, K, K, F16) == (64 + 1) * slot
    assert ask(1 << 20, 10, K, K, F16) == (64 + 10) * slot
    assert ask(1 << 20, 1000, K, K, F16) == (64 + 64) * slot
    assert ask(300, 1, K, K, F16) == 0
