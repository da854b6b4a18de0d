"""A bias that asks for a gradient reaches the kernels in rows side by side: the library writes its gradient's rows as far apart as the
bias's, into a tensor whose rows are side by side."""
import pytest
import torch

from pope_amd import _lib
from pope_amd.hip_pope import _prep
from pope_amd.hip_pope_flash_attn import _prep_pope

VIEWS = {"repeated": lambda: torch.rand(1, 16).expand(4, -1), "of_wider_rows": lambda: torch.rand(4, 40)[:, 8:24], "transposed": lambda: torch.rand(16, 4).mT,
         "side_by_side": lambda: torch.rand(4, 16)}


@pytest.mark.parametrize("view", VIEWS)
def test_rows_side_by_side(view):
    freqs, qk = torch.rand(10, 16), torch.rand(1, 4, 10, 16)
    for prep in (_prep_pope, lambda f, b: _prep(qk, qk, f, b)):
        bias = VIEWS[view]().detach().requires_grad_()
        rows = prep(freqs, bias)[1]
        assert rows.is_contiguous() and torch.equal(rows, bias) and rows.requires_grad
        assert (rows is bias) == (view == "side_by_side")
        with torch.no_grad():   # nothing is copied where there is no gradient to write
            rows = prep(freqs, bias)[1]
            assert rows.stride(-1) == 1 and (view == "transposed" or rows.stride(0) == bias.stride(0))
    rows = _lib.bias_rows(VIEWS[view]())
    assert rows.stride() == (16, 1)
