"""What the Python face of the key/value cache refuses before anything reaches the GPU."""
import pytest
import torch

from xsched_b200 import pk


def test_rows_that_overlap_are_refused():
    """An expanded tensor has one row of memory; a step of 0 would be taken for dense rows behind it."""
    for x in (torch.zeros(1, 4, 8).expand(3, 4, 8), torch.zeros(64).as_strided((3, 4, 8), (16, 8, 1)), torch.zeros(32).expand(5, 32)):
        with pytest.raises(ValueError, match="overlap"):
            pk._rows("q", x, 32)
    assert pk._rows("q", torch.zeros(1, 4, 8).expand(1, 4, 8), 32) == (1, 0)
    assert pk._rows("q", torch.zeros(3, 6, 8)[:, 1:5], 32) == (3, 48)
    assert pk._rows("q", torch.zeros(3, 4, 8), 32) == (3, 0)
    with pytest.raises(ValueError, match="apart"):
        pk._rows("q", torch.zeros(3, 1, 8).expand(3, 4, 8), 32)


def test_tensors_that_require_a_gradient_are_refused_under_grad_mode():
    """No backward pass is recorded: without the refusal their gradients would silently be missing."""
    x = torch.zeros(2, 8, requires_grad=True)
    for y in (x, x * 2, (x * 2)[:1]):
        with pytest.raises(ValueError, match="no_grad"):
            pk._no_gradient("q", y)
    with torch.no_grad():
        pk._no_gradient("q", x)
    pk._no_gradient("q", x.detach())
    cache = pk.KvCache.__new__(pk.KvCache)
    cache.dtype, cache.device = x.dtype, x.device
    with pytest.raises(ValueError, match="qkv requires a gradient"):
        cache._data("qkv", x)
    assert cache._data("qkv", x.detach()) == x.data_ptr()
