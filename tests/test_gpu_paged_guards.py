"""What PagedKVCache refuses or reports of the calls between a layer's staging and the commit."""

import pytest
import torch

from _paged import Requests

pytestmark = pytest.mark.gpu


def test_a_staged_descriptor_needs_a_staged_layer(gpu):
    """Outside of an append it would describe the lengths of the last one, whose pages may be another's by now."""
    r = Requests(gpu, [40, 64], h=1, d=64, page=32, layers=2)
    c = r.cache

    def refused(layer):
        with pytest.raises(RuntimeError, match="not staged"):
            c.prefix(layer, staged=True)

    refused(0)
    k, v = (x.to(gpu) for x in r.block([1, 0], 1))
    c.begin_append(r.i32([1, 0]), 1)
    refused(0)
    c.stage_layer(0, k, v)
    assert c.prefix(0, staged=True).lengths.tolist() == [41, 64]
    refused(1)
    c.stage_layer(1, k, v)
    c.commit_append()
    refused(0)
    c.release(torch.tensor([True, False], device=gpu))
    refused(1)
    for layer in (-1, 2):
        with pytest.raises(IndexError):
            c.prefix(layer, staged=True)
    assert c.prefix(0).lengths.tolist() == [0, 64]
