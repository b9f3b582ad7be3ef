"""A step's rows by adapter, put together by the caller: parts that do not belong together."""

import pytest
import torch

from reflex_b200 import InvalidInput, ops


def test_parts_on_different_devices():
    order, first, tiles = (torch.zeros(s, dtype=torch.int32) for s in ((4,), (4,), (2, 3)))
    for parts in ((order, first, tiles.to("meta")), (order, first.to("meta"), tiles), (order.to("meta"), first, tiles)):
        with pytest.raises(InvalidInput, match="one device"):
            ops.AdapterRows(*parts, 16)
