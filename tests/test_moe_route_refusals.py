"""What the routing entry points refuse, before anything reaches a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

import mmfp4
from mmfp4 import _lib

P = ctypes.c_void_p(4096)


@pytest.mark.parametrize("E,k,groups,keep,msg", [
    (2000, 2, 1, 1, "1024"), (0, 1, 1, 1, "E=0"), (64, 0, 1, 1, "k=0"), (128, 65, 1, 1, "k=65"),
    (64, 9, 8, 1, "k=9"), (64, 2, 7, 1, "groups=7"), (64, 2, 0, 0, "groups=0"),
    (64, 2, 8, 9, "topk_groups=9"), (64, 2, 8, 0, "topk_groups=0"), (256, 2, 128, 8, "groups=128"),
])
def test_route_refuses(E, k, groups, keep, msg):
    with pytest.raises(ValueError, match=msg):
        _lib.call("mm_moe_route", P, 0, None, 4, E, k, 0, groups, keep, 1, 1.0, P, P, None)


def test_other_refusals():
    with pytest.raises(ValueError, match="type 3"):
        _lib.call("mm_moe_route", P, 3, None, 4, 64, 2, 0, 1, 1, 1, 1.0, P, P, None)
    with pytest.raises(ValueError, match="null"):
        _lib.call("mm_moe_route", None, 0, None, 4, 64, 2, 0, 1, 1, 1, 1.0, P, P, None)
    _lib.call("mm_moe_route", None, 0, None, 0, 64, 2, 0, 1, 1, 1, 1.0, None, None, None)
    with pytest.raises(ValueError, match="k=65"):
        _lib.call("mm_moe_route_backward", P, P, 0, P, 4, 128, 65, 0, 1, 1.0, P, None)
    with pytest.raises(ValueError, match="null"):
        _lib.call("mm_moe_route_backward", P, P, 0, None, 4, 128, 6, 0, 1, 1.0, P, None)
    with pytest.raises(ValueError, match="scoring"):
        mmfp4.moe_route(torch.zeros(2, 8), 2, scoring="relu")
    with pytest.raises(RuntimeError, match="GPU"):
        mmfp4.moe_route(torch.zeros(2, 8), 2)
    with pytest.raises(RuntimeError, match="GPU"):
        mmfp4.moe_route_backward(torch.zeros(2, 2), torch.zeros(2, 8), torch.zeros(2, 2).long())
