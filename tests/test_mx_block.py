"""What MxDecodeBlock refuses before it touches a weight (no GPU)."""

from __future__ import annotations

import pytest


@pytest.mark.parametrize("sizes,msg", [(dict(hidden=256, intermediate=500), "blocks of 32"), (dict(hidden=256, intermediate=16), "blocks of 32"),
                                       (dict(hidden=65792, intermediate=512), "65536")])
def test_sizes_that_no_step_can_run(sizes, msg):
    from torch_helion.hip import abi
    from torch_helion.hip.mx import MxDecodeBlock

    with pytest.raises(abi.HipBackendError, match=msg):
        MxDecodeBlock({}, heads=4, kv_heads=2, eps=1e-5, rope_theta=1e4, batch=1, cache=None, **sizes)
