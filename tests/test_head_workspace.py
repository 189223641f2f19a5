"""The class head's `workspace` argument, without a GPU."""
from __future__ import annotations

import numpy as np
import pytest


def test_a_workspace_beside_numpy_arrays_is_refused():
    """Calls on numpy arrays work in memory of the handle's: a workspace would be left unused without a word."""
    from tiny_metal_nn import class_head, logits

    class Calls(class_head._HeadCalls):
        def __init__(self):
            self.made = []

        def _run(self, a, on_host, on_device, packed, stream):
            self.made.append(packed)

    calls, a = Calls(), logits._HostArrays()
    with pytest.raises(ValueError, match="workspace goes with torch tensors"):
        calls._enqueue(a, None, None, None, b"", np.zeros(256, np.uint8), None)
    assert not calls.made
    calls._enqueue(a, None, None, None, b"", None, None)
    assert calls.made == [class_head._NO_WORKSPACE]
