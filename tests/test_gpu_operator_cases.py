"""The timed operator cases' own states: what they load is given back."""
import importlib.util
import os

import pytest
import torch

PATH = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "perf", "operators.py")


@pytest.mark.gpu
def test_states_give_their_layers_back():
    """More states than one context has layers, two alive at a time: all run, and
    device memory stays within two contexts' layers and workspaces."""
    spec = importlib.util.spec_from_file_location("operator_cases", PATH)
    ops = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(ops)
    ops.own = True
    case = {"kind": "window", "heads": 16, "batch": 1, "rows": 1, "length": 40, "sinks": 1, "window": 16, "ragged": False}
    layer = (16 * 256 * 512 + 16 * 512 * 128 + 16 * 8 * 16 * 512) * 2
    states, used, first, free0 = [], [], None, None
    for k in range(4 * ops._LAYERS + 3):
        states = states[-1:] + [ops.prepare(case, 5)]
        out = ops.run(states[-1])
        torch.cuda.synchronize()
        first = out.clone() if first is None else first
        assert torch.equal(out, first), k
        free = torch.cuda.mem_get_info()[0]
        free0 = free if free0 is None else free0
        used.append(free0 - free)
    assert max(used) <= (2 * ops._LAYERS + 2) * max(layer, 2 << 20) + (512 << 20), max(used)
