"""When a SharedInputGroup hands out a kept result and when it computes anew (no GPU: the products are stand-ins)."""

import gc
import weakref

import numpy as np
import pytest
import torch

from conftest import load_package

groups = load_package().groups


class StandIn(groups.SharedInputGroup):
    """A group of three members whose products are multiples of x, counting its computations."""

    def __init__(self):
        torch.nn.Module.__init__(self)
        self._result, self._key, self._handed = None, None, set()
        self.sizes, self.computed = [4, 4, 4], 0

    def forward_all(self, x):
        self.computed += 1
        return [x * (i + 1) for i in range(3)]


@pytest.mark.parametrize("kind", [torch.Tensor.clone, torch.nn.Parameter])
def test_one_computation_for_all_members(kind):
    g, x = StandIn(), kind(torch.randn(2, 4))
    for i in range(3):
        assert torch.equal(g.member_output(i, x), x * (i + 1))
    assert g.computed == 1
    g.member_output(0, x)  # asked again: computed again
    assert g.computed == 2 and not g.state_dict()


def test_another_tensor_is_another_input():
    """The next x may get the freed one's object, address and version; a member not yet called must not see the old product."""
    g, memory = StandIn(), np.ones((2, 4), dtype=np.float32)
    x = torch.from_numpy(memory)
    g.member_output(0, x)
    old, others = id(x), []
    del x
    memory[:] = 2.0
    for _ in range(1000):  # the memory is the old one's; so is the object, as soon as its place is given out again
        y = torch.from_numpy(memory)
        if id(y) == old:
            break
        others.append(y)
    assert torch.equal(g.member_output(1, y), torch.full((2, 4), 4.0)) and g.computed == 2


@pytest.mark.parametrize("change", [lambda x: x.add_(1), lambda x: x.__setattr__("data", x.data + 1)])
def test_a_changed_tensor_is_another_input(change):
    g, x = StandIn(), torch.zeros(2, 4)
    g.member_output(0, x)
    change(x)
    assert torch.equal(g.member_output(1, x), torch.full((2, 4), 2.0))


def test_nothing_is_kept_once_all_members_have_been_called():
    g, x = StandIn(), torch.zeros(2, 4)
    held = weakref.ref(x)
    out = [g.member_output(i, x) for i in range(3)]
    del x
    gc.collect()
    assert held() is None and g._result is None and len(out) == 3
