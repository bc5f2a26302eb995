"""What a network keeps of its weights (resnet18_var._made) follows them: on the CPU, with a stand-in for what the kernels make of them."""
import copy
import io

import pytest
import torch

import resnet18_var
from resnet18_var import _made


class _Owner(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.w = torch.nn.Parameter(torch.arange(6.0).view(2, 3), requires_grad=False)
        self.register_buffer("s", torch.tensor(2.0))
        self.calls = 0

    def _double(self, w, s):
        self.calls += 1
        return w * s, w.sum(1)

    def get(self):
        return _made(self, "_kept", self._double, self.w, self.s)

    def right(self):
        got = self.get()
        return torch.equal(got[0], self.w * self.s) and torch.equal(got[1], self.w.sum(1))


def test_made_once():
    o = _Owner()
    assert o.right() and o.right() and o.get() is o.get() and o.calls == 1
    with torch.inference_mode():
        assert o.right()
    assert o.calls == 1 and "_kept" not in o.state_dict()


def _replace(o):
    o.w = torch.nn.Parameter(torch.full((2, 3), 7.0), requires_grad=False)


def _same_memory(o):
    """another parameter over the same memory, written to as often as the first one was"""
    o.w = torch.nn.Parameter(o.w.data, requires_grad=False)
    while o.w._version < o._kept.seen[0][3]:
        o.w.add_(1)


def _back(o):
    """memory of its own and, in time, memory at the address of before"""
    at = o.w.data_ptr()
    o.w.data = o.w.data + 1
    for _ in range(100):
        o.w.data = o.w.data + 1
        if o.w.data_ptr() == at:
            break


def _in_inference_mode(o):
    with torch.inference_mode():
        o.w.mul_(3)


CHANGES = [lambda o: o.w.mul_(3), lambda o: o.s.fill_(5.0), lambda o: o.w[1].zero_(), lambda o: o.load_state_dict({"w": torch.ones(2, 3), "s": torch.tensor(4.0)}),
           lambda o: o.load_state_dict({"w": torch.ones(2, 3), "s": torch.tensor(4.0)}, assign=True), _replace, _same_memory, _back, _in_inference_mode,
           lambda o: setattr(o.w, "data", torch.full((2, 3), -1.0)), lambda o: setattr(o, "w", torch.nn.Parameter(torch.ones(4, 3), requires_grad=False)),
           lambda o: o.double(), lambda o: torch.nn.init.normal_(o.w)]


@pytest.mark.parametrize("change", range(len(CHANGES)))
def test_follows(change):
    for written_before in (0, 2):
        o = _Owner()
        for _ in range(written_before):
            o.w.add_(1)
        assert o.right()
        CHANGES[change](o)
        assert o.right() and o.right() and o.calls <= 2


def test_same_memory_where_the_shape_is():
    o = _Owner()
    at = [t.data_ptr() for t in o.get()]
    o.w.mul_(2)
    assert o.right() and [t.data_ptr() for t in o.get()] == at
    _replace(o)
    assert o.right() and [t.data_ptr() for t in o.get()] == at


def test_uncounted_writes_are_told():
    net = resnet18_var.ResNet18Var(num_classes=3, pointwise="int8")
    make = lambda w: (w + 1,)  # noqa: E731
    first = _made(net, "_one", make, net.fc_w)
    at = first[0].data_ptr()
    net.fc_w.data.mul_(2)
    net.weights_changed()
    again = _made(net, "_one", make, net.fc_w)
    assert torch.equal(again[0], net.fc_w + 1) and again[0].data_ptr() == at and _made(net, "_one", make, net.fc_w) is again


def test_weights_made_in_inference_mode():
    """torch counts no writes to them: nothing is kept"""
    with torch.inference_mode():
        o = _Owner()
        assert o.right()
        o.w.mul_(3)
        assert o.right()
    assert o.right()


def test_copies_make_their_own():
    o = _Owner()
    kept = o.get()
    for c in (copy.deepcopy(o), torch.load(_saved(o), weights_only=False)):
        c.w.zero_()
        assert c.right() and o.right() and o.get() is kept


def _saved(o):
    f = io.BytesIO()
    torch.save(o, f)
    f.seek(0)
    return f


def test_made_in_inference_mode_renewed_outside():
    o = _Owner()
    with torch.inference_mode():
        assert o.right()
    o.w.mul_(3)
    assert o.right() and not o.get()[0].is_inference()


def test_other_types_are_made_in_memory_of_their_own():
    o = _Owner()
    before = o.get()
    copied = before[0].clone()
    o.double()
    assert o.right() and o.get()[0].dtype == torch.float64 and torch.equal(before[0], copied)
    o.float()
    assert o.right() and o.get()[0].dtype == torch.float32
