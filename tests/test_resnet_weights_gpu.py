"""ResNet18Var keeps what its kernels take of the weights: it follows the weights, on any stream, and inside and outside of captured graphs."""
import pytest
import torch

import resnet18_var

pytestmark = pytest.mark.gpu


def _image(seed=1):
    return torch.randn((2, 3, 64, 64), generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def _net(**how):
    return resnet18_var.ResNet18Var(num_classes=60, **how).cuda().eval()


def _fresh(net, image, **how):
    """The logits of a network that has never seen other weights"""
    new = _net(**how)
    new.load_state_dict(net.state_dict())
    return new(image)


def _scale(t):
    t.mul_(torch.linspace(0.5, 1.5, t.numel(), device=t.device).view(t.shape))


def _pointwise(seed):
    """Shortcuts and classifier of another network"""
    return {n: t for n, t in _net(seed=seed, **INT8).state_dict().items() if "short" in n or "bn1" in n or "fc_" in n}


INT8 = dict(pointwise="int8", fused=False)


@pytest.mark.parametrize("layout", ["NCHW", "NHWC"])
@pytest.mark.parametrize("name", ["fc_w", "blocks.0.0.short", "blocks.3.0.short", "blocks.1.0.bn1.scale"])
def test_codes_follow_writes(name, layout):
    how = dict(INT8, layout=layout)
    net, image = _net(**how), _image()
    before = net(image)
    _scale(net.state_dict()[name])
    after = net(image)
    assert not torch.equal(after, before) and torch.equal(after, _fresh(net, image, **how)) and torch.equal(net(image), after)


def test_codes_follow_loaded_and_replaced_weights():
    net, image = _net(**INT8), _image()
    net(image)
    net.load_state_dict(_pointwise(5), strict=False)
    assert torch.equal(net(image), _fresh(net, image, **INT8))
    net.fc_w = torch.nn.Parameter(torch.randn_like(net.fc_w), requires_grad=False)
    assert torch.equal(net(image), _fresh(net, image, **INT8))
    net.fc_w = torch.nn.Parameter(torch.randn((7, 512), device="cuda"), requires_grad=False)        # a head of another size
    net.fc_b = torch.nn.Parameter(torch.randn(7, device="cuda"), requires_grad=False)
    assert net(image).shape == (2, 7)
    net.fc_w.data.mul_(2)                      # (torch counts no such writes)
    net.weights_changed()
    net.fc_b.zero_()
    a = net(image)
    net.fc_w.mul_(0.5)
    assert torch.equal(net(image) * 2, a)      # (a power of two: every rounding alike)


def test_first_call_on_another_stream():
    net, image = _net(**INT8), _image()
    want = _fresh(net, image, **INT8)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    with torch.cuda.stream(a):
        torch.cuda._sleep(20_000_000)          # (some 10 ms in front of the codes of the weights)
        net(image)
    with torch.cuda.stream(b):
        y = net(image)
    torch.cuda.synchronize()
    assert torch.equal(y, want)


def test_first_call_inside_a_capture():
    net, image = _net(**INT8), _image()
    want = _fresh(net, image, **INT8)          # (also what torch itself sets up)
    net.pointwise = None
    net(image)
    net.pointwise = "int8"                     # (the codes alone are still to be made)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = net(image)
    assert torch.equal(net(image), want)       # before the graph has run
    graph.replay()
    assert torch.equal(y, want)


def test_captured_graph_and_changed_weights():
    """A graph uses what is kept: after a change, the next call outside of a capture renews that where it is"""
    net, image = _net(**INT8), _image()
    want = net(image)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = net(image)
    graph.replay()
    assert torch.equal(y, want)
    for other in (5, 6):
        net.load_state_dict(_pointwise(other), strict=False)
        want = net(image)
        junk = [torch.full((1 << 18,), 1e9, device="cuda") for _ in range(20)]        # (into whatever memory has been given back)
        graph.replay()
        assert torch.equal(y, want) and torch.equal(want, _fresh(net, image, **INT8))
        del junk


def test_round_tf32_inside_a_capture():
    import wg2x2
    x = torch.randn(1000, device="cuda")
    x[::7] = float("nan")
    want = wg2x2.round_tf32(x)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = wg2x2.round_tf32(x)
    graph.replay()
    assert torch.equal(y.view(torch.int32), want.view(torch.int32)) and torch.equal(want.isnan(), x.isnan()) and not want[~x.isnan()].view(torch.int32).bitwise_and(0x1FFF).any()


WAYS = [dict(), dict(layout="NHWC"), dict(fused=False), dict(pointwise="int8"), dict(pointwise="int8", layout="NHWC"), dict(pointwise="int8", fused=False)]


@pytest.mark.parametrize("how", WAYS, ids=str)
def test_every_weight_is_followed(how):
    net, image = _net(**how), _image()
    y = net(image)
    names = [n for n in net.state_dict() if not n.endswith("mask")]
    for name in [n for n in names if n.split(".")[0] != "blocks" or n[7] in "03"]:          # (first and last stage: every kind there is)
        _scale(net.state_dict()[name]) if name != "fc_b" else net.fc_b.add_(1)
        before, y = y, net(image)
        assert not torch.equal(y, before), name
    assert torch.equal(y, _fresh(net, image, **how))
    net.load_state_dict(_net(seed=5, **how).state_dict())
    assert torch.equal(net(image), _fresh(net, image, **how))
    for name, t in list(net.named_parameters()):
        owner, last = net.get_submodule(name.rpartition(".")[0]), name.rpartition(".")[2]
        setattr(owner, last, torch.nn.Parameter(torch.randn_like(t) * t.std(), requires_grad=False))
    assert torch.equal(net(image), _fresh(net, image, **how))


@pytest.mark.parametrize("how", WAYS, ids=str)
def test_first_call_of_a_network_inside_a_capture(how):
    net, image = _net(**how), _image()
    want = _fresh(net, image, **how)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = net(image)
    assert torch.equal(net(image), want)
    graph.replay()
    assert torch.equal(y, want)
    again = torch.cuda.CUDAGraph()             # (now of what is kept)
    with torch.cuda.graph(again):
        y = net(image)
    for seed in (5, 6):
        net.load_state_dict(_net(seed=seed, **how).state_dict())
        want = net(image)
        again.replay()
        assert torch.equal(y, want)


def test_loaded_winograd_weights_in_a_graph():
    net, image = _net(), _image()
    net(image)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        y = net(image)
    weights = {n: layer.W.cpu().numpy() * 0.5 for n, layer in net.winograd_layers().items()}
    net.load_winograd_weights(weights)
    want = net(image)
    graph.replay()
    assert torch.equal(y, want) and torch.equal(want, _fresh(net, image))


def test_network_made_in_inference_mode():
    with torch.inference_mode():
        net, image = _net(), _image()
        net(image)
        net.load_state_dict(_net(seed=5).state_dict())
        assert torch.equal(net(image), _fresh(net, image))


def test_network_of_two_devices_in_turn():
    """Moved to the CPU and back: made anew there"""
    net, image = _net(pointwise="int8"), _image()
    want = net(image)
    net.cpu().cuda()
    assert torch.equal(net(image), want)
