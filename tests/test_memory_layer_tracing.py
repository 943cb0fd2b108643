"""The memory layer with a graph where its operations are recorded or only imagined: fake tensors, make_fx, export,
torch.jit.trace, a dispatch mode that counts.  Every operation must then be torch's own."""
import pytest
import torch
from torch.utils._python_dispatch import TorchDispatchMode

from oracle import ref_cpu as R


def layer_of(dim=48, heads=2, hd=64):
    from vit_amd import surgical_world_model as swm
    layer = swm.GatedDeltaLayer(dim, num_heads=heads, head_dim=hd)
    P = R.fill_state_dict_({f"tr.{k}": v for k, v in layer.state_dict().items()})
    layer.load_state_dict({k[3:]: v for k, v in P.items()})
    return layer.eval()


class Counting(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func))
        return func(*args, **(kwargs or {}))


def test_where_torch_must_see_every_operation():
    from torch._subclasses import FakeTensorMode
    from torch.fx.experimental.proxy_tensor import make_fx
    from vit_amd import module_ops
    assert not module_ops.by_torch_alone()
    seen = []

    def look(x):
        seen.append(module_ops.by_torch_alone())
        return x * 2

    with FakeTensorMode():
        fake = torch.ones(2)
        look(fake)
    for mode in ("real", "fake", "symbolic"):
        make_fx(look, tracing_mode=mode)(torch.ones(2))
    torch.jit.trace(look, torch.ones(2), check_trace=False)
    with Counting():
        look(torch.ones(2))

    class Looks(torch.nn.Module):
        def forward(self, x):
            return look(x)

    torch.export.export(Looks(), (torch.ones(2),), strict=False)
    assert seen and all(seen)
    assert not module_ops.by_torch_alone()
    assert module_ops.by_torch_alone(fake) and not module_ops.by_torch_alone(torch.ones(2), torch.nn.Parameter(torch.ones(2)), None)


@pytest.mark.parametrize("device", ["cpu", "cuda"])
def test_fake_tensors_pass_through_the_layer(device):
    """Shapes of a device layer, also without a device: outputs, and gradients where torch's backward engine finds its device."""
    from torch._subclasses import FakeTensorMode
    from vit_amd import surgical_world_model as swm
    with FakeTensorMode():
        with torch.device(device):
            layer = swm.GatedDeltaLayer(48, num_heads=2, head_dim=64)
        x = torch.empty(2, 6, 48, device=device, requires_grad=True)
        out, state = layer(x)
        assert out.shape == x.shape and state.shape == (2, 2, 64, 64) and out.device.type == device
        if device == "cuda" and not torch.cuda.is_available():
            return
        (out.sum() + state.sum()).backward()
        assert x.grad.shape == x.shape and layer.o_norm.weight.grad.shape == (128,)


@pytest.mark.gpu
def test_recorded_graphs_compute_what_the_layer_does():
    from torch.fx.experimental.proxy_tensor import make_fx
    layer = layer_of().cuda()
    x, other = (R.hashed_uniform(f"tr.{n}", (2, 9, 48), 1.0).cuda() for n in "xy")
    params = dict(layer.named_parameters())

    def call(values, y):
        return torch.func.functional_call(layer, values, (y,))

    traced = make_fx(call)(params, x)
    jit = torch.jit.trace(layer, x.clone().requires_grad_(), check_trace=False)
    for y in (x, other):
        want = layer(y.clone().requires_grad_())
        for got in (traced(params, y), jit(y)):
            for a, b in zip(got, want):
                # f32 sums in another order: products of up to 128 terms, eight layers deep
                assert (a - b).norm() <= 1e-4 * b.norm()
    with Counting() as counted:
        layer(x)
    assert any("sigmoid" in n or "silu" in n for n in counted.names)
    assert any("native_layer_norm" in n for n in counted.names)      # the mode sees the output stage too
