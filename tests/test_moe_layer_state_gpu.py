"""The example layer's 8-bit servers beside its 16-bit ones while the parameters
change."""
import pytest

pytestmark = pytest.mark.gpu


def test_8_bit_serving_follows_the_parameters(device):
    """Served in 8 bits, changed in place, served again: by a server of before and by
    a new one. 8-bit operands are off by up to 2^-4 of a value, 3 roundings in all."""
    import torch
    from mini_triton_nvgpu_v1_amd import moe_layer
    layer = moe_layer.ExpertLayer(width=256, hidden=384, experts=8, top_k=2, seed=9)
    g = torch.Generator(device="cuda")
    g.manual_seed(10)
    x = torch.randn((13, 256), generator=g, device="cuda").to(layer.dtype)
    plain, before = layer.server(13), layer.server(13, f8=True)
    for _ in range(2):
        want = plain.run(x).double()
        for server in (before, layer.server(13, f8=True)):
            got = server.run(x).double()
            assert float((got - want).norm() / want.norm()) < 3 * 2.0 ** -4
        layer.up.mul_(-1.5)
        layer.down.copy_(layer.down.flip(0))
