"""A top_k of each row in every whole type gives what int32 gives."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int8, torch.uint8, torch.int16, torch.int64])
@pytest.mark.parametrize("V", [700, 5000])
def test_top_k_of_every_whole_type(dtype, V):
    from nerf_amd import ops
    gen = torch.Generator(device="cuda").manual_seed(V)
    x = torch.randn(6, V, generator=gen, device="cuda")
    u = torch.rand(6, 3, generator=gen, device="cuda")
    k = torch.tensor([0, 1, 5, 40, 100, 127], device="cuda")
    want = ops.sample_logits(x, 3, top_k=k.int(), u=u)
    got = ops.sample_logits(x, 3, top_k=k.to(dtype), u=u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(TypeError, match="whole numbers"):
        ops.sample_logits(x, 3, top_k=k.float(), u=u)
