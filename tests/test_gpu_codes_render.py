"""One image's code through render(): the query function repeats it for each chunk of rays."""
import pytest
import torch

import nerf_fixtures as fx

pytestmark = pytest.mark.gpu


def test_a_code_of_one_image_through_render():
    from nerf_amd.codes import CodeTable
    from nerf_amd.network import NeRF
    from nerf_amd.positional_encoding import get_embedder
    from nerf_amd.render import render, run_network
    torch.manual_seed(5)
    H = W = 12
    K, _ = fx.intrinsics(H, W)
    pose = torch.tensor(fx.pose_spherical(40.0, -30.0, 4.0)[:3, :4], dtype=torch.float32, device="cuda")
    codes = CodeTable(3, 5, init_std=0.5).cuda()
    net = NeRF(4, 64, 63, 27 + 5, 4, [2], True).cuda()
    e10, _ = get_embedder(10, 0)
    e4, _ = get_embedder(4, 0)

    def image(i, chunk):
        code = codes(torch.tensor([i], device="cuda"))
        query = lambda pts, dirs, fn: run_network(pts, dirs, fn, e10, e4, codes=code.expand(dirs.shape[0], -1))  # noqa: E731
        with torch.no_grad():
            return render(H, W, K, chunk=chunk, c2w=pose, ndc=False, near=2.0, far=6.0, use_viewdirs=True, network_fn=net,
                          network_query_fn=query, N_samples=16)[0]
    whole, other = image(1, H * W), image(2, H * W)
    # chunks change the sizes of the library's matrix products, and so the order of their f32 sums: 63 + 64 + ... terms of order one
    torch.testing.assert_close(image(1, 50), whole, rtol=0, atol=1e-5)
    assert whole.shape == (H, W, 3) and torch.isfinite(whole).all() and not torch.equal(whole, other)
