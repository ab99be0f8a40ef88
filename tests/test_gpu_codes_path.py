"""Drawing a batch by an error map, the codes of the images its rays come from, and the training step through them: the operators of
sampling.sample_logits and codes.CodeTable as raybatch, render and optim use them together."""
import numpy as np
import pytest
import torch

import nerf_fixtures as fx
from test_gpu_lookup import check_bwd
from test_gpu_sample_logits import reference

pytestmark = pytest.mark.gpu

H, W, M = 40, 30, 5


def scene(seed=0):
    rng = np.random.RandomState(seed)
    images = rng.rand(M, H, W, 3).astype(np.float32)
    poses = np.stack([fx.pose_spherical(a, -30.0, 4.0)[:3, :4] for a in np.linspace(0, 300, M)]).astype(np.float32)
    K, _ = fx.intrinsics(H, W)
    return images, poses, K, rng


def test_pixels_drawn_by_an_error_map():
    from nerf_amd.raybatch import ImageRaySampler
    images, poses, K, rng = scene()
    sampler = ImageRaySampler(images, poses, H, W, K)
    error = rng.rand(H, W).astype(np.float32) ** 4 + 1e-4
    logits = torch.log(torch.from_numpy(error)).cuda()
    u = torch.from_numpy(rng.rand(500).astype(np.float32)).cuda()
    rays, rgb, pix, prob = sampler.sample_weighted(2, 500, logits, u=u, temperature=0.7, top_p=0.9)
    ids, p = reference(logits.reshape(-1).cpu().numpy(), u.cpu().numpy(), float(np.float32(0.7)), 0, float(np.float32(0.9)), 0.0)
    assert np.array_equal(pix.cpu().numpy(), ids) and np.allclose(prob.cpu().numpy(), p, rtol=2.0 ** -23, atol=0)
    want_rays, want_rgb = sampler.sample(2, 500, select_inds=pix)
    assert torch.equal(rays, want_rays) and torch.equal(rgb, want_rgb)
    assert torch.equal(rgb.cpu(), torch.from_numpy(images[2].reshape(-1, 3))[pix.cpu()])
    # inside the centre crop, and a map that leaves nothing
    cand = sampler.crop_pixels(0.5)
    rays, rgb, pix, prob = sampler.sample_weighted(1, 64, torch.zeros(cand.numel(), device="cuda"), precrop_frac=0.5)
    assert torch.isin(pix, cand).all() and torch.equal(prob, torch.full_like(prob, 1.0 / cand.numel()))
    assert torch.equal(rays, sampler.sample(1, 64, select_inds=pix)[0])
    rays, rgb, pix, prob = sampler.sample_weighted(3, 8, torch.full((H * W,), -float("inf"), device="cuda"))
    assert (pix == -1).all() and (prob == 0).all() and torch.isnan(rays).all() and torch.isnan(rgb).all()
    with pytest.raises(ValueError, match="candidate pixel"):
        sampler.sample_weighted(0, 8, logits[:-1])


def test_slots_name_the_training_image():
    from nerf_amd.raybatch import RayBatcher
    images, poses, K, _ = scene(1)
    i_train = [4, 0, 3]
    batch = RayBatcher(images, poses, H, W, K, i_train, N_rand=700)
    for _ in range(6):                       # past the end of an epoch
        rays, rgb, slots = batch.next(return_slots=True)
        assert slots.shape == (rays.shape[1],) and int(slots.min()) >= 0 and int(slots.max()) < 3
        origin = torch.from_numpy(poses[:, :3, 3]).cuda()[torch.tensor(i_train, device="cuda")[slots]]
        torch.testing.assert_close(rays[0], origin, rtol=0, atol=1e-6)
    assert torch.equal(batch.slots(torch.tensor([0, H * W - 1, H * W], device="cuda")), torch.tensor([0, 0, 1], device="cuda"))


def test_a_training_step_through_codes():
    from nerf_amd.codes import CodeTable
    from nerf_amd.network import NeRF
    from nerf_amd.optim import FusedAdam
    from nerf_amd.positional_encoding import get_embedder
    from nerf_amd.raybatch import RayBatcher
    from nerf_amd.render import raw2outputs, run_network
    from nerf_amd import ops
    images, poses, K, rng = scene(2)
    torch.manual_seed(3)
    dim, N, S = 5, 96, 16
    batch = RayBatcher(images, poses, H, W, K, range(M), N_rand=N)
    codes = CodeTable(M, dim, init_std=0.5).cuda()
    net = NeRF(4, 64, 63, 27 + dim, 4, [2], True).cuda()
    e10, _ = get_embedder(10, 0)
    e4, _ = get_embedder(4, 0)
    params = [codes.weight] + list(net.parameters())
    opt = FusedAdam(params, lr=1e-2)
    twin = [p.detach().clone().requires_grad_() for p in params]
    adam = torch.optim.Adam(twin, lr=1e-2)
    for _ in range(3):
        rays, target, slots = batch.next(return_slots=True)
        o, d = rays
        viewdirs = d / torch.linalg.vector_norm(d, dim=-1, keepdim=True)
        z = ops.sample_coarse(torch.cat([o, d, torch.full((N, 1), 2.0, device="cuda"), torch.full((N, 1), 6.0, device="cuda")], -1), S)
        pts = o[:, None] + d[:, None] * z[..., None]
        c = codes(slots)
        c.retain_grad()
        raw = run_network(pts, viewdirs, net, e10, e4, codes=c)
        rgb = raw2outputs(raw, z, d)[0]
        loss = ((rgb - target) ** 2).mean()
        opt.zero_grad()
        loss.backward()
        check_bwd(c.grad, slots, M, 1.0, None, codes.weight.grad)
        assert float(codes.weight.grad.abs().max()) > 0
        for p, q in zip(params, twin):
            q.grad = p.grad.detach().clone()
        opt.step()
        adam.step()
        torch.testing.assert_close(codes.weight.detach(), twin[0].detach(), rtol=1e-5, atol=1e-6)
    # the code is what tells two images' rays apart
    with torch.no_grad():
        one = run_network(pts, viewdirs, net, e10, e4, codes=codes(torch.zeros_like(slots)))
        two = run_network(pts, viewdirs, net, e10, e4, codes=codes(torch.ones_like(slots)))
    assert not torch.equal(one, two) and torch.equal(one[..., 3], two[..., 3])       # colour depends on it, density does not
    for bad in (c[:-1], c[:, None]):
        with pytest.raises(ValueError, match="one row per ray"):
            run_network(pts, viewdirs, net, e10, e4, codes=bad)
