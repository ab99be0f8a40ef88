"""What the weights 1 / (n prob) of ImageRaySampler.sample_weighted estimate: the mean over the n candidate pixels where all of them can be
drawn, and the kept pixels' share of it under a filter.

The draws are taken at the midpoints u = (j + 1/2) / N.  A sum over midpoints of a function of u that is constant over each pixel's interval
is off by at most its total variation / (2 N): here that of g = f / (n p) over the pixels in order.  prob is rounded to f32 (2^-24)."""
import numpy as np
import pytest
import torch

from test_gpu_codes_path import H, W, scene

pytestmark = pytest.mark.gpu

N = 1 << 18          # midpoints are exact in f32


@pytest.mark.parametrize("frac", [None, 0.5])
def test_weighted_means(frac):
    from nerf_amd.raybatch import ImageRaySampler
    images, poses, K, rng = scene(4)
    sampler = ImageRaySampler(images, poses, H, W, K)
    cand = sampler.crop_pixels(frac)
    n = H * W if cand is None else cand.numel()
    error = rng.rand(n).astype(np.float32) + np.float32(0.1)
    logits = np.log(error)
    u = (torch.arange(N, device="cuda", dtype=torch.float32) + 0.5) / N
    e = np.exp((logits.astype(np.float64) - logits.max()) / 0.5)
    for filters in (dict(), dict(top_p=0.9), dict(top_k=n // 2), dict(min_p=0.2)):
        _, _, pix, prob = sampler.sample_weighted(1, N, torch.from_numpy(logits).cuda(), precrop_frac=frac, u=u, temperature=0.5, **filters)
        place = pix if cand is None else torch.searchsorted(cand, pix)
        f = torch.from_numpy(error).cuda().double()[place]
        got = float((f / (prob.double() * n)).mean())
        kept = np.zeros(n, bool)
        kept[place.unique().cpu().numpy()] = True
        if not filters:
            assert kept.all()
        p = np.where(kept, e, 0.0) / e[kept].sum()
        want = float(error[kept].astype(np.float64).sum() / n)
        g = np.where(kept, error / (n * np.where(kept, p, 1.0)), 0.0)[kept]
        tol = np.abs(np.diff(g)).sum() / (2 * N) + want * 2.0 ** -23
        assert tol < 0.01 * want and abs(got - want) <= tol, (filters, got, want, tol)
        if filters:                                              # what a filter leaves out is missing from the mean
            assert want < 0.99 * float(error.mean())
