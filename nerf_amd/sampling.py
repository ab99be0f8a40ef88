"""Hierarchical sampling -- counterpart of the reference's sampling.py:5-60, on the HIP kernel
nrf_sample_pdf (bit-exact with the reference's CPU path on identical inputs).

`sample_logits` is the same rule for a discrete distribution given by logits: pixels by an error map, classes, tokens."""
import numpy as np
import torch

from . import ops


def sample_pdf(bins, weights, N_samples, det=False, pytest=False):
    u = None
    lead = list(bins.shape[:-1])
    if pytest:
        # the reference's fixed-random route (sampling.py:32-40): numpy f64 values rounded to f32
        np.random.seed(0)
        if det:
            u = np.broadcast_to(np.linspace(0., 1., N_samples), lead + [N_samples])
        else:
            u = np.random.rand(*(lead + [N_samples]))
        u = torch.tensor(np.ascontiguousarray(u), dtype=torch.float32, device=bins.device)
    elif not det:
        u = torch.rand(lead + [N_samples], device=bins.device)
    return ops.sample_pdf(bins, weights, N_samples, u)


def sample_logits(logits, N_samples=1, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=None):
    """Indices drawn from softmax(logits / temperature) [..., V] after top-k, top-p and min-p -> (ids, prob), both
    [..., N_samples]; ops.sample_logits describes the filters and `u`."""
    return ops.sample_logits(logits, N_samples, temperature, top_k, top_p, min_p, u)
