"""Token sampling (reference: utils/sampler.py:26-57).

The reference draws softmax(logits / T) divided by Exp(1) noise and takes the argmax: a sample of the
categorical distribution.  On the GPU that is one kernel (``ops.sample``: the same race in the log
domain, counter-based random numbers); the tensor-op form below is kept for CPU tensors and as the
definition.  The reference forbids T = 0; here a row with T = 0 is decoded greedily (argmax of the
raw logits, first maximum), which the benchmark configurations require.

With filters (top-k, top-p, min-p per row; None: off for all) the token is drawn by ``ops.sample_filtered`` with one uniform random
number per row from a generator of the sampler's own; ``filtered_tokens`` is its definition in tensor operations.
"""
from __future__ import annotations

import torch
from torch import nn


def filtered_tokens(logits: torch.Tensor, uniforms: torch.Tensor, temperatures: torch.Tensor, top_k: torch.Tensor | None = None,
                    top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None) -> torch.Tensor:
    """``ops.sample_filtered`` in tensor operations, in 64 bits: the borders lie between sums of many tokens."""
    x = torch.where(torch.isnan(logits), -torch.inf, logits.double())
    x, order = torch.sort(x, dim=1, descending=True, stable=True)          # of equal logits the lower token first
    t = temperatures.double()[:, None]
    top = x[:, :1]
    gap = torch.where(x == top, torch.zeros_like(x), x - top)              # also for two infinities
    w = torch.exp(gap / torch.where(t > 0, t, torch.ones_like(t)))
    keep = torch.ones_like(w, dtype=torch.bool)
    if top_k is not None:
        k = top_k.long()[:, None]
        keep &= (torch.arange(x.shape[1], device=x.device)[None] < k) | (k <= 0)
    if top_p is not None:
        p = top_p.double()[:, None]
        mass = w * keep
        near = (torch.cumsum(mass, 1) - mass < p * mass.sum(1, keepdim=True)) | (p >= 1)
        near[:, 0] = True
        keep &= near
    if min_p is not None:
        keep &= w >= min_p.double()[:, None].clamp(max=1)
    mass = torch.zeros_like(w).scatter_(1, order, w * keep)
    upto = torch.cumsum(mass, 1)
    drawn = (upto <= uniforms.double()[:, None].clamp(min=0) * upto[:, -1:]).sum(1)
    last = x.shape[1] - 1 - (mass.flip(1) > 0).to(torch.uint8).argmax(1)
    greedy = (t[:, 0] <= 0) | (top[:, 0] == -torch.inf)
    return torch.where(greedy, order[:, 0], torch.minimum(drawn, last))


class Sampler(nn.Module):
    def __init__(self, seed: int | None = None):
        super().__init__()
        self.seed = seed          # None: taken from torch.initial_seed() at the first draw
        self.calls = 0            # one random stream offset per call
        self.generators: dict[torch.device, torch.Generator] = {}     # of the random numbers behind filters

    def uniforms(self, n: int, device: torch.device) -> torch.Tensor:
        """One random number in [0, 1) for each of n rows."""
        if device not in self.generators:
            self.generators[device] = torch.Generator(device).manual_seed(torch.initial_seed() if self.seed is None else self.seed)
        return torch.rand(n, device=device, generator=self.generators[device])

    def forward(self, logits: torch.Tensor, temperatures: torch.Tensor | None, top_k: torch.Tensor | None = None,
                top_p: torch.Tensor | None = None, min_p: torch.Tensor | None = None) -> torch.Tensor:
        if temperatures is not None and not (top_k is None and top_p is None and min_p is None):
            move = lambda x, dtype: None if x is None else x.to(logits.device, dtype).contiguous()
            args = (self.uniforms(logits.shape[0], logits.device), move(temperatures, torch.float32), move(top_k, torch.int32),
                    move(top_p, torch.float32), move(min_p, torch.float32))
            if logits.is_cuda:
                from .. import ops
                return ops.sample_filtered(logits, *args)
            return filtered_tokens(logits, *args)
        if logits.is_cuda and logits.dim() == 2 and logits.stride(1) == 1 and logits.dtype in (torch.float32,
                                                                                               torch.bfloat16):
            from .. import ops
            if self.seed is None:
                self.seed = torch.initial_seed()
            self.calls += 1
            t = None if temperatures is None else temperatures.to(logits.device, torch.float32).contiguous()
            return ops.sample(logits, t, self.seed, self.calls)
        greedy = logits.argmax(dim=-1)
        if temperatures is None:
            return greedy
        t = temperatures.to(logits.device, torch.float32)
        safe = torch.where(t > 0, t, torch.ones_like(t))
        probs = torch.softmax(logits.float() / safe.unsqueeze(1), dim=-1)
        noise = torch.empty_like(probs).exponential_(1).clamp_min_(1e-10)
        sampled = (probs / noise).argmax(dim=-1)
        return torch.where(t > 0, sampled, greedy)
