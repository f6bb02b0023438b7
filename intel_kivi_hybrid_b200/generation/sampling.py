"""Next-token choice for the generate() loop (reference:
src/kivi_sycl/generation/sampling.py:10-25): argmax unless ``do_sample``;
otherwise temperature scaling, optional top-k cut, softmax, one multinomial
draw.  Returns ids of shape [batch, 1].

Beyond the reference, ``top_p`` keeps the most probable entries that hold that much
of what the top-k cut leaves, and ``min_p`` those with at least that much of the largest
one's probability; ties stay together.  Such draws are ``kivi_sample_filtered``, from
random numbers of torch's generator of the logits' device.

Logits that live on a CUDA device are handled by one kernel of the library
(``kivi_sample_tokens``): the ids stay on the device, so the decode loop needs no
host round trip per token.  Its draws come from a counter-based generator whose
key is taken, call by call, from torch's default CPU generator (so
``torch.manual_seed`` makes a run repeatable, as it does for the reference's
``torch.multinomial``, and drawing the key touches no device).  Logits on the
CPU (a model kept on the host, as in the reference's own set-up) go through the
same torch operations the reference uses.
"""
from typing import Optional

import torch

__all__ = ["sample_token", "DeviceSampler"]


class DeviceSampler:
    """(seed, step) bookkeeping of the device-side draws.  With a fixed ``seed``
    every call advances ``step``; without one, each sampling call draws a fresh
    62-bit key from torch's default CPU generator."""

    def __init__(self, seed: Optional[int] = None):
        self.seed = None if seed is None else int(seed)
        self.step = 0

    def __call__(self, logits: torch.Tensor, temperature: float, top_k: Optional[int], do_sample: bool, top_p: float = 1.0, min_p: float = 0.0) -> torch.Tensor:
        from .. import cabi
        if logits.dtype not in (torch.float32, torch.bfloat16):
            logits = logits.float()
        if logits.stride(-1) != 1:
            logits = logits.contiguous()
        if do_sample and (top_p < 1.0 or min_p > 0.0):
            B, dev = logits.shape[0], logits.device
            if self.seed is None:
                u = torch.rand(B, device=dev)
            else:
                u = torch.rand(B, device=dev, generator=torch.Generator(device=dev).manual_seed((self.seed + 0x9E3779B97F4A7C15 * self.step) % 2 ** 63))
                self.step += 1
            row = lambda x, dtype=torch.float32: torch.full((B,), x, dtype=dtype, device=dev)  # noqa: E731
            cut = row(min(max(int(top_k or 0), 0), 2 ** 31 - 1), torch.int32)
            return cabi.sample_filtered(logits, u, row(max(temperature, 1e-8)), cut, row(top_p), row(min_p)).unsqueeze(1)
        if self.seed is None:       # a fresh key per call: the counter stays at 0
            seed, step = (int(torch.randint(0, 2 ** 62, (1,)).item()) if do_sample else 0), 0
        else:
            seed, step = self.seed, self.step
            self.step += 1
        return cabi.sample_tokens(logits, temperature, top_k or 0, do_sample, seed, step).unsqueeze(1)


_default = None


def sample_token(logits: torch.Tensor, temperature: float, top_k: Optional[int], do_sample: bool, top_p: float = 1.0, min_p: float = 0.0) -> torch.Tensor:
    global _default
    if logits.is_cuda:
        if _default is None:
            _default = DeviceSampler()
        return _default(logits, temperature, top_k, do_sample, top_p, min_p)
    if not do_sample:
        return torch.argmax(logits, dim=-1, keepdim=True)
    filtered = top_p < 1.0 or min_p > 0.0
    if filtered and logits.dtype in (torch.float16, torch.bfloat16):
        logits = logits.float()              # (in 8 or 11 bits different probabilities become ties, and their sums stand still)
    scaled = logits / max(temperature, 1e-8)
    if top_k is not None:
        kth = torch.topk(scaled, top_k, dim=-1).values[:, -1:]
        scaled = scaled.masked_fill(scaled < kth, float("-inf"))
    probs = torch.softmax(scaled, dim=-1)
    if filtered:
        # what lies above an entry: the mass of the strictly larger ones, the same for ties
        largest = probs.amax(-1, keepdim=True)
        ordered, order = probs.sort(dim=-1, descending=True)
        first = torch.searchsorted(-ordered, -ordered)                   # first entry of each run of ties
        above = (ordered.cumsum(-1) - ordered).gather(-1, first)
        keep = torch.zeros_like(probs, dtype=torch.bool).scatter_(-1, order, (above < top_p) if top_p < 1.0 else torch.ones_like(above, dtype=torch.bool))
        keep &= probs >= min_p * largest
        probs = probs.masked_fill(~(keep | (probs == largest)), 0.0)
    return torch.multinomial(probs, num_samples=1)
