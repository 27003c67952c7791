"""Device op tables.  `default_ops(device)` returns the sm_100a kernel table on a
CUDA device (and raises if the extension is missing there: a silent fallback
would hide that the kernels are not running) and the plain-torch table on CPU."""

from __future__ import annotations

import torch

from .torch_ops import TorchOps

_cache = {}
_tables = {}                          # the same by the argument itself: a call per operator is on the hot path of small ones


def default_ops(device):
    table = _tables.get(device)
    if table is None:
        table = _tables[device] = _find_table(torch.device(device))
    return table


def _find_table(device):
    key = (device.type, device.index)
    if key not in _cache:
        if device.type == "cuda":
            from .cuda_ops import CudaOps
            _cache[key] = CudaOps(device)
        else:
            _cache[key] = TorchOps()
    return _cache[key]


from .packed import TokenLogprobs, cached_attention, packed_attention, token_logprobs  # noqa: E402  (needs default_ops)

__all__ = ["TorchOps", "default_ops", "packed_attention", "cached_attention", "token_logprobs", "TokenLogprobs"]
