"""The models' layer norms with a HIP mode beside PyTorch's, chosen as the experts containers choose theirs: by
``forward_mode``.

``'torch'`` (the default) is ``F.layer_norm``, and the residual addition ahead of a block's second norm a tensor addition of
its own.  ``'hip'`` runs the layer-norm kernels, forward and backward, with that addition inside (``add_norm``).  Both modes
store the same tensors in the same element types.  The residual stream has the same bits; the norm's output differs by the
float32 roundings of the row's sums, taken in another order: a few 2^-24 of |n w| + |b|, so 16-bit values now and then by
a step, float32 ones in their last bits, and by more of their own size where n w + b comes near zero.

Hooks on a norm that ``add_norm`` calls see what the mode passes: (x) and the output in ``'torch'`` mode, (x, residual) with
the sum not yet taken, and the pair (output, sum), in ``'hip'`` mode."""
from __future__ import annotations

import torch
from torch import nn
from torch.nn import functional as F

from . import functional
from .hip_abi import D2DMoEError


class NormModes:
    """Mixin of the layer-norm modules: `weight`, `bias` and `norm_eps()` come from the module."""
    MODES = ('torch', 'hip')
    forward_mode = 'torch'

    def norm_eps(self) -> float:
        return 1e-5

    def _hip(self, x) -> bool:
        if self.forward_mode not in self.MODES:
            raise NotImplementedError(f'Unsupported forward_mode: {self.forward_mode}')
        if self.forward_mode == 'torch':
            return False
        if not x.is_cuda:
            raise D2DMoEError("forward_mode 'hip' needs a ROCm device; use 'torch' on the CPU")
        return True

    def _forward_hip(self, x, residual):
        """The kernels take one element type; what the 'torch' mode takes beside that is brought to it here: a sum of two types
        has the wider one (autocast: a 16-bit branch on a float32 stream), and autocast runs a norm in float32."""
        weight, bias = self.weight, self.bias
        if residual is not None and residual.dtype != x.dtype:
            wide = torch.promote_types(x.dtype, residual.dtype)
            x, residual = x.to(wide), residual.to(wide)
        if torch.is_autocast_enabled('cuda'):
            weight, bias = (None if p is None else p.float() for p in (weight, bias))
            if x.dtype != torch.float32:
                h = x if residual is None else x + residual
                out = functional.layer_norm(h.float(), weight, bias, self.norm_eps())
                return out if residual is None else (out, h)
        return functional.layer_norm(x, weight, bias, self.norm_eps(), residual)

    def forward(self, x, residual=None):
        """norm(x), or (norm(x + residual), x + residual)."""
        if self._hip(x):
            return self._forward_hip(x, residual)
        h = x if residual is None else x + residual
        out = F.layer_norm(h, (h.size(-1),), self.weight, self.bias, self.norm_eps())
        return out if residual is None else (out, h)


def add_norm(norm: nn.Module, x, residual):
    """(norm(h), h) of the residual stream h = x + residual, where a block's next half begins.  In one call where the norm runs
    on the HIP kernels; any other module sees the sum alone."""
    if isinstance(norm, NormModes) and norm.forward_mode == 'hip':
        return norm(x, residual)
    h = x + residual
    return norm(h), h


def set_norm_mode(model: nn.Module, mode: str) -> int:
    """Sets forward_mode of every layer norm of this package in `model`; returns how many there are."""
    if mode not in NormModes.MODES:
        raise ValueError(f'mode is one of {NormModes.MODES}, got {mode!r}')
    norms = [m for m in model.modules() if isinstance(m, NormModes)]
    for m in norms:
        m.forward_mode = mode
    return len(norms)
