"""Host-side mirror of the step between two blocks of a Transformer on top of the C ABI: SharpNet's LayerNorm / RMSNorm
kernels (Prod/GPU/Kernels/SinglePrecision.cu:32-297,1345) and its AddLayer as one pass over the rows each way."""
import torch

from . import _capi
from ._capi import check
from .tensor import GPUTensor

_KINDS = {"none": _capi.NORM_NONE, "layer": _capi.NORM_LAYER, "rms": _capi.NORM_RMS}
_PARAMETERS = ("gamma", "beta", "post_gamma", "post_beta", "gate")


def _at(t):
    return None if t is None else t.storage.data_ptr()


class ResidualNorm:
    """r = residual_scale * x + block_scale * gate * post_norm(block) ;  y = norm(r)

    over rows of ``dim`` elements; ``norm`` and ``post_norm`` are 'none', 'layer' or 'rms', ``gate_rows`` the rows of the
    gate (0: no gate; each serves as many consecutive rows of the batch).  Without a block it is a norm alone.

    ``Parameters`` and ``Gradients`` hold a tensor, or None, for each of gamma, beta, post_gamma, post_beta [dim] and gate
    [gate_rows, dim].  By default a norm has a gamma of ones, a LayerNorm a beta of zeros as well, and a gate is ones;
    ``parameters`` / ``gradients`` replace all of them (None: the parameter is not there, the gradient is not wanted).
    The statistics of the forward pass and the scratch memory of the backward pass belong to the layer: passes of one
    layer that may run at the same time on the GPU (two streams, two captured graphs) need a layer each.  Make the first
    passes, which allocate, before capturing a graph."""

    def __init__(self, dim, wrapper, norm="layer", post_norm="none", gate_rows=0, residual_scale=1.0, block_scale=1.0,
                 epsilon=1e-5, parameters=None, gradients=None):
        for kind in (norm, post_norm):
            if kind not in _KINDS:
                raise ValueError(f"a norm is one of {sorted(_KINDS)}, not {kind!r}")
        self.dim, self.w, self.gate_rows = int(dim), wrapper, int(gate_rows)
        self._desc = _capi.NormDesc(0, self.dim, _KINDS[norm], _KINDS[post_norm], self.gate_rows, residual_scale, block_scale, epsilon)
        shapes = {p: [self.gate_rows if p == "gate" else 1, self.dim] for p in _PARAMETERS}
        if parameters is None:
            there = {"gamma": norm != "none", "beta": norm == "layer", "post_gamma": post_norm != "none",
                     "post_beta": post_norm == "layer", "gate": gate_rows > 0}
            parameters = {p: GPUTensor(shapes[p], None, wrapper, torch.full((shapes[p][0] * self.dim,), float("beta" not in p),
                                                                           device=wrapper.device)) if there[p] else None
                          for p in _PARAMETERS}
        if gradients is None:
            gradients = {p: GPUTensor(parameters[p].Shape, None, wrapper) if parameters.get(p) is not None else None for p in _PARAMETERS}
        self.Parameters = {p: parameters.get(p) for p in _PARAMETERS}
        self.Gradients = {p: gradients.get(p) for p in _PARAMETERS}
        for tensors in (self.Parameters, self.Gradients):
            for p, t in tensors.items():
                if t is not None and t.Count != shapes[p][0] * self.dim:
                    raise ValueError(f"{p} must hold {shapes[p]} elements, not {t.Shape}")
        self._stats = self._post_stats = None
        self._kept = []             # buffers that were outgrown: kernels queued earlier may still use them
        self._scratch = None
        torch.cuda.current_stream(wrapper.device).synchronize()     # what was filled above, before the handle's stream reads it

    def SetStatistics(self, stats, post_stats):
        """The [rows, 2] tensors that the forward pass writes and the backward pass reads (new ones by default)."""
        self._stats, self._post_stats = stats, post_stats

    @staticmethod
    def _structure(tensors):
        return _capi.NormParams(*[_at(tensors[p]) for p in _PARAMETERS])

    def _buffer(self, count, shape):
        self._kept.append(GPUTensor(shape, None, self.w, torch.empty(max(count, 4), dtype=torch.float32, device=self.w.device)))
        return self._kept[-1]

    def _rows(self, **tensors):
        count = None
        for name, t in tensors.items():
            if t is None:
                continue
            if count is None:
                count = t.Count
            if t.Count != count or t.Shape[-1] != self.dim:
                raise ValueError(f"{name} must have the batch's rows of {self.dim} elements, not {t.Shape}")
        if count is None:
            raise ValueError("no input")
        self._desc.rows = count // self.dim if self.dim else 0
        return self._desc.rows

    def ForwardPropagation(self, x, block, r, y):
        """``block`` None: a norm alone; ``r`` may then be None, and may always be ``x``."""
        w, rows = self.w, self._rows(x=x, block=block, r=r, y=y)
        if self._desc.norm and (self._stats is None or self._stats.Count < 2 * rows):
            self._stats = self._buffer(2 * rows, (rows, 2))
        if self._desc.post_norm and (self._post_stats is None or self._post_stats.Count < 2 * rows):
            self._post_stats = self._buffer(2 * rows, (rows, 2))
        check(w.handle, w.lib.snb200_residual_norm_fwd(w.handle, self._desc, self._structure(self.Parameters), _at(x), _at(block),
                                                       _at(r), _at(y), _at(self._stats), _at(self._post_stats)))

    def BackwardPropagation(self, r, block, dy, dr, dx, dblock):
        """dx, dblock and ``Gradients`` from ``dy`` (of y) and ``dr`` (what reaches r past y, or None); ``r`` and ``block``
        are those of the forward pass (``r``: x itself where there was none).  dx may be dr."""
        w, rows = self.w, self._rows(r=r, block=block, dy=dy, dr=dr, dx=dx, dblock=dblock)
        for needed, stats in ((self._desc.norm, self._stats), (self._desc.post_norm, self._post_stats)):
            if needed and (stats is None or stats.Count < 2 * rows):
                raise ValueError("no statistics of a forward pass over these rows")
        need = w.lib.snb200_residual_norm_scratch_floats(self._desc)
        if self._scratch is None or self._scratch.Count < need:
            self._scratch = self._buffer(need, (need,))
        check(w.handle, w.lib.snb200_residual_norm_bwd(
            w.handle, self._desc, self._structure(self.Parameters), _at(r), _at(block), _at(dy), _at(dr), _at(self._stats),
            _at(self._post_stats), _at(self._scratch), _at(dx), _at(dblock),
            self._structure(self.Gradients)))
