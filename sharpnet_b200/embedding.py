"""Host-side mirror of SharpNet's word embedding on top of the C ABI (GPU kernels WordEmbeddingForwardPropagation /
WordEmbeddingBackwardPropagation, Prod/GPU/Kernels/SinglePrecision.cu:617,650).

The word indices come as a ``GPUTensor`` (floats, as SharpNet's tensors hold them) or as a contiguous int32 or int64
tensor on the wrapper's device."""
import torch

from . import _capi
from ._capi import check
from .tensor import GPUTensor

_INDEX_TYPES = {torch.int32: _capi.INDEX_INT32, torch.int64: _capi.INDEX_INT64}


def _indices(x, wrapper):
    """(index type, number of tokens, address) of the word indices."""
    if isinstance(x, GPUTensor):
        return _capi.INDEX_FP32, x.Count, x.storage.data_ptr()
    if x.dtype not in _INDEX_TYPES:
        raise ValueError(f"word indices are int32, int64, or floats in a GPUTensor, not {x.dtype}")
    if x.device != wrapper.device or not x.is_contiguous():
        raise ValueError("word indices must be contiguous and on the wrapper's device")
    return _INDEX_TYPES[x.dtype], x.numel(), x.data_ptr()


class EmbeddingLayer:
    """y[t, :] = scale * Weights[x[t], :], and its gradient.

    ``paddingIndex``: tokens with this index receive no gradient (-1: none).  ``weights`` / ``weightGradients`` are
    tensors of shape [vocabularySize, embeddingDim] to use in place of new ones of zeros (a table shared with another
    layer).  Make the first pass, which allocates, before capturing a graph.
    The scratch memory of the backward pass belongs to the layer: passes of one layer that may run at the same time on
    the GPU (two streams, two captured graphs) need a layer each."""

    def __init__(self, vocabularySize, embeddingDim, wrapper, scale=1.0, paddingIndex=-1, weights=None, weightGradients=None):
        self.vocabularySize, self.embeddingDim, self.w = int(vocabularySize), int(embeddingDim), wrapper
        self.scale, self.paddingIndex = float(scale), int(paddingIndex)
        shape = [self.vocabularySize, self.embeddingDim]
        for t in (weights, weightGradients):
            if t is not None and list(t.Shape) != shape:
                raise ValueError(f"the table must be {shape}, not {t.Shape}")
        self._weights, self._weightGradients = weights, weightGradients
        self._scratch = []          # the last one is in use; kernels queued earlier may still read the others

    def _new_table(self):
        t = GPUTensor((self.vocabularySize, self.embeddingDim), None, self.w)
        torch.cuda.current_stream(self.w.device).synchronize()      # its zeros, before the handle's stream reads it
        return t

    @property
    def Weights(self):
        if self._weights is None:
            self._weights = self._new_table()
        return self._weights

    @property
    def WeightGradients(self):
        if self._weightGradients is None:
            self._weightGradients = self._new_table()
        return self._weightGradients

    def ForwardPropagation(self, x, y):
        """``y``: [tokens, embeddingDim] (any shape with that many elements)."""
        w = self.w
        kind, tokens, at = _indices(x, w)
        if y.Count != tokens * self.embeddingDim:
            raise ValueError(f"y must hold {tokens} x {self.embeddingDim} elements, not {y.Shape}")
        check(w.handle, w.lib.snb200_embedding_fwd(w.handle, kind, tokens, self.vocabularySize, self.embeddingDim, at,
                                                   self.scale, self.Weights.storage.data_ptr(), y.storage.data_ptr()))

    def BackwardPropagation(self, x, dy, accumulate=False):
        """WeightGradients = (accumulate ? WeightGradients : 0) + the sums of ``dy`` by word."""
        w = self.w
        kind, tokens, at = _indices(x, w)
        if dy.Count != tokens * self.embeddingDim:
            raise ValueError(f"dy must hold {tokens} x {self.embeddingDim} elements, not {dy.Shape}")
        need = w.lib.snb200_embedding_scratch_bytes(tokens, self.vocabularySize, self.embeddingDim)
        if not self._scratch or self._scratch[-1].numel() < need:
            self._scratch.append(torch.empty(max(need, 16), dtype=torch.uint8, device=w.device))
        check(w.handle, w.lib.snb200_embedding_bwd(
            w.handle, kind, tokens, self.vocabularySize, self.embeddingDim, at, self.scale, self.paddingIndex, int(bool(accumulate)),
            dy.storage.data_ptr(), self._scratch[-1].data_ptr(), self.WeightGradients.storage.data_ptr()))
