"""Host-side mirror of SharpNet's optimizers for the parameters of a Dense layer
(Prod/Optimizers/VanillaSgd.cs, Sgd.cs, Adam.cs).  Each ``UpdateWeights`` keeps the reference's
argument list and issues one fused update kernel per tensor through the C ABI; ``AdamGroup`` takes all
tensors of a model in one."""
import torch

from . import _capi
from ._capi import check
from .tensor import GPUTensor


def PonderedLearning(learningRate, batchSize):
    """lr / batchSize (Prod/Optimizers/Optimizer.cs:26-29)."""
    return float(learningRate) / batchSize


class VanillaSgd:
    """W -= lr/batch * dW   (Prod/Optimizers/VanillaSgd.cs:12-21)."""

    def UpdateWeights(self, learningRate, maxLearningRate, batchSize, weights, weightGradients, bias, biasGradients):
        lr = PonderedLearning(learningRate, batchSize)
        weights.UpdateSGDOptimizer(lr, 0.0, False, weightGradients, None)
        if bias is not None:
            bias.UpdateSGDOptimizer(lr, 0.0, False, biasGradients, None)


class Sgd:
    """SGD with (Nesterov) momentum   (Prod/Optimizers/Sgd.cs:18-52)."""

    def __init__(self, wrapper, SGD_momentum, nesterov, weightShape, biasShapeIfAny):
        self.momentum, self.nesterov = SGD_momentum, nesterov
        self._velocityWeight = GPUTensor(weightShape, None, wrapper)
        self._velocityBias = None if biasShapeIfAny is None else GPUTensor(biasShapeIfAny, None, wrapper)

    def UpdateWeights(self, learningRate, maxLearningRate, batchSize, weights, weightGradients, bias, biasGradients):
        lr = PonderedLearning(learningRate, batchSize)
        weights.UpdateSGDOptimizer(lr, self.momentum, self.nesterov, weightGradients, self._velocityWeight)
        if bias is not None:
            bias.UpdateSGDOptimizer(lr, self.momentum, self.nesterov, biasGradients, self._velocityBias)


class Adam:
    """Adam / AdamW   (Prod/Optimizers/Adam.cs:30-72)."""

    def __init__(self, wrapper, adam_beta1, adam_beta2, adam_eps, weight_decay, weightShape, biasShapeIfAny):
        self.beta1, self.beta2, self.eps, self.weight_decay = adam_beta1, adam_beta2, adam_eps, weight_decay
        self._timestep = 0
        self._adam_VW, self._adam_SW = GPUTensor(weightShape, None, wrapper), GPUTensor(weightShape, None, wrapper)
        self._adam_VB = self._adam_SB = None
        if biasShapeIfAny is not None:
            self._adam_VB, self._adam_SB = GPUTensor(biasShapeIfAny, None, wrapper), GPUTensor(biasShapeIfAny, None, wrapper)

    def UpdateWeights(self, learningRate, maxLearningRate, batchSize, weights, weightGradients, bias, biasGradients):
        self._timestep += 1
        pondered_weight_decay = (learningRate / maxLearningRate) * self.weight_decay
        weights.UpdateAdamOptimizer(learningRate, self.beta1, self.beta2, self.eps, pondered_weight_decay,
                                    weightGradients, self._adam_VW, self._adam_SW, self._timestep)
        if bias is not None:
            bias.UpdateAdamOptimizer(learningRate, self.beta1, self.beta2, self.eps, pondered_weight_decay,
                                     biasGradients, self._adam_VB, self._adam_SB, self._timestep)


class AdamGroup:
    """Adam / AdamW over all parameter tensors of a model as one launch (the loop over the layers' ``Adam.UpdateWeights``,
    Prod/Optimizers/Adam.cs:59-72), with the moments in 32 or in 8 bits.

    ``decays``: a factor of ``weight_decay`` per tensor (1 by default; 0 for biases and norms is customary).  ``states``:
    moments to go on with, one tuple (adam_vW, adam_sW), with 8 bits (adam_vW, adam_sW, v_scale, s_scale), of flat tensors
    per weight tensor, with the ``timestep`` they were left at; zeros by default.  The weights, gradients and moments are
    the tensors given, updated in place, and must not be replaced while the group lives."""

    def __init__(self, wrapper, adam_beta1, adam_beta2, adam_eps, weight_decay, weights, weightGradients, decays=None,
                 state_bits=32, states=None, timestep=0):
        if state_bits not in (8, 32):
            raise ValueError(f"moments of {state_bits} bits: 8 or 32")
        if len(weights) != len(weightGradients) or any(a.Count != b.Count for a, b in zip(weights, weightGradients)):
            raise ValueError("weights and gradients do not match")
        self.w, self.state_bits = wrapper, state_bits
        self.beta1, self.beta2, self.eps, self.weight_decay = adam_beta1, adam_beta2, adam_eps, weight_decay
        self.timestep = int(timestep)
        decays = [1.0] * len(weights) if decays is None else [float(d) for d in decays]
        if states is None:
            def zeros(n, dtype):
                return torch.zeros(n, dtype=dtype, device=wrapper.device)
            moment = torch.float32 if state_bits == 32 else torch.uint8
            states = [(zeros(t.Count, moment), zeros(t.Count, moment)) +
                      ((zeros(-(-t.Count // 256), torch.float32), zeros(-(-t.Count // 256), torch.float32)) if state_bits == 8 else ())
                      for t in weights]
        if len(decays) != len(weights) or len(states) != len(weights):
            raise ValueError("decays and states must have an entry for each weight tensor")
        for t, s in zip(weights, states):
            blocks = -(-t.Count // 256)
            if ([p.numel() for p in s] != [t.Count] * 2 + ([blocks] * 2 if state_bits == 8 else []) or
                    any(not p.is_contiguous() or p.device != wrapper.device for p in s) or
                    any(p.element_size() != 1 if state_bits == 8 else p.dtype != torch.float32 for p in s[:2]) or
                    any(p.dtype != torch.float32 for p in s[2:])):
                raise ValueError(f"the moments do not match a weight tensor of {t.Count} elements")
        torch.cuda.current_stream(wrapper.device).synchronize()      # the zeros above, before the handle's stream reads them
        self._tensors, self.states = (list(weights), list(weightGradients)), list(states)
        self._table = (_capi.AdamTensor * len(weights))(*[
            _capi.AdamTensor(t.Count, g.storage.data_ptr(), t.storage.data_ptr(), *[p.data_ptr() for p in s],
                             *([None] * (4 - len(s))), d)
            for t, g, s, d in zip(weights, weightGradients, self.states, decays)])

    def UpdateWeights(self, learningRate, maxLearningRate):
        """One step; the decay is pondered as in ``Adam.UpdateWeights``.  The stochastic rounding of 8-bit moments takes
        the time step as its seed."""
        self.timestep += 1
        w = self.w
        check(w.handle, w.lib.snb200_adam_group_update(
            w.handle, len(self._table), self._table, self.state_bits, learningRate, self.beta1, self.beta2, self.eps,
            (learningRate / maxLearningRate) * self.weight_decay, self.timestep, self.timestep & 0xFFFFFFFF))
