"""Norm over the channels of a row, in tflib's manner (beside layernorm.py, whose moments run over a whole sample as in the reference)."""
import numpy as np

from ... import autograd as A
from ... import tflib as lib


def Rownorm(name, inputs, kind='layer', eps=1e-5, save8=None):
    """Layer norm (`kind` 'layer': variables `<name>.offset`, `<name>.scale`) or RMS norm ('rms': `<name>.scale` alone) over the last axis of
    `inputs` [..., C].  `save8` ('e4m3' | 'int8'): the normed values kept in 8 bits for the backward pass."""
    n_neurons = inputs.shape[-1]
    offset = lib.param(name + '.offset', np.zeros(n_neurons, dtype='float32')) if kind == 'layer' else None
    scale = lib.param(name + '.scale', np.ones(n_neurons, dtype='float32'))
    return A.rownorm(inputs, scale, offset, eps, kind, save8)
