"""Activations of a taped forward kept in 8 bits until the reverse pass (encoder.checkpoint_bits: 8).

The tape refers to activations by tensor.  Keep8 encodes a tensor that the forward has no further use for
(mmb_checkpoint_rows: 32 features share a power-of-two step) and gives its memory back by shrinking the storage to nothing;
the tensor object stays what the tape and the gradient store know it by.  In the reverse pass weight gradients read the
codes themselves (mmb_grad_weight_rows_q8); what needs the values (attention, LayerNorm, the ReLU gate) gets the rows
restored into the same storage for as long as it runs.  No counterpart in the reference.
"""
from contextlib import contextmanager

from mmb_hip import ops


def storage_id(t):
    """Identity of a tensor's storage, also while the storage is shrunk to nothing."""
    return t.untyped_storage()._cdata


class Keep8:
    def __init__(self):
        self._kept = {}                                     # storage -> (tensor, Q8Rows)

    def __bool__(self):
        return bool(self._kept)

    def keep(self, t, gate=False):
        """Encode t (a matrix that owns its whole storage) and free its memory; anything else is left alone.  gate: the
        reverse pass asks which values are positive, so none may round to zero."""
        if t is None or t.dim() != 2 or not t.is_contiguous() or t.storage_offset() != 0 or \
                storage_id(t) in self._kept or t.untyped_storage().nbytes() != t.numel() * t.element_size():
            return
        self._kept[storage_id(t)] = (t, ops.checkpoint_rows(t, keep_nonzero=gate))
        t.untyped_storage().resize_(0)

    def rows(self, t):
        """The Q8Rows of t, None if t was not kept here (or is a part of what was)."""
        e = self._kept.get(storage_id(t))
        return e[1] if e is not None and e[0].shape == t.shape else None

    @contextmanager
    def restored(self, *tensors):
        """The kept ones among the tensors hold their (decoded) values inside the block."""
        back = []
        try:
            for t in tensors:
                e = self._kept.get(storage_id(t)) if t is not None else None
                if e is not None and t.untyped_storage().nbytes() == 0:
                    t.untyped_storage().resize_(e[0].numel() * e[0].element_size())
                    back.append(t)
                    ops.restore_rows(e[1], out=e[0])
            yield
        finally:
            for t in back:
                t.untyped_storage().resize_(0)


def activations(entries):
    """(tensor, whether it is the output of a ReLU) for the activations that tape entries of transformer layers refer to; a
    tensor's own entry, where it is an output, comes before those that read it."""
    for e in entries:
        if e[0] == "plinear":
            for t, _ in e[3]:
                yield t, False
            for t in (e[5], e[7], e[8]):
                yield t, False
            for t in (e[9], e[10]):
                yield t, e[4] == "relu"
        elif e[0] in ("attn", "ln"):
            yield e[1], False
            yield e[2], False
