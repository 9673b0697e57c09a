"""What the state space operators of ``Backend`` take: the batch of sequences whose tokens ``causal_conv`` and ``selective_scan`` mix."""
import numpy as np


class StateBatch:
    """The sequences of a call: int32 device tensors ``offsets`` [sequences + 1] and, where states are kept between calls, ``lengths``, ``slots`` and ``out_slots``
    [sequences] (``out_slots`` None: the same as ``slots``), and the host's bound of a sequence's new tokens.

    A sequence whose length is no more than its new tokens begins with them; others continue the state in their slot of the pool.  What a call writes
    to a slot no other sequence of the call may read or write."""

    def __init__(self, offsets, max_new, lengths=None, slots=None, out_slots=None):
        if out_slots is None:
            out_slots = slots
        seqs = offsets.shape[0] - 1 if len(offsets.shape) == 1 else -1
        kept = [t for t in (lengths, slots, out_slots) if t is not None]
        if not 0 <= seqs < 2 ** 31 or len(kept) not in (0, 3) or any(tuple(t.shape) != (seqs,) for t in kept) or any(t.dtype != "int32" for t in (offsets, *kept)):
            raise ValueError("a batch is int32 offsets [sequences + 1] and no or both of lengths and slots [sequences], not %s %s"
                             % (offsets.shape, [getattr(t, "shape", None) for t in (lengths, slots, out_slots)]))
        if int(max_new) < 0:
            raise ValueError("a bound of %d new tokens" % int(max_new))
        self.offsets, self.lengths, self.slots, self.out_slots, self.max_new = offsets, lengths, slots, out_slots, min(int(max_new), 2 ** 31 - 1)  # (an int of the library)
        self.arguments = (offsets.address, *(t.address if t is not None else None for t in (lengths, slots, out_slots)), seqs, self.max_new)

    def unkept(self):
        """The same sequences, whose states go nowhere."""
        return StateBatch(self.offsets, self.max_new, self.lengths, self.slots, self.slots.backend.array(np.full(self.slots.shape, -1), "int32"))
