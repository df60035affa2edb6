"""What the ranks of a multi-process CPU test send to their parent.

torch.multiprocessing sends a CPU tensor as a file descriptor of shared memory, which the receiver fetches
from the sender when it unpickles it: a rank that has put its results on a queue and ended by then
leaves nothing to fetch from. Results are small; here they go by value, so that a rank may end as soon
as its queue has been flushed.
"""

from multiprocessing.reduction import ForkingPickler

import torch
from torch.multiprocessing import reductions


def _rebuild(data, dtype, shape):
    if not data:
        return torch.empty(shape, dtype=dtype)
    return torch.frombuffer(bytearray(data), dtype=dtype).reshape(shape)


def _by_value(t):
    if t.device.type != "cpu" or t.layout != torch.strided or t.is_quantized:
        return reductions.reduce_tensor(t)
    flat = t.detach().resolve_conj().resolve_neg().contiguous().reshape(-1)
    return _rebuild, (flat.view(torch.uint8).numpy().tobytes(), t.dtype, tuple(t.shape))


def send_by_value():
    """From now on this process pickles CPU tensors for other processes by value (detached)."""
    ForkingPickler.register(torch.Tensor, _by_value)
