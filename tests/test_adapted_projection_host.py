"""Host side of the adapted 4-bit projections, on CPU tensors (no kernel launches): who is served, what
is refused, what a call leaves behind."""

import threading
from types import SimpleNamespace

import torch

from talm_b200 import qgroup


def _served(rows=1):
    """Whether a CUDA tensor of that many rows would be served now."""
    x = SimpleNamespace(is_cuda=True, shape=(rows, 64), numel=lambda: rows * 64)
    with torch.no_grad():
        return qgroup.takes_matvec(x)


# ------------------------------------------------------------------------------------------
# serving
# ------------------------------------------------------------------------------------------
def test_serving_of_two_threads_that_overlap():
    """A enters, B enters, A leaves, B leaves: each has its own route until it leaves, and nothing stays
    on behind them."""
    turn = [threading.Event() for _ in range(4)]
    seen = {}

    def first():
        with qgroup.serving(4):
            seen["a"] = (_served(4), _served(5))
            turn[0].set()
            turn[1].wait(30)
        seen["a left"] = _served()
        turn[2].set()

    def second():
        turn[0].wait(30)
        seen["b before"] = _served()
        with qgroup.serving(8):
            turn[1].set()
            turn[2].wait(30)
            seen["b"] = (_served(8), _served(9))
        seen["b left"] = _served()

    threads = [threading.Thread(target=f) for f in (first, second)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert seen == {"a": (True, False), "a left": False, "b before": False, "b": (True, False),
                    "b left": False}
    assert not _served()


def test_serving_blocks_that_end_out_of_order():
    """Two blocks of one thread, left in the order in which they were entered."""
    outer, inner = qgroup.serving(4), qgroup.serving(8)
    outer.__enter__()
    inner.__enter__()
    assert _served(8)
    outer.__exit__(None, None, None)
    assert _served(8)
    inner.__exit__(None, None, None)
    assert not _served()
