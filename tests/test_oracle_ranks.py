"""The hand-over from a rank of a CPU test to its parent."""

import pytest
import torch
import torch.multiprocessing as mp


def _tensors():
    g = torch.Generator().manual_seed(3)
    return {"half": torch.randn(5, 7, generator=g).half(), "bf16": torch.randn(3, generator=g).bfloat16(),
            "scalar": torch.tensor(2.5), "empty": torch.zeros(0, 4), "bool": torch.tensor([True, False]),
            "strided": torch.arange(24).view(4, 6).t()[1:4], "double": torch.randn(2, 2, generator=g).double()}


def _rank(queue):
    import oracle  # noqa: F401 - as the ranks of the tests do

    queue.put((7, _tensors()))


@pytest.mark.parametrize("count", [1, 3])
def test_results_outlive_their_rank(count):
    """The parent takes the results off the queue after every rank has ended."""
    context = mp.get_context("spawn")
    queue = context.Queue()
    ranks = [context.Process(target=_rank, args=(queue,)) for _ in range(count)]
    for rank in ranks:
        rank.start()
    for rank in ranks:
        rank.join(240)
        assert rank.exitcode == 0
    want = _tensors()
    for _ in ranks:
        number, got = queue.get(timeout=60)
        assert number == 7 and got.keys() == want.keys()
        for name, t in want.items():
            assert got[name].dtype == t.dtype and torch.equal(got[name], t), name
