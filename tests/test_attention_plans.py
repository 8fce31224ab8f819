"""What the attention operators plan before a call, on the host: no GPU needed."""
import contextlib

import pytest
import torch

from memfabric_hybrid_b200.ops import attention as A

BF = torch.bfloat16


def test_the_workspace_is_sized_on_the_gpu_of_the_tensors(monkeypatch):
    """Its size goes by the number of SMs; the current GPU may be another one with fewer."""
    entered = []

    class Plan:
        def __init__(self, *args):
            pass

        def workspace(self):
            return 4096 if entered == [3] else 64

    @contextlib.contextmanager
    def launch_on(device, stream):
        entered.append(device)
        yield
        entered.pop()

    class Meta(torch.Tensor):
        device = torch.device("cuda", 3)

    monkeypatch.setattr(A, "launch_on", launch_on)
    monkeypatch.setattr(A, "on_gpu", lambda *args, **kw: None)
    monkeypatch.setattr(A._ops, "DecodePlan", Plan)
    q, pages = torch.zeros(3, 8, 64, dtype=BF).as_subclass(Meta), torch.zeros(5, 2, 16, 64, dtype=BF)
    key = object()
    try:
        _, words, _ = A._plan_decode(key, q, pages, pages, torch.zeros(3, 40, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), None, None, None, None, None, None)
    finally:
        A._decode_plans._known.pop(key, None)
    assert words == 1024 and entered == []


@pytest.mark.parametrize("dim", [64, 128])
def test_a_workspace_that_is_too_small_is_refused(dim):
    # q, out and page strides; B 3, 8 query heads to each of 2, pages of 16, 5 of them, 40 to a sequence of 3
    plan = A._ops.DecodePlan(16 * dim, dim, 16 * dim, dim, 32 * dim, 16 * dim, dim, 40, 3, 2, 8, 16, 5, 40, 3, dim, A._ops.BF16, A._ops.BF16)
    need = plan.workspace()
    assert need > 0
    for given in (0, 4, need - 4):
        # refused before anything is launched: the addresses are none
        assert plan.run(0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 4096, given, 1.0, 0) == -2
