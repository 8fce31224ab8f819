"""What the attention operators plan before a call, on the host: no GPU needed."""
import contextlib

import pytest
import torch
from torch.autograd import forward_ad

from memfabric_hybrid_b200.ops import attention as A
from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache

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


def _decode(**kw):
    a = {"q": torch.zeros(3, 8, 64, dtype=BF), "k": torch.zeros(5, 2, 16, 64).to(torch.float8_e4m3fn), "k_scale": torch.ones(2), "v_scale": torch.ones(2)} | kw
    k = a.pop("k")
    return A.decode_attention(a.pop("q"), k, k, torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), **a)


def _prefill(**kw):
    a = {"q": torch.zeros(10, 8, 64, dtype=BF), "k": torch.zeros(10, 2, 64, dtype=BF), "v": torch.zeros(10, 2, 64, dtype=BF)} | kw
    return A.prefill_attention(a.pop("q"), a.pop("k"), a.pop("v"), torch.zeros(3, dtype=torch.int32), **a)


def _write(**kw):
    cache = PagedKVCache.__new__(PagedKVCache)  # without a GPU there is none
    cache.layers, cache._writes = 1, A.Plans()
    cache._plan_write = lambda *args: (0,)
    a = {"k": torch.zeros(10, 2, 64, dtype=BF), "v": torch.zeros(10, 2, 64, dtype=BF), "k_scale": torch.ones(2), "v_scale": torch.ones(2)} | kw
    cache.write(0, a.pop("k"), a.pop("v"), torch.zeros(10, dtype=torch.int64), **a)


CALLS = [(_decode, "q", (3, 8, 64), BF), (_decode, "k_scale", (2,), torch.float32), (_decode, "v_scale", (2,), torch.float32), (_decode, "out", (3, 8, 64), BF),
         (_decode, "lse", (3, 8), torch.float32), (_prefill, "q", (10, 8, 64), BF), (_prefill, "k", (10, 2, 64), BF), (_prefill, "v", (10, 2, 64), BF),
         (_prefill, "out", (10, 8, 64), BF), (_prefill, "lse", (10, 8), torch.float32), (_write, "k", (10, 2, 64), BF), (_write, "v", (10, 2, 64), BF),
         (_write, "k_scale", (2,), torch.float32), (_write, "v_scale", (2,), torch.float32)]


@pytest.mark.parametrize("call,name,shape,dtype", CALLS)
def test_whatever_wants_a_gradient_is_refused(call, name, shape, dtype):
    with pytest.raises(RuntimeError, match="backward"):
        call(**{name: torch.zeros(shape, dtype=dtype, requires_grad=True)})


@pytest.mark.parametrize("call,name,shape,dtype", CALLS)
def test_tangents_are_not_dropped(call, name, shape, dtype):
    with forward_ad.dual_level():
        x = forward_ad.make_dual(torch.zeros(shape, dtype=dtype), torch.ones(shape, dtype=dtype))
        with pytest.raises(RuntimeError, match="forward-mode"):
            call(**{name: x})


@pytest.mark.parametrize("scale", [1e39, 1.8e38, 2.0 ** 127 * 1.01, 1e-38, 1e-45, 1e-50])
@pytest.mark.parametrize("call", [_decode, _prefill])
def test_scales_that_fp32_does_not_hold_are_refused(call, scale):
    """As fp32 numbers, with the factor to powers of two and its inverse: infinite, 0 or without all their bits."""
    with pytest.raises(ValueError, match="scale must"):
        A._scale(scale, 64)
    for fine in (2.0 ** 127, 2.0 ** -125, 1.0, None):
        A._scale(fine, 64)
    with pytest.raises(ValueError, match="scale must|GPU"):
        call(scale=scale)
