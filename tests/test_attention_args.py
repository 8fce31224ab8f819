"""What the attention operators and the paged cache refuse, before anything is launched: no GPU needed."""
import pytest
import torch

from memfabric_hybrid_b200.ops import attention as A
from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache

BF, F8 = torch.bfloat16, torch.float8_e4m3fn


def _decode(**kw):
    a = {"q": torch.zeros(3, 8, 64, dtype=BF), "k_pages": torch.zeros(5, 2, 16, 64, dtype=BF), "v_pages": torch.zeros(5, 2, 16, 64, dtype=BF),
         "table": torch.zeros(3, 4, dtype=torch.int32), "lengths": torch.zeros(3, dtype=torch.int32)} | kw
    return A.decode_attention(a.pop("q"), a.pop("k_pages"), a.pop("v_pages"), a.pop("table"), a.pop("lengths"), **a)


def _pages(dtype=BF, pages=5, kv=2, page=16, dim=64):
    x = torch.zeros(pages, kv, page, dim)
    return {"k_pages": x.to(dtype), "v_pages": x.to(dtype)}


def _scales(n=2, dtype=torch.float32):
    return {"k_scale": torch.ones(n, dtype=dtype), "v_scale": torch.ones(n, dtype=dtype)}


@pytest.mark.parametrize("kw", [
    {"q": torch.zeros(3, 8, 128, dtype=BF)}, {"q": torch.zeros(3, 8 * 64, dtype=BF)}, {"q": torch.zeros(3, 7, 64, dtype=BF)}, {"q": torch.zeros(3, 8, 64)},
    {"q": torch.zeros(3, 8, 64, dtype=torch.float16)}, {"q": torch.zeros(3, 0, 64, dtype=BF)}, {"q": torch.zeros(4, 8, 64, dtype=BF)},
    {"q": torch.zeros(3, 8, 96, dtype=BF), **_pages(dim=96)}, {"q": torch.zeros(3, 8, 256, dtype=BF), **_pages(dim=256)},
    _pages(F8), {**_pages(F8), "k_scale": torch.ones(2)}, _scales(), {**_pages(F8), **_scales(3)}, {**_pages(F8), **_scales(2, BF)}, _pages(torch.float8_e5m2),
    _pages(torch.int8), {"v_pages": torch.zeros(5, 2, 16, 64, dtype=torch.float16)}, {"v_pages": torch.zeros(6, 2, 16, 64, dtype=BF)},
    {"v_pages": torch.zeros(5, 16, 2, 64, dtype=BF).transpose(1, 2)}, _pages(page=0), _pages(kv=0),
    {"table": torch.zeros(3, 4, dtype=torch.int64)}, {"table": torch.zeros(12, dtype=torch.int32)}, {"table": torch.zeros(4, 3, dtype=torch.int32).T},
    {"table": torch.zeros(3, 2 ** 28, dtype=torch.int32, device="meta")}, {"lengths": torch.zeros(3)}, {"lengths": torch.zeros(2, dtype=torch.int32)},
    {"rows": torch.zeros(2, dtype=torch.int32)}, {"rows": torch.zeros(3, dtype=torch.int64)}, {"scale": 0.0}, {"scale": -1.0}, {"scale": float("nan")},
    {"scale": float("inf")}, {"out": torch.zeros(3, 8, 64)}, {"out": torch.zeros(3, 8, 128, dtype=BF)}, {"out": torch.zeros(3, 1, 64, dtype=BF).expand(3, 8, 64)},
    {"lse": torch.zeros(3, 8, dtype=BF)}, {"lse": torch.zeros(8, 3)}, {"status": torch.zeros(2, dtype=torch.int32)}, {"status": torch.zeros(1)},
    {"q": torch.zeros(3, 8, 65, dtype=BF)[:, :, 1:]}, {"q": torch.zeros(3, 8, 128, dtype=BF)[:, :, ::2]}, {"q": torch.zeros(3, 8, 68, dtype=BF)[:, :, :64]},
    {"k_pages": torch.zeros(5, 2, 16, 72, dtype=BF)[..., :64]}, {"q": torch.zeros(3 * 8 * 64 + 1, dtype=BF)[1:].view(3, 8, 64)},
])
def test_decode_refuses(kw):
    with pytest.raises(ValueError):
        _decode(**kw)


def test_what_is_not_on_a_gpu_and_what_wants_a_gradient():
    with pytest.raises(ValueError, match="GPU"):
        _decode()
    with pytest.raises(RuntimeError, match="backward"):
        _decode(q=torch.zeros(3, 8, 64, dtype=BF, requires_grad=True))
    with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
        _decode(q=torch.zeros(3, 8, 64, dtype=BF, requires_grad=True))
    with pytest.raises(RuntimeError, match="backward"):
        _prefill(v=torch.zeros(10, 2, 64, dtype=BF, requires_grad=True))
    with pytest.raises(ValueError, match="GPU"):
        _prefill()


def _prefill(**kw):
    a = {"q": torch.zeros(10, 8, 64, dtype=BF), "k": torch.zeros(10, 2, 64, dtype=BF), "v": torch.zeros(10, 2, 64, dtype=BF),
         "cu_q": torch.zeros(3, dtype=torch.int32)} | kw
    return A.prefill_attention(a.pop("q"), a.pop("k"), a.pop("v"), a.pop("cu_q"), **a)


@pytest.mark.parametrize("kw", [
    {"q": torch.zeros(10, 8, 128, dtype=BF)}, {"q": torch.zeros(10, 9, 64, dtype=BF)}, {"q": torch.zeros(10, 8, 64)}, {"q": torch.zeros(1, 10, 8, 64, dtype=BF)},
    {"k": torch.zeros(10, 2, 64, dtype=torch.float16)}, {"v": torch.zeros(9, 2, 64, dtype=BF)}, {"v": torch.zeros(10, 2, 64, dtype=torch.float16)},
    {"k": torch.zeros(10, 0, 64, dtype=BF), "v": torch.zeros(10, 0, 64, dtype=BF)}, {"cu_q": torch.zeros(3)}, {"cu_q": torch.zeros(3, dtype=torch.int64)},
    {"cu_q": torch.zeros(0, dtype=torch.int32)}, {"cu_k": torch.zeros(4, dtype=torch.int32)}, {"cu_k": torch.zeros(3, dtype=torch.int64)}, {"scale": 0.0},
    {"scale": -0.1}, {"scale": float("nan")}, {"out": torch.zeros(10, 8, 64)}, {"out": torch.zeros(1, 8, 64, dtype=BF).expand(10, 8, 64)},
    {"lse": torch.zeros(8, 10)}, {"k": torch.zeros(10, 2, 68, dtype=BF)[..., :64]}, {"k": torch.zeros(10, 64, 2, dtype=BF).transpose(1, 2)},
    {"v": torch.zeros(10, 2, 65, dtype=BF)[..., 1:]},
    {"q": torch.zeros(10, 8, 96, dtype=BF), "k": torch.zeros(10, 2, 96, dtype=BF), "v": torch.zeros(10, 2, 96, dtype=BF)},
])
def test_prefill_refuses(kw):
    with pytest.raises(ValueError):
        _prefill(**kw)


@pytest.mark.parametrize("kw", [
    {"data": torch.zeros(2, 5, 3, 2, 4, 16, dtype=BF)}, {"data": torch.zeros(2, 5, 2, 2, 4, 24, dtype=BF)}, {"data": torch.zeros(2, 5, 2, 2, 4, 16)},
    {"data": torch.zeros(2, 5, 2, 4, 2, 16, dtype=BF).transpose(3, 4)}, {"data": torch.zeros(5, 2, 2, 4, 16, dtype=BF)}, {"data": torch.zeros(0, 5, 2, 2, 4, 16, dtype=BF)},
    {"table": torch.zeros(3, 6, dtype=torch.int64)}, {"table": torch.zeros(3, 12, dtype=torch.int32)[:, :6]}, {"table": torch.zeros(0, 6, dtype=torch.int32)},
    {"table": torch.zeros(3, 2 ** 30, dtype=torch.int32, device="meta")}, {"lengths": torch.zeros(4, dtype=torch.int32)}, {"refs": torch.zeros(6, dtype=torch.int32)},
    {"refs": torch.zeros(6, dtype=torch.int32)[1:]}, {"status": torch.zeros(1)}, {},
])
def test_cache_refuses(kw):
    a = {"data": torch.zeros(2, 5, 2, 2, 4, 16, dtype=BF), "table": torch.zeros(3, 6, dtype=torch.int32), "lengths": torch.zeros(3, dtype=torch.int32),
         "refs": torch.zeros(5, dtype=torch.int32)} | kw
    with pytest.raises(ValueError):
        PagedKVCache(**a)


def test_a_stream_of_another_gpu_is_refused():
    from types import SimpleNamespace

    from memfabric_hybrid_b200.ops.attention import launch_on

    with pytest.raises(ValueError, match="the stream belongs to cuda:1"):
        launch_on(0, SimpleNamespace(device=torch.device("cuda", 1)))
