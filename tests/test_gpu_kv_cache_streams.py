"""The paged cache used on other streams than the current one."""
import pytest

pytestmark = pytest.mark.gpu


def test_check_status_waits_for_calls_on_every_stream():
    """A call that another stream has not come to yet is told of, too, and what comes after the check is not wiped out by it."""
    import torch

    from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache

    cache = PagedKVCache.allocate(1, 8, 4, 1, 16, 3, 4)
    none, first = (torch.tensor([n], dtype=torch.int32, device="cuda") for n in (7, 0))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            torch.cuda._sleep(50_000_000)  # about 30 ms
        cache.free(none, stream=side)
        assert cache.check_status() == 2
        torch.cuda._sleep(20_000_000)
        assert cache.check_status() == 0
        cache.free(first, stream=side)
        cache.free(none, stream=side)
        assert cache.check_status() == 2 and cache.check_status() == 0
