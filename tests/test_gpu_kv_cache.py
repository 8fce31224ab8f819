"""The paged cache's book-keeping against a plain model of it on the host, word for word; writes against torch; and a run of the operators
together, as a serving loop uses them."""
import random

import pytest

pytestmark = pytest.mark.gpu


class Model:
    """The rules in Python: the lowest-numbered free page first, in the order of the request."""

    def __init__(self, cache):
        self.data = cache.data.cpu()
        self.refs = cache.refs.tolist()
        self.table = cache.table.tolist()
        self.lengths = cache.lengths.tolist()
        self.ps, self.width, self.seqs = cache.page_size, cache.width, cache.seqs

    def _pages(self, n):
        return -(-n // self.ps)

    def reserve(self, seqs, counts, total):
        free = [p for p, r in enumerate(self.refs) if r <= 0]
        none = [-1] * total
        if len(set(seqs)) < len(seqs) or any(not 0 <= s < self.seqs for s in seqs) or any(c < 0 for c in counts) or sum(counts) > total:
            return none, 2
        if any(self.lengths[s] + c > self.width * self.ps for s, c in zip(seqs, counts)):
            return none, 2
        shared = [c > 0 and self.lengths[s] % self.ps > 0 and self.refs[self.table[s][self.lengths[s] // self.ps]] > 1 for s, c in zip(seqs, counts)]
        need = [self._pages(self.lengths[s] + c) - self._pages(self.lengths[s]) + sh for s, c, sh in zip(seqs, counts, shared)]
        if sum(need) > len(free):
            return none, 2
        slots, copies = [], []
        for s, c, sh, n in zip(seqs, counts, shared, need):
            old = self.lengths[s]
            mine, free = free[:n], free[n:]
            at = self._pages(old)
            if sh:
                copies.append((self.table[s][at - 1], mine[0], old % self.ps))
                self.refs[self.table[s][at - 1]] -= 1
                self.table[s][at - 1] = mine[0]
                self.refs[mine[0]] = 1
                mine = mine[1:]
            for p in mine:
                self.table[s][at], self.refs[p] = p, 1
                at += 1
            self.lengths[s] = old + c
            slots += [self.table[s][t // self.ps] * self.ps + t % self.ps for t in range(old, old + c)]
        for a, b, rows in copies:
            self.data[:, b, :, :, :rows] = self.data[:, a, :, :, :rows]
        return slots + [-1] * (total - len(slots)), 0

    def fork(self, src, dst):
        status, before = 0, list(self.lengths)
        for i, (a, b) in enumerate(zip(src, dst)):
            if not (0 <= a < self.seqs and 0 <= b < self.seqs) or b in dst[:i] or b in src or a in dst or before[b]:
                status = 2
                continue
            n = self._pages(before[a])
            self.table[b][:n] = self.table[a][:n]
            for p in self.table[a][:n]:
                self.refs[p] += 1
            self.lengths[b] = before[a]
        return status

    def free(self, seqs):
        status = 0
        for s in seqs:
            if not 0 <= s < self.seqs:
                status = 2
                continue
            for j in range(self._pages(self.lengths[s])):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lengths[s] = 0
        return status

    def compact(self):
        live = [p for p, r in enumerate(self.refs) if r > 0]
        n = len(live)
        remap = [p if self.refs[p] > 0 and p < n else -1 for p in range(len(self.refs))]
        for a, b in zip([p for p in live if p >= n], [p for p in range(n) if self.refs[p] <= 0]):
            remap[a] = b
            self.data[:, b] = self.data[:, a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[remap[p] if p >= 0 else p for p in row] for row in self.table]
        return remap

    def check(self, cache):
        import torch

        assert cache.refs.tolist() == self.refs and cache.lengths.tolist() == self.lengths and cache.table.tolist() == self.table
        assert torch.equal(cache.data.view(torch.uint8).cpu(), self.data.view(torch.uint8))


def _ints(x):
    import torch

    return torch.tensor(x, dtype=torch.int32, device="cuda")


def _cache(layers, pages, page, kv, dim, seqs, width, dtype="bfloat16"):
    import torch

    from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache

    cache = PagedKVCache.allocate(layers, pages, page, kv, dim, seqs, width, getattr(torch, dtype))
    cache.data.view(torch.uint8).copy_(torch.randint(0, 100, cache.data.view(torch.uint8).shape, dtype=torch.uint8, device="cuda"))
    return cache


# pages: fewer and more than one step of the scan (4096), odd; page sizes of one token, odd ones, 16; three types
@pytest.mark.parametrize("layers,pages,page,kv,dim,seqs,width,dtype", [(1, 40, 4, 1, 16, 9, 9, "bfloat16"), (3, 57, 1, 2, 64, 12, 17, "float16"), (2, 131, 7, 3, 16, 33, 6, "float8_e4m3fn"),
                                                                    (1, 9001, 16, 1, 16, 300, 40, "bfloat16"), (5, 64, 16, 2, 128, 8, 20, "bfloat16")])
def test_random_calls_match_the_model(layers, pages, page, kv, dim, seqs, width, dtype):
    cache = _cache(layers, pages, page, kv, dim, seqs, width, dtype)
    model, rng = Model(cache), random.Random(pages)
    for turn in range(60):
        what = rng.choice(["reserve", "reserve", "reserve", "fork", "free", "compact"])
        n = rng.randint(1, seqs)
        some = rng.sample(range(seqs), n)
        if what == "reserve":
            counts = [rng.choice([0, 1, 1, rng.randint(0, page * 3)]) for _ in some]
            total = sum(counts) + rng.choice([0, 0, 5])
            slots = cache.reserve(_ints(some), _ints(counts), total)
            want, status = model.reserve(some, counts, total)
            assert slots.tolist() == want and cache.check_status() == status, (turn, what)
        elif what == "fork":
            src = [rng.choice(some) for _ in range(n)]
            dst = [rng.randrange(-1, seqs + 1) if rng.random() < 0.1 else rng.randrange(seqs) for _ in range(n)]
            cache.fork(_ints(src), _ints(dst))
            assert cache.check_status() == model.fork(src, dst), (turn, what)
        elif what == "free":
            some = some[:max(1, n // 2)] + some[:1] + ([seqs, -4] if rng.random() < 0.2 else [])  # one of them twice
            cache.free(_ints(some))
            assert cache.check_status() == model.free(some), (turn, what)
        else:
            remap = cache.compact()
            assert remap.tolist() == model.compact(), (turn, what)
        model.check(cache)


def test_reserve_is_all_or_nothing():
    cache = _cache(1, 8, 4, 1, 16, 4, 5)
    model = Model(cache)
    calls = [([0, 1], [9, 4], 13), ([2], [17], 17), ([2], [21], 40), ([0, 0], [1, 1], 2), ([4], [1], 1), ([-1], [1], 1), ([3], [-1], 4), ([3], [5], 4), ([2, 3], [16, 4], 20),
             ([2 ** 31 - 1], [1], 1), ([3], [2 ** 31 - 1], 2 ** 10), ([2], [16], 16), ([3], [1], 1), ([3], [0], 0)]
    for seqs, counts, total in calls:
        slots = cache.reserve(_ints(seqs), _ints(counts), total)
        want, status = model.reserve(seqs, counts, total)
        assert slots.tolist() == want and cache.check_status() == status, (seqs, counts)
        model.check(cache)
    assert cache.reserve(_ints([]), _ints([]), 3).tolist() == [-1] * 3


def test_fork_chains_and_sharing_of_a_page_by_many():
    cache = _cache(2, 40, 4, 2, 16, 10, 6)
    model = Model(cache)
    for step in ([("reserve", [0], [6])], [("fork", [0] * 6, [1, 2, 3, 4, 5, 6])], [("reserve", [0, 1, 2, 3], [1, 1, 3, 0])], [("fork", [1, 7], [7, 8])], [("fork", [1], [7])],
                 [("fork", [7, 7], [8, 8])], [("free", [0, 1, 1, 2])], [("reserve", [3, 4, 5, 6, 7, 8], [1] * 6)], [("free", [3, 4, 5, 6, 7, 8, 9])]):
        for name, *args in step:
            if name == "reserve":
                assert cache.reserve(*(_ints(x) for x in args), sum(args[1])).tolist() == model.reserve(*args, sum(args[1]))[0]
                cache.check_status()
            else:
                getattr(cache, name)(*(_ints(x) for x in args))
                assert cache.check_status() == getattr(model, name)(*args)
            model.check(cache)
    assert cache.refs.sum().item() == 0


def test_calls_replay_from_a_graph():
    cache = _cache(2, 64, 4, 1, 16, 6, 8)
    model = Model(cache)
    rows, counts = _ints([0, 2, 5]), _ints([1, 1, 1])
    import torch

    graph = torch.cuda.CUDAGraph()
    cache.reserve(rows, counts, 3)
    model.reserve([0, 2, 5], [1, 1, 1], 3)
    with torch.cuda.graph(graph):
        slots = cache.reserve(rows, counts, 3)
    for _ in range(9):
        graph.replay()
        assert slots.tolist() == model.reserve([0, 2, 5], [1, 1, 1], 3)[0]
        model.check(cache)


@pytest.mark.parametrize("src,dtype", [("bfloat16", "bfloat16"), ("float16", "float16"), ("bfloat16", "float8_e4m3fn"), ("float16", "float8_e4m3fn")])
@pytest.mark.parametrize("tokens,kv,dim,page", [(1, 1, 16, 1), (37, 3, 48, 5), (300, 8, 128, 16), (2, 1, 64, 64)])
def test_write(src, dtype, tokens, kv, dim, page):
    import torch

    cache = _cache(2, -(-tokens // page) + 9, page, kv, dim, 1, 1, dtype)
    g = torch.Generator(device="cuda").manual_seed(tokens)
    qkv = (3 * torch.randn(tokens, 4 + 2 * kv, dim, generator=g, device="cuda")).to(getattr(torch, src))
    k, v = qkv[:, 4:4 + kv], qkv[:, 4 + kv:]
    if tokens > 5:
        k[1, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 6e4], dtype=qkv.dtype)
    slots = torch.randperm(cache.pages * page, generator=g, device="cuda")[:tokens].contiguous()
    if tokens > 5:
        slots[3], slots[4] = -1, -5
    scales = {}
    want = cache.data.clone()
    rows = [i for i in range(tokens) if int(slots[i]) >= 0]
    if dtype == "float8_e4m3fn":
        scales = {"k_scale": 0.01 + torch.rand(kv, generator=g, device="cuda"), "v_scale": 0.01 + torch.rand(kv, generator=g, device="cuda")}
        k8, v8 = ((x.float() * (1 / s)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for x, s in ((k, scales["k_scale"]), (v, scales["v_scale"])))
    else:
        k8, v8 = k, v
    bits = want.view(torch.uint8 if dtype == "float8_e4m3fn" else torch.int16)
    for i in rows:
        p, o = int(slots[i]) // page, int(slots[i]) % page
        bits[1, p, 0, :, o], bits[1, p, 1, :, o] = k8[i].contiguous().view(bits.dtype), v8[i].contiguous().view(bits.dtype)
    cache.write(1, k, v, slots, **scales)
    assert cache.check_status() == 0
    got = cache.data.view(bits.dtype)
    if dtype == "float8_e4m3fn":  # one NaN is as good as another
        same = (got == bits) | (cache.data.float().isnan() & want.float().isnan())
        assert bool(same.all())
    else:
        assert torch.equal(got, bits)
    slots[0] = cache.pages * page
    cache.write(0, k, v, slots, **scales)
    assert cache.check_status() == 2


@pytest.mark.parametrize("dtype", ["bfloat16", "float8_e4m3fn"])
def test_serving_loop(dtype):
    """Prompts, their candidates, a few tokens each, a candidate dropped, the cache compacted in between: every decoded row against attention over
    the keys and values that its sequence has been given."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A
    from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache

    layers, heads, kv, dim, page = 2, 8, 2, 64, 16
    cache = PagedKVCache.allocate(layers, 200, page, kv, dim, 8, 40, getattr(torch, dtype))
    g = torch.Generator(device="cuda").manual_seed(0)
    scales = {"k_scale": torch.full((kv,), 0.01, device="cuda"), "v_scale": torch.full((kv,), 0.02, device="cuda")} if dtype != "bfloat16" else {}
    history = {}

    def fresh(n):
        return torch.randn(layers, n, heads + 2 * kv, dim, generator=g, device="cuda").to(torch.bfloat16)

    def step(seqs, counts, prompt):
        total = sum(counts)
        x = fresh(total)
        slots = cache.reserve(_ints(seqs), _ints(counts), total)
        cu = torch.tensor([0] + counts, dtype=torch.int32, device="cuda").cumsum(0).to(torch.int32)
        for layer in range(layers):
            q, k, v = x[layer, :, :heads], x[layer, :, heads:heads + kv], x[layer, :, heads + kv:]
            cache.write(layer, k, v, slots, **scales)
            if prompt:
                out = A.prefill_attention(q, k, v, cu)
            else:
                out = cache.decode(layer, q, _ints(seqs), **scales)
            for i, s in enumerate(seqs):
                rows = slice(int(cu[i]), int(cu[i + 1]))
                past = history.get((s, layer))
                new = x[layer, rows, heads:]
                if dtype != "bfloat16" and not prompt:
                    pass
                history[s, layer] = new if past is None else torch.cat([past, new])
                kept = history[s, layer].double()
                kk, vv = kept[:, :kv], kept[:, kv:]
                if scales and not prompt:
                    kk, vv = (((y.float() * (1 / sc)[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).double() * sc.double()[:, None])
                              for y, sc in ((kk, scales["k_scale"]), (vv, scales["v_scale"])))
                n = kept.shape[0]
                seen = torch.arange(n, device="cuda") <= torch.arange(counts[i], device="cuda")[:, None] + n - counts[i]
                ref, _ = A._attend_reference(q[rows], kk, vv, seen, dim ** -0.5)
                assert float((out[rows].double() - ref).abs().max()) < 0.03, (s, layer, n)
        assert cache.check_status() == 0

    step([0, 1, 2], [37, 5, 160], True)
    cache.fork(_ints([0, 0, 2]), _ints([3, 4, 5]))
    for a, b in ((0, 3), (0, 4), (2, 5)):
        for layer in range(layers):
            history[b, layer] = history[a, layer]
    step([3, 0, 4, 5, 1], [1] * 5, False)
    cache.free(_ints([0, 2]))
    for s in (0, 2):
        for layer in range(layers):
            del history[s, layer]
    remap = cache.compact()
    assert int((remap >= 0).sum()) == int((cache.refs > 0).sum())
    for _ in range(18):
        step([5, 1, 3, 4], [1] * 4, False)
    step([0], [50], True)
    cache.compact()
    step([0, 4, 3], [1] * 3, False)
    assert cache.check_status() == 0


def test_cache_in_pooled_memory_whose_pages_are_moved_by_batch_copies(port):
    """Two caches in one rank's pooled HBM, as a prefill and a decode instance have them: a sequence's blocks go from one to the other by one batch
    call, and are decoded there."""
    import torch

    from memfabric_hybrid_b200 import bm
    from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache
    from memfabric_hybrid_b200.parallel.pool import open_pool
    from memfabric_hybrid_b200.utils.tensors import device_tensor_from_gva

    torch.cuda.set_device(0)
    pool = open_pool(0, 1, 0, 64 << 20, store_url=f"tcp://127.0.0.1:{port}")
    try:
        layers, pages, page, kv, dim = 3, 40, 16, 2, 64
        shape = (layers, pages, 2, kv, page, dim)
        nbytes = 2 * layers * pages * 2 * kv * page * dim
        caches = []
        for i in range(2):
            data = device_tensor_from_gva(pool.hbm() + i * (32 << 20), nbytes, torch.bfloat16).view(shape)
            data.zero_()
            caches.append(PagedKVCache(data, torch.full((3, 8), -1, dtype=torch.int32, device="cuda"), torch.zeros(3, dtype=torch.int32, device="cuda"),
                                       torch.zeros(pages, dtype=torch.int32, device="cuda")))
        there, here = caches
        g = torch.Generator(device="cuda").manual_seed(3)
        slots = there.reserve(_ints([2, 1]), _ints([19, 100]), 119)
        for layer in range(layers):
            there.write(layer, *(torch.randn(119, kv, dim, generator=g, device="cuda").to(torch.bfloat16) for _ in range(2)), slots)
        here.reserve(_ints([0, 1]), _ints([40, 100]), 140)
        q = torch.randn(1, 8, dim, generator=g, device="cuda").to(torch.bfloat16)
        want = [there.decode(layer, q, _ints([1])) for layer in range(layers)]
        torch.cuda.synchronize()
        moves = [(there.block(layer, a), here.block(layer, b)) for layer in range(layers) for a, b in zip(there.table[1, :7].tolist(), here.table[1, :7].tolist())]
        assert pool.handle.copy_data_batch([a for (a, _), _ in moves], [b for _, (b, _) in moves], [n for (_, n), _ in moves], len(moves), bm.BmCopyType.G2G, 0) == 0
        for layer in range(layers):
            assert torch.equal(here.decode(layer, q, _ints([1])), want[layer])
        assert there.check_status() == 0 and here.check_status() == 0
        del there, here, caches, data, want
    finally:
        torch.cuda.synchronize()
        pool.close()


def test_caches_of_other_kinds_do_not_take_what_one_has_taken():
    import torch

    k = torch.ones(5, 2, 64, dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(5, device="cuda")
    one, alike, fewer, longer, narrow = (_cache(1, 8, 4, *kind) for kind in
                                         ((2, 64, 3, 4), (2, 64, 9, 2), (1, 64, 3, 4), (2, 128, 3, 4), (2, 64, 3, 4, "float8_e4m3fn")))
    for cache in (one, alike):
        for _ in range(2):
            cache.write(0, k, k, slots)
        assert torch.equal(cache.k_pages(0).transpose(1, 2).reshape(-1, 2, 64)[:5], k)
    for cache in (fewer, longer, narrow):
        with pytest.raises(ValueError):
            cache.write(0, k, k, slots)
    assert alike.reserve(_ints([8]), _ints([3]), 3).tolist() == [0, 1, 2] and alike.check_status() == 0
    with pytest.raises(ValueError):
        one.reserve(_ints([0, 1, 2, 0]), _ints([1, 1, 1, 1]), 4)
    alike.reserve(_ints([0, 1, 2, 8]), _ints([1, 1, 1, 0]), 3)
    assert alike.lengths.tolist() == [1, 1, 1, 0, 0, 0, 0, 0, 3] and alike.check_status() == 0


FIRST_CALLS = """
import torch
from memfabric_hybrid_b200.ops.attention import prefill_attention, prefill_attention_reference
from memfabric_hybrid_b200.ops.kv_cache import PagedKVCache

ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
x = torch.randn(700, 12, 128, device="cuda", dtype=torch.bfloat16)
q, k, v = x[:, :8], x[:, 8:10], x[:, 10:]
cu, seqs, counts, third, one, rows = map(ints, ([0, 300, 700], [0, 1], [300, 400], [3], [1], [1, 1, 1]))
cache = PagedKVCache.allocate(2, 64, 16, 2, 128, 6, 40)
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    prompt = prefill_attention(q, k, v, cu)
    cache.write(0, k, v, cache.reserve(seqs, counts, 700))
    cache.fork(one, third)
    cache.write(0, k[:1], v[:1], cache.reserve(third, one, 1))
    step = cache.decode(0, q[:3], rows)
    cache.free(one)
    moved = cache.compact()
graph.replay()
torch.cuda.synchronize()
assert cache.check_status() == 0 and cache.lengths.tolist() == [300, 0, 0, 401, 0, 0]
assert int((cache.refs > 0).sum()) == 19 + 26 and bool((cache.refs[:45] == 1).all())
want = prefill_attention_reference(q, k, v, cu)[0]
assert float((prompt.double() - want).abs().max()) < 0.03
keys, values = (t[300:].double().repeat_interleave(4, 1) for t in (k, v))
weights = torch.softmax(torch.einsum("bhd,nhd->bhn", q[:3].double(), keys) * 128 ** -0.5, -1)
assert float((step.double() - torch.einsum("bhn,nhd->bhd", weights, values)).abs().max()) < 0.03
"""


def test_a_process_may_begin_with_a_capture():
    """Nothing that a first call sets up (attributes of kernels, plans) disturbs the capture of a graph."""
    import subprocess
    import sys
    from pathlib import Path

    r = subprocess.run([sys.executable, "-c", FIRST_CALLS], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stderr[-2000:]
