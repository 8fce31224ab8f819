"""What a row of a prompt may not see must not reach it, whatever stands there; and what it does see must."""
import pytest

pytestmark = pytest.mark.gpu


def _values(shape, dtype, seed):
    import torch

    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda").to(dtype)


def _largest(dtype):
    import torch

    return float(torch.finfo(dtype).max)


# sequences, then rows of the key buffer that belong to none
ROWS, KEYS, TAIL = [150, 160, 20, 300], [150, 290, 9, 300], 90


def _packed(dtype, dim, heads=8, kv=2):
    import torch

    cu = [torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32, device="cuda") for n in (ROWS, KEYS)]
    return (_values((sum(ROWS), heads, dim), dtype, 1), _values((sum(KEYS) + TAIL, kv, dim), dtype, 2), _values((sum(KEYS) + TAIL, kv, dim), dtype, 3), *cu)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", ["bfloat16", "float16"])
def test_large_values_that_no_row_sees(name, dim, causal):
    """The largest number of the type in the next sequence, in later tokens and behind the last sequence: the same bits as with zeros there."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    dtype = getattr(torch, name)
    q, k, v, cu_q, cu_k = _packed(dtype, dim)
    at = torch.arange(sum(ROWS), device="cuda")
    places = [(slice(sum(KEYS), None), at >= 0),                     # behind the last sequence
              (slice(150, 440), (at < 150) | (at >= 310))]           # all of the second one
    if causal:
        places += [(slice(100, 150), (at < 100) | (at >= 150)),      # the end of the first
                   (slice(441, 449), (at < 322) | (at >= 330))]      # nine keys of twenty rows: eleven rows see none of them, the next one the first
    for where, rows in places:
        got = []
        for x in (0.0, _largest(dtype), -_largest(dtype)):
            v2 = v.clone()
            v2[where] = x
            got.append(A.prefill_attention(q, k, v2, cu_q, cu_k, causal=causal, lse=True))
        assert bool(got[0][0][rows].isfinite().all())
        for out, lse in got[1:]:
            same = torch.equal(out[rows], got[0][0][rows]) and torch.equal(lse[rows], got[0][1][rows])
            assert same


@pytest.mark.parametrize("dim", [64, 128])
def test_seen_keys_whose_weight_is_next_to_nothing(dim):
    """One key takes all: the others' logits lie 200 and more below it (weights below 2^-288), and their values of 1e36 count no more than 1e-50."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    n = 400
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q = torch.ones(n, 2, dim, dtype=torch.bfloat16, device="cuda")
    k = torch.full((n, 1, dim), -16.0, dtype=torch.bfloat16, device="cuda")
    k[0] = 16.0  # logits of 16 * sqrt(dim) and its opposite
    v = torch.full((n, 1, dim), 1e36, dtype=torch.bfloat16, device="cuda")
    v[0] = _values((dim,), torch.bfloat16, 4)
    for causal in (True, False):
        out = A.prefill_attention(q, k, v, cu, causal=causal)
        same = torch.equal(out, v[:1].expand(n, 2, dim))
        assert same


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", ["bfloat16", "float16"])
def test_nan_and_infinities_that_no_row_sees(name, dim, causal):
    """In keys and values alike: the same bits as with zeros there."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    dtype = getattr(torch, name)
    q, k, v, cu_q, cu_k = _packed(dtype, dim)
    at = torch.arange(sum(ROWS), device="cuda")
    places = [(slice(sum(KEYS), None), at >= 0), (slice(150, 440), (at < 150) | (at >= 310))]
    if causal:
        places += [(slice(100, 150), (at < 100) | (at >= 150)), (slice(441, 449), (at < 322) | (at >= 330)), (slice(100, 101), (at < 100) | (at >= 150))]
    for where, rows in places:
        v2, k2 = v.clone(), k.clone()
        v2[where] = k2[where] = 0
        want, want_lse = A.prefill_attention(q, k2, v2, cu_q, cu_k, causal=causal, lse=True)
        for x in (float("nan"), float("inf"), -float("inf")):
            v2[where] = k2[where] = x
            out, lse = A.prefill_attention(q, k2, v2, cu_q, cu_k, causal=causal, lse=True)
            same = torch.equal(out[rows], want[rows]) and torch.equal(lse[rows], want_lse[rows])
            assert same
        v2[where] = 0  # a key alone, seen or not
        out = A.prefill_attention(q, k2, v2, cu_q, cu_k, causal=causal)
        same = torch.equal(out[rows], want[rows])
        assert same


@pytest.mark.parametrize("heads,kv", [(8, 2), (1, 1), (7, 1), (256, 1)])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("name", ["bfloat16", "float16"])
def test_single_values_that_are_not_finite(name, dim, heads, kv):
    """One of each kind here and there: exactly the rows and columns that see them become NaN or infinite, as the definition has it, and the others keep
    their bits."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    dtype = getattr(torch, name)
    rows, keys = [300, 1, 140, 260], [300, 130, 511, 260]
    cu = [torch.tensor([0, *torch.tensor(n).cumsum(0).tolist()], dtype=torch.int32, device="cuda") for n in (rows, keys)]
    q, k, v = _values((sum(rows), heads, dim), dtype, 1), _values((sum(keys), kv, dim), dtype, 2), _values((sum(keys), kv, dim), dtype, 3)
    g = torch.Generator().manual_seed(dim + heads)
    for causal in (True, False):
        want, want_lse = A.prefill_attention(q, k, v, *cu, causal=causal, lse=True)
        for _ in range(3):
            v2 = v.clone()
            for x in (float("nan"), float("inf"), -float("inf")) * 4:
                v2[int(torch.randint(0, sum(keys), (1,), generator=g)), int(torch.randint(0, kv, (1,), generator=g)), int(torch.randint(0, dim, (1,), generator=g))] = x
            v2[40, 0, 5], v2[250, 0, 5], v2[200, 0, 33] = float("inf"), -float("inf"), float("nan")
            out, lse = A.prefill_attention(q, k, v2, *cu, causal=causal, lse=True)
            ref, _ = A.prefill_attention_reference(q, k, v2, *cu, causal)
            same = [torch.equal(out.isnan(), ref.isnan()), torch.equal(out == float("inf"), ref == float("inf")), torch.equal(out == -float("inf"), ref == -float("inf")),
                    torch.equal(out[ref.isfinite()], want[ref.isfinite()]), torch.equal(lse, want_lse)]
            assert all(same), same


@pytest.mark.parametrize("count", [64, 65, 150])
def test_values_that_are_not_finite_in_many_sequences(count):
    """More and fewer sequences than are ranked, several units of work to a CTA, of which many are done once more."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    g = torch.Generator().manual_seed(count)
    rows = torch.randint(0, 400, (count,), generator=g)
    keys = rows + torch.randint(0, 200, (count,), generator=g)
    cu = [torch.tensor([0, *n.cumsum(0).tolist()], dtype=torch.int32, device="cuda") for n in (rows, keys)]
    q, k, v = (_values((int(n.sum()), heads, 64), torch.bfloat16, heads + 5) for n, heads in ((rows, 4), (keys, 2), (keys, 2)))
    want, want_lse = A.prefill_attention(q, k, v, *cu, lse=True)
    bad = torch.randint(0, v.numel(), (count // 2,), generator=g).cuda()
    for x in (float("nan"), float("inf")):
        v.view(-1)[bad] = x
        out, lse = A.prefill_attention(q, k, v, *cu, lse=True)
        ref, _ = A.prefill_attention_reference(q, k, v, *cu)
        same = [torch.equal(out.isnan(), ref.isnan()), torch.equal(out.isinf(), ref.isinf()), torch.equal(out[ref.isfinite()], want[ref.isfinite()]),
                torch.equal(lse, want_lse)]
        assert all(same), same


@pytest.mark.parametrize("where", ["first value", "first key", "a query", "all values", "behind the end"])
def test_what_is_not_finite_costs_a_few_times_the_call(where):
    """2049 tokens with something that is not finite. Computed again row by row, key by key, they take some hundred times as long."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    n = 2049
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q, k, v = (_values((n + 127, heads, 128), torch.bfloat16, heads) for heads in (8, 2, 2))
    bad = [t.clone() for t in (q, k, v)]
    if where == "behind the end":
        bad[1][n:], bad[2][n:] = float("nan"), float("nan")
    elif where == "all values":
        bad[2][:] = float("nan")
    else:
        bad[{"a query": 0, "first key": 1, "first value": 2}[where]][0, 0] = float("nan")

    def took(*x):
        best = []
        for _ in range(5):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            for _ in range(4):
                A.prefill_attention(*x, cu, causal=where != "behind the end")
            b.record()
            b.synchronize()
            best.append(a.elapsed_time(b))
        return min(best)

    took(q, k, v)
    clean, odd = took(q, k, v), took(*bad)
    print(f"{where}: {clean * 250:.0f} us, {odd * 250:.0f} us")
    assert odd < 20 * clean, (clean, odd)


def test_replays_and_streams_with_values_that_are_not_finite():
    """A captured call whose values become NaN and finite again between replays, beside calls on other streams."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    cu = torch.tensor([0, 700, 701, 1900, 2000], dtype=torch.int32, device="cuda")
    q, k, v = (_values((2100, heads, 128), torch.bfloat16, heads) for heads in (8, 2, 2))
    odd = v.clone()
    odd[650], odd[1300, 1, 3:40], odd[1999], odd[2000:] = float("nan"), float("inf"), float("-inf"), float("nan")
    want = {id(x): A.prefill_attention(q, k, x, cu)[:2000].clone() for x in (v, odd)}
    assert bool(want[id(v)].isfinite().all()) and not bool(want[id(odd)].isfinite().all())
    taken = v.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.prefill_attention(q, k, taken, cu)
    streams, got = [torch.cuda.Stream() for _ in range(3)], []
    torch.cuda.synchronize()
    for turn in range(6):
        x = odd if turn % 2 else v
        taken.copy_(x)
        graph.replay()
        for i, s in enumerate(streams):
            y = odd if (turn + i) % 2 else v
            got.append((A.prefill_attention(q, k, y, cu, stream=s), y))
        torch.cuda.synchronize()
        same = torch.equal(out[:2000].nan_to_num(5.0), want[id(x)].nan_to_num(5.0))
        assert same
    for z, y in got:
        same = torch.equal(z[:2000].nan_to_num(5.0), want[id(y)].nan_to_num(5.0))
        assert same
