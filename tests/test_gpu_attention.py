"""Attention operators against a plain implementation in 64 bits: lengths at the edges of tiles and pages, head layouts, strides, masks that
leave a row empty, infinities and NaN where nothing may look."""
import pytest

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _tol(ref, mass, dtype, dim, n, logit, p_eps):
    """What the roundings of a pass may add up to. The result is rounded once (eps / 2 of it) and so is each weight (p_eps / 2 of its part of
    sum p |v| / sum p, `mass`); logits of size `logit` err by their dim products' and sums' fp32 roundings, which move a weight and the sum by as
    much; n weights and products are added up in fp32, and 2^x is off by a few units of 2^-22."""
    import torch

    h, u = torch.finfo(dtype).eps / 2, 2.0 ** -24
    return (h * ref.abs() + (p_eps / 2 + (2 * (dim + 2) * logit + 2 * n + 64) * u) * mass) * (1 + 4 * h) + 1e-30


def _check(out, ref, mass, dtype, dim, n, logit, p_eps=None):
    import torch

    err = (out.double() - ref).abs()
    tol = _tol(ref, mass, dtype, dim, n, logit, torch.finfo(dtype).eps if p_eps is None else p_eps)
    assert out.isfinite().all()
    assert bool((err <= tol).all()), f"{float((err / tol).max()):.2f} of what is allowed"


def _pool(lengths, page, kv, dim, dtype, width=None, spare=3, seed=0, scales=None):
    """Pages in random order, table and lengths; what no sequence reaches is NaN (e4m3: its NaN)."""
    import torch

    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    pages = sum(need) + spare
    data = torch.randn(pages, 2, kv, page, dim, generator=g, device="cuda")
    if dtype == torch.float8_e4m3fn:
        data = (data * 100).clamp(-448, 448)
    order = torch.randperm(pages, generator=g, device="cuda")
    width = max(need + [1]) if width is None else width
    table = torch.full((len(lengths), width), -7, dtype=torch.int32, device="cuda")  # entries behind the length are not looked at
    at = 0
    for i, n in enumerate(lengths):
        table[i, :need[i]] = order[at:at + need[i]].to(torch.int32)
        at += need[i]
        if n % page:
            data[order[at - 1], :, :, n % page:] = NAN
    data[order[at:]] = NAN
    data = data.to(dtype)
    return data[:, 0], data[:, 1], table, torch.tensor(lengths, dtype=torch.int32, device="cuda")


def _q(shape, dtype, seed=1):
    import torch

    return (1.5 * torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")).to(dtype)


def _decode_case(lengths, page, heads, kv, dim, dtype, cache=None, rows=None, **kw):
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    cache = cache or dtype
    k, v, table, lens = _pool(lengths, page, kv, dim, cache, **kw)
    scales = {}
    if cache == torch.float8_e4m3fn:
        scales = {"k_scale": (1 + torch.rand(kv, device="cuda")) / 100, "v_scale": (1 + torch.rand(kv, device="cuda")) / 100}
    B = len(rows) if rows is not None else len(lengths)
    rows = torch.tensor(rows, dtype=torch.int32, device="cuda") if rows is not None else None
    q = _q((B, heads, dim), dtype)
    out, lse = A.decode_attention(q, k, v, table, lens, rows=rows, lse=True, **scales)
    ref, ref_lse = A.decode_attention_reference(q, k, v, table, lens, rows, **scales)
    mass, _ = A.decode_attention_reference(q, k, v.abs() if not scales else v.float().abs(), table, lens, rows, **scales)
    # 8-bit caches are widened to fp16, and so are the weights
    _check(out, ref, mass, dtype, dim, max(lengths), 40, 2.0 ** -10 if scales else None)
    empty = ref_lse == -INF
    assert torch.equal(lse == -INF, empty)
    assert float((lse.double() - ref_lse)[~empty].abs().max() if (~empty).any() else 0) < (2 * (dim + 2) * 40 + 2 * max(lengths) + 64) * 2.0 ** -24
    again, _ = A.decode_attention(q, k, v, table, lens, rows=rows, lse=True, **scales)
    assert torch.equal(out, again)


EDGES = [0, 1, 2, 15, 16, 17, 63, 64, 65, 127, 128, 255, 256, 257, 700, 0]


@pytest.mark.parametrize("name,cache", [("bfloat16", None), ("float16", None), ("bfloat16", "float8_e4m3fn"), ("float16", "float8_e4m3fn")])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_lengths_at_edges(name, cache, dim):
    import torch

    _decode_case(EDGES, 16, 8, 2, dim, getattr(torch, name), getattr(torch, cache) if cache else None)


# one row; rows of at most four tiles; more rows than CTAs; one row over all CTAs; two of very different length
@pytest.mark.parametrize("lengths", [[1], [137], [256] * 3, list(range(1, 300)), [20011], [9000, 3], [0, 0], [0, 0, 5000, 0]])
def test_decode_splits(lengths):
    import torch

    _decode_case(lengths, 16, 8, 2, 128, torch.bfloat16)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (7, 1), (16, 1), (17, 1), (40, 1), (64, 2), (32, 8)])
@pytest.mark.parametrize("cache", [None, "float8_e4m3fn"])
def test_decode_head_layouts(heads, kv, cache):
    import torch

    _decode_case([5, 300, 1111], 32, heads, kv, 128, torch.bfloat16, getattr(torch, cache) if cache else None)


@pytest.mark.parametrize("page", [1, 3, 16, 48, 100, 512])
@pytest.mark.parametrize("dim", [64, 128])
def test_decode_page_sizes(page, dim):
    import torch

    _decode_case([0, 1, page, page + 1, 3 * page - 1, 400], page, 4, 2, dim, torch.float16)


@pytest.mark.parametrize("lengths", [[256, 255, 1], [257, 256, 3], [511, 512, 0, 12], [513, 512], [512] * 40, [1024, 700, 1025], [640] * 9])
@pytest.mark.parametrize("page", [16, 64, 9])
@pytest.mark.parametrize("dim,cache", [(64, None), (64, "float8_e4m3fn"), (128, "float8_e4m3fn")])
def test_decode_at_the_lengths_from_which_rows_are_cut(lengths, page, dim, cache):
    import torch

    _decode_case(lengths, page, 8, 2, dim, torch.bfloat16, cache=getattr(torch, cache) if cache else None)


def test_decode_values_that_lie_before_the_keys():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    for dtype in (torch.float16, torch.float8_e4m3fn):
        k, v, table, lens = _pool([300, 77, 1200], 16, 2, 64, dtype)
        scales = {"k_scale": torch.full((2,), 0.01, device="cuda"), "v_scale": torch.full((2,), 0.02, device="cuda")} if dtype == torch.float8_e4m3fn else {}
        q = _q((3, 8, 64), torch.float16)
        want = A.decode_attention(q, k.view(torch.uint8).contiguous().view(dtype), v.view(torch.uint8).contiguous().view(dtype), table, lens, **scales)
        turned = torch.stack((v.view(torch.uint8), k.view(torch.uint8)), 1).view(dtype)
        assert turned[:, 0].data_ptr() < turned[:, 1].data_ptr()
        assert torch.equal(A.decode_attention(q, turned[:, 1], turned[:, 0], table, lens, **scales), want)


def test_decode_rows_in_any_order_and_twice():
    import torch

    _decode_case([100, 0, 1300, 64, 7], 16, 8, 2, 128, torch.bfloat16, rows=[2, 2, 1, 4, 0, 2, 3])


def test_decode_token_major_pages_strided_queries_and_out():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    k, v, table, lens = _pool([300, 1, 77], 16, 4, 128, torch.bfloat16, spare=0)
    ref, _ = A.decode_attention_reference(_q((3, 8, 128), torch.bfloat16), k, v, table, lens)
    kt, vt = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (k, v))
    wide = torch.zeros(3, 12, 160, dtype=torch.bfloat16, device="cuda")
    q = wide[:, 2:10, 16:144]
    q.copy_(_q((3, 8, 128), torch.bfloat16))
    room = torch.full((3, 10, 136), 5.0, dtype=torch.bfloat16, device="cuda")
    got = A.decode_attention(q, kt, vt, table, lens, out=room[:, 1:9, :128])
    assert got.data_ptr() == room[:, 1:9, :128].data_ptr()
    assert torch.equal(got, A.decode_attention(q.contiguous(), k, v, table, lens))
    assert float((got.double() - ref).abs().max()) < 0.05
    assert bool((room[:, 0] == 5).all() and (room[:, 9] == 5).all() and (room[:, :, 128:] == 5).all())


def test_decode_large_and_small_queries_of_an_8_bit_cache():
    """Queries that fp16 could not hold: each head is scaled by a power of two of its own."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    k, v, table, lens = _pool([200], 16, 2, 64, torch.float8_e4m3fn, spare=0)
    one = torch.ones(2, device="cuda")
    q = _q((1, 4, 64), torch.bfloat16) * torch.tensor([1e6, 1e-30, 0.0, 1.0], device="cuda", dtype=torch.bfloat16)[:, None]
    for scale in (1e-8, 1e-3):
        out = A.decode_attention(q, k, v, table, lens, scale=scale, k_scale=one, v_scale=one)
        ref, _ = A.decode_attention_reference(q, k, v, table, lens, None, scale, one, one)
        mass, _ = A.decode_attention_reference(q, k, v.float().abs(), table, lens, None, scale, one, one)
        logit = float((q.double().abs().amax() * 64 * 448 * scale))
        _check(out, ref, mass, torch.bfloat16, 64, 200, logit, 2.0 ** -10)


def test_decode_keys_that_are_infinite_or_nan():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    k, v, table, lens = _pool([50, 50, 50], 16, 1, 64, torch.bfloat16, spare=0)
    v[int(table[0, 1]), 0, 3, 5] = NAN  # seen: this column of the first sequence
    v[int(table[1, 1]), 0, 3, 5] = INF
    k[int(table[2, 0]), 0, 2, 1] = NAN  # all of the third
    out = A.decode_attention(_q((3, 2, 64), torch.bfloat16), k, v, table, lens)
    ref, _ = A.decode_attention_reference(_q((3, 2, 64), torch.bfloat16), k, v, table, lens)
    assert torch.equal(out.isnan(), ref.isnan()) and bool(out[0, :, 5].isnan().all()) and bool((out[1, :, 5] == INF).all())


def test_decode_reports_pages_and_rows_that_do_not_exist():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    k, v, table, lens = _pool([40, 300], 16, 2, 64, torch.bfloat16, spare=0)
    q = _q((2, 4, 64), torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = A.decode_attention(q, k, v, table, lens, status=status)
    assert int(status) == 0
    for bad in (-1, k.shape[0], 2 ** 31 - 1, -2 ** 31):
        status.zero_()
        broken = table.clone()
        broken[1, 3] = bad
        out = A.decode_attention(q, k, v, broken, lens, status=status)
        assert int(status) == 2 and torch.equal(out[0], good[0])
        zeroed_k, zeroed_v = k.clone(), v.clone()
        zeroed_k[int(table[1, 3])] = 0
        zeroed_v[int(table[1, 3])] = 0
        assert torch.equal(out, A.decode_attention(q, zeroed_k, zeroed_v, table, lens))
    status.zero_()
    out = A.decode_attention(q, k, v, table, lens, rows=torch.tensor([2, 1], dtype=torch.int32, device="cuda"), status=status)
    # what else is in a batch decides where rows are cut, so bits are compared with a batch of the same lengths
    same = A.decode_attention(q, k, v, table, torch.tensor([0, 300], dtype=torch.int32, device="cuda"))
    assert int(status) == 2 and torch.equal(out, same) and bool((out[0] == 0).all())
    # lengths beyond the table's width are cut off, negative ones are none
    long = torch.tensor([-5, 10 ** 9], dtype=torch.int32, device="cuda")
    full = torch.tensor([0, table.shape[1] * 16], dtype=torch.int32, device="cuda")
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    assert torch.equal(A.decode_attention(q, k, v, table, long), A.decode_attention(q, k, v, table, full))


def test_decode_cache_offsets_past_32_bits():
    """Pages more than 2^32 bytes apart."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    data = torch.empty(40000, 2, 8, 64, 128, dtype=torch.bfloat16, device="cuda")  # 10.5 GB
    table = torch.tensor([[39999, 3, 20001, 35000]], dtype=torch.int32, device="cuda")
    for p in table[0].tolist():
        data[p].normal_()
    lens = torch.tensor([250], dtype=torch.int32, device="cuda")
    q = _q((1, 16, 128), torch.bfloat16)
    out = A.decode_attention(q, data[:, 0], data[:, 1], table, lens)
    small = data[table[0].long()]
    order = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    assert torch.equal(out, A.decode_attention(q, small[:, 0], small[:, 1], order, lens))


def test_decode_graph_replays_with_other_lengths_and_beside_another_graph():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    k, v, table, lens = _pool([3000, 900], 16, 2, 128, torch.bfloat16, spare=0)
    k, v = torch.nan_to_num(k), torch.nan_to_num(v)
    q = [_q((2, 8, 128), torch.bfloat16, seed) for seed in (5, 6)]
    length = [lens.clone(), lens.clone()]
    A.decode_attention(q[0], k, v, table, lens)
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(A.decode_attention(q[i], k, v, table, length[i]))
        graphs.append(graph)
    for new in ([3000, 900], [1, 0], [64, 899], [2999, 257]):
        length[0].copy_(torch.tensor(new, dtype=torch.int32))
        length[1].copy_(torch.tensor(new[::-1], dtype=torch.int32).clamp(max=900))
        torch.cuda.synchronize()
        for _ in range(3):
            for i in range(2):
                with torch.cuda.stream(streams[i]):
                    graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], A.decode_attention(q[i], k, v, table, length[i]))


def test_calls_on_a_stream_of_the_callers():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    k, v, table, lens = _pool([3000, 900], 16, 2, 128, torch.bfloat16, spare=0)
    q = _q((2, 8, 128), torch.bfloat16)
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    x = _q((200, 8, 128), torch.bfloat16)
    want, want_p = A.decode_attention(q, k, v, table, lens), A.prefill_attention(x, x[:, :2], x[:, 2:4], cu)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    for _ in range(20):
        got, got_p = A.decode_attention(q, k, v, table, lens, stream=side), A.prefill_attention(x, x[:, :2], x[:, 2:4], cu, stream=side)
        junk = [torch.full((1 << 20,), 7.0, device="cuda") for _ in range(4)]  # takes what the current stream's allocator would give away
        del junk
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(got_p, want_p)


# ------------------------------------------------------------------------------------------------ prefill


def _prefill_case(rows, keys, heads, kv, dim, dtype, causal, head=0, tail=0, spoil=True):
    """Sequences of rows[i] queries on keys[i] keys; `head` rows before and `tail` rows behind belong to no sequence."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    cu_q, cu_k = ([s] for s in (head, 0))
    for n, m in zip(rows, keys):
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + m)
    T, S = cu_q[-1] + tail, cu_k[-1]
    q = _q((T, heads, dim), dtype, 3)
    kvs = _q((max(S, 1), 2 * kv, dim), dtype, 4) / 1.5
    k, v = kvs[:S, :kv], kvs[:S, kv:]
    cq, ck = (torch.tensor(c, dtype=torch.int32, device="cuda") for c in (cu_q, cu_k))
    out = torch.full((T, heads, dim), 7.0, dtype=dtype, device="cuda")
    lse = torch.full((T, heads), 7.0, device="cuda")
    A.prefill_attention(q, k, v, cq, ck, causal=causal, out=out, lse=lse)
    ref, ref_lse = A.prefill_attention_reference(q, k, v, cq, ck, causal)
    mass, _ = A.prefill_attention_reference(q, k, v.abs(), cq, ck, causal)
    inside = slice(head, cu_q[-1])
    _check(out[inside], ref[inside], mass[inside], dtype, dim, max(list(keys) + [1]), 40)
    empty = ref_lse[inside] == -INF
    assert torch.equal(lse[inside] == -INF, empty)
    d = (lse.double() - ref_lse)[inside][~empty].abs()
    assert d.numel() == 0 or float(d.max()) < (2 * (dim + 2) * 40 + 2 * max(keys) + 64) * 2.0 ** -24
    assert bool((out[:head] == 7).all() and (out[cu_q[-1]:] == 7).all() and (lse[:head] == 7).all() and (lse[cu_q[-1]:] == 7).all())
    again = A.prefill_attention(q, k, v, cq, ck, causal=causal)
    assert torch.equal(again[inside], out[inside])


PROMPTS = [1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 1]


@pytest.mark.parametrize("name", ["bfloat16", "float16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_lengths_at_edges(name, dim, causal):
    import torch

    _prefill_case(PROMPTS, PROMPTS, 8, 2, dim, getattr(torch, name), causal)


@pytest.mark.parametrize("heads,kv", [(1, 1), (3, 3), (5, 1), (6, 2), (7, 1), (8, 8), (16, 1), (24, 2), (128, 1), (256, 1)])
def test_prefill_head_layouts(heads, kv):
    import torch

    _prefill_case([150, 3, 40], [150, 3, 40], heads, kv, 64, torch.bfloat16, True)


# chunks behind a cached part, fewer keys than rows (the first rows see none), no keys, no rows, empty sequences in between
@pytest.mark.parametrize("rows,keys", [([40, 1, 130], [300, 257, 130]), ([200, 70], [129, 5]), ([5, 0, 7, 0], [0, 9, 7, 0]), ([0], [0]), ([0, 0], [5, 0]), ([1], [1]),
                                       ([1] * 150, [1 + 7 * i for i in range(150)])])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_chunks_and_empty_rows(rows, keys, causal):
    import torch

    _prefill_case(rows, keys, 4, 2, 128, torch.bfloat16, causal)


def test_prefill_rows_of_no_sequence_stay():
    import torch

    _prefill_case([70, 130], [70, 130], 4, 2, 64, torch.float16, True, head=5, tail=90)


@pytest.mark.parametrize("rows,keys,heads,kv,dim", [([2048], [2048], 8, 2, 128), ([1500, 900], [1500, 2900], 4, 4, 64)])
def test_prefill_long(rows, keys, heads, kv, dim):
    import torch

    _prefill_case(rows, keys, heads, kv, dim, torch.bfloat16, True)


def test_prefill_sharp_and_growing_logits():
    """Maxima that grow from key to key, and one key that takes all: the running maximum moves in every tile."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    n = 700
    cu = torch.tensor([0, n], dtype=torch.int32, device="cuda")
    q = torch.ones(n, 2, 64, dtype=torch.bfloat16, device="cuda")
    ramp = torch.linspace(-30, 30, n, device="cuda")[:, None, None].expand(n, 1, 64)
    v = _q((n, 1, 64), torch.bfloat16)
    for k in (ramp, -ramp, torch.where(torch.arange(n, device="cuda")[:, None, None] % 97 == 5, 40.0, -40.0).expand(n, 1, 64)):
        k = k.to(torch.bfloat16).contiguous()
        for causal in (True, False):
            out = A.prefill_attention(q, k, v, cu, causal=causal)
            ref, _ = A.prefill_attention_reference(q, k, v, cu, None, causal)
            mass, _ = A.prefill_attention_reference(q, k, v.abs(), cu, None, causal)
            _check(out, ref, mass, torch.bfloat16, 64, n, 64 * 40 / 8)


def test_prefill_infinities_and_nan_in_masked_places():
    """What a row may not see must not reach it: keys and values of later tokens and of other sequences."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    cu = torch.tensor([0, 150, 310, 330], dtype=torch.int32, device="cuda")
    q, k, v = _q((330, 8, 128), torch.bfloat16, 1), _q((330, 2, 128), torch.bfloat16, 2), _q((330, 2, 128), torch.bfloat16, 3)
    clean, _ = A.prefill_attention_reference(q, k, v, cu)
    k, v = k.clone(), v.clone()
    k[100], v[100, :, ::3], v[120, 1, 7], k[310:], v[310:] = NAN, NAN, INF, INF, NAN
    out = A.prefill_attention(q, k, v, cu)
    keep = torch.ones(330, dtype=torch.bool, device="cuda")
    keep[100:150] = False
    keep[310:] = False
    assert float((out.double() - clean)[keep].abs().max()) < 0.05 and bool(out[keep].isfinite().all())
    assert bool(out[100:150].isnan().any(-1).all()) and bool(out[310:].isnan().all())


def test_prefill_strides_scale_and_graph():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    qkv = _q((330, 12, 128), torch.bfloat16)
    cu = torch.tensor([0, 150, 310, 330], dtype=torch.int32, device="cuda")
    q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
    want = A.prefill_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu, scale=0.3)
    ref, _ = A.prefill_attention_reference(q, k, v, cu, scale=0.3)
    assert float((want.double() - ref).abs().max()) < 0.06
    room = torch.full((340, 16, 128), 3.0, dtype=torch.bfloat16, device="cuda")
    A.prefill_attention(q, k, v, cu, scale=0.3, out=room[5:335, 4:12])
    assert torch.equal(room[5:335, 4:12], want)
    room[5:335, 4:12] = 3
    assert bool((room == 3).all())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = A.prefill_attention(q, k, v, cu, scale=0.3)
    for new in ([0, 150, 310, 330], [0, 1, 2, 330], [0, 330, 330, 330]):
        cu.copy_(torch.tensor(new, dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, A.prefill_attention(q, k, v, cu, scale=0.3))


@pytest.mark.parametrize("count,most", [(64, 300), (65, 300), (200, 40), (7, 1500)])
@pytest.mark.parametrize("causal", [True, False])
def test_prefill_many_sequences_of_random_lengths(count, most, causal):
    """Every row tile of every sequence is done once, however the work is dealt out: few sequences are ranked by what they take, many are not."""
    import random

    import torch

    r = random.Random(count)
    rows = [r.choice([0, 1, r.randint(1, most)]) for _ in range(count)]
    keys = [r.choice([n, n, 0, n + r.randint(0, most), max(0, n - 40)]) for n in rows]
    _prefill_case(rows, keys, 6, 2, 64, torch.bfloat16, causal)


@pytest.mark.parametrize("heads,kv", [(12, 1), (40, 4), (100, 1), (14, 2), (11, 1)])
def test_prefill_heads_packed_into_tiles_that_they_do_not_fill(heads, kv):
    import torch

    _prefill_case([1, 130, 37, 300], [1, 130, 200, 300], heads, kv, 128, torch.float16, True)


def test_prefill_head_major_tensors():
    """Heads before tokens in memory: strides in the other order."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    cu = torch.tensor([0, 150, 310], dtype=torch.int32, device="cuda")
    q, k, v = (_q((n, 310, 64), torch.bfloat16, s).transpose(0, 1) for n, s in ((6, 1), (2, 2), (2, 3)))
    want = A.prefill_attention(q.contiguous(), k.contiguous(), v.contiguous(), cu)
    assert torch.equal(A.prefill_attention(q, k, v, cu), want)
    out = torch.empty(6, 310, 64, dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    assert torch.equal(A.prefill_attention(q, k, v, cu, out=out), want)


def test_prefill_of_nothing():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    cu = torch.zeros(1, dtype=torch.int32, device="cuda")
    x = _q((5, 4, 64), torch.bfloat16)
    out = torch.full_like(x, 2.0)
    assert torch.equal(A.prefill_attention(x, x, x, cu, out=out), torch.full_like(x, 2.0))
    none = x[:0]
    assert A.prefill_attention(none, x, x, torch.zeros(3, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)
    out, lse = A.prefill_attention(x, none, none, torch.tensor([0, 5], dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda"), lse=True)
    assert bool((out == 0).all()) and bool((lse == -INF).all())
    d = torch.zeros(1, 2, 4, 16, 64, dtype=torch.bfloat16, device="cuda")
    assert A.decode_attention(x[:0], d[:, 0], d[:, 1], torch.zeros(0, 3, dtype=torch.int32, device="cuda"), torch.zeros(0, dtype=torch.int32, device="cuda")).shape == (0, 4, 64)
    one = A.decode_attention(x, d[:, 0], d[:, 1], torch.zeros(5, 0, dtype=torch.int32, device="cuda"), torch.full((5,), 9, dtype=torch.int32, device="cuda"))
    assert bool((one == 0).all())


def test_offsets_that_leave_the_tensors_are_cut_off():
    """cu_q and cu_k that say more than there are tokens, or begin below zero: nothing outside is read or written."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    q, k, v = _q((100, 4, 64), torch.bfloat16, 1), _q((90, 2, 64), torch.bfloat16, 2), _q((90, 2, 64), torch.bfloat16, 3)
    room = torch.full((140, 4, 64), 5.0, dtype=torch.bfloat16, device="cuda")
    cu = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    A.prefill_attention(q, k, v, cu(0, 60, 1000), cu(0, 60, 2 ** 31 - 1), out=room[20:120])
    want = A.prefill_attention(q, k, v, cu(0, 60, 100), cu(0, 60, 90))
    assert torch.equal(room[20:120], want)
    for bad in (cu(-8, 60, 100), cu(2 ** 31 - 1, -5, 7), cu(100, 60, 0)):
        A.prefill_attention(q, k, v, bad, cu(0, 60, 90), out=room[20:120])
        A.prefill_attention(q, k, v, cu(0, 60, 100), bad, out=room[20:120])
    torch.cuda.synchronize()
    assert bool((room[:20] == 5).all() and (room[120:] == 5).all())


@pytest.mark.parametrize("batch", [3, 64, 65, 700])
def test_offsets_of_any_content_stay_inside(batch):
    """Offsets in no order, out of range and at the ends of their type: nothing outside is written. (What lies inside is not defined then.)"""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    g = torch.Generator().manual_seed(batch)
    for heads, kv_heads in ((4, 2), (6, 2), (7, 7)):
        q, k, v = _q((300, heads, 64), torch.bfloat16, 1), _q((290, kv_heads, 64), torch.bfloat16, 2), _q((290, kv_heads, 64), torch.bfloat16, 3)
        room, lse = torch.full((340, heads, 64), 5.0, dtype=torch.bfloat16, device="cuda"), torch.full((340, heads), 5.0, device="cuda")
        for _ in range(4):
            cu = []
            for _ in range(2):
                x = torch.randint(-50, 400, (batch + 1,), generator=g)
                odd = torch.randint(0, 6, (batch + 1,), generator=g)
                x = torch.where(odd == 0, -2 ** 31, torch.where(odd == 1, 2 ** 31 - 1, x))
                cu.append(x.to(torch.int32).cuda())
            A.prefill_attention(q, k, v, *cu, out=room[20:320], lse=lse[20:320])
            torch.cuda.synchronize()
        assert bool((room[:20] == 5).all() and (room[320:] == 5).all() and (lse[:20] == 5).all() and (lse[320:] == 5).all())


def test_prefill_offsets_past_32_bits():
    """Queries, keys, values and results of more than 2^32 bytes each: the last prompts of many against the same ones alone."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    count, n = 4200, 128
    x = torch.empty(count * n, 32, 128, dtype=torch.bfloat16, device="cuda")  # 4.4 GB
    last = slice((count - 3) * n, count * n)
    x.zero_()
    x[last].normal_(generator=torch.Generator(device="cuda").manual_seed(0))
    cu = torch.arange(count + 1, device="cuda", dtype=torch.int32) * n
    out = A.prefill_attention(x, x, x, cu)
    assert torch.equal(out[last], A.prefill_attention(x[last], x[last], x[last], cu[:4].contiguous()))
    assert bool((out[:n] == 0).all())


def test_decode_thousands_of_sequences():
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    g = torch.Generator(device="cuda").manual_seed(2)
    lens = torch.randint(0, 600, (5000,), generator=g, device="cuda", dtype=torch.int32)
    data = torch.randn(997, 2, 2, 16, 64, generator=g, device="cuda").to(torch.bfloat16)
    table = torch.randint(0, 997, (5000, 38), generator=g, device="cuda", dtype=torch.int32)
    q = _q((5000, 8, 64), torch.bfloat16)
    out = A.decode_attention(q, data[:, 0], data[:, 1], table, lens)
    for rows in (slice(0, 7), slice(2500, 2507), slice(4993, 5000)):
        ref, _ = A.decode_attention_reference(q[rows], data[:, 0], data[:, 1], table[rows], lens[rows])
        mass, _ = A.decode_attention_reference(q[rows], data[:, 0], data[:, 1].abs(), table[rows], lens[rows])
        _check(out[rows], ref, mass, torch.bfloat16, 64, 600, 40)


def test_calls_on_several_streams_at_once():
    """Prompts and decode steps that run side by side: nothing is shared between calls."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    x = _q((3000, 12, 128), torch.bfloat16)
    cu = torch.tensor([0, 1100, 1101, 3000], dtype=torch.int32, device="cuda")
    k, v, table, lens = _pool([5000, 900, 0, 333], 16, 2, 128, torch.bfloat16, spare=0)
    q = _q((4, 8, 128), torch.bfloat16)
    want_p, want_d = A.prefill_attention(x[:, :8], x[:, 8:10], x[:, 10:], cu), A.decode_attention(q, k, v, table, lens)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(4)], []
    for turn in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((A.prefill_attention(x[:, :8], x[:, 8:10], x[:, 10:], cu) if (i + turn) % 2 else A.decode_attention(q, k, v, table, lens), (i + turn) % 2))
    torch.cuda.synchronize()
    for out, prompt in got:
        assert torch.equal(out, want_p if prompt else want_d)
