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
