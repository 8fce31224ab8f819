"""Decoding over an 8-bit cache with queries whose elements lie far apart: they are brought into fp16's range, and must not lose what counts."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("heads", [2, 12])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("large,small", [(2.0 ** 20, 2.0 ** -6), (2.0 ** 30, 1.0), (1.0, 2.0 ** -26), (2.0 ** 127, 2.0 ** 100), (2.0 ** -70, 2.0 ** -96), (2.0 ** 4, 2.0 ** -22)])
def test_small_elements_beside_a_large_one(heads, dim, large, small):
    """The large element meets keys of zero, the small ones meet keys that differ: the logits are theirs alone. A query of bf16 spans 26 binary places here,
    which the sums of the products hold exactly enough: products of 4 and 8 bits, added up in fp32."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    g = torch.Generator(device="cuda").manual_seed(dim + heads)
    n, page, group = 300, 16, heads // 2
    pages = -(-n // page)
    data = torch.randint(-7, 8, (pages, 2, 2, page, dim), generator=g, device="cuda").float() * 64  # e4m3 holds them all
    data[:, 0, :, :, 0] = 0
    data = data.to(torch.float8_e4m3fn)
    q = torch.randint(-8, 9, (3, heads, dim), generator=g, device="cuda").float() * (small / 8)
    q[:, :, 0] = large
    q = q.to(torch.bfloat16)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32).expand(3, pages).contiguous()
    lens = torch.tensor([n, 1, 177], dtype=torch.int32, device="cuda")
    one = torch.ones(2, device="cuda")
    scale = 2.0 ** -10 / small / dim ** 0.5  # logits of some units
    scale = min(scale, 2.0 ** 100)
    out, lse = A.decode_attention(q, data[:, 0], data[:, 1], table, lens, scale=scale, k_scale=one, v_scale=one, lse=True)
    args = (table, lens, None, scale, one, one)
    ref, ref_lse = A.decode_attention_reference(q, data[:, 0], data[:, 1], *args)
    mass, _ = A.decode_attention_reference(q, data[:, 0], data[:, 1].float().abs(), *args)
    # the result is rounded to bf16, the weights to fp16; logits up to 7 * 64 * dim * 2^-10 / sqrt(dim) err by the dim roundings of their sum and a few more
    logit, u = 7 / 16 * dim ** 0.5, 2.0 ** -24
    weights = 2.0 ** -11 + (2 * (dim + 2) * logit + 2 * n + 64) * u
    assert bool(((out.double() - ref).abs() <= (2.0 ** -9 * ref.abs() + weights * mass) * 1.01 + 1e-30).all())
    assert float((lse.double() - ref_lse).abs().max()) <= (2 * (dim + 2) * logit + 2 * n + 64) * u


@pytest.mark.parametrize("cache", ["bfloat16", "float8_e4m3fn"])
def test_an_infinite_element(cache):
    """Every logit is infinite then: a row whose logits are all -inf has nothing to weigh, one with +inf or 0 * inf is NaN."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    data = torch.ones(4, 2, 1, 16, 64, device="cuda")
    data[:, 0, :, :, 0] = -1
    data[1, 0, 0, 3, 0], data[2, 0, 0, 3, 0] = 1, 0
    data = data.to(getattr(torch, cache))
    scales = {"k_scale": torch.ones(1, device="cuda"), "v_scale": torch.ones(1, device="cuda")} if cache == "float8_e4m3fn" else {}
    q = torch.full((3, 2, 64), 1000.0, dtype=torch.bfloat16, device="cuda")
    q[:, 0, 0] = float("inf")
    q[:, 1, 0] = 1.0
    table = torch.tensor([[0], [1], [2]], dtype=torch.int32, device="cuda")
    lens = torch.full((3,), 16, dtype=torch.int32, device="cuda")
    out, lse = A.decode_attention(q, data[:, 0], data[:, 1], table, lens, lse=True, **scales)
    assert bool((out[0, 0] == 0).all()) and float(lse[0, 0]) == -float("inf")
    assert bool(out[1:, 0].isnan().all()) and bool((out[:, 1] == 1).all())
