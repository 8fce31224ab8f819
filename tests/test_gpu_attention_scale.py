"""The smallest and the largest scale that the attention operators take."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", ["bfloat16", "float16"])
@pytest.mark.parametrize("power", [-125, -100, 100, 120])
def test_extreme_scales(name, power):
    """Logits of about one, from elements that make up for the scale as far as the type reaches; next to nothing otherwise, which gives means."""
    import torch

    from memfabric_hybrid_b200.ops import attention as A

    dtype, scale = getattr(torch, name), 2.0 ** power
    g = torch.Generator(device="cuda").manual_seed(0)
    q, k, v = (torch.randn(200, heads, 64, generator=g, device="cuda") for heads in (4, 2, 2))
    half = 2.0 ** (-power // 2) if name == "bfloat16" else 2.0 ** max(-14, min(12, -power // 2))  # fp16 holds no more, as normal numbers
    if power > 0 and name == "float16":
        k[:] = 0  # logits that would not be finite otherwise
    q, k, v = (q * half / 8).to(dtype), (k * half).to(dtype), v.to(dtype)
    cu = torch.tensor([0, 200], dtype=torch.int32, device="cuda")
    out, lse = A.prefill_attention(q, k, v, cu, scale=scale, lse=True)
    ref, ref_lse = A.prefill_attention_reference(q, k, v, cu, None, True, scale)
    mass, _ = A.prefill_attention_reference(q, k, v.abs(), cu, None, True, scale)
    h, u = torch.finfo(dtype).eps / 2, 2.0 ** -24
    fuzz = (2 * 66 * 20 + 2 * 200 + 64) * u  # logits below 20; the polynomial of some weights errs by 1.01e-4 for bf16, 2.9e-6 for fp16
    weights = h + fuzz + 2 * (1.01e-4 if name == "bfloat16" else 2.9e-6)
    assert bool(((out.double() - ref).abs() <= h * ref.abs() + weights * mass * 1.01 + 1e-30).all())
    assert float((lse.double() - ref_lse).abs().max()) <= fuzz + (1.01e-4 if name == "bfloat16" else 2.9e-6)
    pages = torch.zeros(13, 2, 2, 16, 64, dtype=dtype, device="cuda")
    pages[:, 0] = torch.nn.functional.pad(k, (0, 0, 0, 0, 0, 8)).view(13, 16, 2, 64).transpose(1, 2)
    pages[:, 1] = torch.nn.functional.pad(v, (0, 0, 0, 0, 0, 8)).view(13, 16, 2, 64).transpose(1, 2)
    table, lens = torch.arange(13, dtype=torch.int32, device="cuda")[None], torch.tensor([200], dtype=torch.int32, device="cuda")
    one = A.decode_attention(q[199:], pages[:, 0], pages[:, 1], table, lens, scale=scale)
    assert bool(((one.double() - ref[199:]).abs() <= h * ref[199:].abs() + (h + fuzz) * mass[199:] * 1.01 + 1e-30).all())
