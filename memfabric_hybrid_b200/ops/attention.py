"""Attention over keys and values that are cached or have just been computed (csrc/kernels/mf_decode_attention.cu,
csrc/kernels/mf_prefill_attention.cu):

* ``decode_attention`` - one new token per sequence over a paged cache (``ops.kv_cache.PagedKVCache``, or any pages with a table);
* ``prefill_attention`` - whole prompts, or chunks of prompts behind what is already there, packed one behind the other.

Both are forward passes for serving: bf16 or fp16, head dimensions 64 and 128, any number of query heads per key head, sums and softmax
statistics in fp32. All tensors are on one GPU; lengths and offsets stay on the device, so the calls can be captured into a CUDA graph.
"""
from __future__ import annotations

import contextlib
import math

from .. import _loader  # noqa: F401
from .._loader import _pymf
from ..utils.tensors import current_stream_handle

_ops = _pymf.ops
_types = None


def type_code(dtype):
    """The kernels' number of an element type, None for one that they do not know."""
    global _types
    if _types is None:
        import torch

        _types = {torch.bfloat16: _ops.BF16, torch.float16: _ops.FP16, torch.float8_e4m3fn: _ops.E4M3}
    return _types.get(dtype)


def strides(name, t, *dims):
    """Strides of `dims` in elements (0 where there is one entry). The rows have to be contiguous and to begin at multiples of 16 bytes."""
    size, shape, step = t.element_size(), t.shape, t.stride()
    got = tuple(step[d] if shape[d] > 1 else 0 for d in dims)
    if (shape[-1] > 1 and step[-1] != 1) or t.data_ptr() % 16 or any(s * size % 16 or s < 0 for s in got):
        raise ValueError(f"{name}: the last dimension must be contiguous, rows must begin at multiples of 16 bytes (strides {step})")
    return got


def on_gpu(first, **tensors):
    """All tensors on the GPU of `first`."""
    if not first.is_cuda:
        raise ValueError("the tensors must be on a GPU")
    dev = first.device
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, not on {dev}")


@contextlib.contextmanager
def _elsewhere(device, stream):
    import torch

    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


_here = contextlib.nullcontext()


def launch_on(device, stream):
    """A context in which what is allocated belongs to the stream that will use it, on the tensors' GPU."""
    import torch

    if stream is None and torch._C._cuda_getDevice() == device.index:
        return _here
    return _elsewhere(device, stream)


def no_gradient(*tensors):
    import torch

    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError("this operator has no backward pass: call it under torch.no_grad(), or detach its inputs")


def _int32(name, t, dims):
    import torch

    if t.dtype != torch.int32 or t.dim() != dims or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be an int32 tensor of {dims} dimension(s), contiguous in the last one")


def _result(out, like, lse, lse_shape):
    import torch

    if out is None:
        out = torch.empty(like.shape, dtype=like.dtype, device=like.device)
    elif out.shape != like.shape or out.dtype != like.dtype:
        raise ValueError(f"out must be {tuple(like.shape)} {like.dtype}")
    if lse is True:
        lse = torch.empty(lse_shape, dtype=torch.float32, device=like.device)
    return out, lse


def _check_out(out, lse, lse_shape):
    import torch

    if out is not None and ((out.shape[1] > 1 and out.stride(1) < out.shape[2]) or (out.shape[0] > 1 and out.stride(0) < out.shape[1] * out.stride(1))):
        raise ValueError("out must not overlap itself")
    if lse is not None and lse is not True and lse is not False:
        if lse.dtype != torch.float32 or tuple(lse.shape) != lse_shape or not lse.is_contiguous():
            raise ValueError(f"lse must be a contiguous fp32 tensor {lse_shape}")


def _scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    if not (scale > 0 and math.isfinite(scale)):
        raise ValueError("scale must be positive and finite")
    return float(scale)


def decode_attention(q, k_pages, v_pages, table, lengths, *, rows=None, scale=None, k_scale=None, v_scale=None, out=None, lse=None, status=None,
                     stream=None):
    """Attention of one new token per sequence over its cached keys and values, the token's own among them.

    q [B, heads, dim]; k_pages, v_pages [pages, kv_heads, page_size, dim] (any strides, the same for both; pass `.transpose(1, 2)` of pages that
    are kept token by token), heads a multiple of kv_heads; table int32 [seqs, width]: the pages of each sequence; lengths int32 [seqs]: its
    tokens (no more than width * page_size count). rows int32 [B]: the sequence of each query, by default the first B; else B sequences
    in order. Pages in q's type, or float8_e4m3fn with k_scale, v_scale fp32 [kv_heads] (value = e4m3 * scale). scale: of the logits,
    1 / sqrt(dim) by default. Returns out [B, heads, dim]; with lse=True (or a tensor for it) also the logarithm of the sum of
    exponentials, fp32 [B, heads]. A sequence without tokens gives zeros and -inf. What lies in a page behind a sequence's
    length does not matter.

    status: int32 tensor of one element, receives MF_DEV_ERR_BOUNDS (2) where a length reaches a page number that does not exist (its
    keys and values then count as zeros) or rows names no sequence (which then has no tokens)."""
    import torch

    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape or k_pages.shape[3] != q.shape[2]:
        raise ValueError("q must be [B, heads, dim], k_pages and v_pages [pages, kv_heads, page_size, dim]")
    B, heads, dim = q.shape
    pages, kv_heads, page_size, _ = k_pages.shape
    q_type, cache_type = type_code(q.dtype), type_code(k_pages.dtype)
    if dim not in (64, 128) or kv_heads == 0 or heads == 0 or heads % kv_heads or page_size == 0:
        raise ValueError("head dimensions are 64 or 128, heads is a multiple of kv_heads, pages hold a token at least")
    if q_type not in (_ops.BF16, _ops.FP16) or v_pages.dtype != k_pages.dtype or cache_type not in (q_type, _ops.E4M3):
        raise ValueError("q is bf16 or fp16, the pages are of its type or float8_e4m3fn")
    if (cache_type == _ops.E4M3) != (k_scale is not None) or (k_scale is None) != (v_scale is None):
        raise ValueError("k_scale and v_scale come with float8_e4m3fn pages, and only with them")
    if k_scale is not None:
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or s.shape != (kv_heads,) or not s.is_contiguous():
                raise ValueError(f"k_scale and v_scale must be contiguous fp32 tensors of {kv_heads} elements")
    _int32("table", table, 2)
    _int32("lengths", lengths, 1)
    if rows is not None:
        _int32("rows", rows, 1)
    if lengths.shape[0] != table.shape[0] or (rows.shape[0] != B if rows is not None else table.shape[0] < B):
        raise ValueError("table and lengths have an entry for each sequence, rows (or they) for each query")
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1):
        raise ValueError("status must be an int32 tensor of one element")
    if table.shape[1] * page_size > 0x7fffff00:
        raise ValueError("a sequence may have 2^31 - 256 tokens at most")
    _check_out(out, lse, (B, heads))
    factor = _scale(scale, dim)
    qs, step = strides("q", q, 0, 1), strides("k_pages", k_pages, 0, 1, 2)
    if strides("v_pages", v_pages, 0, 1, 2) != step:
        raise ValueError("k_pages and v_pages must have the same strides")
    no_gradient(q)
    on_gpu(q, k_pages=k_pages, v_pages=v_pages, table=table, lengths=lengths, rows=rows, k_scale=k_scale, v_scale=v_scale, out=out,
           lse=lse if isinstance(lse, torch.Tensor) else None, status=status)
    with launch_on(q.device, stream):
        given, (out, lse) = out, _result(out, q, lse, (B, heads))
        os = strides("out", out, 0, 1) if given is not None else (heads * dim, dim)
        group = heads // kv_heads
        ws = torch.empty(_ops.decode_attention_workspace(B, kv_heads, group, dim, table.shape[1] * page_size), dtype=torch.uint8, device=q.device)
        rc = _ops.decode_attention(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(), lengths.data_ptr(),
                                   rows.data_ptr() if rows is not None else 0, k_scale.data_ptr() if k_scale is not None else 0,
                                   v_scale.data_ptr() if v_scale is not None else 0, out.data_ptr(), lse.data_ptr() if isinstance(lse, torch.Tensor) else 0,
                                   status.data_ptr() if status is not None else 0, ws.data_ptr(), *qs, *os, *step, table.stride(0), B, kv_heads, group, page_size,
                                   pages, table.shape[1], table.shape[0], factor, dim, q_type, cache_type, current_stream_handle())
    if rc != 0:
        raise RuntimeError(f"decode_attention launch failed ({rc})")
    return (out, lse) if isinstance(lse, torch.Tensor) else out


def prefill_attention(q, k, v, cu_q, cu_k=None, *, causal=True, scale=None, out=None, lse=None, status=None, stream=None):
    """Attention of packed prompts. q [tokens, heads, dim], k and v [keys, kv_heads, dim] (any strides, rows contiguous), heads a multiple of
    kv_heads; cu_q int32 [B + 1]: the rows of sequence b are cu_q[b] to cu_q[b + 1], ascending from 0 or more; cu_k the same for keys,
    by default cu_q. With `causal` the last row of a sequence sees all of its keys, each row before it one less: a chunk of a prompt is given as
    its rows with all keys up to its end. scale: of the logits, 1 / sqrt(dim) by default.

    Returns out [tokens, heads, dim]; with lse=True (or a tensor for it) also the logarithm of the sum of exponentials, fp32
    [tokens, heads]. Rows that see no key give zeros and -inf; rows that belong to no sequence are left as they are. status: int32 tensor of one
    element, receives GEMM_PIPELINE_EXPIRED (3) if a bounded wait inside the kernel ran out."""
    import torch

    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError("q must be [tokens, heads, dim], k and v [keys, kv_heads, dim]")
    tokens, heads, dim = q.shape
    keys, kv_heads, _ = k.shape
    kind = type_code(q.dtype)
    if dim not in (64, 128) or kv_heads == 0 or heads == 0 or heads % kv_heads or heads > 65535:
        raise ValueError("head dimensions are 64 or 128, heads is a multiple of kv_heads")
    if kind not in (_ops.BF16, _ops.FP16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v are all bf16 or all fp16")
    if tokens > 0x7fffff00 or keys > 0x7fffff00:
        raise ValueError("2^31 - 256 tokens at most")
    cu_k = cu_q if cu_k is None else cu_k
    _int32("cu_q", cu_q, 1)
    _int32("cu_k", cu_k, 1)
    if cu_q.shape[0] < 1 or cu_k.shape != cu_q.shape:
        raise ValueError("cu_q and cu_k have one entry more than there are sequences")
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1):
        raise ValueError("status must be an int32 tensor of one element")
    _check_out(out, lse, (tokens, heads))
    factor = _scale(scale, dim)
    qs, ks, vs = strides("q", q, 0, 1), strides("k", k, 0, 1), strides("v", v, 0, 1)
    for t, step in ((q, qs), (k, ks), (v, vs)):
        if any(n > 1 and s == 0 for n, s in zip(t.shape, step)):
            raise ValueError("q, k and v must not be expanded: the rows are fetched by strides of their own")
    no_gradient(q, k, v)
    on_gpu(q, k=k, v=v, cu_q=cu_q, cu_k=cu_k, out=out, lse=lse if isinstance(lse, torch.Tensor) else None, status=status)
    with launch_on(q.device, stream):
        given, (out, lse) = out, _result(out, q, lse, (tokens, heads))
        os = strides("out", out, 0, 1) if given is not None else (heads * dim, dim)
        rc = _ops.prefill_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), out.data_ptr(),
                                    lse.data_ptr() if isinstance(lse, torch.Tensor) else 0, status.data_ptr() if status is not None else 0, *qs, *ks, *vs, *os, cu_q.shape[0] - 1, kv_heads, heads // kv_heads,
                                    tokens, keys, int(causal), factor, dim, kind, current_stream_handle())
    if rc != 0:
        raise RuntimeError(f"prefill_attention launch failed ({rc})")
    return (out, lse) if isinstance(lse, torch.Tensor) else out


def _attend_reference(q, k, v, seen, scale):
    """One sequence in fp64: q [rows, heads, dim], k and v [keys, kv_heads, dim], seen bool [rows, keys]. Only what is seen counts."""
    import torch

    group = q.shape[1] // k.shape[1]
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    if k.shape[0] == 0:
        return out, lse
    for h in range(q.shape[1]):
        logits = (q[:, h].double() @ k[:, h // group].double().T) * scale
        logits = torch.where(seen, logits, float("-inf"))
        lse[:, h] = torch.logsumexp(logits, 1)
        p = torch.where(seen, torch.exp(logits - torch.where(lse[:, h:h + 1] == float("-inf"), 0.0, lse[:, h:h + 1])), 0.0)
        bad = ~torch.isfinite(v[:, h // group])
        if bool(bad.any()):  # 0 * inf is not a part of the sum
            out[:, h] = torch.where(seen[:, :, None], p[:, :, None] * v[None, :, h // group].double(), 0.0).sum(1)
        else:
            out[:, h] = p @ v[:, h // group].double()
    return out, lse


def decode_attention_reference(q, k_pages, v_pages, table, lengths, rows=None, scale=None, k_scale=None, v_scale=None):
    """fp64 PyTorch oracle of decode_attention: (out, lse)."""
    import torch

    scale = q.shape[2] ** -0.5 if scale is None else scale
    outs, lses = [], []
    for b in range(q.shape[0]):
        r = int(rows[b]) if rows is not None else b
        n = max(0, min(int(lengths[r]), table.shape[1] * k_pages.shape[2]))
        used = table[r, :-(-n // k_pages.shape[2])].tolist()
        k, v = (torch.stack([x[p].double() for p in used]).permute(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:n] if n else q.new_zeros(0, x.shape[1], x.shape[3])
                for x in (k_pages, v_pages))
        if k_scale is not None:
            k, v = k * k_scale.double()[:, None], v * v_scale.double()[:, None]
        o, l = _attend_reference(q[b:b + 1], k, v, torch.ones(1, n, dtype=torch.bool, device=q.device), scale)
        outs.append(o)
        lses.append(l)
    return torch.cat(outs), torch.cat(lses)


def prefill_attention_reference(q, k, v, cu_q, cu_k=None, causal=True, scale=None):
    """fp64 PyTorch oracle of prefill_attention: (out, lse), zeros and -inf for rows of no sequence."""
    import torch

    scale = q.shape[2] ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=q.device)
    cq, ck = cu_q.tolist(), (cu_q if cu_k is None else cu_k).tolist()
    for b in range(len(cq) - 1):
        n, m = cq[b + 1] - cq[b], ck[b + 1] - ck[b]
        seen = torch.ones(n, m, dtype=torch.bool, device=q.device)
        if causal:
            seen = torch.arange(m, device=q.device) <= torch.arange(n, device=q.device)[:, None] + (m - n)
        out[cq[b]:cq[b + 1]], lse[cq[b]:cq[b + 1]] = _attend_reference(q[cq[b]:cq[b + 1]], k[ck[b]:ck[b + 1]], v[ck[b]:ck[b + 1]], seen, scale)
    return out, lse
