"""Attention over keys and values that are cached or have just been computed (csrc/kernels/mf_decode_attention.cu,
csrc/kernels/mf_prefill_attention.cu):

* ``decode_attention`` - one new token per sequence over a paged cache (``ops.kv_cache.PagedKVCache``, or any pages with a table);
* ``prefill_attention`` - whole prompts, or chunks of prompts behind what is already there, packed one behind the other.

Both are forward passes for serving: bf16 or fp16, head dimensions 64 and 128, any number of query heads per key head, sums and softmax
statistics in fp32. All tensors are on one GPU; lengths and offsets stay on the device, so the calls can be captured into a CUDA graph.
"""
from __future__ import annotations

import contextlib

import torch
from torch.autograd import forward_ad

from .. import _loader  # noqa: F401
from .._loader import _pymf
from ..utils.tensors import current_stream_handle

_ops = _pymf.ops
_types = None


def type_code(dtype):
    """The kernels' number of an element type, None for one that they do not know."""
    global _types
    if _types is None:
        _types = {torch.bfloat16: _ops.BF16, torch.float16: _ops.FP16, torch.float8_e4m3fn: _ops.E4M3}
    return _types.get(dtype)


def strides(name, t, *dims):
    """Strides of `dims` in elements (0 where there is one entry). Rows have to be contiguous and a multiple of 16 bytes apart."""
    size, shape, step = t.element_size(), t.shape, t.stride()
    got = tuple(step[d] if shape[d] > 1 else 0 for d in dims)
    if (shape[-1] > 1 and step[-1] != 1) or any(s * size % 16 or s < 0 for s in got):
        raise ValueError(f"{name}: the last dimension must be contiguous, rows must begin at multiples of 16 bytes (strides {step})")
    return got


def on_gpu(device, **tensors):
    """All tensors on this GPU."""
    if device.type != "cuda":
        raise ValueError("the tensors must be on a GPU")
    for name, t in tensors.items():
        if t is not None and t.device != device:
            raise ValueError(f"{name} is on {t.device}, not on {device}")


@contextlib.contextmanager
def _elsewhere(device, stream):
    with torch.cuda.device(device), torch.cuda.stream(stream):
        yield


_here = contextlib.nullcontext()


def launch_on(device, stream):
    """A context in which what is allocated belongs to the stream that will use it, on GPU number `device`."""
    if stream is None:
        if torch._C._cuda_getDevice() == device:
            return _here
    elif stream.device.index != device:
        raise ValueError(f"the stream belongs to {stream.device}, the tensors are on cuda:{device}")
    return _elsewhere(device, stream)


def no_gradient(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                raise RuntimeError("this operator has no backward pass: call it under torch.no_grad(), or detach its inputs")
    if forward_ad._current_level >= 0:  # within a dual_level()
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise RuntimeError("this operator has no forward-mode derivative: call it with the primals (torch.autograd.forward_ad.unpack_dual)")


def int32(name, t, dims):
    if t.dtype != torch.int32 or t.dim() != dims or (t.shape[-1] > 1 and t.stride(-1) != 1):
        raise ValueError(f"{name} must be an int32 tensor of {dims} dimension(s), contiguous in the last one")


def head_scales(k_scale, v_scale, heads, wanted):
    if wanted != (k_scale is not None) or (k_scale is None) != (v_scale is None):
        raise ValueError("k_scale and v_scale come with a float8_e4m3fn cache, and only with it")
    if wanted:
        for s in (k_scale, v_scale):
            if s.dtype != torch.float32 or s.shape != (heads,) or not s.is_contiguous():
                raise ValueError(f"k_scale and v_scale must be contiguous fp32 tensors of {heads} elements")


def one_word(status):
    if status is not None and (status.dtype != torch.int32 or status.numel() != 1):
        raise ValueError("status must be an int32 tensor of one element")


class Plans:
    """What the checks of a call have found, by the shapes, strides, types and devices of its tensors: a call like one before it is launched
    without being looked at again (the checks take longer than a small kernel). Nothing of the tensors themselves is kept."""

    def __init__(self, most=512):
        self._most, self._known = most, {}

    @staticmethod
    def of(t):
        return None if t is None else (t.shape, t.stride(), t.dtype, t.get_device())

    def get(self, key):
        return self._known.get(key)

    def put(self, key, plan):
        if len(self._known) >= self._most:  # a program whose shapes never repeat
            self._known.clear()
        self._known[key] = plan
        return plan


def _check_result(out, like_shape, like_dtype, lse, lse_shape):
    if out is not None:
        if out.shape != like_shape or out.dtype != like_dtype:
            raise ValueError(f"out must be {tuple(like_shape)} {like_dtype}")
        taken = out.shape[2]
        for step, n in sorted((out.stride(d), out.shape[d]) for d in (0, 1) if out.shape[d] > 1):
            if step < taken:
                raise ValueError("out must not overlap itself")
            taken = step * n
    if lse is not None and (lse.dtype != torch.float32 or tuple(lse.shape) != lse_shape or not lse.is_contiguous()):
        raise ValueError(f"lse must be a contiguous fp32 tensor {lse_shape}")


def _scale(scale, dim):
    if scale is None:
        return dim ** -0.5
    if not 2.0 ** -125 <= scale <= 2.0 ** 127:  # times log2(e), and 6 divided by that, are fp32 numbers in the kernels
        raise ValueError("scale must be positive, from 2^-125 to 2^127")
    return float(scale)


_decode_plans, _prefill_plans = Plans(), Plans()
_misaligned = "tensors must begin at multiples of 16 bytes"


def _plan_decode(key, q, k_pages, v_pages, table, lengths, rows, k_scale, v_scale, out, lse, status):
    if q.dim() != 3 or k_pages.dim() != 4 or v_pages.shape != k_pages.shape or k_pages.shape[3] != q.shape[2]:
        raise ValueError("q must be [B, heads, dim], k_pages and v_pages [pages, kv_heads, page_size, dim]")
    B, heads, dim = q.shape
    pages, kv_heads, page_size, _ = k_pages.shape
    q_type, cache_type = type_code(q.dtype), type_code(k_pages.dtype)
    if dim not in (64, 128) or kv_heads == 0 or heads == 0 or heads % kv_heads or page_size == 0:
        raise ValueError("head dimensions are 64 or 128, heads is a multiple of kv_heads, pages hold a token at least")
    if q_type not in (_ops.BF16, _ops.FP16) or v_pages.dtype != k_pages.dtype or cache_type not in (q_type, _ops.E4M3):
        raise ValueError("q is bf16 or fp16, the pages are of its type or float8_e4m3fn")
    head_scales(k_scale, v_scale, kv_heads, cache_type == _ops.E4M3)
    int32("table", table, 2)
    int32("lengths", lengths, 1)
    if rows is not None:
        int32("rows", rows, 1)
    if lengths.shape[0] != table.shape[0] or (rows.shape[0] != B if rows is not None else table.shape[0] < B):
        raise ValueError("table and lengths have an entry for each sequence, rows (or they) for each query")
    one_word(status)
    capacity = table.shape[1] * page_size
    if capacity > 0x7fffff00:
        raise ValueError("a sequence may have 2^31 - 256 tokens at most")
    _check_result(out, q.shape, q.dtype, lse, (B, heads))
    qs, step = strides("q", q, 0, 1), strides("k_pages", k_pages, 0, 1, 2)
    if strides("v_pages", v_pages, 0, 1, 2) != step:
        raise ValueError("k_pages and v_pages must have the same strides")
    os = strides("out", out, 0, 1) if out is not None else (heads * dim, dim)
    on_gpu(q.device, k_pages=k_pages, v_pages=v_pages, table=table, lengths=lengths, rows=rows, k_scale=k_scale, v_scale=v_scale, out=out, lse=lse,
           status=status)
    native = _ops.DecodePlan(*qs, *os, *step, table.stride(0), B, kv_heads, heads // kv_heads, page_size, pages, table.shape[1], table.shape[0], dim, q_type,
                             cache_type)
    with launch_on(q.device.index, None):  # its size goes by the GPU that the call runs on, whichever is the current one
        words = (native.workspace() + 3) // 4
    return _decode_plans.put(key, (native, words, dim ** -0.5))


def decode_attention(q, k_pages, v_pages, table, lengths, *, rows=None, scale=None, k_scale=None, v_scale=None, out=None, lse=None, status=None,
                     stream=None):
    """Attention of one new token per sequence over its cached keys and values, the token's own among them.

    q [B, heads, dim]; k_pages, v_pages [pages, kv_heads, page_size, dim] (any strides, the same for both; pass `.transpose(1, 2)` of pages that
    are kept token by token), heads a multiple of kv_heads; table int32 [seqs, width]: the pages of each sequence; lengths int32 [seqs]: its
    tokens (no more than width * page_size count). rows int32 [B]: the sequence of each query, by default the first B. Pages in q's type, or
    float8_e4m3fn with k_scale, v_scale fp32 [kv_heads] (value = e4m3 * scale). scale: of the logits, 2^-125 to 2^127, 1 / sqrt(dim) by
    default. Returns out [B, heads, dim]; with lse=True (or a tensor for it) also the logarithm of the sum of exponentials, fp32 [B, heads].
    A sequence without tokens gives zeros and -inf. What lies in a page behind a sequence's length does not matter. The last bits of a row
    may depend on what else is in the batch (that decides where long rows are cut), and on nothing else. out must not overlap the inputs.

    status: int32 tensor of one element, receives MF_DEV_ERR_BOUNDS (2) where a length reaches a page number that does not exist (its
    keys and values then count as zeros) or rows names no sequence (which then has no tokens)."""
    with_lse = lse is not None and lse is not False
    if lse is True or lse is False:
        lse = None
    no_gradient(q, k_pages, v_pages, k_scale, v_scale, out, lse)
    # the required tensors one by one and the others by name, as a call takes no longer than a few of these look-ups
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k_pages.shape, k_pages.stride(), k_pages.dtype, k_pages.get_device(), v_pages.shape, v_pages.stride(),
           v_pages.dtype, v_pages.get_device(), table.shape, table.stride(), table.dtype, table.get_device(), lengths.shape, lengths.stride(), lengths.dtype,
           lengths.get_device(), *(() if rows is k_scale is v_scale is out is lse is status is None else
                                   map(Plans.of, (rows, k_scale, v_scale, out, lse, status))))
    native, words, factor = _decode_plans.get(key) or _plan_decode(key, q, k_pages, v_pages, table, lengths, rows, k_scale, v_scale, out, lse, status)
    if scale is not None:
        factor = _scale(scale, 0)
    with launch_on(key[3], stream):
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if with_lse and lse is None:
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        ws = table.new_empty(words) if words else None
        at = q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), out.data_ptr()
        if (at[0] | at[1] | at[2] | at[3]) & 15:
            raise ValueError(_misaligned)
        rc = native.run(*at, table.data_ptr(), lengths.data_ptr(), 0 if rows is None else rows.data_ptr(), 0 if k_scale is None else k_scale.data_ptr(),
                        0 if v_scale is None else v_scale.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if status is None else status.data_ptr(),
                        0 if ws is None else ws.data_ptr(), 4 * words, factor, current_stream_handle())
    if rc != 0:
        raise RuntimeError(f"decode_attention launch failed ({rc})")
    return (out, lse) if with_lse else out


def _plan_prefill(key, q, k, v, cu_q, cu_k, out, lse, status):
    if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.shape[2] != q.shape[2]:
        raise ValueError("q must be [tokens, heads, dim], k and v [keys, kv_heads, dim]")
    tokens, heads, dim = q.shape
    keys, kv_heads, _ = k.shape
    kind = type_code(q.dtype)
    if dim not in (64, 128) or kv_heads == 0 or heads == 0 or heads % kv_heads:
        raise ValueError("head dimensions are 64 or 128, heads is a multiple of kv_heads")
    if kind not in (_ops.BF16, _ops.FP16) or k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError("q, k and v are all bf16 or all fp16")
    if tokens > 0x7fffff00 or keys > 0x7fffff00:
        raise ValueError("2^31 - 256 tokens at most")
    int32("cu_q", cu_q, 1)
    int32("cu_k", cu_k, 1)
    if cu_q.shape[0] < 1 or cu_k.shape != cu_q.shape:
        raise ValueError("cu_q and cu_k have one entry more than there are sequences")
    one_word(status)
    _check_result(out, q.shape, q.dtype, lse, (tokens, heads))
    qs, ks, vs = strides("q", q, 0, 1), strides("k", k, 0, 1), strides("v", v, 0, 1)
    for t, step in ((q, qs), (k, ks), (v, vs)):
        if any(n > 1 and s == 0 for n, s in zip(t.shape, step)):
            raise ValueError("q, k and v must not be expanded: the rows are fetched by strides of their own")
    os = strides("out", out, 0, 1) if out is not None else (heads * dim, dim)
    on_gpu(q.device, k=k, v=v, cu_q=cu_q, cu_k=cu_k, out=out, lse=lse, status=status)
    return _prefill_plans.put(key, (_ops.PrefillPlan(*qs, *ks, *vs, *os, cu_q.shape[0] - 1, kv_heads, heads // kv_heads, tokens, keys, dim, kind), dim ** -0.5))


def prefill_attention(q, k, v, cu_q, cu_k=None, *, causal=True, scale=None, out=None, lse=None, status=None, stream=None):
    """Attention of packed prompts. q [tokens, heads, dim], k and v [keys, kv_heads, dim] (any strides, rows contiguous, not expanded), heads a multiple
    of kv_heads; cu_q int32 [B + 1]: the rows of sequence b are cu_q[b] to cu_q[b + 1], ascending from 0 or more; cu_k the same for keys,
    by default cu_q. With `causal` the last row of a sequence sees all of its keys, each row before it one less: a chunk of a prompt is given as
    its rows with all keys up to its end. scale: of the logits, 2^-125 to 2^127, 1 / sqrt(dim) by default.

    Returns out [tokens, heads, dim]; with lse=True (or a tensor for it) also the logarithm of the sum of exponentials, fp32
    [tokens, heads]. Rows that see no key give zeros and -inf; rows that belong to no sequence are left as they are. out must not overlap the
    inputs. What a row may not see does not change a bit of it, NaN and infinities included. status: int32 tensor of one element, receives
    GEMM_PIPELINE_EXPIRED (3) if a bounded wait inside the kernel ran out; rows may be unwritten then, and nothing else tells."""
    with_lse = lse is not None and lse is not False
    if lse is True or lse is False:
        lse = None
    no_gradient(q, k, v, out, lse)
    cu_k = cu_q if cu_k is None else cu_k
    key = (q.shape, q.stride(), q.dtype, q.get_device(), k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype, v.get_device(), cu_q.shape,
           cu_q.stride(), cu_q.dtype, cu_q.get_device(), cu_k.shape, cu_k.stride(), cu_k.dtype, cu_k.get_device(),
           *(() if out is lse is status is None else map(Plans.of, (out, lse, status))))
    native, factor = _prefill_plans.get(key) or _plan_prefill(key, q, k, v, cu_q, cu_k, out, lse, status)
    if scale is not None:
        factor = _scale(scale, 0)
    with launch_on(key[3], stream):
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        if with_lse and lse is None:
            lse = torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        at = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        if (at[0] | at[1] | at[2] | at[3]) & 15:
            raise ValueError(_misaligned)
        rc = native.run(*at, cu_q.data_ptr(), cu_k.data_ptr(), 0 if lse is None else lse.data_ptr(), 0 if status is None else status.data_ptr(),
                        bool(causal), factor, current_stream_handle())
    if rc != 0:
        raise RuntimeError(f"prefill_attention launch failed ({rc})")
    return (out, lse) if with_lse else out


def _attend_reference(q, k, v, seen, scale):
    """One sequence in fp64: q [rows, heads, dim], k and v [keys, kv_heads, dim], seen bool [rows, keys]. Only what is seen counts."""
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
