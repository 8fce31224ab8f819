"""A paged key-value cache whose book-keeping lives on the GPU (csrc/kernels/mf_kv_cache.cu).

    cache = PagedKVCache.allocate(layers, pages, page_size, kv_heads, head_dim, seqs, width)
    slots = cache.reserve(seqs, counts, total)            # once per step: pages and slots for the new tokens
    cache.write(layer, k, v, slots)                       # per layer
    out = cache.decode(layer, q, rows)                    # per layer: ops.attention.decode_attention over the sequences `rows`
    cache.fork(src, dst); cache.free(seqs); cache.compact()

Every call is a launch or two on the current stream, with nothing read back, so a step can be captured into a CUDA graph. Free pages are
handed out from the lowest number on, in the order of the request, so a run can be repeated bit by bit. The block of a page in one layer
is contiguous (`block`): what `bm.copy_data_batch` moves between pools, if the data lies in one.
"""
from __future__ import annotations

import functools

import torch

from .attention import Plans, _misaligned, _ops, decode_attention, head_scales, int32, launch_on, no_gradient, on_gpu, one_word, strides, type_code
from ..utils.tensors import current_stream_handle


@functools.lru_cache(maxsize=64)
def _plans(device, kind, kv_heads, head_dim):
    """What the checks of writes and of requests have found, for all caches that they go by alike: a new one does not begin from nothing."""
    return Plans(), Plans()


class PagedKVCache:
    """Around tensors that the caller keeps, all on one GPU and contiguous:

    data [layers, pages, 2 (key, value), kv_heads, page_size, head_dim], bf16, fp16 or float8_e4m3fn, head_dim a multiple of 16; table int32
    [seqs, width]: the pages of each sequence, -1 where there is none; lengths int32 [seqs]: its tokens; refs int32 [pages]: how many
    sequences hold a page, 0 for a free one. status int32 [1] (made here if not given): check_status()."""

    def __init__(self, data, table, lengths, refs, status=None):
        if data.dim() != 6 or data.shape[2] != 2 or 0 in data.shape or not data.is_contiguous():
            raise ValueError("data must be contiguous [layers, pages, 2, kv_heads, page_size, head_dim]")
        self.layers, self.pages, _, self.kv_heads, self.page_size, self.head_dim = data.shape
        self._type = type_code(data.dtype)
        if self._type is None or self.head_dim % 16:
            raise ValueError("data is bf16, fp16 or float8_e4m3fn, head_dim a multiple of 16")
        int32("table", table, 2)
        int32("lengths", lengths, 1)
        int32("refs", refs, 1)
        if not table.is_contiguous() or table.shape[0] == 0 or lengths.shape[0] != table.shape[0] or refs.shape[0] != self.pages:
            raise ValueError("table [seqs, width] and lengths [seqs] have a row for each sequence, refs [pages] an entry for each page")
        if table.shape[0] > _ops.KV_MAX_SEQS or table.shape[1] * self.page_size > 0x7fffff00:
            raise ValueError(f"{_ops.KV_MAX_SEQS} sequences and 2^31 - 256 tokens of one at most")
        if data.data_ptr() % 16 or refs.data_ptr() % 16:
            raise ValueError("data and refs must begin at multiples of 16 bytes")
        one_word(status)
        on_gpu(data.device, table=table, lengths=lengths, refs=refs, status=status)
        self.data, self.table, self.lengths, self.refs = data, table, lengths, refs
        self.status = status if status is not None else torch.zeros(1, dtype=torch.int32, device=data.device)
        self.seqs, self.width = table.shape
        self._device = data.device
        self._writes, self._requests = _plans(data.device, self._type, self.kv_heads, self.head_dim)
        self._native = _ops.KvCache(data.data_ptr(), table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), self.status.data_ptr(), self.layers, self.pages,
                                    self.page_size, self.kv_heads, self.head_dim * data.element_size(), self.seqs, self.width)

    @classmethod
    def allocate(cls, layers, pages, page_size, kv_heads, head_dim, seqs, width, dtype=None, device="cuda"):
        """An empty cache in memory of its own (bf16 by default)."""
        data = torch.zeros(layers, pages, 2, kv_heads, page_size, head_dim, dtype=dtype or torch.bfloat16, device=device)
        return cls(data, torch.full((seqs, width), -1, dtype=torch.int32, device=device), torch.zeros(seqs, dtype=torch.int32, device=device),
                   torch.zeros(pages, dtype=torch.int32, device=device))

    def k_pages(self, layer):
        return self.data[layer, :, 0]

    def v_pages(self, layer):
        return self.data[layer, :, 1]

    def block(self, layer, page):
        """(address, bytes) of what one layer keeps in a page, keys and values."""
        if not (0 <= layer < self.layers and 0 <= page < self.pages):
            raise ValueError("no such layer or page")
        n = 2 * self.kv_heads * self.page_size * self.head_dim * self.data.element_size()
        return self.data.data_ptr() + (layer * self.pages + page) * n, n

    def check_status(self) -> int:
        """0, or MF_DEV_ERR_BOUNDS (2) if a call since the last check was refused on the device, wholly or in part. Waits for the GPU, whatever
        streams the calls were given."""
        torch.cuda.synchronize(self._device)  # the calls may have been given other streams than the current one
        s = int(self.status.item())
        if s:
            self.status.zero_()
            torch.cuda.current_stream(self._device).synchronize()  # before another stream's next call
        return s

    def _request(self, name, t):
        key = (t.shape, t.stride(), t.dtype, t.get_device())
        n = self._requests.get(key)
        if n is None:
            int32(name, t, 1)
            if t.device != self._device:
                raise ValueError(f"{name} is on {t.device}, not on {self._device}")
            n = self._requests.put(key, (t.shape[0],))
        return n[0]

    def _at_most_all(self, n):
        if n > self.seqs:
            raise ValueError(f"{n} entries: the cache has {self.seqs} sequences")

    def reserve(self, seqs, counts, total, stream=None):
        """Lengthens each sequence seqs[i] by counts[i] tokens (int32 [n] both) and returns the new tokens' slots, int64 [total], request by
        request; total is their number, known on the host, or more: slots behind the last token are -1. A last page that is partly
        filled and held by others as well is copied first, its filled rows in all layers. All or nothing: where pages or the
        table's width do not suffice, the tokens are more than total, or a sequence does not exist or is named twice, nothing changes,
        all slots are -1 and the status is set."""
        n = self._request("seqs", seqs)
        if self._request("counts", counts) != n:
            raise ValueError("seqs and counts have the same length")
        self._at_most_all(n)
        if not 0 <= total <= 0x7fffffff:
            raise ValueError("total must be the number of new tokens")
        with launch_on(self._device.index, stream):
            if n == 0:
                return torch.full((total,), -1, dtype=torch.int64, device=self._device)
            slots = torch.empty(total, dtype=torch.int64, device=self._device)
            ws = seqs.new_empty(self._native.reserve_workspace(n, total) // 4)
            rc = self._native.reserve(seqs.data_ptr(), counts.data_ptr(), n, total, slots.data_ptr(), ws.data_ptr(), current_stream_handle())
        if rc != 0:
            raise RuntimeError(f"kv_reserve launch failed ({rc})")
        return slots

    def write(self, layer, k, v, slots, *, k_scale=None, v_scale=None, stream=None):
        """Puts keys and values [tokens, kv_heads, head_dim] (any strides, rows contiguous) of one layer into their slots (int64 [tokens], from
        reserve(), or page * page_size + place). A slot below 0 leaves its token out; one behind the last page too, and sets the status;
        what one holds that is named twice is not defined.
        A float8_e4m3fn cache takes bf16 or fp16 and k_scale, v_scale fp32 [kv_heads]: it holds x * (1 / scale), rounded to nearest and
        saturated at 448; any other cache takes its own type."""
        key = (k.shape, k.stride(), k.dtype, k.get_device(), v.shape, v.stride(), v.dtype, v.get_device(), slots.shape, slots.stride(), slots.dtype,
               slots.get_device(), *(() if k_scale is v_scale is None else map(Plans.of, (k_scale, v_scale))))
        plan = self._writes.get(key) or self._writes.put(key, self._plan_write(k, v, slots, k_scale, v_scale))
        if not 0 <= layer < self.layers:
            raise ValueError(f"there are {self.layers} layers")
        no_gradient(k, v, k_scale, v_scale)
        with launch_on(self._device.index, stream):
            at = k.data_ptr(), v.data_ptr()
            if (at[0] | at[1]) & 15:
                raise ValueError(_misaligned)
            rc = self._native.write(layer, *at, slots.data_ptr(), k_scale.data_ptr() if k_scale is not None else 0,
                                    v_scale.data_ptr() if v_scale is not None else 0, *plan, current_stream_handle())
        if rc != 0:
            raise RuntimeError(f"kv_write launch failed ({rc})")

    def _plan_write(self, k, v, slots, k_scale, v_scale):
        shape = (slots.shape[0] if slots.dim() == 1 else -1, self.kv_heads, self.head_dim)
        if k.shape != shape or v.shape != shape or slots.dtype != torch.int64 or not slots.is_contiguous():
            raise ValueError(f"k and v must be [tokens, {self.kv_heads}, {self.head_dim}], slots contiguous int64 [tokens]")
        kind, wide = type_code(k.dtype), self._type == _ops.E4M3
        if v.dtype != k.dtype or kind not in (_ops.BF16, _ops.FP16) or not (wide or kind == self._type):
            raise ValueError(f"a cache of {self.data.dtype} does not take {k.dtype} and {v.dtype}")
        head_scales(k_scale, v_scale, self.kv_heads, wide)
        ks, vs = strides("k", k, 0, 1), strides("v", v, 0, 1)
        on_gpu(self._device, k=k, v=v, slots=slots, k_scale=k_scale, v_scale=v_scale)
        return (*ks, *vs, shape[0], self.head_dim, kind, self._type)

    def decode(self, layer, q, rows=None, *, scale=None, k_scale=None, v_scale=None, out=None, lse=None, stream=None):
        """decode_attention of q [B, heads, head_dim] over the sequences rows (int32 [B], by default the first B) of one layer."""
        if not 0 <= layer < self.layers:
            raise ValueError(f"there are {self.layers} layers")
        return decode_attention(q, self.k_pages(layer), self.v_pages(layer), self.table, self.lengths, rows=rows, scale=scale, k_scale=k_scale,
                                v_scale=v_scale, out=out, lse=lse, status=self.status, stream=stream)

    def fork(self, src, dst, stream=None):
        """Each dst[i], an empty sequence, gets the tokens of src[i] and shares its pages (int32 [n] both; one source may be named many times). A pair
        that is out of range, or whose destination is in use, was named before it or is a source of this call, is left out and sets the status."""
        n = self._request("src", src)
        if self._request("dst", dst) != n:
            raise ValueError("src and dst have the same length")
        self._at_most_all(n)
        with launch_on(self._device.index, stream):
            rc = self._native.fork(src.data_ptr(), dst.data_ptr(), n, current_stream_handle())
        if rc != 0:
            raise RuntimeError(f"kv_fork launch failed ({rc})")

    def free(self, seqs, stream=None):
        """Empties the sequences (int32 [n]); pages that nobody else holds are free then. Empty ones stay as they are, whoever is named twice is
        emptied once, numbers out of range set the status."""
        n = self._request("seqs", seqs)
        with launch_on(self._device.index, stream):
            rc = self._native.free(seqs.data_ptr(), n, current_stream_handle())
        if rc != 0:
            raise RuntimeError(f"kv_free launch failed ({rc})")

    def compact(self, stream=None):
        """Moves the n pages in use to the places 0 to n - 1: those behind go, in ascending order, into the free ones before. Tables and refs follow.
        Returns int32 [pages]: the new number of each page that was in use, -1 for the others."""
        with launch_on(self._device.index, stream):
            remap = torch.empty_like(self.refs)
            ws = remap.new_empty(self._native.compact_workspace() // 4)
            rc = self._native.compact(remap.data_ptr(), ws.data_ptr(), current_stream_handle())
        if rc != 0:
            raise RuntimeError(f"kv_compact launch failed ({rc})")
        return remap
