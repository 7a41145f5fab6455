"""Keys and values of many sequences in pages, and one new token's attention over them.

No counterpart in the reference, whose text encoder's block
(patches/tp_qwen3vl.py:259-281) runs whole prompts and keeps nothing. A cache holds keys and values
16-bit as they are, or as INT8 codes with one FP32 scale per token and head
(the framework's row quantizer), half the bytes of every token's attention.

Key j of sequence b lies in page page_table[b, j // page_size] at token
j % page_size. The table and the lengths live on the GPU and nothing here reads
them back, so a step may be captured into a graph and replayed with other
contents. A table entry outside of the cache (-1, say) is a page that is not
there: nothing is written to it, zeros are read from it, and its keys take no
part in an attention.
"""
from dataclasses import dataclass

import torch

from . import _abi, kernels


@dataclass(frozen=True)
class KVCache:
    """k and v [pages, heads, page_size, dim]: float16, bfloat16 or int8 codes
    with k_scale and v_scale fp32 [pages, heads, page_size]. k and v may be views
    of larger buffers, both with the same strides (channels contiguous, the
    others multiples of 8 elements); so may the scales (tokens contiguous, the
    others multiples of 4). To be written to, no two places may share memory."""
    k: torch.Tensor
    v: torch.Tensor
    k_scale: torch.Tensor = None
    v_scale: torch.Tensor = None

    def __post_init__(self):
        k, v = self.k, self.v
        if k.ndim != 4 or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
            raise ValueError('k and v must be [pages, heads, page_size, dim] of the same shape, type and strides')
        if k.dtype not in (torch.float16, torch.bfloat16, torch.int8):
            raise ValueError('k and v must be float16, bfloat16 or int8')
        pages, heads, page_size, dim = k.shape
        if pages == 0 or heads == 0 or page_size == 0 or page_size % 16 or page_size > 4096:
            raise ValueError('a cache has pages and heads, and pages of 16 to 4096 tokens, a multiple of 16')
        if not 8 <= dim <= 256 or dim % 8:
            raise ValueError('dim must be a multiple of 8, 8 to 256')
        if k.stride(3) != 1 or any(s % 8 for s in k.stride()[:3]) or k.stride(2) < dim or \
                any(t.data_ptr() % 16 for t in (k, v)):
            raise ValueError('k and v must have contiguous channels, 16-byte alignment and strides of 8 elements')
        scales = (self.k_scale, self.v_scale)
        if not self.codes:
            if any(t is not None for t in scales):
                raise ValueError('scales go with int8 codes')
            return
        for t in scales:
            if t is None or t.dtype != torch.float32 or tuple(t.shape) != (pages, heads, page_size):
                raise ValueError('codes need k_scale and v_scale, float32 [pages, heads, page_size]')
            if t.stride(2) != 1 or any(s % 4 for s in t.stride()[:2]) or t.data_ptr() % 16 or \
                    t.stride() != scales[0].stride():
                raise ValueError('scales must have the same strides, contiguous tokens and 16-byte alignment')

    @classmethod
    def allocate(cls, pages, page_size, heads, dim, *, dtype=torch.float16, device=None):
        """A cache of zeros; dtype float16, bfloat16 or int8 (codes)."""
        dev = torch.device(device) if device is not None else torch.device('cuda', 0)
        k, v = (torch.zeros((pages, heads, page_size, dim), dtype=dtype, device=dev) for _ in range(2))
        if dtype != torch.int8:
            return cls(k, v)
        return cls(k, v, *(torch.zeros((pages, heads, page_size), dtype=torch.float32, device=dev) for _ in range(2)))

    @property
    def codes(self):
        return self.k.dtype == torch.int8

    @property
    def heads(self):
        return self.k.shape[1]

    @property
    def page_size(self):
        return self.k.shape[2]

    @property
    def dim(self):
        return self.k.shape[3]


def write(cache, k, v, page_table, lengths, starts=None):
    """Write new keys and values [rows, heads, dim] (fp16 or bf16).

    page_table int32 [sequences, width]; lengths int32 [sequences]: each
    sequence's keys with the new ones; starts int32 [sequences + 1], from 0:
    sequence b's new rows are [starts[b], starts[b + 1]), its last keys in
    order. Without starts every sequence has one row. Rows behind the last
    sequence, and keys outside of the table, are not written. If two rows name
    one place (a page that is listed twice), either may remain, or a mixture.
    Codes are those of the activation quantizer; a row that holds an infinity
    or a NaN gets the scale NaN."""
    if not _abi.native().cache_write(cache.k, cache.v, cache.k_scale, cache.v_scale, k, v, page_table, lengths, starts):
        kernels.cache_write(cache, k, v, page_table, lengths, starts)


def read(cache, page_table, starts, rows, *, dtype=None, out=None):
    """The first keys and values of every sequence as packed rows (k, v), each
    [rows, heads, dim]: rows [starts[b], starts[b + 1]) take sequence b's keys 0,
    1, ... (zeros where its table has no page). dtype: fp16 or bf16 of what codes
    stand for (a 16-bit cache gives its own). out: (k, v) to write into, whose
    rows behind the last sequence stay as they are; new outputs have zeros
    there. What packed_attention takes for a prompt's next part."""
    if out is None:
        r = _abi.native().cache_read(cache.k, cache.v, cache.k_scale, cache.v_scale, page_table, starts, rows, dtype)
        if r is not None:
            return r
    return kernels.cache_read(cache, page_table, starts, rows, dtype=dtype, out=out)


def attend(q, cache, page_table, lengths, *, scale=None, out=None):
    """Attention of one new token of every sequence, q [sequences, heads, dim],
    over the first lengths[b] keys of its pages (the new token's own included,
    once written): softmax(scale q . k) v, query head h with the cache's head
    h // (heads / cache.heads). scale: 1 / sqrt(dim) by default. A sequence
    without keys gives 0, one whose scores are all -inf NaN, an infinite value
    an infinity or, where its weight is rounded to 0, NaN. Inference only."""
    y = _abi.native().cache_attend(cache.k, cache.v, cache.k_scale, cache.v_scale, q, page_table, lengths, scale, out)
    if y is not None:
        return y
    return kernels.cache_attend(q, cache, page_table, lengths, scale=scale, out=out)
