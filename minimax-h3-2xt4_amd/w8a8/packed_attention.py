"""Attention of packed sequences of different lengths, causal or not.

The attention of the text encoder's block, whose projections tp_qwen3vl mirrors
(patches/tp_qwen3vl.py:259 takes its output), and of image encoders. The INT8
attention (int8_attention) takes equal lengths without a mask; this one the
prompts of several requests, or the images of an encoder, as they lie one behind
the other, in fp16 or bf16.
"""
from . import _abi, kernels


def packed_attention(q, k, v, starts, k_starts=None, *, causal=True, scale=None, out=None):
    """softmax(scale q . k) v of every sequence, [rows, heads, dim].

    q [rows, heads, dim], k and v [keys, kv_heads, dim], fp16 or bf16, head h
    with key head h // (heads / kv_heads); dim a multiple of 8 up to 256.
    starts int32 [sequences + 1], from 0: sequence b's queries are rows
    [starts[b], starts[b + 1]); k_starts the same of its keys (starts by
    default). causal: of nq queries and nk keys, query i sees the keys up to
    i + nk - nq (a prompt's next part behind its cached keys); a query that sees
    none gives 0, and what it does not see has no effect, infinities and NaNs
    included. A query whose scores are all -inf gives NaN; an infinite value that
    it sees gives an infinity or, where its weight is rounded to 0, NaN. scale: 1 / sqrt(dim) by default. out: to write into, its rows
    behind the last sequence staying as they are; a new output has zeros there.
    Inference only."""
    y = _abi.native().packed_attention(q, k, v, starts, k_starts, causal, scale, out)
    if y is not None:
        return y
    return kernels.packed_attention(q, k, v, starts, k_starts, causal=causal, scale=scale, out=out)
