"""The residual stream between two blocks: update, norms and quantization in one pass.

The reference updates the stream with gated_add / residual_add
(patches/h3_tensor_flow.py:130-152) and then normalizes it for the next
projection (:134-142). Here the update rides in a GEMM's epilogue where it
can; where it cannot (after the SUM exchange of rank partials, or when the
branch has an RMS norm of its own, which the reference's blocks have not),
residual_norm does both in one kernel, down to the next projection's INT8
codes.
"""
from . import _abi, kernels
from .h3_tensor_flow import _norm_args


def residual_norm(x, branch, *, weight=None, eps=None, post_weight=None, post_eps=None, gate=None, shift=None,
                  scale=None, labels=None, residual_scale=1.0, branch_scale=1.0, quantize=False, convrot=True,
                  round_rotated=True, want_normalized=False, signs=None, out=None):
    """kernels.residual_norm: x' = x * residual_scale + norm(branch) *
    branch_scale * gate[label], then norm_quantize of x'. Inference only.

    A branch that a norm follows cannot carry the residual divisor c in its
    projection's weight scale: pass branch_scale=1/c. ``out=x`` updates the
    stream in place."""
    if signs is None:
        r = _abi.native().residual_norm(x, branch, weight, eps, post_weight, post_eps, gate, shift, scale, labels,
                                        residual_scale, branch_scale, quantize, convrot, round_rotated,
                                        want_normalized, out)
        if r is not None:
            return r
    return kernels.residual_norm(x, branch, weight=weight, eps=eps, post_weight=post_weight, post_eps=post_eps,
                                 gate=gate, shift=shift, scale=scale, labels=labels, residual_scale=residual_scale,
                                 branch_scale=branch_scale, quantize=quantize, convrot=convrot,
                                 round_rotated=round_rotated, want_normalized=want_normalized, signs=signs, out=out)


def update_and_prepare(x, branch, gate, segments, norm, shift, scale, *, post_norm=None, branch_scale=1.0,
                       convrot=True, out=None):
    """One block's update and the next sublayer's activation: (x', (codes,
    row_scale)), the codes being modulated_norm_quantize(norm, x', shift,
    scale, segments)'s. gate, shift and scale are [R, hidden] modulation
    tables, segments [(a, b, row)] tile the rows, norm is the next sublayer's
    and post_norm the branch's own RMSNorm (or None). Inference only: the norms'
    weights are taken as constants, any other input that requires a gradient is
    refused."""
    if any(t is None or t.ndim != 2 for t in (gate, shift, scale)):
        raise ValueError('gate, shift and scale must be tables [R, hidden]')
    weight, eps, labels, shift, scale = _norm_args(norm, x, shift, scale, segments)
    if any(row >= gate.shape[0] for _, _, row in segments):
        raise ValueError('segments name a row that the gate table has not')
    post_weight = post_eps = None
    if post_norm is not None:
        post_weight, post_eps, _, _, _ = _norm_args(post_norm, x, None, None, None)
    r = kernels.residual_norm(x, branch, weight=weight, eps=eps, post_weight=post_weight, post_eps=post_eps,
                              gate=gate.float(), shift=shift, scale=scale, labels=labels,
                              branch_scale=branch_scale, quantize=True, convrot=convrot, out=out)
    return r['x'], (r['q'], r['scale'])
