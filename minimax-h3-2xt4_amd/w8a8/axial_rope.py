"""Rotary positions with several axes (time, height, width) for images and video.

The reference is handed rotation matrices (patches/tp_dit.py:296-309 and
tilelang_fp32_rms_rope.py:45-66 take freqs [1, S, 1, half, 2, 2]); here they
come from the rows' positions: ``rotate`` turns Q and K directly, with the
per-head RMS norm where the block has one, and ``freqs`` writes the matrices
that rms_rope.execute and the QKV projection's epilogue read.

A table of turns is two vectors over the pairs of a head: inv_freq (fp64
angle of one step) and axis (which coordinate of a row's position turns the
pair). ``ladder`` builds the usual ones.
"""
import torch

from . import _abi, kernels


def ladder(sections, theta=10000.0, *, shared=False, interleaved=False, device=None):
    """(inv_freq fp64 [pairs], axis int32 [pairs]) for sections[a] pairs of axis a.

    Pairs of axis a are a run of sections[a] in the order of the axes, each
    run a geometric ladder of its own, theta ** (-j / sections[a]); with
    shared one ladder theta ** (-p / pairs) goes over all pairs instead.
    interleaved (with shared): the axes take pairs in turn, a, a + n, a + 2 n,
    .. for n axes, until an axis has its sections; what is left is axis 0's.
    """
    sections = [int(s) for s in sections]
    pairs, n = sum(sections), len(sections)
    if not sections or min(sections) < 0 or not 1 <= pairs <= 128 or n > 16:
        raise ValueError('1 to 16 sections of at most 128 pairs in all required')
    if interleaved and not shared:
        raise ValueError('interleaved axes share one ladder')
    if interleaved:
        axis = [p % n if p < n * sections[p % n] else 0 for p in range(pairs)]
        if any(axis.count(a) != sections[a] for a in range(n)):
            raise ValueError('the sections cannot be interleaved: an axis runs out of pairs before the end')
    else:
        axis = [a for a in range(n) for _ in range(sections[a])]
    if shared:
        inv = [float(theta) ** (-p / pairs) for p in range(pairs)]
    else:
        inv = [float(theta) ** (-j / s) for s in sections for j in range(s)]
    return (torch.tensor(inv, dtype=torch.float64, device=device),
            torch.tensor(axis, dtype=torch.int32, device=device))


def grid_positions(frames, height, width, *, start=(0, 0, 0), device=None):
    """int32 [frames * height * width, 3] positions (time, height, width) of a
    clip's patches in row order, from ``start``."""
    t, h, w = (torch.arange(s, s + n, dtype=torch.int32, device=device)
               for s, n in zip(start, (frames, height, width)))
    return torch.stack(torch.meshgrid(t, h, w, indexing='ij'), -1).reshape(-1, 3)


def rotate(q, k, positions, inv_freq, axis, *, pairing='half', q_gain=None, k_gain=None, eps=1e-6, out=None):
    """q [rows, heads, dim] and k [rows, k_heads, dim] (or None) turned by
    their rows' positions [rows, axes]; see kernels.axial_rope. pairing:
    'half' (p with p + pairs) or 'adjacent' (2 p with 2 p + 1). Inference only."""
    if pairing not in ('half', 'adjacent'):
        raise ValueError('pairing must be half or adjacent')
    q_out, k_out = out if out is not None else (None, None)
    r = _abi.native().axial_rope(q, k, positions, inv_freq, axis, pairing == 'adjacent', q_gain, k_gain, eps, q_out,
                                 k_out)
    if r is not None:
        return r
    return kernels.axial_rope(q, k, positions, inv_freq, axis, adjacent=pairing == 'adjacent', q_gain=q_gain,
                              k_gain=k_gain, eps=eps, out=out)


def freqs(positions, inv_freq, axis, *, dtype=torch.float16):
    """(1, rows, 1, pairs, 2, 2) rotation matrices of the positions, the
    layout of the reference's freqs argument."""
    f = kernels.axial_freqs(positions, inv_freq, axis, dtype=dtype)
    return f.view(1, f.shape[0], 1, f.shape[1], 2, 2)


def freqs_pairs(positions, inv_freq, axis, *, dtype=torch.float16):
    """rms_rope.pack_freqs(freqs(...)) without the matrices in between."""
    return kernels.axial_freqs(positions, inv_freq, axis, dtype=dtype, pairs_layout=True)
