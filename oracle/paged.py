"""CPU restatement, in 64 bits, of the operators around the paged KV cache (test infrastructure; see package docstring).

The reference has none of them, so the definitions here are the operators' own.  A ragged batch: rows
cu[b] .. cu[b+1]-1 are the last tokens of sequence b, whose length with them is lens[b]; row t is at position
lens[b] - cu[b+1] + t.  Page p of sequence b is pool page table[b, p]; a page holds 64 rows.
"""

from __future__ import annotations

import torch

PAGE = 64


def norm_rope(x, weight, positions, inv_freq, eps: float, interleaved: bool):
    """x [n, heads, D] at positions [n]; returns (result, the rows' sizes that its rounding errors scale with), fp64."""
    y = x.double()
    if weight is not None:
        y = y / torch.sqrt(y.pow(2).mean(-1, keepdim=True) + eps) * weight.double()
    half = inv_freq.shape[0]
    a = positions.double()[:, None, None] * inv_freq.double()
    if interleaved:
        first, second = slice(0, 2 * half, 2), slice(1, 2 * half, 2)
    else:
        first, second = slice(0, half), slice(half, 2 * half)
    out, size = y.clone(), y.abs().clone()
    out[..., first] = y[..., first] * a.cos() - y[..., second] * a.sin()
    out[..., second] = y[..., second] * a.cos() + y[..., first] * a.sin()
    size[..., first] = size[..., second] = y[..., first].abs() + y[..., second].abs()
    return out, size


def positions_of(cu, lens):
    """(row, sequence, position) of every row of the batch."""
    return [(t, b, lens[b] - cu[b + 1] + t) for b in range(len(lens)) for t in range(cu[b], cu[b + 1])]


def attn_paged(q, k_pages, v_pages, table, cu, lens, scale: float):
    """q [T, Hq, D]; returns fp64 [T, Hq, D] (rows of no sequence NaN), sum_j w_j |v_j| and max_j scale * sum |q_i k_ji|."""
    T, Hq, D = q.shape
    Hkv = k_pages.shape[1]
    group = Hq // Hkv
    out = torch.full((T, Hq, D), float("nan"), dtype=torch.float64, device=q.device)
    spread, score = torch.zeros_like(out), 0.0
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        used = max(0, min(length, table.shape[1] * PAGE))
        pages = table[b, :(used + PAGE - 1) // PAGE].long()
        k = k_pages[pages].transpose(1, 2).reshape(-1, Hkv, D)[:used].double()
        v = v_pages[pages].transpose(1, 2).reshape(-1, Hkv, D)[:used].double()
        pos = length - n + torch.arange(n, device=q.device)
        sees = torch.arange(used, device=q.device)[None] <= pos[:, None]
        for h in range(Hq):
            qh, kh, vh = q[cu[b]:cu[b + 1], h].double(), k[:, h // group], v[:, h // group]
            x = (qh @ kh.T * scale).masked_fill(~sees, float("-inf"))
            w = torch.softmax(x, -1) if used else x
            w = torch.where(sees.any(-1, keepdim=True), w, torch.zeros_like(w))
            out[cu[b]:cu[b + 1], h] = w @ vh
            spread[cu[b]:cu[b + 1], h] = w @ vh.abs()
            if used:
                score = max(score, (qh.abs() @ kh.abs().T).max().item() * scale)
    return out, spread, score
