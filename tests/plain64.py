"""Plain 64-bit restatements of the attention calls and of the multi-axis rotation, and the error a 16-bit kernel may
make against them.  Written from the formulas, request by request."""
from __future__ import annotations

import math

import torch

# Half a rounding step, relative to the value.
HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def kv_lens(kv_indptr, last, page_size):
    n = [int(kv_indptr[b + 1] - kv_indptr[b]) for b in range(len(kv_indptr) - 1)]
    return [(c - 1) * page_size + int(last[b]) if c > 0 else 0 for b, c in enumerate(n)]


def attend(q, pool, qo_indptr, kv_indptr, kv_indices, last, sm_scale=None, causal=True, window_left=-1, first_tokens=0,
           sinks=None):
    """(out, spread, lse) in 64 bits: softmax over the visible keys, spread = the same softmax over |v|, which scales
    every error that a rounding of the probabilities makes.  A query that sees nothing gives zeros and -inf."""
    n, hq, d = q.shape
    page_size, hkv = pool.shape[2], pool.shape[3]
    group = hq // hkv
    scale = sm_scale if sm_scale is not None else 1.0 / math.sqrt(d)
    out = torch.zeros((n, hq, d), dtype=torch.float64)
    spread = torch.zeros((n, hq, d), dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    lens = kv_lens(kv_indptr, last, page_size)
    for b, kv in enumerate(lens):
        r0, r1 = int(qo_indptr[b]), int(qo_indptr[b + 1])
        if kv == 0 or r1 == r0:
            continue
        t = torch.arange(kv)
        pages = torch.as_tensor(kv_indices[int(kv_indptr[b]): int(kv_indptr[b + 1])]).long().clamp_min(0)
        k = pool[pages, 0].reshape(-1, hkv, d)[:kv].double()
        v = pool[pages, 1].reshape(-1, hkv, d)[:kv].double()
        pos = torch.arange(kv - (r1 - r0), kv)[:, None]
        see = (t[None] <= pos) if causal else torch.ones((r1 - r0, kv), dtype=torch.bool)
        if window_left >= 0:
            see &= (t[None] >= pos - window_left) | (t[None] < first_tokens)
        used = see.any(0)  # what nobody sees may hold anything
        k, v = torch.where(used[:, None, None], k, 0.0), torch.where(used[:, None, None], v, 0.0)
        for h in range(hq):
            s = (q[r0:r1, h].double() @ k[:, h // group].T) * scale
            s = s.masked_fill(~see, -math.inf)
            top = s.amax(1, keepdim=True)
            alive = torch.isfinite(top)
            p = torch.where(see, (s - torch.where(alive, top, 0.0)).exp(), 0.0)
            total = p.sum(1, keepdim=True)
            if sinks is not None:
                total = total + torch.where(alive, (float(sinks[h]) - top).exp(), 0.0)
            w = torch.where(alive, p / total.clamp_min(1e-300), 0.0)
            out[r0:r1, h] = w @ v[:, h // group]
            spread[r0:r1, h] = w @ v[:, h // group].abs()
            lse[r0:r1, h] = torch.where(alive, top + total.clamp_min(1e-300).log(), -math.inf)[:, 0]
    return out, spread, lse


def attention_tolerance(dtype, out, spread, keys, q_k):
    """What a kernel that accumulates in 32 bits may be off by, per element.

    Output rounding: half a step of |out|.  16-bit kernels also round the probabilities before they meet v: half a
    step of the spread.  A score is a 32-bit sum of d <= 256 products whose magnitudes add up to `q_k` (scaled):
    with one rounding (or truncation, 2^-23) per term it is off by at most d * 2^-23 * q_k, an exponential's argument
    by 2^-23 of itself more; numerator and denominator both carry that.  The sums over `keys` probabilities add at most
    keys * 2^-24 of themselves."""
    half = HALF_STEP[dtype]
    # Below the smallest normal number the steps stay tiny * eps: half of one, for the output and for each of the
    # probabilities (their sum is at least 1 in the units of the running maximum, |v| at most 8 here).
    under = half * torch.finfo(dtype).tiny * (1 + 8 * keys)
    fuzz = 2 * (256 + 8) * 2.0 ** -23 * q_k + 2 * (keys + 64) * 2.0 ** -24
    probability = half if dtype != torch.float32 else 0.0
    return half * out.abs() + (probability + fuzz) * spread + under


def score_magnitude(q, pool, scale):
    """A bound of sum |q_i k_i| * scale over all heads and keys (finite ones): the largest row norms' product."""
    k = pool[:, 0].float()
    k = torch.where(torch.isfinite(k), k, torch.zeros_like(k))
    return float(q.float().norm(dim=-1).max() * k.norm(dim=-1).max()) * scale


def check_attention(got, got_lse, q, pool, ref, scale=None, keys=None):
    out, spread, lse = ref
    s = scale if scale is not None else 1.0 / math.sqrt(q.shape[-1])
    q_k = score_magnitude(q, pool, s)
    tol = attention_tolerance(q.dtype, out, spread, keys or 4096, q_k)
    diff = (got.cpu().double() - out).abs()
    assert torch.isfinite(got.cpu().float()).all()
    worst = (diff - tol).max().item() if diff.numel() else -1.0
    assert worst <= 0, f"{int((diff > tol).sum())} of {diff.numel()} elements off, worst by {worst:.3g}"
    if got_lse is not None:
        a, b = got_lse.cpu().double(), lse
        assert torch.equal(torch.isinf(a), torch.isinf(b))
        fin = torch.isfinite(b)
        # the score's own error, and the 32-bit value's half step
        bound = (256 + 8) * 2.0 ** -23 * q_k + 2.0 ** -22 * (1 + b[fin].abs()) + 2 * (keys or 4096) * 2.0 ** -24
        assert ((a[fin] - b[fin]).abs() <= bound).all()


def pair_axes(sections, cyclic):
    half, axes = sum(sections), len(sections)
    if cyclic:
        return [i % axes if i < axes * sections[i % axes] and i % axes > 0 else 0 for i in range(half)]
    return [a for a, n in enumerate(sections) for _ in range(n)]


def rotate_axes(x, pos, sections, cyclic, theta, interleave, scale=1.0, table=None):
    """x [n, heads, d] rotated in 64 bits; pos [axes, n]."""
    half = sum(sections)
    axis = torch.tensor(pair_axes(sections, cyclic))
    own = pos.long()[axis].T  # [n, half]
    if table is None:
        freq = torch.tensor([theta ** (-2.0 * i / (2 * half)) / scale for i in range(half)], dtype=torch.float64)
        cos, sin = (own.double() * freq).cos(), (own.double() * freq).sin()
    else:
        i = torch.arange(half)
        cos, sin = table[own, i].double(), table[own, half + i].double()
    cos, sin = cos[:, None], sin[:, None]
    out = x.double().clone()
    if interleave:
        a, b = x[..., 0: 2 * half: 2].double(), x[..., 1: 2 * half: 2].double()
        out[..., 0: 2 * half: 2], out[..., 1: 2 * half: 2] = a * cos - b * sin, a * sin + b * cos
    else:
        a, b = x[..., :half].double(), x[..., half: 2 * half].double()
        out[..., :half], out[..., half: 2 * half] = a * cos - b * sin, a * sin + b * cos
    size = out.abs().clone()
    mag = (a.abs() + b.abs())
    if interleave:
        size[..., 0: 2 * half: 2] = size[..., 1: 2 * half: 2] = mag
    else:
        size[..., :half] = size[..., half: 2 * half] = mag
    return out, size


def rotation_tolerance(dtype, out, size):
    """One rounding to the storage type, on top of 32-bit arithmetic: cos and sin are within 2 units of 2^-24 plus the
    angle's own 2^-27 turns, each product and the sum round once: less than 2^-21 of |a| + |b|.  Below the smallest
    normal number the type's steps stay tiny * eps (16-bit floats: 2^-24 under 2^-14), half of one of them is
    HALF_STEP * tiny."""
    return HALF_STEP[dtype] * (out.abs() + torch.finfo(dtype).tiny) + 2.0 ** -21 * size
