"""The attention operators from their definitions, in 64 bits, one sequence and one head at a time (torch on the CPU)."""
import math

import torch

HALF_STEP = {torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def rotary(x, cos, sin, positions, sections, interleaved):
    """x [T, H, D]; returns (out, magnitude): the result and |a c| + |b s| of every element."""
    x, cos, sin = x.double(), cos.double(), sin.double()
    positions = positions.reshape(len(sections), -1)
    pairs = cos.shape[1]
    out, size = x.clone(), torch.zeros_like(x)
    pair = 0
    for axis, count in enumerate(sections):
        for _ in range(count):
            c, s = cos[positions[axis], pair][:, None], sin[positions[axis], pair][:, None]
            i, j = (2 * pair, 2 * pair + 1) if interleaved else (pair, pair + pairs)
            a, b = x[..., i], x[..., j]
            out[..., i], out[..., j] = a * c - b * s, b * c + a * s
            size[..., i] = (a * c).abs() + (b * s).abs()
            size[..., j] = (b * c).abs() + (a * s).abs()
            pair += 1
    assert pair == pairs
    return out, size


def round_half_even(x):
    return torch.round(x)


def quantize(x, block, zero_points):
    """Rows [..., D] -> (codes, fp16 scales, zero points), all per the header's formulas."""
    b = x.double().unflatten(-1, (-1, block))
    clean = torch.nan_to_num(b, nan=0.0, posinf=math.inf, neginf=-math.inf)
    lo, hi = clean.amin(-1).clamp(max=0), clean.amax(-1).clamp(min=0)
    step = (hi - lo) / 15 if zero_points else torch.maximum(hi / 7, -lo / 8)
    scale = step.float().clamp(max=65504).half()
    s = scale.double()
    safe = torch.where(s > 0, s, torch.ones_like(s))
    zero = torch.round(-lo / safe).clamp(0, 15) * (s > 0) if zero_points else torch.full_like(s, 8)
    code = (torch.round(clean / safe[..., None]).clamp(-32, 32) * (s > 0)[..., None] + zero[..., None]).clamp(0, 15)
    return code.flatten(-2).to(torch.uint8), scale, zero.to(torch.uint8)


def dequantize(code, scale, zero):
    b = code.double().unflatten(-1, (scale.shape[-1], -1))
    return ((b - zero.double()[..., None]) * scale.double()[..., None]).flatten(-2)


def row_sizes(code, scale, zero):
    """code * s + zero * s of every element."""
    b = code.double().unflatten(-1, (scale.shape[-1], -1))
    return ((b + zero.double()[..., None]) * scale.double()[..., None]).flatten(-2)


def unpack(packed, n):
    return torch.stack((packed & 15, packed >> 4), -1).flatten(-2)[..., :n]


def attend(q, k, v, scale, causal, window, p_error, q_error=0.0, k_size=None):
    """One head: q [N, D], k and v [L, D] in 64 bits; k_size: the size of what is summed where that is not |k| (a 4-bit key
    is summed as code * s and zero * s apart).  Returns (out, bound): the result and the error that f32 arithmetic
    may add, from the sizes of what is summed:
      a score is a sum of D products, each rounded once and added once: (D + 3) 2^-23 of sum |q||k| scale;
      a weight 2^x carries twice that (numerator and denominator), 2^-22 of the exponential itself, and p_error of its
      rounding; sums over L keys add L 2^-23 of sum p |v|."""
    n, total, d = q.shape[0], k.shape[0], q.shape[1]
    if total == 0 or n == 0:
        return torch.zeros(n, d, dtype=torch.float64), torch.zeros(n, d, dtype=torch.float64)
    at = torch.arange(total - n, total)[:, None]
    key = torch.arange(total)[None]
    keep = torch.ones(n, total, dtype=torch.bool)
    if causal:
        keep &= key <= at
    if window:
        keep &= key > at - window
    out, bound = torch.zeros(n, d, dtype=torch.float64), torch.zeros(n, d, dtype=torch.float64)
    k_size = k.abs() if k_size is None else k_size
    for i in range(n):
        j = keep[i].nonzero().flatten()
        if j.numel() == 0:
            continue
        x = (k[j] @ q[i]) * scale
        p = torch.softmax(x, 0)
        out[i] = p @ v[j]
        size = ((k_size[j] @ q[i].abs()) * abs(scale)).max().item()
        delta = size * ((d + 3) * 2.0 ** -23 + q_error) + 2.0 ** -22
        bound[i] = (p @ v[j].abs()) * (2 * delta + p_error + (j.numel() + 8) * 2.0 ** -23)
    return out, bound


def check(got, want, bound, what):
    """|got - want| within the bound plus half a step of the output's type; subnormal fp16 results have a fixed step."""
    got64 = got.double().cpu()
    tol = bound + HALF_STEP[got.dtype] * (want.abs() + bound) + (2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -149)
    bad = ~((got64 - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst {float(((got64 - want).abs() / tol).max()):.3g} of the "
                           f"bound at {[int(v) for v in bad.nonzero()[0]]}: {float(got64[tuple(bad.nonzero()[0])])} for "
                           f"{float(want[tuple(bad.nonzero()[0])])}")
