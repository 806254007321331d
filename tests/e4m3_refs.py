"""Plain implementations, in 64 bits, of the sequence cache in 8 bits: a code per element and a power of two per page, plane and head."""
from __future__ import annotations

import math

import numpy as np
import torch

PAGE, LOW, HIGH, TOP = 64, -112, 119, 448.0


def round_code(x: torch.Tensor) -> torch.Tensor:
    """float64 -> the nearest e4m3 value, ties to even; too large ones, and infinities, to +-448; NaN stays."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, TOP))) - 3)
    return (torch.round(x / step) * step).clamp(-TOP, TOP)


def exponent(rows: torch.Tensor) -> int:
    """Of one plane and head: the least e in the range under which every finite element lies within 448 * 2^e."""
    finite = rows[torch.isfinite(rows)].abs()
    amax = float(finite.max()) if finite.numel() else 0.0
    if amax == 0.0:
        return LOW
    m, k = math.frexp(amax)
    return min(max(k - 9 if m <= 0.875 else k - 8, LOW), HIGH)


def rotate(x: torch.Tensor, pos: torch.Tensor, inv_freq, rot_dim: int) -> torch.Tensor:
    """x float64 [T, heads, D]; split halves of the first rot_dim components."""
    if inv_freq is None:
        return x
    angle = pos.double()[:, None, None] * inv_freq.double()
    a, b = x[..., :rot_dim // 2], x[..., rot_dim // 2:rot_dim]
    return torch.cat((a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin(), x[..., rot_dim:]), -1)


def write(qkv, bias, cu_q, tok_pos, slots, inv_freq, rot_dim, n_heads, kv_heads, dim, codes, scales, table):
    """All on the CPU. codes float64 [pages, 2, kv_heads, 64, dim], scales float64 [pages, 2, kv_heads]: updated in place. Returns the queries and the
    new rows [T, 2, kv_heads, dim], both before rounding."""
    x = qkv[:, :(n_heads + 2 * kv_heads) * dim].double()
    if bias is not None:
        x = x + bias.double()
    x = x.view(len(x), n_heads + 2 * kv_heads, dim)
    turned = rotate(x[:, :n_heads + kv_heads], tok_pos, inv_freq, rot_dim)
    rows = torch.stack((turned[:, n_heads:], x[:, n_heads + kv_heads:]), 1)
    for s, slot in enumerate(slots):
        t = cu_q[s]
        while slot >= 0 and t < cu_q[s + 1]:
            pos = int(tok_pos[t])
            n, at, page = min(cu_q[s + 1] - t, PAGE - pos % PAGE), pos % PAGE, int(table[slot, pos // PAGE])
            for plane in range(2):
                for h in range(kv_heads):
                    e = exponent(rows[t:t + n, plane, h])
                    if at > 0:
                        before = int(math.log2(float(scales[page, plane, h])))
                        if e > before:
                            codes[page, plane, h, :at] = round_code(codes[page, plane, h, :at] * 2.0 ** (before - e))
                        e = max(e, before)
                    scales[page, plane, h] = 2.0 ** e
                    codes[page, plane, h, at:at + n] = round_code(rows[t:t + n, plane, h] * 2.0 ** -e)
            t += n
    return turned[:, :n_heads].reshape(len(x), -1), rows


def attend(q, cu_q, tok_pos, slots, values, table, n_heads, scale, window):
    """q [T, n_heads * dim]; values float64 [pages, 2, kv_heads, 64, dim] (codes times scales). Returns (output, sum of weights times |value|, largest
    sum of |q k| times scale over a row's keys), float64 [T, n_heads, dim], the last [T, n_heads, 1]."""
    kv_heads, dim = values.shape[2], values.shape[4]
    group = n_heads // kv_heads
    out = torch.zeros((len(q), n_heads, dim), dtype=torch.float64)
    size, far = torch.zeros_like(out), torch.zeros((len(q), n_heads, 1), dtype=torch.float64)
    for s, slot in enumerate(slots):
        for t in range(cu_q[s], cu_q[s + 1]):
            if slot < 0:
                continue
            p = int(tok_pos[t])
            lo = max(0, p - window + 1) if window > 0 else 0
            at = np.arange(lo, p + 1)
            pages = torch.from_numpy(np.asarray(table)[slot, at // PAGE].astype(np.int64))
            rows = values[pages, :, :, torch.from_numpy(at % PAGE)]                  # [keys, 2, kv heads, dim]
            for h in range(n_heads):
                k, v = rows[:, 0, h // group], rows[:, 1, h // group]
                x = q[t, h * dim:(h + 1) * dim].double()
                w = torch.softmax(k @ x * scale, 0)
                out[t, h], size[t, h] = w @ v, w @ v.abs()
                far[t, h] = float((k.abs() @ x.abs()).max()) * scale
    return out, size, far


def attend_tolerance(out, size, far, dtype):
    """How far a kernel's output may be from `attend`'s, element by element.
    A score is a sum of products whose operands float32 queries leave 2^-22 short (two float16 of 11 bits, the second one's rounding) and whose
    float32 sums lose at most 2^-23 of the sizes at each of some tens of additions: within 2^-17 * far. A weight is off by that much and by 2^-21 of the
    base-2 exponential; rounded to float16 by 2^-11 more for bfloat16 outputs, by 2^-22 for float32. The weights' error counts twice, in the sum of
    values and in the sum of weights. The sums in float32, of up to some thousands of tiles, lose 2^-18 of the sizes."""
    weight = 2.0 ** -17 * far + 2.0 ** -18 + (2.0 ** -11 if dtype == torch.bfloat16 else 2.0 ** -22)
    return torch.finfo(dtype).eps / 2 * out.abs() + 2 * weight * size + 1e-30
