"""A serving step's operators restated on the CPU in 64 bits (test infrastructure)."""

import numpy as np
import torch


def reserve(stack, count, tables, lens, new, block_size, max_tokens):
    """Sequence after sequence, as a host allocator does it: (tables, starts,
    slots, positions, lens, count, status)."""
    tables, width = tables.copy(), tables.shape[1]
    lens, new = [int(c) for c in lens], [int(n) for n in new]
    slots, positions = np.full(max_tokens, -1, np.int64), np.zeros(max_tokens, np.int32)
    starts = np.zeros(len(lens) + 1, np.int32)
    status = 0
    if any(c < 0 for c in lens) or any(n < 0 for n in new) or not 0 <= count <= len(stack):
        status = 4
    elif any(c + n > width * block_size for c, n in zip(lens, new)):
        status = 2
    elif sum(new) > max_tokens:
        status = 3
    elif sum(-(-(c + n) // block_size) + (-c // block_size) for c, n in zip(lens, new)) > count:
        status = 1
    if status:
        return tables, starts, slots, positions, np.array(lens), count, status
    left = [int(i) for i in stack[:count]]
    for b, (c, n) in enumerate(zip(lens, new)):
        for j in range(-(-c // block_size), -(-(c + n) // block_size)):
            tables[b, j] = left.pop()
        t = starts[b]
        for p in range(c, c + n):
            slots[t] = int(tables[b, p // block_size]) * block_size + p % block_size
            positions[t] = p
            t += 1
        starts[b + 1] = t
    return tables, starts, slots, positions, np.array([c + n for c, n in zip(lens, new)]), len(left), 0


def release(stack, count, tables, lens, finished, block_size):
    """(stack, lens, count, status)."""
    stack, lens = stack.copy(), np.array(lens)
    blocks = [-(-int(c) // block_size) if f else 0 for c, f in zip(lens, finished)]
    if any(f and c < 0 for c, f in zip(lens, finished)) or not 0 <= count <= len(stack):
        return stack, lens, count, 4
    if any(n > tables.shape[1] for n in blocks):
        return stack, lens, count, 2
    if sum(blocks) > len(stack) - count:
        return stack, lens, count, 1
    for b, n in enumerate(blocks):
        stack[count : count + n] = tables[b, :n]
        count += n
        lens[b] = 0 if finished[b] else lens[b]
    return stack, lens, count, 0


def rope(x, positions, freq, factor, interleaved):
    """x [T, H, D] float64 numpy, rotated."""
    y = x.copy()
    half = len(freq)
    angle = positions.astype(np.float64)[:, None] * freq[None, :]
    c, s = np.cos(angle)[:, None] * factor, np.sin(angle)[:, None] * factor
    first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved \
        else (slice(0, half), slice(half, 2 * half))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * c - b * s, b * c + a * s
    return y


def extend(q, k, v, length, *, scale, softcap=0.0, slopes=None, window=0, prefix=0, eps_dot=2.0**-24, eps_p=0.0,
           eps_tanh=2.0**-20):
    """One sequence's new tokens q [n, H, D] against its keys k, v [c, H_kv, D]
    (float64 tensors on the CPU), and how far a kernel that sums in float32 may
    be off: (out, bound), both [n, H, D].

    A score of D products is off by at most (D + 4) eps_dot sum |q_i k_i| scale
    (every product and partial sum rounded once); the cap's tanh is off by
    eps_tanh times the cap; the distance term and each later sum are rounded
    once.  A weight exp(s) then is off by the score's error d relatively (e^d - 1
    <= 2 d for d <= 1), the same for the sum it is divided by, and by 2^-22 for
    the exponential; eps_p for a rounding of the weights; n terms summed add
    n 2^-24."""
    n, heads, dim = q.shape
    group = heads // k.shape[1]
    out, bound = torch.zeros_like(q), torch.zeros_like(q)
    if n == 0 or length == 0:
        return out, bound
    j, p = torch.arange(length)[None], torch.arange(length - n, length)[:, None]
    ok = (j <= p) | (j < prefix)
    if window:
        ok &= j > p - window
    seen = ok.sum(-1, keepdim=True)
    for h in range(heads):
        kk, vv = k[:, h // group], v[:, h // group]
        s = q[:, h] @ kk.T * scale
        d = (dim + 4) * eps_dot * (q[:, h].abs() @ kk.abs().T) * abs(scale)
        if softcap:
            s = softcap * torch.tanh(s / softcap)
            d = d + softcap * eps_tanh
        if slopes is not None:
            far = float(slopes[h]) * (p - j).abs().double()
            s = s - far
            d = d + 3 * eps_dot * far
        d = torch.where(ok, d + 4 * eps_dot * s.abs(), 0.0)
        w = torch.softmax(s.masked_fill(~ok, float("-inf")), dim=-1)
        w = torch.where(seen > 0, w, 0.0)
        out[:, h] = w @ vv
        rel = 4 * d.amax(-1, keepdim=True) + 2.0**-21 + eps_p + (seen + 16) * 2.0**-24
        bound[:, h] = rel * (w @ vv.abs())
    return out, bound
