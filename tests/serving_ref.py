"""Plain float64 forms of the serving operators, on the CPU, written from their
definitions, and the error that float32 kernels with one rounding of the output
(and, on the tensor cores, of the probabilities) may add."""

import math

import torch

# half a step of each type, relative to the value
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def visible(n, m, window, sinks):
    """[n, m]: query i stands at m - n + i."""
    p = torch.arange(m - n, m)[:, None]
    j = torch.arange(m)[None, :]
    sees = j <= p
    if window is not None:
        sees &= (j > p - window) | (j < sinks)
    return sees


def attention(q, k, v, sees, scale):
    """softmax over the visible keys, and its error bound per element.

    q [h, n, d], k [h, m, d], v [h, m, dv] float64, sees [n, m].  Returns out and
    the two magnitudes that errors scale with: spread = sum_j p_j |v_j| (every
    relative error of a probability or of the sums is at most that times it) and
    score = max_j scale sum_c |q_c k_jc| (a float32 dot product of d terms is off
    by at most (d + 2) 2^-24 of that)."""
    x = torch.einsum("hnd,hmd->hnm", q, k) * scale
    x = torch.where(sees, x, torch.full((), -math.inf, dtype=torch.float64))
    top = x.amax(-1, keepdim=True) if x.shape[-1] else x.new_full(x.shape[:-1] + (1,), -math.inf)
    w = torch.exp(x - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    w = torch.where(sees, w, torch.zeros_like(w))
    total = w.sum(-1, keepdim=True)
    w = w / torch.where(total > 0, total, torch.ones_like(total))
    vz = torch.where(sees.any(0)[None, :, None], v, torch.zeros_like(v))
    kz = torch.where(sees.any(0)[None, :, None], k, torch.zeros_like(k))
    size = torch.einsum("hnd,hmd->hnm", q.abs(), kz.abs()) * abs(scale)
    size = torch.where(sees, size, torch.zeros_like(size))
    score = size.amax(-1, keepdim=True) if size.shape[-1] else size.new_zeros(size.shape[:-1] + (1,))
    return torch.einsum("hnm,hmd->hnd", w, vz), torch.einsum("hnm,hmd->hnd", w, vz.abs()), score


def attention_bound(ref, spread, score, dim, keys, dtype, p_half):
    """Half a step of the output's type; of each probability: p_half for its
    rounding, twice the score's float32 error (numerator and sum both move), 4
    2^-22 for exp and the scaled query, and 2^-23 for each of the at most `keys`
    additions of the running sums.  fp16 outputs below 2^-14 have a fixed step of
    2^-24, bf16 and fp32 ones no such floor that matters here."""
    rel = p_half + 2 * (dim + 2) * 2.0 ** -24 * score + 4 * 2.0 ** -22 + keys * 2.0 ** -23
    return HALF[dtype] * (ref.abs() + rel * spread) + rel * spread + (2.0 ** -25 if dtype == torch.float16 else 1e-37)


def code_span(dtype):
    """How much larger the terms of a score over 4-bit codes are than |q k|, at most,
    for rows that are not far off zero.  A value is s c' + x, c' the code plus an
    offset, and both products are summed on their own.  Rows of roughly normal values
    of deviation 1 have s = 5 / 15 and mean |k| = 0.8: float32 takes c' = code - 8, so
    8 s + |x| <= 2.7 + 0.5 = 4 * 0.8; 16-bit types take c' = code + 16, so 31 s + |x| <=
    10.3 + 7.8 + 0.5 < 24 * 0.8."""
    return 4 if dtype == torch.float32 else 24


def assert_close(got, ref, bound):
    got = got.double().cpu()
    assert got.shape == ref.shape, (got.shape, ref.shape)
    assert torch.isfinite(got).all()
    over = ((got - ref).abs() - bound).max().item() if got.numel() else -1.0
    assert over <= 0, f"off by {over:.3e} more than the bound (largest error {(got - ref).abs().max().item():.3e})"


# ---------------------------------------------------------------- 4-bit rows

def padded(dim):
    return max(32, 1 << (dim - 1).bit_length())


def quantise(x):
    """Rows x [..., d] float64 -> codes (uint8), scale, least (float64 values of bfloat16)."""
    ok = torch.isfinite(x).all(-1, keepdim=True)
    xs = torch.where(torch.isfinite(x), x, torch.zeros_like(x))
    low, high = xs.amin(-1, keepdim=True), xs.amax(-1, keepdim=True)
    least = low.float().to(torch.bfloat16)
    scale = ((high - low) / 15.0).float().to(torch.bfloat16)
    ok &= torch.isfinite(least.float())
    nan = torch.full((), float("nan"), dtype=torch.float64)
    s, m = scale.double(), least.double()
    t = torch.where(s > 0, (xs - m) / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(xs))
    codes = torch.where(ok, t.round().clamp(0, 15), torch.zeros_like(t)).to(torch.uint8)
    return codes, torch.where(ok, s, nan), torch.where(ok, m, nan)


def value_of(codes, scale, least):
    """The float32 value a code stands for."""
    return (codes.double() * scale + least).float()


def k_rows(k_codes, slots, dim):
    """Codes [T, H, dim] of slots from k_codes [P, H, page, dp / 2]."""
    c = k_codes.cpu()
    page = c.shape[2]
    b = c[slots // page, :, slots % page].to(torch.int64)
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)[..., :dim].to(torch.uint8)


def v_rows(v_codes, slots, dim):
    c = v_codes.cpu()
    page = c.shape[2] * 4
    off = slots % page
    b = c[slots // page, :, off // 4, :, off % 4].to(torch.int64)
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)[..., :dim].to(torch.uint8)


def params(p, slots):
    c = p.cpu().double()
    page = c.shape[2]
    return c[slots // page, :, slots % page]


# ---------------------------------------------------------------- page plans

def plan(lengths, new, tables, free, count, page):
    """Token by token: (lengths, offsets, positions, slots, tables, free count)."""
    tables = [list(r) for r in tables]
    left, positions, slots, offsets = count, [], [], [0]
    for r, (have, add) in enumerate(zip(lengths, new)):
        for i in range(add):
            pos = have + i
            row = pos // page
            if row < len(tables[r]) and pos % page == 0:
                left -= 1
                tables[r][row] = free[left] if left >= 0 else -1
            entry = tables[r][row] if row < len(tables[r]) else -1
            positions.append(pos)
            slots.append(entry * page + pos % page if entry >= 0 else -1)
        offsets.append(offsets[-1] + add)
    return [a + b for a, b in zip(lengths, new)], offsets, positions, slots, tables, max(left, 0)


def rotary(x, positions, weight, freq, eps, interleaved):
    """x [T, H, d] float64 -> rotated rows."""
    d, half = x.shape[-1], freq.shape[0]
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    if weight is not None:
        y = y * weight.double()
    angle = positions.double()[:, None, None] * freq
    c, s = torch.cos(angle), torch.sin(angle)
    out = y.clone()
    ia = torch.arange(half) * 2 if interleaved else torch.arange(half)
    ib = ia + 1 if interleaved else ia + half
    out[..., ia] = y[..., ia] * c - y[..., ib] * s
    out[..., ib] = y[..., ib] * c + y[..., ia] * s
    return out


def rng(seed):
    g = torch.Generator()
    g.manual_seed(seed)
    return g

