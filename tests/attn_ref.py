"""Plain 64-bit forms of the attention operators, on the CPU, with the error that a bf16 kernel may make.

Every function returns (value, bound) in float64. The bounds, with u = 2^-24 (fp32) and a bf16 output rounding
of half a step:

* norm and rotation of a head of D elements: the sum of squares is D/32 (at most 16) fmas and 5 adds of
  positive terms in fp32, so off by at most 21 u, its root by half of that; the mean, the reciprocal root, the
  weight's and the scale's products and the rotation's two operations add at most 8 u, the reduced angle pi u
  and the hardware sine and cosine 2^-21.2 = 7 u: below 2^-19 = 32 u of |y_i| + |y_j| of the pair.
* attention: each score is a sum of D exact products in fp32, off by at most D 2^-23 sum|q k|, the sum's
  running value being at most that; the exponential and the running rescaling add 2^-20 relative. A weight is
  rounded to bf16, p (1 + e) with |e| <= 2^-8. With the sum of the rounded weights below, the output is off by
  sum(p e (v - o)), at most 2^-8 (sum(p |v|) + |o|); with the sum of the weights as they were (chunks), by
  sum(p e v), which is less. The scores' error, of numerator and denominator, counts twice in sum(p |v|).
"""
import torch


def half_step(x: torch.Tensor) -> torch.Tensor:
    """Half a bf16 step at |x|."""
    e = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -126)))
    return 2.0 ** (e - 8)


def norm(x, weight, eps):
    x = x.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    return y if weight is None else y * weight.double()


def rotate(y, positions, inv_freq, rotary):
    """Pairs (i, i + rotary / 2) turned by position * inv_freq. Returns (value, |y_i| + |y_j|)."""
    h = rotary // 2
    a = positions.double()[:, None, None] * torch.tensor(inv_freq, dtype=torch.float64)
    c, s = torch.cos(a), torch.sin(a)
    lo, hi, rest = y[..., :h], y[..., h:rotary], y[..., rotary:]
    mag = lo.abs() + hi.abs()
    return (torch.cat([lo * c - hi * s, hi * c + lo * s, rest], -1), torch.cat([mag, mag, rest.abs()], -1))


def norm_rope(x, positions, inv_freq, rotary, weight, eps):
    v, mag = rotate(norm(x, weight, eps), positions, inv_freq, rotary)
    return v, half_step(v) + 2.0 ** -19 * mag


def tokens(q_offsets, kv_lens):
    """(row, sequence, position) of every row that belongs to a sequence."""
    out = []
    for b, n in enumerate(kv_lens):
        q0, q1 = q_offsets[b], q_offsets[b + 1]
        out += [(r, b, n - (q1 - q0) + r - q0) for r in range(q0, q1)]
    return out


def attention(q, k_pages, v_pages, q_offsets, kv_lens, table, scale, window):
    """q [rows, hq, D], pages [n, hk, page, D] (CPU). Rows of no sequence come back as NaN with bound NaN."""
    rows, hq, d = q.shape
    hk, page = k_pages.shape[1], k_pages.shape[2]
    out = torch.full((rows, hq, d), float("nan"), dtype=torch.float64)
    bound = torch.full_like(out, float("nan"))
    for b, n in enumerate(kv_lens):
        q0, q1 = q_offsets[b], q_offsets[b + 1]
        if q1 == q0:
            continue
        pos = torch.arange(n - (q1 - q0), n)[:, None]
        j = torch.arange(n)[None]
        seen = (j <= pos) & ((j > pos - window) if window else torch.ones_like(j, dtype=torch.bool))
        any_seen = seen.any(0)
        k = torch.zeros(n, hk, d, dtype=torch.float64)
        v = torch.zeros_like(k)
        for p in range(-(-n // page)):
            lo, hi = p * page, min(n, (p + 1) * page)
            if not any_seen[lo:hi].any():
                continue                               # its table entry may be anything
            k[lo:hi] = k_pages[table[b][p], :, : hi - lo].transpose(0, 1).double()
            v[lo:hi] = v_pages[table[b][p], :, : hi - lo].transpose(0, 1).double()
        k[~any_seen], v[~any_seen] = 0, 0
        for h in range(hq):
            kh = h // (hq // hk)
            x = q[q0:q1, h].double()
            s = (x @ k[:, kh].T) * scale
            s_err = d * 2.0 ** -23 * scale * (x.abs() @ k[:, kh].abs().T).masked_fill(~seen, 0).amax(-1, keepdim=True) \
                if n else torch.zeros(q1 - q0, 1, dtype=torch.float64)
            s = s.masked_fill(~seen, -float("inf"))
            p = torch.exp(s - s.amax(-1, keepdim=True).clamp(min=-1e300)) if n else s
            total = p.sum(-1, keepdim=True)
            p = p / torch.where(total > 0, total, 1.0)
            o = p @ v[:, kh]
            out[q0:q1, h] = o
            bound[q0:q1, h] = half_step(o) + (p @ v[:, kh].abs()) * (2.0 ** -8 + 2.0 ** -20 + 2 * s_err) \
                + 2.0 ** -8 * o.abs() + 2.0 ** -126
    return out, bound
