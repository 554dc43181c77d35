"""64-bit reference of the fp4_ds_mla format and its attention (torch, any device)."""

import torch

LEVELS = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _nearest_even(x, grid):
    """Index of the grid value nearest to x (float64, >= 0), the even index of two
    as near; beyond the last value, the last."""
    hi = torch.searchsorted(grid, x.contiguous()).clamp(max=len(grid) - 1)
    lo = (hi - 1).clamp(min=0)
    dh, dl = (grid[hi] - x).abs(), (x - grid[lo]).abs()
    return torch.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)


def quantize(kv_c, k_pe):
    """bf16 [n, 512], [n, 64] -> uint8 rows [n, 416]; NaN groups get scale byte 0x7F
    (their codes are unspecified)."""
    dev = kv_c.device
    x = kv_c.double().view(-1, 32, 16)
    nan = x.isnan().any(2)
    scales = torch.arange(127, dtype=torch.uint8, device=dev).view(torch.float8_e4m3fn).double()
    amax = torch.where(x.isnan(), 0.0, x.abs()).amax(2)
    want = (amax / 6).clamp(2.0 ** -9, 448.0)
    sb = _nearest_even(want, scales)                       # the byte is the index
    s = scales[sb][:, :, None]
    mag = torch.where(x.isnan(), 0.0, x.abs()) / s
    code = _nearest_even(mag.clamp(max=6.0), torch.tensor(LEVELS, dtype=torch.float64, device=dev))
    code = (code + 8 * torch.signbit(x).long()).view(-1, 256, 2)
    packed = (code[:, :, 0] + 16 * code[:, :, 1]).to(torch.uint8)
    sb = torch.where(nan, 127, sb).to(torch.uint8)
    return torch.cat([packed, sb, k_pe.contiguous().view(torch.uint8)], 1)


def values(rows):
    """uint8 rows [n, 416] -> float64 [n, 576]."""
    lv = torch.tensor(LEVELS + [-v for v in LEVELS], dtype=torch.float64, device=rows.device)
    b = rows[:, :256].long()
    lat = lv[torch.stack([b % 16, b // 16], 2)].view(-1, 32, 16)
    s = rows[:, 256:288].contiguous().view(torch.float8_e4m3fn).double()
    rope = rows[:, 288:].contiguous().view(torch.bfloat16).double()
    return torch.cat([(lat * s[:, :, None]).view(-1, 512), rope], 1)


def attend(q, pool, slots, sm_scale, G=1):
    """q [T, H, 576], pool [n, 416], slots [T, G, k] (-1 masked, also outside the
    pool) -> out [T, H, 512], lse [T, H] in float64, and the bounds of the
    kernel's error.

    Bounds.  Products of the score are exact in fp32 (11 x 6 bits), their 576-term
    sum is off by at most 576 * 2^-23 * A with A = scale * sum |q k| (one ulp a
    term), the exponent's rounding and the exp2 add less than 2^-20 (1 + A).  P is
    rounded to fp16 (2^-11).  So each weight is off by e = 2^-11 + d relative with
    d = A (576 * 2^-23 + 2^-20) + 2^-20, the output by (e + d) * sum p |v| / l
    (numerator and sum) plus its own bf16 rounding 2^-8 |out|, the lse by d plus
    its fp32 arithmetic 2^-20 (1 + |lse|).  P is stored times 2^6, so a weight
    below fp16's normal range (2^-20 of the largest) is off by up to half its
    smallest step, 2^-25 2^-6 = 2^-31 of the largest weight, instead of 2^-11 of
    itself.  The reference maximum is never above the largest score met, so the
    sum is at least the weight 1 that this is relative to: 2^-31 sum |v| more."""
    T, H, _ = q.shape
    out = torch.zeros(T, H, 512, dtype=torch.float64, device=q.device)
    lse = torch.full((T, H), float("-inf"), dtype=torch.float64, device=q.device)
    tol_o, tol_l = torch.zeros_like(out), torch.zeros_like(lse)
    hpg = H // G
    for t in range(T):
        for g in range(G):
            sl = slots[t, g].long()
            sl = sl[(sl >= 0) & (sl < len(pool))]
            if len(sl) == 0:
                continue
            k = values(pool[sl])
            hs = slice(g * hpg, (g + 1) * hpg)
            qd = q[t, hs].double()
            z = qd @ k.T * sm_scale
            lse[t, hs] = torch.logsumexp(z, 1)
            p = torch.softmax(z, 1)
            out[t, hs] = p @ k[:, :512]
            a = (qd.abs() @ k.abs().T * abs(sm_scale)).amax(1)
            d = a * (576 * 2.0 ** -23 + 2.0 ** -20) + 2.0 ** -20
            tol_l[t, hs] = d + 2.0 ** -20 * (1 + lse[t, hs].abs())
            tol_o[t, hs] = (2.0 ** -11 + 2 * d)[:, None] * (p @ k[:, :512].abs()) + 2.0 ** -8 * out[t, hs].abs()
            tol_o[t, hs] += 2.0 ** -31 * k[:, :512].abs().sum(0)
    return out, lse, tol_o, tol_l


def check(got, want):
    """got (out, lse) against attend()'s four tensors."""
    o, l = got[0].double(), got[1].double()
    out, lse, tol_o, tol_l = want
    assert torch.equal(torch.isneginf(l), torch.isneginf(lse)), "-inf pattern of lse"
    fin = ~torch.isneginf(lse)
    assert torch.isfinite(o).all() and torch.isfinite(l[fin]).all()
    assert (o[~fin] == 0).all(), "rows without entries are zero"
    assert ((l - lse).abs()[fin] <= tol_l[fin]).all(), f"lse off by {(l - lse).abs()[fin].max():.3e}"
    over = (o - out).abs() - tol_o
    assert (over <= 0).all(), f"out over its bound by {over.max():.3e} at {int(over.argmax())}"
