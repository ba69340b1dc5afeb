"""Plain 64-bit forms of the attention half's operators, on the CPU with torch:
what include/noor_moe.h states, written out, for the tests."""
import math

import torch

F8 = torch.float8_e4m3fn
QMAX = {"int8": 127.0, "e4m3": 448.0}
E4M3 = torch.arange(127, dtype=torch.uint8).view(F8).double()  # the finite magnitudes, ascending


def rotate(x, positions, inv_freq, layout, factor=1.0, sign=1.0):
    """x [T, H, D] in f64; positions [T]; inv_freq the f32 table."""
    x = x.double()
    half = inv_freq.numel()
    y = x.clone()
    ang = positions.double()[:, None] * inv_freq.double()[None]
    c, s = (torch.cos(ang) * factor)[:, None], (torch.sin(ang) * factor * sign)[:, None]
    if layout == "interleaved":
        i0, i1 = torch.arange(half) * 2, torch.arange(half) * 2 + 1
    else:
        i0, i1 = torch.arange(half), torch.arange(half) + half
    y[..., i0] = x[..., i0] * c - x[..., i1] * s
    y[..., i1] = x[..., i0] * s + x[..., i1] * c
    return y


def scale_for(amax, fmt):
    """Smallest power of two >= 2^-126 with amax <= Q s; NaN if not finite."""
    if not math.isfinite(amax):
        return math.nan
    e = -126
    if amax > 0:
        e = max(e, math.ceil(math.log2(amax / QMAX[fmt])))
        while e > -126 and amax <= QMAX[fmt] * 2.0 ** (e - 1):
            e -= 1
        while amax > QMAX[fmt] * 2.0 ** e:
            e += 1
    return 2.0 ** e


def code(x, fmt):
    """x (f64, in steps) rounded to the nearest code value, ties to even."""
    if fmt == "int8":
        return x.round().clamp(-127, 127)
    mid = (E4M3[1:] + E4M3[:-1]) / 2
    i = torch.searchsorted(mid, x.abs().contiguous())
    at = i.clamp(max=mid.numel() - 1)
    i = i + ((x.abs() == mid[at]) & (i < mid.numel()) & (i % 2 == 1))
    return E4M3[i] * torch.sign(x)


class RefCache:
    """The pages of one pool (k or v) as values: vals [P, H, block, D] code
    values and scale [P, H]."""

    def __init__(self, P, H, blk, D, fmt):
        self.vals = torch.zeros((P, H, blk, D), dtype=torch.float64)
        self.scale = torch.zeros((P, H), dtype=torch.float64)
        self.blk, self.fmt = blk, fmt

    def append(self, x, row0, n, end, pages):
        """Rows row0 .. row0 + n - 1 of x [rows, H, D] are tokens end - n .. end - 1."""
        pos = end - n
        while pos < end:
            j, slot = pos // self.blk, pos % self.blk
            m = min(end - pos, self.blk - slot)
            page = int(pages[j])
            for h in range(x.shape[1]):
                new = x[row0:row0 + m, h].double()
                s = scale_for(float(new.abs().max()) if bool(torch.isfinite(new).all()) else math.inf, self.fmt)
                old = float(self.scale[page, h]) if slot else 0.0
                if slot and math.isnan(old):
                    s = math.nan
                elif slot and not math.isnan(s):
                    s = max(s, old)
                if math.isnan(s):
                    self.vals[page, h, slot:slot + m] = 0.0
                else:
                    if slot and s != old:
                        self.vals[page, h, :slot] = code(self.vals[page, h, :slot] * (old / s), self.fmt)
                    self.vals[page, h, slot:slot + m] = code(new / s, self.fmt)
                self.scale[page, h] = s
            row0, pos = row0 + m, pos + m

    def tokens(self, pages, n):
        """Values [n, H, D] of a sequence's first n tokens."""
        p = torch.as_tensor(pages[:max(1, -(-n // self.blk))]).long()
        v = self.vals[p] * self.scale[p][:, :, None, None]
        return v.transpose(1, 2).reshape(-1, v.shape[1], v.shape[3])[:n]


def attend(q, k, v, pos, scale, window):
    """q [n, Hq, D] at positions pos [n] over k, v [L, Hkv, D], all f64.
    Returns out, lse, mag (sum p |v| / sum p), smax (largest scale |q|.|k|) and
    vsum (sum |v| over the tokens that any row sees)."""
    n, Hq, D = q.shape
    L, Hkv, _ = k.shape
    g = Hq // Hkv
    kk, vv = k.repeat_interleave(g, 1), v.repeat_interleave(g, 1)
    s = torch.einsum("nhd,lhd->hnl", q, kk) * scale
    key = torch.arange(L)
    hidden = key[None] > pos[:, None]
    if window > 0:
        hidden |= pos[:, None] - key[None] > window
    s = s.masked_fill(hidden[None], -math.inf)
    top = s.amax(-1, keepdim=True) if L else torch.full((Hq, n, 1), -math.inf, dtype=q.dtype)
    p = torch.exp(s - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    p = p.masked_fill(hidden[None], 0.0)
    tot = p.sum(-1, keepdim=True)
    w = p / torch.where(tot == 0, torch.ones_like(tot), tot)
    vz = torch.where(hidden.all(0)[:, None, None], torch.zeros_like(vv), vv)  # nobody sees it: whatever it holds
    out = torch.einsum("hnl,lhd->nhd", w, vz)
    mag = torch.einsum("hnl,lhd->nhd", w, vz.abs())
    lse = (top.squeeze(-1) + torch.log(tot.squeeze(-1))).transpose(0, 1)
    smax = (torch.einsum("nhd,lhd->hnl", q.abs(), kk.abs()) * abs(scale)).masked_fill(hidden[None], 0).nan_to_num().amax(-1)
    return out, lse, mag, smax.transpose(0, 1), vz.abs().sum(0)


def attend_tolerance(dtype, out, mag, smax, vsum, D, L):
    """Largest error of one output.  Its own rounding; each p off by its f16
    parts (one part 2^-11, two 2^-21), and by its score: a sum of D + 8 products
    and factors in f32, whose error (2^-23 a step, the tensor core cuts rather than
    rounds) is relative to scale |q|.|k| and doubles through the quotient; the
    sums over L tokens.  And f16's own floor: a p below 2^-14 of its format is off by
up to 2^-25 whatever its size, and the largest p is at least 2^7 there (2^7 in
the many-row kernel, 2^14 in the other, where F32's second part reaches as
far), so each token adds up to 2^-32 |v| (F32 2^-39 |v|) of the row's largest
weight, which is at most 1."""
    bf = dtype == torch.bfloat16
    own = 2.0 ** -8 if bf else 2.0 ** -24
    p = 2.0 ** -11 if bf else 2.0 ** -21
    rel = p + 2 * (D + 8) * 2.0 ** -23 * smax[..., None] + (L + 64) * 2.0 ** -23
    return own * out.abs() + mag * rel + (2.0 ** -32 if bf else 2.0 ** -39) * vsum + 1e-30
