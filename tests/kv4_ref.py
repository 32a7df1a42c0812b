"""The 4-bit cache and the attention over it, stated in 64 bits with torch: what the tests of the kernels compare with."""
import math

import torch

DIM, GROUP, KVH, GQA = 128, 32, 4, 8


def quantise(x16):
    """x16 half [..., 128] -> (codes, d, lo) as float64 [..., 4, 32], [..., 4, 1], [..., 4, 1]."""
    g = x16.double().reshape(*x16.shape[:-1], DIM // GROUP, GROUP)
    fine = torch.isfinite(g).all(-1, keepdim=True)
    lo, hi = g.amin(-1, keepdim=True), g.amax(-1, keepdim=True)
    d = ((hi - lo) / 15).to(torch.float16).double()
    code = torch.where(d > 0, torch.round((g - lo) / torch.where(d > 0, d, 1.0)), 0.0).clamp(0, 15)
    bad = torch.full_like(d, math.nan)
    return torch.where(fine, code, 0.0), torch.where(fine, d, bad), torch.where(fine, lo, 0.0)


def kept(x16):
    """The values a 4-bit cache keeps of half rows, in 64 bits."""
    code, d, lo = quantise(x16)
    return (lo + code * d).reshape(x16.shape)


def norm_rope(x, w, pos, rope):
    """x [n][heads][128] float64; the angle is the fp32 product of position and inverse frequency, as in the model."""
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + 1e-6) * w.double()
    if not rope:
        return x
    freq = torch.tensor([10000.0 ** (-2.0 * i / DIM) for i in range(64)], dtype=torch.float64, device=x.device).float()
    ang = (pos.float()[:, None] * freq).double()[:, None]
    a, b = x[..., :64], x[..., 64:]
    return torch.cat((a * ang.cos() - b * ang.sin(), a * ang.sin() + b * ang.cos()), -1)


def split_rows(qkv, weights, pos, rope):
    """Raw rows [n][5120] -> q [n][32][128] float64, k and v [n][4][128] half."""
    qn, kn, _ = weights
    x = qkv.double().view(-1, 40, DIM)
    q = norm_rope(x[:, :32], qn, pos, rope)
    k = norm_rope(x[:, 32:36], kn, pos, rope).to(torch.float16)
    return q, k, x[:, 36:].to(torch.float16)


def visible(q_pos, k_pos, is_swa, first):
    """[queries][keys] truth values."""
    seen = k_pos[None] <= q_pos[:, None]
    if is_swa:
        seen &= (k_pos[None] > q_pos[:, None] - 513) | (k_pos[None] < first)
    return seen


def attend(q, k, v, seen, sinks):
    """q [n][32][128], k and v [4][m][128], seen [n][m] -> out [n][32][128], and a bound on what roundings may do to it.

    The kernels round q, the keys of a call and probabilities to half (2^-11 relative each), and probabilities times d or
    the staged values once more.  A score's error is then at most 3 * 2^-11 * sum |q_i k_i| / sqrt(128) (keys that went
    through norm and rotation in 32 bits may land on the neighbouring half: 2 * 2^-11), which moves every probability by at
    most twice that, relatively; three more roundings sit on the products p v.  32-bit sums add less than 2^-16.

    A cached value is lo + d code, and its product the sum of p' lo and r(p' d) code, with p' the rounded probability and r
    one more rounding: p' lo + p' d code (1 + e) = p' v + e p' (v - lo), |e| <= 2^-11.  So where lo and d code nearly cancel
    (a query that sees two keys: v = 0.002 from terms of 1.3) the error is 2^-11 p |v - lo|, however small v is, and the
    32-bit sums are relative to those terms too.  A group's least value has code 0, so lo is its minimum."""
    n, m = q.shape[0], k.shape[1]
    qh = q.view(n, KVH, GQA, DIM)
    s = torch.einsum("nhgd,hmd->nhgm", qh, k) / math.sqrt(DIM)
    mag = torch.einsum("nhgd,hmd->nhgm", qh.abs(), k.abs()) / math.sqrt(DIM)
    s = s.masked_fill(~seen[:, None, None], -math.inf)
    mag = mag.masked_fill(~seen[:, None, None], 0.0)
    sink = sinks.double().view(1, KVH, GQA, 1).expand(n, KVH, GQA, 1)
    p = torch.cat((s, sink), -1).softmax(-1)[..., :m]
    out = torch.einsum("nhgm,hmd->nhgd", p, v)
    g = v.unflatten(-1, (DIM // GROUP, GROUP))
    off = torch.einsum("nhgm,hmd->nhgd", p, (g - g.amin(-1, keepdim=True)).flatten(-2)) * (2**-11 + 2**-16)
    room = off + torch.einsum("nhgm,hmd->nhgd", p, v.abs()) * (2 * 3 * 2**-11 * mag.amax(-1, keepdim=True) + 3 * 2**-11 + 2**-16)
    return out.reshape(n, 32, DIM), room.reshape(n, 32, DIM) + 1e-6


def assert_near(got, want, room, what):
    """got bf16 or fp32; `room` from attend().  Each output within its bound; over all of them the roundings are random:
    about 2^-11 / sqrt(3) from each of five (q, k, p, p d, v), each with a weight of about one, 6.3e-4 together and at
    most double that through the softmax, 1.3e-3 (+ 2^-8 / sqrt(3) = 2.3e-3 from a bf16 output)."""
    half_step = 2.0**-8 if got.dtype == torch.bfloat16 else 2.0**-24
    g, w, r = got.double().reshape(-1), want.reshape(-1), room.reshape(-1)
    assert torch.isfinite(g).all(), what
    over = (g - w).abs() - (r + half_step * (w.abs() + r))
    assert over.max() <= 0, f"{what}: {int((over > 0).sum())} outputs beyond their bound, worst by {float(over.max()):.3e}"
    rel = float((g - w).norm() / w.norm())
    assert rel <= 1.3e-3 + (2.3e-3 if got.dtype == torch.bfloat16 else 0), f"{what}: relative error {rel:.3e}"
    return rel


def assert_kept(got, half_rows, what):
    """Values read back (fp32) of rows whose K went through norm and rotation in 32 bits: a value next to a border between
    two halves may land on the other one, and that may move one code, or the d or lo of its group by a half step.  So: most
    equal, the rest within a step and a half-precision step."""
    code, d, lo = quantise(half_rows)
    want = (lo + code * d).reshape(half_rows.shape)
    step = d.expand_as(code).reshape(half_rows.shape)
    diff = (got.double() - want).abs()
    assert (diff <= step * 1.01 + 16 * 2.0**-10 * (want.abs() + step)).all(), f"{what}: {float((diff / step).max()):.3f} steps off"
    far = float((diff > 2.0**-24 * want.abs()).double().mean())
    assert far <= 0.02, f"{what}: {far:.4f} of the values differ"
