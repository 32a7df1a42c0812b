"""Decode over a 4-bit cache whose V rows are of any size, beside keys that take most of the softmax, against the 64-bit
statement and against a prefill of the same row over the same cache."""
import math

import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    import flint_mac_b200 as fa

    fa.load_library()
    return fa


def _rand(torch, seed, *shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def _weights(torch):
    g = torch.Generator().manual_seed(3)
    return (1 + 0.1 * torch.randn(128, generator=g), 1 + 0.1 * torch.randn(128, generator=g), torch.randn(32, generator=g))


def _peaked(torch, seed, n, keys, gap, tops):
    """Raw rows [2][n][5120] of a token and the one after it, and K [n][4][keys][128] in half: the scores of the first
    token's heads are about normal with unit deviation in base 2, those of the keys `tops` [n][keys] about `gap` higher."""
    sign = torch.sign(_rand(torch, seed, n, 4, 1, 128))  # what a group's eight queries have in common
    qkv = _rand(torch, seed + 1, 2, n, 5120)
    qkv[0, :, :4096] += 3 * sign.expand(n, 4, 8, 128).reshape(n, 4096)
    k = _rand(torch, seed + 2, n, 4, keys, 128) * (1 / math.log2(math.e))
    # q is 3 / sqrt(10) of sqrt(128) long along the signs: q . sign / sqrt(128) = 10.7
    k += tops[:, None, :, None] * sign * (gap / (10.7 * math.log2(math.e)))
    return qkv, k.to(torch.float16)


def _first_tiles(fa, torch, n, keys, target):
    """One key in each of the first eight tiles of every piece that the plan makes."""
    tops = torch.zeros(n, keys)
    for piece in fa.plan_decode_int4([keys] * n, False, 0, target):
        for t in range(piece[1], min(piece[1] + 8, piece[2])):
            tops[piece[0], min(64 * t + (7 * t) % 64, keys - 1)] = 1
    return tops.cuda()


def _check(fa, torch, n, keys, target, qkv, k, v, extra=0.0, scale=1.0, prefill=True):
    w = _weights(torch)
    with fa.Attn([False], [False], n, keys + 2, kv_format=fa.KV_INT4) as h:
        h.set_layer(0, *(x.numpy() for x in w))
        h._lib.flint_attn_set_target_items(h._h, target)
        h.store_kv_dev(0, list(range(n)), [0] * n, keys, k, v, fa.F16)
        for s in range(n):
            h.set_pos(s, keys)
        out = torch.empty(n, 4096, device="cuda")
        h.decode_dev(0, list(range(n)), qkv[0], fa.F32, out, fa.F32)
        h.check()
        two = torch.empty(n, 2, 4096, device="cuda")
        for s in range(n if prefill else 0):
            h.prefill_dev(0, s, 2, qkv[:, s].contiguous(), fa.F32, two[s], fa.F32)
        h.check()
    w = tuple(x.cuda() for x in w)
    at = torch.full((n,), keys, device="cuda")
    q, kn, vn = ref.split_rows(qkv[0], w, at, False)
    for s in range(n):
        kk = torch.cat((ref.kept(k[s]), kn[s].double()[:, None]), 1)
        vv = torch.cat((ref.kept(v[s]), vn[s].double()[:, None]), 1)
        want, room = ref.attend(q[s:s + 1], kk, vv, torch.ones(1, keys + 1, dtype=torch.bool, device="cuda"), w[2])
        room = room - 1e-6 + 1e-6 * scale  # the part that does not follow the values is for values of about one
        ref.assert_near(out[s:s + 1], want, room + extra, f"decode {s}")
        if prefill:  # staged values are halves: below the least normal one they are off by up to 2^-25, however small they are
            ref.assert_near(two[s, :1], want, room + 2.0**-25, f"prefill {s}")


@pytest.mark.parametrize("exponent", [-14, -12, -9, -6, 0, 5, 12])
@pytest.mark.parametrize("gap", [0, 8, 11, 13, 18])
@pytest.mark.parametrize("n,keys,target", [(1, 8192, 296), (1, 8192, 4), (1, 32768, 296), (1, 32768, 32), (3, 8192, 12), (2, 2000, 1)])
def test_one_size(fa, exponent, gap, n, keys, target):
    import torch

    scale = 2.0**exponent
    qkv, k = _peaked(torch, 61, n, keys, gap, _first_tiles(fa, torch, n, keys, target))
    v = (_rand(torch, 67, n, 4, keys, 128) * scale).to(torch.float16)
    qkv[:, :, 36 * 128:] *= scale
    _check(fa, torch, n, keys, target, qkv, k, v, scale=scale)


# Rows of mixed sizes.  The products' operand is the probability, 2^11 times its size relative to a reference P that some key
# seen exceeds at least twofold, and d times 2^b, with b such that the largest d of a tile lies between 2^-6 and 4 (b <= 14; b >=
# -12, and the probability takes it where it is negative).  Beside the relative roundings that attend() counts, an operand
# below the least normal half is off by 2^-25 at most.  In the output, whose denominator is at least 2 P, that makes for each
# key seen
#   15 codes * 2^-25 * 2^-b * 2^-11 / 2 * (1, for the product; d_j, for the probability where b < 0)
# with 2^-b <= min(max(2^6 * largest d of the tile, 2^-14), 2^12); and 2^-37 (|lo_j| + 15 d_j) for the probability itself.
def _extra(torch, v):
    _, d, lo = ref.quantise(v)  # [n][4][keys][4][1]
    n, kvh, keys = d.shape[:3]
    pad = torch.zeros(n, kvh, -keys % 64, 4, device="cuda", dtype=torch.float64)
    most = torch.cat((d[..., 0], pad), 2).reshape(n, kvh, -1, 64 * 4).amax(-1)
    unit = (most * 64).clamp(2.0**-14, 2.0**12).repeat_interleave(64, 2)[:, :, :keys, None]
    per_key = 15 * 2.0**-37 * unit * (1 + d[..., 0]) + 2.0**-37 * (lo[..., 0].abs() + 15 * d[..., 0])
    return float(per_key.sum(2).max())


@pytest.mark.parametrize("low,high,by", [(-9, 0, "row"), (-14, 3, "row"), (-9, 0, "tile"), (-14, 12, "tile"), (-14, 10, "group")])
@pytest.mark.parametrize("gap", [0, 11, 15])
@pytest.mark.parametrize("n,keys,target", [(1, 8192, 4), (1, 32768, 296), (2, 3000, 1)])
def test_mixed_sizes(fa, low, high, by, gap, n, keys, target):
    """Sizes drawn anew for each row, each tile of 64 rows, or each group of 32 values of a row."""
    import torch

    qkv, k = _peaked(torch, 71, n, keys, gap, _first_tiles(fa, torch, n, keys, target))
    shape = {"row": (n, 4, keys, 1), "tile": (n, 4, keys, 1), "group": (n, 4, keys, 4)}[by]
    e = torch.empty(shape, device="cuda").uniform_(low, high, generator=torch.Generator(device="cuda").manual_seed(73))
    if by == "tile":
        e = e[:, :, torch.arange(keys, device="cuda") // 64 * 64]
    v = (_rand(torch, 79, n, 4, keys, 4, 32) * torch.exp2(e).expand(n, 4, keys, 4)[..., None]).reshape(n, 4, keys, 128).to(torch.float16)
    _check(fa, torch, n, keys, target, qkv, k, v, extra=_extra(torch, v), prefill=False)


def test_outlier_tiles_without_weight(fa):
    """Tiles of values near the end of the range that nothing attends to, between tiles of small ones that have all the
    weight: the small ones keep their accuracy."""
    import torch

    n, keys, target = 2, 4096, 1
    tops = (torch.arange(keys, device="cuda") // 64 % 2 == 0).float().expand(n, keys)
    qkv, k = _peaked(torch, 83, n, keys, 30, tops)
    v = (_rand(torch, 89, n, 4, keys, 128) * torch.where(tops > 0, 2.0**-8, 2.0**12)[:, None, :, None]).to(torch.float16)
    qkv[:, :, 36 * 128:] *= 2.0**-8
    # (the large rows' probabilities are below 2^-20 of a denominator that 2048 keys make up: attend() has them)
    _check(fa, torch, n, keys, target, qkv, k, v, extra=2.0**-37 * 15 * 64 * 2.0**-8 * keys, scale=2.0**-8, prefill=False)
