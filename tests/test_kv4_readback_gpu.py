"""Rows of a 4-bit cache read right behind the calls that write them, with nothing on the host in between."""
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    import flint_mac_b200 as fa

    fa.load_library()
    return fa


def _open(fa, torch, is_swa, n, n_ctx, **kw):
    h = fa.Attn([is_swa], [False], n, n_ctx, kv_format=fa.KV_INT4, **kw)
    g = torch.Generator().manual_seed(3)
    w = (1 + 0.1 * torch.randn(128, generator=g), 1 + 0.1 * torch.randn(128, generator=g), torch.randn(32, generator=g))
    h.set_layer(0, *(x.numpy() for x in w))
    return h


def _rand(torch, seed, *shape):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


@pytest.mark.parametrize("is_swa,paged", [(False, False), (False, True), (True, False)])
@pytest.mark.parametrize("n,pos", [(1, 5000), (16, 639), (128, 200)])
def test_load_decode_load(fa, is_swa, paged, n, pos):
    """Load, decode another row into the same position, load: each second load has the row of its own decode.  The grids of
    such a chain overlap: the second load may be resident while the first one still reads the blocks."""
    import torch

    seqs, rounds, rows = list(range(n)), 8, 70
    x = _rand(torch, 51, 2, n, 4, pos, 128).to(torch.float16)
    qkv = _rand(torch, 53, rounds, n, 5120)
    back = torch.empty(rounds, 2, 2, n, 4, rows, 128, device="cuda")
    out = torch.empty(n, 4096, device="cuda")
    with _open(fa, torch, is_swa, n, pos + 64, kv_pages=n * (pos // 64 + 2) if paged else 0) as h:
        h.store_kv_dev(0, seqs, [0] * n, pos, x[0], x[1], fa.F16)
        for s in seqs:
            h.set_pos(s, pos)
        at = [pos + 1 - rows] * n
        h.decode_dev(0, seqs, qkv[-1], fa.F32, out, fa.F32)
        h.check()
        before = [h.prepared_load_kv_dev(0, seqs, at, rows, back[i, 0, 0], back[i, 0, 1], fa.F32) for i in range(rounds)]
        after = [h.prepared_load_kv_dev(0, seqs, at, rows, back[i, 1, 0], back[i, 1, 1], fa.F32) for i in range(rounds)]
        decode = h.prepared_decode_dev(0, seqs, fa.F32, out, fa.F32)
        for i in range(rounds):
            before[i]()
            decode(qkv[i].data_ptr())
            after[i]()
        h.check()
    new = ref.kept(qkv[:, :, 36 * 128:].reshape(rounds, n, 4, 128).to(torch.float16)).float()
    old = ref.kept(x[1][:, :, pos + 1 - rows:]).float()
    for i in range(rounds):
        assert torch.equal(back[i, 0, 1, :, :, :-1], old) and torch.equal(back[i, 1, 1, :, :, :-1], old)
        assert torch.equal(back[i, 0, 1, :, :, -1], new[i - 1]), i
        assert torch.equal(back[i, 1, 1, :, :, -1], new[i]), i
        # K rows: the same in every load between two decodes, another one behind each
        assert torch.equal(back[i, 0, 0, :, :, -1], back[i - 1, 1, 0, :, :, -1]) or i == 0
        assert not torch.equal(back[i, 0, 0, :, :, -1], back[i, 1, 0, :, :, -1])


@pytest.mark.parametrize("is_swa,first", [(False, 0), (True, 0), (True, 5)])
def test_chunk_behind_a_chunk(fa, is_swa, first):
    """Two chunks of a prompt, and again with another first chunk, back to back: each second chunk attends to the rows of the
    chunk in front of it, as it does when the host waits between the calls."""
    import torch

    p0, n1, n2, rounds = 700, 37, 150, 6
    k, v = _rand(torch, 55, 2, 1, 4, p0, 128)
    a, b = _rand(torch, 57, rounds, n1, 5120), _rand(torch, 59, n2, 5120)
    outs = []
    for wait in (True, False):
        out1, out2 = torch.empty(rounds, n1, 4096, device="cuda"), torch.empty(rounds, n2, 4096, device="cuda")
        with _open(fa, torch, is_swa, 1, 1000, first_tokens=first) as h:
            h.store_kv_dev(0, [0], [0], p0, k, v, fa.F32)
            for i in range(rounds):
                h.set_pos(0, p0)
                h.prefill_dev(0, 0, n1, a[i], fa.F32, out1[i], fa.F32)
                if wait:
                    h.check()
                h.set_pos(0, p0 + n1)
                h.prefill_dev(0, 0, n2, b, fa.F32, out2[i], fa.F32)
                if wait:
                    h.check()
            h.check()
        outs.append((out1, out2))
    for x, y in zip(*outs):
        assert torch.isfinite(x).all() and torch.equal(x, y)
    assert not torch.equal(outs[0][1][0], outs[0][1][1])


def test_codes_beside_a_border(fa):
    """Values as near to the border between two codes as halves get, tiny ones beside a large least value: whichever code they
    get, they are within half a step and 2^-19 of one of what it stands for (the difference x - lo and its quotient by d are
    below 16 steps and rounded to 32 bits, 2^-24 relative each: 2^-19 steps)."""
    import torch

    g = torch.Generator().manual_seed(101)
    n = 6400
    code = torch.randint(1, 14, (n, 4, 1), generator=g).double() + 0.5
    d = (0.1 + 0.4 * torch.rand(n, 4, 1, generator=g)).half().double()
    lo = (-code * d).half().double()
    x = torch.empty(n, 4, 32, dtype=torch.float64)
    x[..., 0:1], x[..., 1:2] = lo, (lo + 15 * d).half().double()
    c = torch.arange(1, 15) + 0.5
    x[..., 2:16] = (lo + c * d).half().double()          # beside every border
    x[..., 16:32] = (lo + code * d).half().double()      # beside the one that lies next to zero
    rows = x.reshape(n, 128).half()
    rows[-1, :2] = torch.tensor([-2.01171875, 1.5390625])
    rows[-1, 2:32] = 0.00018322467803955078              # x - lo is a tie of 32-bit floats, on a border of d = 0.2366943359375
    back = torch.empty(2, 1, 4, n // 4, 128, device="cuda")
    given = rows.cuda().view(1, 4, n // 4, 128)
    with _open(fa, torch, False, 1, n // 4) as h:
        h.store_kv_dev(0, [0], [0], n // 4, given, given, fa.F16)
        h.load_kv_dev(0, [0], [0], n // 4, back[0], back[1], fa.F32)
        h.check()
    assert torch.equal(back[0], back[1])
    _, d, lo = ref.quantise(given)
    value, x = back[0].double().unflatten(-1, (4, 32)), given.double().unflatten(-1, (4, 32))
    inside = (x - lo) / d <= 14.5  # (beyond it the last code's value may lie further off by the rounding of d)
    assert float(inside.double().mean()) > 0.9
    off = (value - x).abs() - d * (0.5 + 2.0**-19) - 2.0**-24 * value.abs()
    assert float(off[inside].max()) <= 0, float((off / d)[inside].max())
    assert float(d[0, -1, -1, 0, 0]) == 0.2366943359375
