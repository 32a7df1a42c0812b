"""4-bit K/V caches, and first tokens that stay visible beside rings of either format, through the C ABI: store, load, decode,
prefill, against 64-bit statements."""
import math

import numpy as np
import pytest

import kv4_ref as ref


@pytest.fixture(scope="module")
def fa():
    import flint_mac_b200 as fa

    fa.load_library()
    return fa


# ------------------------------------------------------------------------------------------------ refusals without a GPU
@pytest.mark.parametrize("kw,match", [
    ({"kv_format": 2}, "kv_format"),
    ({"kv_format": -1}, "kv_format"),
    ({"kv_format": 1, "first_tokens": 65}, "first_tokens"),
    ({"kv_format": 1, "first_tokens": -1}, "first_tokens"),
    ({"first_tokens": 65}, "first_tokens"),
    ({"kv_format": 1, "kv_ranks": 2}, "sharded"),
])
def test_open_refuses(fa, kw, match):
    with pytest.raises(fa.FlintAttnError, match=match):
        fa.Attn([True], [True], 1, 128, **kw)


def test_rows_of_no_handle_are_refused(fa):
    import ctypes as C

    lib, err, zero = fa.load_library(), C.create_string_buffer(200), (C.c_int32 * 1)(0)
    for fn in (lib.flint_attn_store_kv_dev, lib.flint_attn_load_kv_dev):
        assert fn(None, 0, 1, zero, zero, 1, 16, 16, fa.F32, None, err, 200) == -1 and err.value == b"null handle"


def test_statement_keeps_what_it_says():
    """The reference itself: every value within half a step of what it came from, the least and largest of a group exact
    to the rounding of d."""
    import torch

    x = torch.randn(50, 128, generator=torch.Generator().manual_seed(1)).to(torch.float16)
    code, d, lo = ref.quantise(x)
    assert code.max() == 15 and code.min() == 0
    err = (ref.kept(x) - x.double()).abs().reshape(50, 4, 32)
    assert (err <= d * (0.5 + 15 * 2.0**-11)).all()


@pytest.mark.parametrize("is_swa,first", [(False, 0), (True, 0), (True, 5), (True, 64)])
@pytest.mark.parametrize("target", [1, 7, 100, 296])
def test_plan_covers_every_tile_once(fa, is_swa, first, target):
    """Whatever the batch: every tile of every token in one piece, the pieces of a launch longest first, their records and
    counters apart from each other, and windows whole."""
    rng = np.random.default_rng(target)
    batches = [[0], [1], [64], [65], [131072], [0, 0, 0], [8192] * 64, [100] * 300, list(range(0, 2000, 7)), [131072, 0, 5, 5],
               [int(x) for x in np.exp(rng.uniform(0, 11, 200))], [int(x) for x in rng.integers(0, 600, 2048)], [1 << 30, 3, 1 << 20]]
    for pos in batches:
        pcs = fa.plan_decode_int4(pos, is_swa, first, target)
        assert (np.diff(pcs[:, 6]) >= 0).all() and np.bincount(pcs[:, 6]).max() <= 1300
        for launch in set(pcs[:, 6]):
            mine = pcs[pcs[:, 6] == launch]
            assert (np.diff(mine[:, 2] - mine[:, 1]) <= 0).all()
            cut = mine[mine[:, 4] > 1]
            records = cut[:, 5] + cut[:, 3]
            assert sorted(records) == list(range(len(cut))) and (mine[:, 7] == len(cut)).all()
        assert set(pcs[:, 0]) == set(range(len(pos)))
        for i, p in enumerate(pos):
            j0 = max(p - 512, 0) if is_swa else 0
            tiles = (1 if is_swa and min(first, j0) > 0 else 0) + (0 if p == j0 else (p - 1) // 64 - j0 // 64 + 1)
            mine = pcs[pcs[:, 0] == i]
            mine = mine[np.argsort(mine[:, 3])]
            n = len(mine)
            assert (mine[:, 3] == range(n)).all() and (mine[:, 4] == n).all() and len(set(mine[:, 6])) == 1
            assert mine[0, 1] == 0 and mine[-1, 2] == tiles and (mine[1:, 1] == mine[:-1, 2]).all()
            assert n == 1 or (mine[:, 2] > mine[:, 1]).all()
            assert n == 1 or not is_swa
    with pytest.raises(fa.FlintAttnError):
        fa.plan_decode_int4([5, -1], is_swa, first, target)


gpu = pytest.mark.gpu


def _weights(torch, seed):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.1 * torch.randn(128, generator=g), 1 + 0.1 * torch.randn(128, generator=g), torch.randn(32, generator=g))


def _open(fa, torch, is_swa, rope, n, n_ctx, seed=3, n_layers=1, half=False, **kw):
    h = fa.Attn([is_swa] * n_layers, [rope] * n_layers, n, n_ctx, kv_format=fa.KV_F16 if half else fa.KV_INT4, **kw)
    w = _weights(torch, seed)
    for il in range(n_layers):
        h.set_layer(il, *(x.numpy() for x in w))
    return h, tuple(x.cuda() for x in w)


def _keep(half):
    """What a cache of the format keeps of half-precision rows, in 64 bits."""
    return (lambda x: x.double()) if half else ref.kept


def _check_keys(got, half_rows, half, what):
    if half:
        # Norm and rotation in 32 bits: the scale is off by 2^-22 (a sum of 128 squares over seven levels) and four roundings
        # of 2^-24, sine and cosine by 2^-23, the products and their sum by three of 2^-24: below 2^-20 of |a| + |b|, the two
        # values that are turned into each other, which is at most 16 here.  A small result of large ones keeps that error,
        # 2^-16; beyond it a value lands on the same half or its neighbour.
        far = (got.double() - half_rows.double()).abs() > 2.0**-10 * half_rows.double().abs() + 2.0**-16
        assert not bool(far.any()), f"{what}: {int(far.sum())} keys off"
    else:
        ref.assert_kept(got, half_rows, what)


def _rand(torch, seed, *shape, dtype=None):
    x = torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))
    return x if dtype is None else x.to(dtype)


def _kind(fa, torch, dtype):
    return {torch.float32: fa.F32, torch.bfloat16: fa.BF16, torch.float16: fa.F16}[dtype]


# ------------------------------------------------------------------------------------------------ store and load
@gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("n,rows,at", [(1, 1, 0), (1, 64, 0), (3, 65, 63), (5, 7, 130), (150, 3, 61), (1, 1000, 24)])
def test_store_then_load(fa, dtype, paged, n, rows, at):
    import torch

    dt = getattr(torch, dtype)
    x = _rand(torch, 5, 2, n, 4, rows, 128) * torch.tensor([1.0, 7.0], device="cuda").view(2, 1, 1, 1, 1)
    x = x.to(dt)
    starts = [at + i % 4 for i in range(n)]
    with fa.Attn([False], [False], n, 1100, kv_format=fa.KV_INT4, kv_pages=n * 18 if paged else 0) as h:
        seqs = list(reversed(range(n)))
        h.store_kv_dev(0, seqs, starts, rows, x[0], x[1], _kind(fa, torch, dt))
        for back in (torch.float32, dt):
            k, v = torch.full((2, n, 4, rows, 128), 777.0, device="cuda", dtype=back)
            h.load_kv_dev(0, seqs, starts, rows, k, v, _kind(fa, torch, back))
            h.check()
            for got, given in ((k, x[0]), (v, x[1])):
                want = ref.kept(given.to(torch.float16))
                if back == torch.float32:
                    assert torch.equal(got, want.float())
                else:  # rounded to 32 bits and then to `back`: at most the next value from one rounding
                    assert ((got.double() - want).abs() <= torch.finfo(back).eps / 2 * want.abs() * 1.001 + 2.0**-25).all()
        # host copies of the same rows, by slot
        k16, v16 = h.read_kv(0, seqs[-1], starts[-1], rows)
        for got, given in ((k16, x[0, -1]), (v16, x[1, -1])):
            want = ref.kept(given.to(torch.float16)).cpu().numpy()
            g = got.view(np.float16).astype(np.float64)
            assert (np.abs(g - want) <= 2.0**-11 * np.abs(want) * 1.001 + 2.0**-25).all()


@gpu
@pytest.mark.parametrize("is_swa,paged", [(False, False), (False, True), (True, False)])
def test_store_and_load_of_half_precision_caches(fa, is_swa, paged):
    import torch

    x = _rand(torch, 6, 2, 2, 4, 1500, 128)
    with fa.Attn([is_swa], [False], 3, 1600, kv_pages=60 if paged else 0) as h:
        h.store_kv_dev(0, [2, 0], [50, 7], 1500, x[0], x[1], fa.F32)
        k, v = torch.empty(2, 2, 4, 1000, 128, device="cuda")
        h.load_kv_dev(0, [2, 0], [550, 507], 1000, k, v, fa.F32)
        h.check()
        for got, given in ((k, x[0]), (v, x[1])):
            assert torch.equal(got, given[:, :, 500:].to(torch.float16).float())
        slot = 551 & 1023 if is_swa else 551
        assert np.array_equal(h.read_kv(0, 2, slot, 1)[0].view(np.float16), x[0, 0, :, 501:502].to(torch.float16).cpu().numpy())


@gpu
def test_groups_at_the_ends_of_the_range(fa):
    """Constant groups, the widest range, steps below the least normal half, infinities, NaN, signed zeros."""
    import torch

    x = torch.zeros(4, 16, 128, device="cuda", dtype=torch.float16)
    x[:, 0] = 3.25
    x[:, 1, ::2], x[:, 1, 1::2] = 65504, -65504
    x[:, 2] = torch.arange(128, device="cuda") * 2.0**-24
    x[:, 3] = (torch.arange(128, device="cuda") % 3) * 2.0**-24 - 2.0**-24
    x[:, 4, 40] = math.inf
    x[:, 5, 70] = -math.inf
    x[:, 6, 127] = math.nan
    x[:, 7, ::2] = -0.0
    x[:, 8] = 1 + (torch.arange(128, device="cuda") % 32) * 2.0**-10
    x[:, 9] = 2048 + (torch.arange(128, device="cuda") % 31) * 2.0  # ties between two codes: d = 4, distances 2
    x[:, 10:] = _rand(torch, 8, 4, 6, 128) * torch.logspace(-6, 4, 6, device="cuda")[:, None]
    with fa.Attn([False], [False], 1, 64, kv_format=fa.KV_INT4) as h:
        h.store_kv_dev(0, [0], [17], 16, x, x, fa.F16)
        k, v = torch.empty(2, 4, 16, 128, device="cuda")
        h.load_kv_dev(0, [0], [17], 16, k, v, fa.F32)
        want = ref.kept(x).float()
        for got in (k, v):
            assert torch.equal(got.nan_to_num(nan=12345.0), want.nan_to_num(nan=12345.0))
        assert int(torch.isnan(k).sum()) == 4 * 3 * 32
        # values beyond half's range are infinite in half, so the group reads as NaN; the groups beside it stay
        big = torch.ones(1, 4, 1, 128, device="cuda")
        big[..., 5] = 7e4
        h.store_kv_dev(0, [0], [0], 1, big, big, fa.F32)
        h.load_kv_dev(0, [0], [0], 1, k[:, :1].contiguous(), v[:, :1].contiguous(), fa.F32)
        k1, v1 = torch.empty(2, 1, 4, 1, 128, device="cuda")
        h.load_kv_dev(0, [0], [0], 1, k1, v1, fa.F32)
        assert torch.isnan(k1[..., :32]).all() and (k1[..., 32:] == 1).all()


@gpu
@pytest.mark.parametrize("half", [False, True])
@pytest.mark.parametrize("first", [0, 5, 64])
def test_ring_rows_by_position(fa, first, half):
    """A ring keeps the last row of each slot, and the first tokens' rows whatever comes after."""
    import torch

    x = _rand(torch, 9, 2, 4, 2500, 128, dtype=torch.float16)
    with fa.Attn([True], [True], 2, 4000, kv_format=fa.KV_F16 if half else fa.KV_INT4, first_tokens=first) as h:
        assert h.n_slots(0) == 1024 + first
        h.store_kv_dev(0, [1], [0], 2500, x[0], x[1], fa.F16)
        k, v = torch.empty(2, 4, 1024, 128, device="cuda")
        h.load_kv_dev(0, [1], [2500 - 1024], 1024, k, v, fa.F32)
        want = _keep(half)(x)
        assert torch.equal(k, want[0, :, -1024:].float()) and torch.equal(v, want[1, :, -1024:].float())
        if first:
            k, v = torch.empty(2, 4, first, 128, device="cuda")
            h.load_kv_dev(0, [1], [0], first, k, v, fa.F32)
            assert torch.equal(k, want[0, :, :first].float()) and torch.equal(v, want[1, :, :first].float())
            k16, _ = h.read_kv(0, 1, 1024, first)
            assert np.array_equal(k16.view(np.float16), want[0, :, :first].float().to(torch.float16).cpu().numpy())
            # and by slot: the rows in the ring's slot 0.. are later ones
            k16, _ = h.read_kv(0, 1, 0, first)
            assert np.array_equal(k16.view(np.float16), want[0, :, 2048:2048 + first].float().to(torch.float16).cpu().numpy())
        h.write_kv(0, 0, 1000, np.ones((4, 24, 128), np.uint16) * 0x3C00, np.ones((4, 24, 128), np.uint16) * 0x4000)
        k16, v16 = h.read_kv(0, 0, 990, 34)
        assert (k16[:, 10:] == 0x3C00).all() and (v16[:, 10:] == 0x4000).all() and not k16[:, :10].any()


@gpu
def test_rows_refused(fa):
    import torch

    x = torch.zeros(2, 4, 10, 128, device="cuda", dtype=torch.float16)
    with fa.Attn([False, True], [False, True], 2, 200, kv_format=fa.KV_INT4, kv_pages=3) as h:
        for bad, match in [
            (lambda: h.store_kv_dev(2, [0, 1], [0, 0], 10, x, x, fa.F16), "layer"),
            (lambda: h.store_kv_dev(0, [0, 2], [0, 0], 10, x, x, fa.F16), "sequence index"),
            (lambda: h.store_kv_dev(0, [1, 1], [0, 0], 10, x, x, fa.F16), "twice"),
            (lambda: h.store_kv_dev(0, [0, 1], [0, 191], 10, x, x, fa.F16), "row range"),
            (lambda: h.store_kv_dev(0, [0, 1], [-1, 0], 10, x, x, fa.F16), "row range"),
            (lambda: h.store_kv_dev(0, [0, 1], [0, 0], 0, x, x, fa.F16), "row count"),
            (lambda: h.store_kv_dev(0, [0, 1], [0, 0], 10, x, x, 3), "dtype"),
            (lambda: h.store_kv_dev(0, [0, 1], [0, 0], 10, x.data_ptr() + 2, x, fa.F16), "16-byte"),
            (lambda: h.store_kv_dev(0, [0, 1], [0, 0], 10, 0, x, fa.F16), "null"),
            (lambda: h.load_kv_dev(0, [0, 1], [0, 195], 10, x, x, fa.F16), "row range"),
            (lambda: h.store_kv_dev(0, [0, 1], [100, 100], 10, x, x, fa.F16), "pool exhausted"),
            (lambda: h.decode_partial_dev(0, [0], x, fa.F32, x), "not set"),
        ]:
            with pytest.raises(fa.FlintAttnError, match=match):
                bad()
        with pytest.raises(ValueError):
            h.store_kv_dev(0, [0, 1], [0], 10, x, x, fa.F16)
        assert h.pages_free() == 3
        w = _weights(torch, 1)
        h.set_layer(0, *(t.numpy() for t in w))
        big = torch.zeros(1, 5120, device="cuda")
        for rows, out in ((0, big), (big, 0), (big.data_ptr() + 8, big), (big, big.data_ptr() + 2)):
            with pytest.raises(fa.FlintAttnError, match="null|16-byte"):
                h.decode_dev(0, [0], rows, fa.F32, out, fa.F32)
        with pytest.raises(fa.FlintAttnError, match="dtype"):
            h.decode_dev(0, [0], big, fa.F16, big, fa.F32)
        with pytest.raises(fa.FlintAttnError, match="4-bit"):
            h.decode_partial_dev(0, [0], big, fa.F32, big)
        with pytest.raises(fa.FlintAttnError, match="4-bit"):
            h.prefill_partial_dev(0, 0, 1, big, fa.F32, big, big)
        h.set_pos(0, 9)
        for n in (192, 2**31 - 1):
            with pytest.raises(fa.FlintAttnError, match="context full"):
                h.prefill_dev(0, 0, n, big, fa.F32, big, fa.F32)
        prepared = h.prepared_store_kv_dev(0, [0], [0], 1, x, x, fa.F16), lambda f=h.prepared_decode_dev(0, [0], fa.F32, big, fa.F32): f(big.data_ptr())
        # a page that no sequence holds reads as zeros
        k, v = torch.ones(2, 1, 4, 10, 128, device="cuda")
        h.load_kv_dev(0, [1], [60], 10, k, v, fa.F32)
        assert not k.any() and not v.any()
    for call in (*prepared, lambda: h.load_kv_dev(0, [1], [60], 10, k, v, fa.F32)):
        with pytest.raises(fa.FlintAttnError, match="closed"):
            call()


@gpu
@pytest.mark.parametrize("half", [False, True])
def test_pages_given_back_read_as_zeros(fa, half):
    """Pages a sequence gave back belong to another one: its positions there read as zeros, not as the other's rows."""
    import torch

    k, v = _history(torch, 91, 2, 640)
    with fa.Attn([False], [False], 2, 1000, kv_format=fa.KV_F16 if half else fa.KV_INT4, kv_pages=12) as h:
        h.store_kv_dev(0, [0], [0], 640, k[:1], v[:1], fa.F16)
        h.seq_release(0)
        h.store_kv_dev(0, [1], [0], 640, k[1:], v[1:], fa.F16)
        kb, vb = torch.ones(2, 2, 4, 640, 128, device="cuda")
        h.load_kv_dev(0, [0, 1], [0, 0], 640, kb, vb, fa.F32)
        assert not kb[0].any() and not vb[0].any()
        assert torch.equal(vb[1], _keep(half)(v[1]).float())
        h.store_kv_dev(0, [0], [30], 70, k[:1, :, :70].contiguous(), v[:1, :, :70].contiguous(), fa.F16)
        h.load_kv_dev(0, [0, 1], [30, 30], 600, kb2 := torch.ones(2, 4, 600, 128, device="cuda"), torch.empty(2, 4, 600, 128, device="cuda"), fa.F32)
        assert torch.equal(kb2[0, :, :70], _keep(half)(k[0, :, :70]).float()) and not kb2[0, :, 98:].any()
        assert torch.equal(kb2[1], kb[1, :, 30:630])
        k16, v16 = h.read_kv(0, 0, 128, 300)
        assert not k16.any() and not v16.any()


# ------------------------------------------------------------------------------------------------ decode
def _history(torch, seed, n, rows):
    k = _rand(torch, seed, n, 4, rows, 128) * (0.5 + torch.rand(4, 1, 128, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)))
    return k.to(torch.float16), (_rand(torch, seed + 1, n, 4, rows, 128) + 0.25).to(torch.float16)


def _decode_want(torch, qkv, w, rope, is_swa, first, positions, k, v, half=False):
    kept = _keep(half)
    outs, rooms, k_new, v_new = [], [], [], []
    for i, p in enumerate(positions):
        at = torch.tensor([p], device="cuda")
        q, kn, vn = ref.split_rows(qkv[i:i + 1], w, at, rope)
        key_at = torch.arange(p + 1, device="cuda")
        keys = torch.cat((kept(k[i, :, :p]), kn.double().transpose(0, 1)), 1)
        vals = torch.cat((kept(v[i, :, :p]), vn.double().transpose(0, 1)), 1)
        o, r = ref.attend(q, keys, vals, ref.visible(at, key_at, is_swa, first), w[2])
        outs.append(o)
        rooms.append(r)
        k_new.append(kn)
        v_new.append(vn)
    return torch.cat(outs), torch.cat(rooms), torch.cat(k_new), torch.cat(v_new)


POSITIONS = [0, 1, 2, 63, 64, 65, 127, 128, 300, 511, 512, 513, 514, 575, 576, 640, 1023, 1024, 1025, 1100, 1536, 2047, 2500]


@gpu
@pytest.mark.parametrize("in_type,out_type", [("float32", "float32"), ("bfloat16", "bfloat16"), ("float32", "bfloat16")])
@pytest.mark.parametrize("is_swa,rope,paged,first,half", [
    (False, False, False, 0, False), (False, True, True, 0, False), (True, True, False, 0, False), (True, True, False, 1, False),
    (True, True, False, 4, False), (True, False, False, 33, False), (True, True, False, 64, False),
    (True, True, False, 1, True), (True, False, False, 33, True), (True, True, False, 64, True)])
def test_decode(fa, in_type, out_type, is_swa, rope, paged, first, half):
    import torch

    n, dt, ot = len(POSITIONS), getattr(torch, in_type), getattr(torch, out_type)
    k, v = _history(torch, 11, n, 2500)
    qkv = _rand(torch, 13, n, 5120, dtype=dt)
    h, w = _open(fa, torch, is_swa, rope, n + 1, 2600, kv_pages=41 * n if paged else 0, first_tokens=first, half=half)
    with h:
        seqs = [(5 * i + 1) % (n + 1) for i in range(n)]
        assert len(set(seqs)) == n
        for i, p in enumerate(POSITIONS):
            if p:
                h.store_kv_dev(0, [seqs[i]], [0], p, k[i:i + 1, :, :p].contiguous(), v[i:i + 1, :, :p].contiguous(), fa.F16)
            h.set_pos(seqs[i], p)
        out = torch.full((n + 1, 4096), 777.0, device="cuda", dtype=ot)
        h.decode_dev(0, seqs, qkv, _kind(fa, torch, dt), out, _kind(fa, torch, ot))
        h.check()
        want, room, k_new, v_new = _decode_want(torch, qkv, w, rope, is_swa, first, POSITIONS, k, v, half)
        ref.assert_near(out[:n], want, room, f"decode {is_swa} {paged} {first}")
        for i, p in enumerate(POSITIONS):  # each sequence by itself, the short ones above all
            ref_rel = float((out[i].double() - want[i].reshape(-1)).norm() / want[i].norm())
            assert ref_rel <= (4e-3 if ot == torch.bfloat16 else 2e-3), (p, ref_rel)
        assert (out[n] == 777).all()  # rows behind the last sequence
        kb, vb = torch.empty(2, n, 4, 1, 128, device="cuda")
        h.load_kv_dev(0, seqs, POSITIONS, 1, kb, vb, fa.F32)
        assert torch.equal(vb[:, :, 0], _keep(half)(v_new).float())
        _check_keys(kb[:, :, 0], k_new, half, "stored keys")
        if first:  # new tokens below `first` are among the first tokens' rows too
            for i, p in enumerate(POSITIONS):
                if p < first:
                    _, v16 = h.read_kv(0, seqs[i], 1024 + p, 1)
                    assert np.array_equal(v16[:, 0].view(np.float16), _keep(half)(v_new[i]).float().to(torch.float16).cpu().numpy())


@gpu
@pytest.mark.parametrize("n,pos,target", [(700, 130, 0), (1, 1040, 0), (30, 1700, 0), (1, 9000, 0), (2, 40000, 0), (64, 700, 0), (70, 513, 7), (1, 70000, 2000), (200, 90, 0)])
def test_decode_splits(fa, n, pos, target):
    """Long ranges cut into many items and merged in two levels, batches that fill the GPU, work lists that are uploaded."""
    import torch

    k, v = _history(torch, 17, n, pos)
    qkv = _rand(torch, 19, n, 5120)
    h, w = _open(fa, torch, False, False, n, pos + 8)
    with h:
        if target:
            h.set_target_items(target)
        h.store_kv_dev(0, range(n), [0] * n, pos, k, v, fa.F16)
        positions = [pos - (i % 5) * 13 for i in range(n)]
        for i, p in enumerate(positions):
            h.set_pos(i, p)
        out = torch.empty(n, 4096, device="cuda")
        again = torch.empty_like(out)
        h.decode_dev(0, range(n), qkv, fa.F32, out, fa.F32)
        h.decode_dev(0, range(n), qkv, fa.F32, again, fa.F32)
        h.check()
        some = list(range(0, n, max(1, n // 8)))
        want, room, _, _ = _decode_want(torch, qkv[some], w, False, False, 0, [positions[i] for i in some], k[some], v[some])
        ref.assert_near(out[some], want, room, "split decode")
        assert torch.equal(out, again)


@gpu
@pytest.mark.parametrize("is_swa,first", [(False, 0), (True, 0), (True, 4)])
def test_what_masked_rows_hold_does_not_matter(fa, is_swa, first):
    """Rows a query does not see (taken back, or left in the ring) may hold anything, NaN among it."""
    import torch

    p, n_ctx = 1100, 2200
    k, v = _history(torch, 23, 1, p)
    qkv = _rand(torch, 25, 1, 5120)
    outs = []
    for fill in (None, math.nan, 6e4):
        h, w = _open(fa, torch, is_swa, True, 1, n_ctx, first_tokens=first)
        with h:
            if fill is not None:
                junk = torch.full((1, 4, 1024, 128), fill, device="cuda")
                junk[..., ::3] = -fill
                h.store_kv_dev(0, [0], [0], 1024, junk, junk, fa.F32)
                h.store_kv_dev(0, [0], [1024], 1024, junk, junk, fa.F32)
            rows = p if not is_swa else 512
            if first:
                h.store_kv_dev(0, [0], [0], first, k[:, :, :first].contiguous(), v[:, :, :first].contiguous(), fa.F16)
            h.store_kv_dev(0, [0], [p - rows], rows, k[:, :, p - rows:].contiguous(), v[:, :, p - rows:].contiguous(), fa.F16)
            h.set_pos(0, p)
            out = torch.empty(1, 4096, device="cuda")
            h.decode_dev(0, [0], qkv, fa.F32, out, fa.F32)
            h.check()
            outs.append(out)
    want, room, _, _ = _decode_want(torch, qkv, w, True, is_swa, first, [p], k, v)
    ref.assert_near(outs[0], want, room, "masked")
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


@gpu
def test_a_key_that_is_not_a_number_is_seen(fa):
    import torch

    k, v = _history(torch, 27, 2, 300)
    k[1, 2, 100, 7] = math.nan
    h, _ = _open(fa, torch, False, False, 2, 400)
    with h:
        h.store_kv_dev(0, [0, 1], [0, 0], 300, k, v, fa.F16)
        for s in range(2):
            h.set_pos(s, 300)
        out = torch.empty(2, 4096, device="cuda")
        h.decode_dev(0, [0, 1], _rand(torch, 28, 2, 5120), fa.F32, out, fa.F32)
        h.check()
        bad = torch.isnan(out).view(2, 4, 1024)
        assert bad[1, 2].all() and not bad[0].any() and not bad[1, [0, 1, 3]].any()


@gpu
def test_extreme_scales_of_values(fa):
    """Small values keep their relative accuracy, large ones do not overflow."""
    import torch

    for scale in (2.0**-9, 2.0**12):
        k, v = _history(torch, 29, 1, 800)
        v = (v.float() * scale).to(torch.float16)
        qkv = _rand(torch, 31, 1, 5120)
        qkv[:, 36 * 128:] *= scale
        h, w = _open(fa, torch, False, False, 1, 900)
        with h:
            h.store_kv_dev(0, [0], [0], 800, k, v, fa.F16)
            h.set_pos(0, 800)
            out = torch.empty(1, 4096, device="cuda")
            h.decode_dev(0, [0], qkv, fa.F32, out, fa.F32)
            h.check()
            want, room, _, _ = _decode_want(torch, qkv, w, False, False, 0, [800], k, v)
            ref.assert_near(out, want, room + scale * 2.0**-10, "scaled values")


# ------------------------------------------------------------------------------------------------ prefill
@gpu
@pytest.mark.parametrize("in_type,out_type", [("float32", "float32"), ("bfloat16", "bfloat16")])
@pytest.mark.parametrize("is_swa,first,paged,half", [
    (False, 0, False, False), (False, 0, True, False), (True, 0, False, False), (True, 1, False, False), (True, 20, False, False),
    (True, 64, False, False), (True, 3, False, True), (True, 64, False, True)])
@pytest.mark.parametrize("past,tokens", [(0, 1), (0, 33), (0, 700), (63, 2), (510, 7), (700, 130), (1500, 512), (40, 600), (2000, 1), (2000, 700), (2400, 512), (1900, 1100)])
def test_prefill(fa, in_type, out_type, is_swa, first, paged, half, past, tokens):
    import torch

    dt, ot = getattr(torch, in_type), getattr(torch, out_type)
    k, v = _history(torch, 33, 1, max(past, 1))
    qkv = _rand(torch, 35, tokens, 5120, dtype=dt)
    h, w = _open(fa, torch, is_swa, True, 3, 3000, kv_pages=60 if paged else 0, first_tokens=first, half=half)
    kept = _keep(half)
    with h:
        if past:
            h.store_kv_dev(0, [1], [0], past, k, v, fa.F16)
        h.set_pos(1, past)
        out = torch.full((tokens + 1, 4096), 777.0, device="cuda", dtype=ot)
        h.prefill_dev(0, 1, tokens, qkv, _kind(fa, torch, dt), out, _kind(fa, torch, ot))
        h.check()
        at = torch.arange(past, past + tokens, device="cuda")
        q, kn, vn = ref.split_rows(qkv, w, at, True)
        keys = torch.cat((kept(k[0, :, :past]), kn.double().transpose(0, 1)), 1)
        vals = torch.cat((kept(v[0, :, :past]), vn.double().transpose(0, 1)), 1)
        want, room = ref.attend(q, keys, vals, ref.visible(at, torch.arange(past + tokens, device="cuda"), is_swa, first), w[2])
        ref.assert_near(out[:tokens], want, room, "prefill")
        assert (out[tokens] == 777).all()
        rows = min(tokens, 1024) if is_swa else tokens
        kb, vb = torch.empty(2, 4, rows, 128, device="cuda")
        h.load_kv_dev(0, [1], [past + tokens - rows], rows, kb, vb, fa.F32)
        assert torch.equal(vb, kept(vn[-rows:]).transpose(0, 1).float())
        _check_keys(kb, kn[-rows:].transpose(0, 1), half, "prefilled keys")
        for p in range(min(first, past + tokens)):
            want_v = kept(vn[p - past]) if p >= past else kept(v[0, :, p])
            _, v16 = h.read_kv(0, 1, 1024 + p, 1)
            assert np.array_equal(v16[:, 0].view(np.float16), want_v.float().to(torch.float16).cpu().numpy())


@gpu
@pytest.mark.parametrize("in_type", ["float32", "bfloat16"])
@pytest.mark.parametrize("is_swa,first,half", [(False, 0, False), (True, 0, False), (True, 4, False), (True, 64, True)])
@pytest.mark.parametrize("past,tokens", [(600, 300), (0, 700), (20, 560), (1400, 40)])
def test_prefill_keeps_infinities_from_queries_that_do_not_see_them(fa, in_type, is_swa, first, half, past, tokens):
    """Values that are not finite, in padding behind the prompt, in one row of it, in the window's history and in a first
    token: queries that see one get NaN in its heads, all others what they get without them."""
    import torch

    dt = getattr(torch, in_type)
    k, v = _history(torch, 45, 1, max(past, 1))
    qkv = _rand(torch, 47, tokens, 5120, dtype=dt)
    bad_at = {head: set() for head in range(4)}
    v[0, 2, -1, 3], v[0, 2, -1, 4] = 65504, -65504  # d rounds up: lo + 15 d is 65536 in a 4-bit cache
    k2, v2, qkv2 = k.clone(), v.clone(), qkv.clone()
    mid, pad = tokens // 3, tokens - 10
    qkv2[mid, 4608 + 128 + 77] = math.inf  # V of KV head 1, one value
    bad_at[1].add(past + mid)
    qkv2[pad:] = math.nan
    for head in range(4):
        bad_at[head].update(range(past + pad, past + tokens))
    if past > 512:
        v2[0, 0, past - 500, 5] = -math.inf
        bad_at[0].add(past - 500)
    if first and past:
        v2[0, 3, 1, 127] = math.nan
        bad_at[3].add(1)
    outs = []
    for kk, vv, x in ((k, v, qkv), (k2, v2, qkv2)):
        h, _ = _open(fa, torch, is_swa, True, 1, past + tokens, first_tokens=first, half=half)
        with h:
            if past:
                h.store_kv_dev(0, [0], [0], past, kk, vv, fa.F16)
            h.set_pos(0, past)
            out = torch.empty(tokens, 4096, device="cuda")
            h.prefill_dev(0, 0, tokens, x, _kind(fa, torch, dt), out, fa.F32)
            h.check()
            outs.append(out.view(tokens, 4, 1024))
    assert torch.isfinite(outs[0]).all()
    at, keys = torch.arange(past, past + tokens, device="cuda"), torch.arange(past + tokens, device="cuda")
    sees = ref.visible(at, keys, is_swa, first)
    for head in range(4):
        hit = sees[:, sorted(bad_at[head])].any(1)
        assert torch.isnan(outs[1][hit, head]).all(), head
        assert torch.equal(outs[1][~hit, head], outs[0][~hit, head]), head


# ------------------------------------------------------------------------------------------------ together
@gpu
@pytest.mark.parametrize("is_swa,first,paged,half", [(False, 0, True, False), (True, 4, False, False), (True, 4, False, True)])
def test_a_conversation(fa, is_swa, first, paged, half):
    """Prompt in two chunks, tokens one at a time beside another sequence, a rollback, and on: the cache that the calls
    left is what the next one sees, against the 64-bit statement run over the values that it holds."""
    import torch

    P1, P2, N = 590, 100, 40
    h, w = _open(fa, torch, is_swa, True, 2, 1400, kv_pages=44 if paged else 0, first_tokens=first, half=half)
    qkv = _rand(torch, 41, P1 + P2 + N, 5120)
    other = _rand(torch, 43, P1 + P2 + N, 5120)
    with h:
        def held(seq, upto):
            start = max(0, upto - 900)
            k, v = torch.zeros(2, 4, upto, 128, device="cuda")
            kb, vb = torch.empty(2, 4, upto - start, 128, device="cuda")
            h.load_kv_dev(0, [seq], [start], upto - start, kb, vb, fa.F32)
            k[:, start:], v[:, start:] = kb, vb
            return k.double(), v.double()

        out = torch.empty(P1, 4096, device="cuda")
        h.prefill_dev(0, 0, P1, qkv, fa.F32, out, fa.F32)
        h.advance([0], P1)
        k, v = held(0, P1)
        out2 = torch.empty(P2, 4096, device="cuda")
        h.prefill_dev(0, 0, P2, qkv[P1:].contiguous(), fa.F32, out2, fa.F32)
        at = torch.arange(P1, P1 + P2, device="cuda")
        q, kn, vn = ref.split_rows(qkv[P1:P1 + P2], w, at, True)
        want, room = ref.attend(q, torch.cat((k, kn.double().transpose(0, 1)), 1), torch.cat((v, vn.double().transpose(0, 1)), 1),
                                ref.visible(at, torch.arange(P1 + P2, device="cuda"), is_swa, first), w[2])
        ref.assert_near(out2, want, room, "second chunk")
        h.advance([0], P2)
        first_run = []
        for step in range(2):
            for t in range(N):
                p = P1 + P2 + t
                assert h.pos(0) == p
                k, v = held(0, p)
                rows = torch.stack((qkv[p], other[h.pos(1)]))
                o = torch.empty(2, 4096, device="cuda")
                h.decode_dev(0, [0, 1], rows, fa.F32, o, fa.F32)
                at = torch.tensor([p], device="cuda")
                q, kn, vn = ref.split_rows(qkv[p:p + 1], w, at, True)
                want, room = ref.attend(q, torch.cat((k, kn.double().transpose(0, 1)), 1), torch.cat((v, vn.double().transpose(0, 1)), 1),
                                        ref.visible(at, torch.arange(p + 1, device="cuda"), is_swa, first), w[2])
                ref.assert_near(o[:1], want, room, f"token {p}")
                if step == 0:
                    first_run.append(o[0].clone())
                else:
                    assert torch.equal(o[0], first_run[t])  # the same tokens after the rollback
                h.advance([0, 1])
            if step == 0:
                assert h.truncate(0, P1 + P2) == 0
        h.check()


@gpu
def test_host_buffers_blocks_and_other_streams(fa, fo):
    """The host-buffer calls and the attention blocks with projections on a 4-bit handle give what the device calls give;
    a side stream works like the default one."""
    import torch

    T, n = 70, 2
    kinds = [(True, True), (False, False)]
    sw = fo.stack_weights(3, 2, 256, 128, kinds)
    outs = []
    for how in ("host", "pinned", "dev"):
        with fa.Attn([True, False], [True, False], n, 200, kv_format=fa.KV_INT4, first_tokens=4) as h:
            for il in range(2):
                h.set_layer(il, sw["q_norm"][il], sw["k_norm"][il], sw["sinks"][il])
                h.set_projections(il, sw["attn_norm"][il], *(fo.to_bf16_bits(sw[x][il]) for x in ("wq", "wk", "wv", "wo")))
            qkv = _rand(torch, 51, T + 1, 5120)
            out, row = torch.empty(T, 4096), torch.empty(1, 4096)
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            for il in range(2):
                if how != "dev":
                    rows = qkv.cpu()
                    h.prefill(il, 0, T, rows[:T].contiguous(), fa.F32, out, fa.F32)
                else:
                    d = torch.empty(T, 4096, device="cuda")
                    h.prefill_dev(il, 0, T, qkv, fa.F32, d, fa.F32, side.cuda_stream)
                    side.synchronize()
                    out.copy_(d)
            h.advance([0], T)
            for il in range(2):
                if how != "dev":
                    rows = qkv[T:].cpu()
                    if how == "pinned":
                        rows, row = rows.pin_memory(), row.pin_memory()
                    h.decode(il, [0], rows, fa.F32, row, fa.F32)
                else:
                    d = torch.empty(1, 4096, device="cuda")
                    h.decode_dev(il, [0], qkv[T:].contiguous(), fa.F32, d, fa.F32, side.cuda_stream)
                    side.synchronize()
                    row.copy_(d)
            x = torch.from_numpy(sw["embd"][np.arange(T) % 128]).cuda().contiguous()
            for il in range(2):
                h.prefill_block_dev(il, 1, T, x)
            h.advance([1], T)
            y = x[-1:].clone()
            for il in range(2):
                h.decode_block_dev(il, [1], y)
            h.check()
            outs.append([t.cpu().clone() for t in (out, row, x, y)])
    for a, b, c in zip(*outs):
        assert torch.isfinite(a).all() and torch.equal(a, b) and torch.equal(a, c)


@gpu
def test_captured_and_replayed(fa):
    """Store, decode and load in one captured graph, replayed with other rows in the same buffers."""
    import torch

    h, w = _open(fa, torch, True, True, 3, 3000, first_tokens=4)
    with h:
        k, v = _history(torch, 61, 3, 1024)
        rows, out = torch.zeros(3, 5120, device="cuda"), torch.empty(3, 4096, device="cuda")
        kb, vb = torch.empty(2, 3, 4, 1, 128, device="cuda")
        ring_k, ring_v = k.clone(), v.clone()
        for s in range(3):
            h.set_pos(s, 1024)

        def step(stream):
            h.store_kv_dev(0, [0, 1, 2], [0, 0, 0], 1024, ring_k, ring_v, fa.F16, stream)
            h.decode_dev(0, [0, 1, 2], rows, fa.F32, out, fa.F32, stream)
            h.load_kv_dev(0, [0, 1, 2], [1024] * 3, 1, kb, vb, fa.F32, stream)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(side.cuda_stream)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(torch.cuda.current_stream().cuda_stream)
        for seed in (63, 65):
            rows.copy_(_rand(torch, seed, 3, 5120))
            k2, v2 = _history(torch, seed, 3, 1024)
            ring_k.copy_(k2)
            ring_v.copy_(v2)
            out.zero_()
            g.replay()
            torch.cuda.synchronize()
            want, room, _, v_new = _decode_want(torch, rows, w, True, True, 4, [1024] * 3, k2, v2)
            ref.assert_near(out, want, room, "replayed")
            assert torch.equal(vb[:, :, 0], ref.kept(v_new).float())
        h.check()


@gpu
def test_a_graph_outlives_larger_calls(fa):
    """Graphs of one handle, one of them a launch of several rounds, replayed in turn and after larger batches of the
    handle, give what they gave."""
    import torch

    n, p = 300, 1500
    k, v = _history(torch, 93, 1, p)
    rows = _rand(torch, 95, n, 5120)
    h, w = _open(fa, torch, False, True, n, 1600)
    with h:
        for s in range(n):
            h.store_kv_dev(0, [s], [0], p, k, v, fa.F16)
            h.set_pos(s, p)
        outs, many = torch.empty(2, 2, 4096, device="cuda"), torch.empty(n - 50, 4096, device="cuda")
        side = torch.cuda.Stream()
        graphs = []
        for i in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):  # (no call of the handle before the first capture)
                h.decode_dev(0, [0, 1][: i + 1], rows, fa.F32, outs[i], fa.F32, torch.cuda.current_stream().cuda_stream)
            graphs.append(g)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            h.decode_dev(0, range(n - 50), rows, fa.F32, many, fa.F32, torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
        big = torch.empty(n, 4096, device="cuda")
        got = []
        for _ in range(3):
            outs.fill_(777)
            for g in graphs:
                g.replay()
            got.append(outs.clone())
            h.decode_dev(0, range(n - 50), rows, fa.F32, big, fa.F32)
            assert torch.equal(many, big[: n - 50])
            many.zero_()
            h.decode_dev(0, range(n), rows, fa.F32, big, fa.F32)
        torch.cuda.synchronize()
        h.check()
        want, room, _, _ = _decode_want(torch, rows[:2], w, True, False, 0, [p, p], k.expand(2, -1, -1, -1), v.expand(2, -1, -1, -1))
        ref.assert_near(got[0][1], want, room, "graph")
        ref.assert_near(got[0][0, :1], want[:1], room[:1], "graph")
        assert (got[0][0, 1] == 777).all()
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


@gpu
@pytest.mark.parametrize("half,is_swa,first", [(False, False, 0), (False, True, 0), (True, True, 4)])
def test_captures_refused(fa, half, is_swa, first):
    """A prefill is not captured, nor a call that takes pages; the capture goes on and takes the calls that are allowed."""
    import torch

    paged = not is_swa
    x, out = _rand(torch, 97, 40, 5120), torch.empty(40, 4096, device="cuda")
    k, v = _history(torch, 99, 2, 64)
    h, _ = _open(fa, torch, is_swa, True, 2, 400, kv_pages=6 if paged else 0, first_tokens=first, half=half)
    with h:
        h.store_kv_dev(0, [0], [0], 64, k[:1], v[:1], fa.F16)
        h.set_pos(0, 63)
        h.set_pos(1, 0)
        h.decode_dev(0, [0], x, fa.F32, out, fa.F32)
        want = out[0].clone()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            st = torch.cuda.current_stream().cuda_stream
            with pytest.raises(fa.FlintAttnError, match="captured"):
                h.prefill_dev(0, 0, 40, x, fa.F32, out, fa.F32, st)
            if paged:
                for call in (lambda: h.decode_dev(0, [0, 1], x, fa.F32, out, fa.F32, st),
                             lambda: h.prefill_dev(0, 1, 1, x, fa.F32, out, fa.F32, st),
                             lambda: h.store_kv_dev(0, [0], [60], 10, k, v, fa.F16, st)):
                    with pytest.raises(fa.FlintAttnError, match="captured"):
                        call()
                assert h.pages_free() == 5
            h.decode_dev(0, [0], x, fa.F32, out, fa.F32, st)
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        h.check()
        assert torch.equal(out[0], want) and not out[1:].any()


@gpu
def test_positions_past_32_bits_of_bytes(fa):
    """A cache of more than 4 GB: block addresses of the last sequence lie beyond 32 bits."""
    import torch

    n, n_ctx = 56, 131072  # 56 x 4 x 2048 blocks x 10240 B = 4.7 GB
    h, w = _open(fa, torch, False, False, n, n_ctx)
    with h:
        k, v = _history(torch, 71, 2, 300)
        h.store_kv_dev(0, [0, n - 1], [0, 0], 300, k, v, fa.F16)
        far_k, far_v = _history(torch, 73, 1, 3)
        h.store_kv_dev(0, [n - 1], [n_ctx - 3], 3, far_k, far_v, fa.F16)
        for s in (0, n - 1):
            h.set_pos(s, 300)
        rows = _rand(torch, 75, 2, 5120)
        out = torch.empty(2, 4096, device="cuda")
        h.decode_dev(0, [0, n - 1], rows, fa.F32, out, fa.F32)
        want, room, _, _ = _decode_want(torch, rows, w, False, False, 0, [300, 300], k, v)
        ref.assert_near(out, want, room, "far sequence")
        kb, vb = torch.empty(2, 1, 4, 3, 128, device="cuda")
        h.load_kv_dev(0, [n - 1], [n_ctx - 3], 3, kb, vb, fa.F32)
        assert torch.equal(kb, ref.kept(far_k).float()) and torch.equal(vb, ref.kept(far_v).float())


@gpu
def test_serving_loop_on_pages(fa):
    """Requests that join, decode together and leave, on a pool too small for all of them at once: pages that held other
    sequences (not-a-number rows among them) serve the next ones, and each request gets what it gets alone."""
    import torch

    from flint_mac_b200 import ContinuousBatcher

    torch.manual_seed(5)
    reqs = {i: (40 + 97 * i, 5 + i) for i in range(6)}  # prompt tokens, new tokens
    rows = {i: _rand(torch, 100 + i, p + n, 5120) for i, (p, n) in reqs.items()}
    alone = {}
    for i, (p, n) in reqs.items():
        h, _ = _open(fa, torch, False, True, 1, p + n)
        with h:
            out = torch.empty(p + n, 4096, device="cuda")
            h.prefill_dev(0, 0, p, rows[i], fa.F32, out, fa.F32)
            h.advance([0], p)
            for t in range(p, p + n):
                h.decode_dev(0, [0], rows[i][t:t + 1].contiguous(), fa.F32, out[t:t + 1], fa.F32)
                h.advance([0])
            h.check()
            alone[i] = out
    h, _ = _open(fa, torch, False, True, 3, 1024, kv_pages=18)
    with h:
        junk = torch.full((1, 4, 1024, 128), math.nan, device="cuda")
        for s in range(3):  # every page has held something else
            h.store_kv_dev(0, [s], [0], 6 * 64, junk[:, :, :6 * 64].contiguous(), junk[:, :, :6 * 64].contiguous(), fa.F32)
        for s in range(3):
            h.seq_release(s)
        assert h.pages_free() == 18
        b = ContinuousBatcher(max_seqs=3, kv_pages=18, n_ctx=1024)
        for i, (p, n) in reqs.items():
            b.submit(i, p, n)
        got = {i: torch.empty_like(alone[i]) for i in reqs}
        steps = 0
        while not b.idle:
            plan = b.next_step()
            for r in plan.admit:
                p = reqs[r.req_id][0]
                h.prefill_dev(0, r.slot, p, rows[r.req_id], fa.F32, got[r.req_id], fa.F32)
                h.advance([r.slot], p)
            if plan.decode:
                slots = [r.slot for r in plan.decode]
                at = [h.pos(s) for s in slots]
                x = torch.stack([rows[r.req_id][t] for r, t in zip(plan.decode, at)])
                o = torch.empty(len(slots), 4096, device="cuda")
                h.decode_dev(0, slots, x, fa.F32, o, fa.F32)
                h.advance(slots)
                for r, t, y in zip(plan.decode, at, o):
                    got[r.req_id][t] = y
            for r in b.complete(plan):
                h.seq_release(r.slot)
            steps += 1
            assert steps < 200
        h.check()
        assert h.pages_free() == 18
    for i in reqs:
        # the same values, split and summed in another order: 32-bit sums and the probabilities' half rounding
        err = float((got[i] - alone[i]).norm() / alone[i].norm())
        assert err <= 1e-3, (i, err)


@gpu
def test_windows_of_many_sequences_on_half_precision_rings(fa):
    """Work lists of every capacity of the half-precision kernel with first tokens, uploaded ones among them."""
    import torch

    first, n_ctx = 16, 1400
    for n in (1, 12, 40, 120, 200):  # 4 n items
        k, v = _history(torch, 81, n, 1100)
        qkv = _rand(torch, 83, n, 5120)
        positions = [1100 - (37 * i) % 700 for i in range(n)]
        h, w = _open(fa, torch, True, True, n, n_ctx, half=True, first_tokens=first)
        with h:
            h.store_kv_dev(0, range(n), [0] * n, 1100, k, v, fa.F16)
            for i, p in enumerate(positions):
                h.set_pos(i, p)
            # positions whose ring slots hold later rows are stored again, as a shorter sequence would have left them
            for i, p in enumerate(positions):
                h.store_kv_dev(0, [i], [0], p, k[i:i + 1, :, :p].contiguous(), v[i:i + 1, :, :p].contiguous(), fa.F16)
            out = torch.empty(n, 4096, device="cuda")
            h.decode_dev(0, range(n), qkv, fa.F32, out, fa.F32)
            h.check()
            some = list(range(0, n, max(1, n // 9)))
            want, room, _, _ = _decode_want(torch, qkv[some], w, True, True, first, [positions[i] for i in some], k[some], v[some], True)
            ref.assert_near(out[some], want, room, f"{n} windows")
