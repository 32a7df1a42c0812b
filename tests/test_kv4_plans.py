"""Host-side plans of the calls over 4-bit caches: what they cover and what they refuse (no GPU)."""
import pytest


@pytest.fixture(scope="module")
def fa():
    import flint_mac_b200 as fa

    fa.load_library()
    return fa


@pytest.mark.parametrize("first,fine", [(-1, False), (0, True), (64, True), (65, False), (1 << 30, False)])
@pytest.mark.parametrize("is_swa", [False, True])
def test_decode_plan_takes_the_first_tokens_a_handle_can_keep(fa, is_swa, first, fine):
    if fine:
        assert len(fa.plan_decode_int4([5, 2000], is_swa, first)) >= 2
    else:
        with pytest.raises(fa.FlintAttnError):
            fa.plan_decode_int4([5, 2000], is_swa, first)


def _sizes():
    import random

    rng = random.Random(5)
    fixed = [(1, 0), (2, 0), (31, 1), (32, 128), (33, 127), (512, 16384), (640, 6000), (1300, 3000), (700, 2000), (512, 2400), (1100, 1900),
             (5000, 100), (5120, 1), (6000, 0), (40000, 0), (3, 131069), (100, 1 << 20)]
    return fixed + [(int(2 ** rng.uniform(0, 13)), int(2 ** rng.uniform(0, 17)) - 1) for _ in range(400)]


def test_prefill_plan_covers_every_tile_once(fa):
    """Whatever the sizes: each unit's tiles in one piece each, its parts numbered from 0 on in the order of its keys, every CTA's
    pieces together and in order, no CTA's load far from the others', and no piece below four tiles but whole units."""
    import numpy as np

    seen = 0
    for n_sm in (1, 2, 3, 16, 147, 148, 160):
        for n_tok, p0 in _sizes():
            pcs = fa.plan_prefill_int4(n_tok, p0, n_sm)
            if len(pcs) == 0:
                continue
            seen += 1
            cta, unit, part, t0, t1, tiles, q0, kvh = pcs.T
            n_units = (n_tok + 31) // 32 * 4
            assert len(pcs) <= 640 and cta.min() >= 0 and cta.max() < n_sm and (np.diff(cta) >= 0).all()
            assert set(unit) == set(range(n_units)) and (np.diff(unit) >= 0).all() and (t1 > t0).all()
            begins = np.flatnonzero(np.diff(unit, prepend=-1))
            ends = np.append(begins[1:], len(pcs)) - 1
            assert (t0[begins] == 0).all() and (t1[ends] == tiles[ends]).all() and (part[begins] == 0).all()
            inside = np.setdiff1d(np.arange(len(pcs)), begins)
            assert (t0[inside] == t1[inside - 1]).all() and (part[inside] == part[inside - 1] + 1).all()
            assert part.max() >= 1  # something is cut, or it would not be this plan
            short = (t1 - t0 < 4) & (t1 - t0 < tiles)
            assert not short.any(), (n_tok, p0, n_sm, pcs[short])
            # a unit's tiles reach its last query; the four KV heads of a block of queries are alike
            last = np.minimum(q0 + 31, p0 + n_tok - 1)
            assert (tiles == last // 128 + 1).all()
            assert sorted(zip(q0[begins], kvh[begins])) == sorted((p0 + 32 * b, h) for b in range(n_units // 4) for h in range(4))
            # A CTA's stretch ends where total * (cta + 1) / n_sm tiles are handed out, rounded down (1), up to three tiles before
            # where less than four are left of it, up to three behind where less than four would be left of the unit.
            load = np.bincount(cta, t1 - t0, n_sm)
            assert load.max() <= load.sum() / n_sm + 7, (n_tok, p0, n_sm, load)
    assert seen > 300


@pytest.mark.parametrize("n_tok,p0,n_sm", [(0, 5, 148), (-1, 5, 148), (5, -1, 148), (5, 5, 0), (2147483647, 1, 148), (2147483647, 0, 148), (1, 2147483647, 148)])
def test_prefill_plan_refuses(fa, n_tok, p0, n_sm):
    with pytest.raises(fa.FlintAttnError):
        fa.plan_prefill_int4(n_tok, p0, n_sm)


@pytest.mark.parametrize("n_tok,p0,n_sm", [(6000, 0, 148), (512, 16384, 161), (20, 30, 148)])
def test_prefill_plan_leaves_units_alone(fa, n_tok, p0, n_sm):
    """More units than a work list holds, more multiprocessors than it counts, nothing worth a cut."""
    assert len(fa.plan_prefill_int4(n_tok, p0, n_sm)) == 0
