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
