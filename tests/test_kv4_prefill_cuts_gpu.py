"""Prefills behind a 4-bit cache whose units are cut at any key tile, so that all CTAs end together."""
import pytest

import kv4_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def fa():
    import flint_mac_b200 as fa

    fa.load_library()
    return fa


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("tokens,past", [(300, 600), (512, 1500), (700, 2000), (640, 6000), (1300, 3000)])
def test_cut_units(fa, paged, tokens, past):
    import torch

    n_sm = torch.cuda.get_device_properties(0).multi_processor_count
    pieces = fa.plan_prefill_int4(tokens, past, n_sm)
    assert len(pieces) > 0 and pieces[:, 2].max() >= 1  # the launch makes its list with the same call
    g = torch.Generator(device="cuda").manual_seed(91)
    k, v = torch.randn(2, 1, 4, past, 128, device="cuda", generator=g).to(torch.float16)
    qkv = torch.randn(tokens, 5120, device="cuda", generator=g)
    c = torch.Generator().manual_seed(3)
    w = (1 + 0.1 * torch.randn(128, generator=c), 1 + 0.1 * torch.randn(128, generator=c), torch.randn(32, generator=c))
    with fa.Attn([False], [True], 1, past + tokens, kv_format=fa.KV_INT4, kv_pages=(past + tokens) // 64 + 1 if paged else 0) as h:
        h.set_layer(0, *(x.numpy() for x in w))
        h.store_kv_dev(0, [0], [0], past, k, v, fa.F16)
        h.set_pos(0, past)
        out = torch.full((2, tokens, 4096), 777.0, device="cuda")
        for o in out:
            h.prefill_dev(0, 0, tokens, qkv, fa.F32, o, fa.F32)
        h.check()
    assert torch.equal(out[0], out[1])
    at = torch.arange(past, past + tokens, device="cuda")
    q, kn, vn = ref.split_rows(qkv, tuple(x.cuda() for x in w), at, True)
    keys = torch.cat((ref.kept(k[0]), kn.double().transpose(0, 1)), 1)
    vals = torch.cat((ref.kept(v[0]), vn.double().transpose(0, 1)), 1)
    for i in range(0, tokens, 128):  # (the statement's scores of all queries at once would take 10 GB)
        seen = ref.visible(at[i:i + 128], torch.arange(past + tokens, device="cuda"), False, 0)
        want, room = ref.attend(q[i:i + 128], keys, vals, seen, w[2].cuda())
        ref.assert_near(out[0, i:i + 128], want, room, f"queries from {i}")
