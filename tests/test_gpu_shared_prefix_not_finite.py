"""Shared-prefix decode with NaN in the query and in the cache's block scales."""
import numpy as np
import pytest
import torch

from test_gpu_shared_prefix import even, make, rel_fro, run

pytestmark = pytest.mark.gpu

PLANS = [(1, 1), (2, 2), (3, 1), (0, 1), (0, 3)]
NAN = float("nan")


@pytest.mark.parametrize("d,g,page", [(128, 8, 16), (128, 6, 64), (256, 4, 32), (256, 8, 128)])
@pytest.mark.parametrize("lens", [[400, 350, 0, 291, 200], [500], [100]])
def test_nan_blocks_of_the_query_count_as_zeros(cuda_device, d, g, page, lens):
    """The quantisers take a block of NaNs with scale zero, as the plain decode's prologue does: bit for bit the result of
    zeros in its place, whatever the plan, with own tokens and without."""
    kv, q, t = make(cuda_device, lens, 290, 2, g, d, page)
    for heads in ("one block", "one head", "all"):
        zero, bad = t["q"].clone(), t["q"].clone()
        for x, value in ((zero, 0.0), (bad, NAN)):
            if heads == "one block":
                x[:, 1, 16:32] = value
                x[:, g, d - 16:] = value
            elif heads == "one head":
                x[:, 0] = value
                x[:, g + 2] = value
            else:
                x[:] = value
        for ps, sp in PLANS:
            want = run(dict(t, q=zero), kv, 290, d ** -0.5, ps, sp)
            assert torch.isfinite(want).all()
            assert torch.equal(run(dict(t, q=bad), kv, 290, d ** -0.5, ps, sp), want), (heads, ps, sp)


def test_nan_blocks_of_the_query_beside_the_plain_decode(cuda_device):
    """Twice the bound of either against 64 bits, 6e-4, on queries whose residues both kernels settle alike."""
    from resinfer_b200 import ops
    kv, q, t = make(cuda_device, [400, 350, 291, 200], 290, 2, 8, 128, 16)
    t["q"] = even(t["q"])
    t["q"][0, 3], t["q"][1, 9, :16], t["q"][3] = NAN, NAN, NAN
    for ps, sp in PLANS:
        got = run(t, kv, 290, 0.1, ps, sp)
        plain = torch.zeros_like(got)
        ops.resattn_decode(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"].clamp(min=0), t["seq_lens"],
                           0.1 * kv["k_global_scale"], kv["v_global_scale"], plain, splits=2)
        for i in range(4):
            assert rel_fro(got[i].cpu().numpy(), plain[i].cpu().numpy()) < 1.2e-3, (ps, sp, i)


@pytest.mark.parametrize("d,page", [(128, 16), (128, 128), (256, 32)])
@pytest.mark.parametrize("ps,sp", PLANS)
@pytest.mark.parametrize("lo,hi", [(0, 290), (0, 64), (130, 131), (289, 290)])
def test_nan_scores_do_not_vanish(cuda_device, d, page, ps, sp, lo, hi):
    """K block scales of NaN in prefix tokens lo .. hi - 1 of KV head 1: NaN for every row of that head which attends to
    one of them -- also where all scores of a piece are NaN, so that no maximum was ever found -- and nothing else moves."""
    lens, prefix = [400, 291, 290, 120, 0, 290], 290
    kv, q, t = make(cuda_device, lens, prefix, 2, 8, d, page)
    clean = run(t, kv, prefix, 0.1, ps, sp)
    sf = t["k_sf"].clone()
    for i, n in enumerate(lens):                                  # every sequence's copy of the tokens
        for tok in range(lo, min(hi, n)):
            sf[kv["block_tables"][i, tok // page], 1, tok % page] = 0x7F
    got = run(dict(t, k_sf=sf), kv, prefix, 0.1, ps, sp)
    assert torch.equal(got[:, :8], clean[:, :8])
    for i, n in enumerate(lens):
        if n > lo:
            assert torch.isnan(got[i, 8:]).all(), i
        else:
            assert torch.equal(got[i], clean[i]), i


@pytest.mark.parametrize("d,page", [(128, 16), (256, 64)])
@pytest.mark.parametrize("ps,sp", PLANS)
def test_nan_scores_of_own_tokens(cuda_device, d, page, ps, sp):
    """All own tokens of one sequence, and one of another's; a sequence of NaN throughout."""
    lens, prefix = [400, 291, 330, 70], 256
    kv, q, t = make(cuda_device, lens, prefix, 2, 4, d, page)
    clean = run(t, kv, prefix, 0.1, ps, sp)
    sf = t["k_sf"].clone()
    for i, tok in [(0, n) for n in range(256, 400)] + [(1, 290)]:
        sf[kv["block_tables"][i, tok // page], :, tok % page] = 0x7F
    got = run(dict(t, k_sf=sf), kv, prefix, 0.1, ps, sp)
    assert torch.isnan(got[:2]).all() and torch.equal(got[2:], clean[2:])
    got = run(dict(t, k_sf=torch.full_like(sf, 0x7F)), kv, prefix, 0.1, ps, sp)
    assert torch.isnan(got).all()
