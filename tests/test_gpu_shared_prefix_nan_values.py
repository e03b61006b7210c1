"""Shared-prefix decode over a cache with NaN block scales in V: NaN in the block's columns of the rows that attend to the
token, nothing elsewhere -- a row that ends before it, in the same tile of the same launch, is as without."""
import pytest
import torch

from test_gpu_shared_prefix import make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,page", [(128, 16), (128, 48), (128, 128), (256, 32), (256, 128)])
@pytest.mark.parametrize("ps,sp", [(1, 1), (3, 2), (0, 1), (0, 3)])
@pytest.mark.parametrize("toks", [[0], [130], [131, 300, 45], [599]])
def test_in_the_prefix(cuda_device, d, page, ps, sp, toks):
    lens, prefix = [700, 600, 601, 131, 0, 45, 130, 132] + list(range(200, 260)), 600
    kv, q, t = make(cuda_device, lens, prefix, 2, 8, d, page)
    clean = run(t, kv, prefix, 0.1, ps, sp)
    sf, want = t["v_sf"].clone(), clean.clone()
    for k, tok in enumerate(toks):
        blk, byte = (3 + 5 * k) % (d // 16), (0x7F, 0xFF)[k % 2]
        for i, n in enumerate(lens):
            if n > tok:
                sf[kv["block_tables"][i, tok // page], 1, tok % page, blk] = byte
                want[i, 8:, 16 * blk:16 * blk + 16] = float("nan")
    got = run(dict(t, v_sf=sf), kv, prefix, 0.1, ps, sp)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))


@pytest.mark.parametrize("d,page", [(128, 16), (256, 64)])
@pytest.mark.parametrize("ps,sp", [(2, 1), (2, 3), (0, 2)])
def test_in_own_tokens(cuda_device, d, page, ps, sp):
    lens, prefix = [400, 291, 330, 70], 250
    kv, q, t = make(cuda_device, lens, prefix, 2, 4, d, page)
    clean = run(t, kv, prefix, 0.1, ps, sp)
    sf, want = t["v_sf"].clone(), clean.clone()
    for i, tok, blk in ((0, 255, 2), (0, 399, 7), (1, 290, 0)):
        sf[kv["block_tables"][i, tok // page], :, tok % page, blk] = 0x7F
        want[i, :, 16 * blk:16 * blk + 16] = float("nan")
    got = run(dict(t, v_sf=sf), kv, prefix, 0.1, ps, sp)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(torch.nan_to_num(got), torch.nan_to_num(want))
