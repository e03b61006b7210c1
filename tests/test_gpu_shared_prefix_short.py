"""Shared-prefix decode where no sequence reaches the prefix's end: tokens that nobody attends to need not be written.

Tolerance: that of test_gpu_shared_prefix, 6e-4 in FP32."""
import numpy as np
import pytest
import torch

from test_gpu_shared_prefix import TOL_F32, make, reference, rel_fro, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,page", [(128, 16), (128, 48), (128, 128), (256, 16), (256, 128)])
@pytest.mark.parametrize("lens", [[300, 90, 0, 257], [1], [300] * 3 + list(range(1, 60)) + [0] * 9, [0, 0]])
@pytest.mark.parametrize("ps,sp", [(1, 1), (3, 2), (6, 1), (0, 2)])
def test_tokens_beyond_the_longest_sequence(cuda_device, d, page, lens, ps, sp):
    """NaN scales and any codes behind the longest sequence, inside the prefix.  71 sequences of eight heads are five row tiles
    of different longest lengths."""
    prefix, longest = 600, max(lens)
    kv, q, t = make(cuda_device, lens, prefix, 2, 8, d, page)
    want = reference(q, kv, d ** -0.5)
    tokens = np.arange(prefix)
    row = np.zeros(t["block_tables"].shape[1], np.int64)
    row[:] = t["block_tables"][0].cpu().numpy()
    for x, byte in ((t["k_data"], 0x77), (t["k_sf"], 0x7F), (t["v_data"], 0xF7), (t["v_sf"], 0xFF)):
        for tok in tokens[longest:]:
            x[int(row[tok // page]), :, int(tok % page)] = byte
    got = run(t, kv, prefix, d ** -0.5, ps, sp)
    for i, n in enumerate(lens):
        assert (not got[i].any()) if n == 0 else rel_fro(got[i].cpu().numpy(), want[i]) < TOL_F32, (i, n)
