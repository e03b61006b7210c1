"""The query's codes and residues in the tail kernel, for every size of a group and with nothing else to average over.

Tolerance: that of test_gpu_shared_prefix, 6e-4 in FP32."""
import pytest
import torch

from test_gpu_shared_prefix import TOL_F32, make, reference, rel_fro, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("g", [4, 6, 8])
@pytest.mark.parametrize("heat", [0.3, 1.0, 40.0])
def test_tail_alone(cuda_device, d, g, heat):
    """Two tokens and more, queries of different spread: each head's scores show its own codes."""
    lens = [2, 3, 40, 700]
    kv, q, t = make(cuda_device, lens, 0, 2, g, d, 16, heat=heat)
    want = reference(q, kv, d ** -0.5)
    for sp in (1, 2):
        got = run(t, kv, 0, d ** -0.5, 0, sp)
        for i in range(len(lens)):
            for h in range(2 * g):
                assert rel_fro(got[i, h].cpu().numpy(), want[i, h]) < TOL_F32, (sp, i, h)
