"""More pieces of the prefix than it has steps, on more CTAs than there are SMs: empty ones and working ones follow each
other on an SM.

Tolerance: that of test_gpu_shared_prefix, 6e-4 in FP32."""
import pytest
import torch

from test_gpu_shared_prefix import TOL_F32, make, reference, rel_fro, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,page", [(128, 16), (128, 128), (256, 64)])
@pytest.mark.parametrize("prefix,ps", [(300, 256), (300, 40), (1, 64), (0, 7), (128, 3)])
def test_more_pieces_than_steps(cuda_device, d, page, prefix, ps):
    """Eight KV heads, three row tiles: up to 6144 CTAs of which three in 256 have work."""
    lens = [prefix + 1 + i % 60 for i in range(40)]
    lens[7], lens[30] = 0, prefix // 2
    kv, q, t = make(cuda_device, lens, prefix, 8, 8, d, page)
    want = reference(q, kv, d ** -0.5)
    for sp in (1, 2):
        got = run(t, kv, prefix, d ** -0.5, ps, sp)
        assert rel_fro(got.cpu().numpy(), want) < TOL_F32
        assert not got[7].any()
        for _ in range(3):
            assert torch.equal(run(t, kv, prefix, d ** -0.5, ps, sp), got)
