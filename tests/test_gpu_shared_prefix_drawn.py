"""Shared-prefix decode on drawn batches and drawn plans, against the definition in 64 bits (queries as they come, not ones
whose residues suit two kernels alike).

Tolerance: that of test_gpu_shared_prefix, 6e-4 in FP32."""
import numpy as np
import pytest
import torch

from test_gpu_shared_prefix import TOL_F32, make, reference, rel_fro, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed", range(24))
def test_drawn(cuda_device, seed):
    rng = np.random.default_rng(900 + seed)
    d, page = int(rng.choice([128, 256])), int(rng.choice([16, 32, 48, 64, 80, 128, 256]))
    hkv, g, b = int(rng.integers(1, 4)), int(rng.choice([4, 6, 8])), int(np.exp(rng.uniform(0, np.log(60))))
    prefix = int(np.exp(rng.uniform(0, np.log(2500))))
    lens = np.where(rng.random(b) < 0.15, rng.integers(0, prefix + 1, b), prefix + rng.integers(0, 120, b))
    kv, q, t = make(cuda_device, lens.tolist(), prefix, hkv, g, d, page, seed=seed, heat=float(rng.choice([0.3, 1.0, 3.0])))
    row = int(np.argmax(lens))                                    # its table holds the prefix as far as anyone goes
    want = reference(q, kv, d ** -0.5)
    for _ in range(3):
        ps, sp = int(rng.integers(0, 9)), int(rng.integers(1, 6))
        got = run(t, kv, prefix, d ** -0.5, ps, sp, row=row)
        for i, n in enumerate(lens):
            assert (not got[i].any()) if n == 0 else rel_fro(got[i].cpu().numpy(), want[i]) < TOL_F32, (ps, sp, i, n)
