"""Shared-prefix decode when a wait of one CTA runs out: the CTA ends in order, with nothing of its own in flight, the status
word says which wait it was, and nothing else is touched -- not the other rows of the same call, whose CTAs follow on the same
SMs, and not the calls behind it."""
import functools

import pytest
import torch

from test_gpu_shared_prefix import make

pytestmark = pytest.mark.gpu

PS = 8                                                            # pieces of six steps


@functools.lru_cache(maxsize=1)
def _batch(dev, d, page):
    """3 row tiles x 8 KV heads x 8 pieces = 192 CTAs."""
    prefix = PS * 6 * (128 if d == 128 else 64)
    return (prefix, *make(dev, [prefix + 1 + i % 30 for i in range(40)], prefix, 8, 8, d, page))


SITES = [3, 8, 14, 14]                                            # scores, P.V, copies of codes, of scales


@pytest.mark.parametrize("role", range(4))
@pytest.mark.parametrize("step", [0, 1, 2, 4, 5])
@pytest.mark.parametrize("d,page", [(128, 16), (128, 128), (256, 64)])
def test_one_cta_gives_up(cuda_device, d, page, role, step):
    from resinfer_b200 import _cabi, ops
    lib = _cabi.load()
    prefix, kv, q, t = _batch(cuda_device, d, page)

    def call():
        out = torch.zeros(t["q"].shape, device=cuda_device)
        ops.resattn_decode_shared_prefix(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"], t["seq_lens"], prefix,
                                         0.1 * kv["k_global_scale"], kv["v_global_scale"], out, prefix_splits=PS, splits=1, max_kv_len=prefix + 30)
        return out

    clean = call()
    torch.cuda.synchronize()
    ops.check_status(cuda_device)
    other = torch.ones(t["q"].shape[:2], dtype=torch.bool, device=cuda_device)
    other[:16, :8] = False                                        # the first CTA's 128 rows
    lib.ri_resattn_set_prefix_expiry(role, step)
    try:
        outs = [call() for _ in range(3)]
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError, match=rf"\(status {1 + (SITES[role] << 16)}\)"):
            ops.check_status(cuda_device)
    finally:
        lib.ri_resattn_set_prefix_expiry(-1, 0)
    for out in outs:
        assert torch.equal(out[other], clean[other])
    outs = [call() for _ in range(3)]
    torch.cuda.synchronize()
    ops.check_status(cuda_device)
    assert all(torch.equal(out, clean) for out in outs)


def test_no_such_step(cuda_device):
    """The helper names a step that the first CTA does not have: nothing happens."""
    from resinfer_b200 import _cabi, ops
    from test_gpu_shared_prefix import run
    lib = _cabi.load()
    kv, q, t = make(cuda_device, [400, 350], 300, 2, 8, 128, 16)
    want = run(t, kv, 300, 0.1, 2, 1)
    lib.ri_resattn_set_prefix_expiry(1, 1000)
    try:
        assert torch.equal(run(t, kv, 300, 0.1, 2, 1), want)
    finally:
        lib.ri_resattn_set_prefix_expiry(-1, 0)
