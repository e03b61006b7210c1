"""Shared-prefix decode whose inputs the kernels right in front of it write, over and over in the same memory: queries,
lengths, tables and cache rows of one step must never be those of the step before."""
import pytest
import torch

from test_gpu_shared_prefix import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,page,ps,sp", [(128, 16, 2, 1), (128, 64, 3, 2), (256, 32, 1, 1), (128, 16, 0, 2)])
def test_every_step_reads_its_own_inputs(cuda_device, d, page, ps, sp):
    from resinfer_b200 import ops
    prefix, lens = 300, [330, 301, 420, 0, 305, 390]
    sets = []
    for seed in (1, 2):
        kv, q, t = make(cuda_device, lens, prefix, 2, 8, d, page, seed=seed)
        sets.append(t)
        lens = lens[::-1]
    names = ["q", "seq_lens", "block_tables", "k_data", "k_sf", "v_data", "v_sf"]
    sizes = {n: max(t[n].shape[0] for t in sets) for n in names}
    cols = max(t["block_tables"].shape[1] for t in sets)
    for t in sets:                                                # one shape for both
        bt = torch.full((len(lens), cols), -1, dtype=torch.int32, device=cuda_device)
        bt[:, :t["block_tables"].shape[1]] = t["block_tables"]
        t["block_tables"] = bt
        for n in names[3:]:
            x = torch.zeros((sizes[n],) + t[n].shape[1:], dtype=torch.uint8, device=cuda_device)
            x[:t[n].shape[0]] = t[n]
            t[n] = x

    def call(t, out):
        ops.resattn_decode_shared_prefix(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"], t["seq_lens"], prefix,
                                         0.1, 1.0, out, prefix_splits=ps, splits=sp, prefix_row=2, max_kv_len=500)

    want = []
    for t in sets:
        want.append(torch.zeros(t["q"].shape, device=cuda_device))
        call(t, want[-1])
    torch.cuda.synchronize()
    assert not torch.equal(want[0], want[1])
    live = {n: sets[0][n].clone() for n in names}
    outs = [torch.zeros_like(want[0]) for _ in range(100)]
    for i, out in enumerate(outs):
        for n in names:
            live[n].copy_(sets[i % 2][n])
        call(live, out)
    torch.cuda.synchronize()
    ops.check_status(cuda_device)
    for i, out in enumerate(outs):
        assert torch.equal(out, want[i % 2]), i
