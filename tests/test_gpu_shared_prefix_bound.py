"""Sequences longer than the bound that the call was given, as in a graph captured before they grew: no token is left out.

Tolerance: that of test_gpu_shared_prefix, 6e-4 in FP32."""
import pytest
import torch

from test_gpu_shared_prefix import TOL_F32, make, reference, rel_fro, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d,page", [(128, 16), (256, 64)])
@pytest.mark.parametrize("ps,sp", [(2, 1), (2, 4), (0, 1), (0, 3)])
@pytest.mark.parametrize("bound", [1, 250, 256, 400])
def test_longer_than_the_bound(cuda_device, d, page, ps, sp, bound):
    lens, prefix = [900, 251, 0, 400, 130, 577], 250
    kv, q, t = make(cuda_device, lens, prefix, 2, 8, d, page)
    want = reference(q, kv, d ** -0.5)
    got = run(t, kv, prefix, d ** -0.5, ps, sp, max_len=bound)
    for i, n in enumerate(lens):
        assert (not got[i].any()) if n == 0 else rel_fro(got[i].cpu().numpy(), want[i]) < TOL_F32, (i, n)


def test_a_captured_step_whose_sequences_grow(cuda_device):
    from resinfer_b200.nvfp4.cute_attn import NvFp4PagedKVPool, host
    lens, prefix, d, page = [700, 310, 1000], 300, 128, 16
    kv, q, t = make(cuda_device, lens, prefix, 2, 8, d, page)
    pool = NvFp4PagedKVPool(2, d, t["k_data"], t["v_data"], t["k_sf"], t["v_sf"], page_size=page)
    seq_lens, out = torch.tensor([301, 305, 310], dtype=torch.int32, device=cuda_device), torch.zeros_like(t["q"])

    def call(o, bound):
        host.run_paged_fp4_decode_shared_prefix(t["q"], pool, t["block_tables"], seq_lens, prefix, 0.1 * kv["k_global_scale"], o,
                                                max_seq_len=bound, value_scale=kv["v_global_scale"])

    call(out, 310)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(out, 310)
    seq_lens.copy_(t["seq_lens"])
    graph.replay()
    fresh = torch.zeros_like(out)
    call(fresh, 1000)
    # two BF16 results of the same operation: 2 * 2.3e-3 for the output's rounding and 1.2e-3 for P's
    assert rel_fro(out.float().cpu().numpy(), fresh.float().cpu().numpy()) < 6e-3
