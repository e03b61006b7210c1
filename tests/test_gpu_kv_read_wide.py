"""Large reads of a paged NVFP4 cache: several tokens a thread, against the same rows read in small calls (one token a
thread, held against the oracle in test_gpu_kv_cache).  Copies of the same values: compared for equality."""
import pytest
import torch

from test_gpu_kv_cache import _pool

pytestmark = pytest.mark.gpu


def _many(dev, blocks):
    """Tokens of `blocks` 16-value blocks at which a read takes four of them a thread, and a few more: no multiple of
    anything."""
    sms = torch.cuda.get_device_properties(dev).multi_processor_count
    return sms * 2048 * 8 // blocks + 1237


def _filled(dev, pages, hkv, page, d, packed, seed):
    pool = _pool(dev, pages, hkv, page, d, packed)
    pool.k_global_scale, pool.v_global_scale = 0.37, 1.9
    gen = torch.Generator(device=dev).manual_seed(seed)
    for x, top in ((pool.k_data, 256), (pool.v_data, 256), (pool.k_sf, 0x7F), (pool.v_sf, 0x7F)):
        x.copy_(torch.randint(0, top, x.shape, generator=gen, device=dev, dtype=torch.uint8))
    return pool


def _in_small_calls(pool, slots, dtype):
    from resinfer_b200.nvfp4.cute_attn import host
    parts = [host.read_paged_kv(pool, slots[i:i + 2000], dtype=dtype) for i in range(0, slots.numel(), 2000)]
    return tuple(torch.cat(p) for p in zip(*parts))


SHAPES = [(8, 128, 16, True), (3, 112, 48, False), (40, 256, 16, False), (1, 64, 32, True)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv,d,page,packed", SHAPES)
def test_by_slots(cuda_device, hkv, d, page, packed, dtype):
    from resinfer_b200.nvfp4.cute_attn import host
    n = _many(cuda_device, hkv * d // 16)
    pool = _filled(cuda_device, 300, hkv, page, d, packed, 1)
    gen = torch.Generator(device=cuda_device).manual_seed(2)
    slots = torch.randint(-200, 300 * page + 200, (n,), generator=gen, device=cuda_device)   # padding at both ends
    want = _in_small_calls(pool, slots, dtype)
    for s in (slots, slots.int()):
        got = host.read_paged_kv(pool, s, dtype=dtype)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("hkv,d,page,packed", SHAPES)
@pytest.mark.parametrize("form", ["short", "mixed", "one"])
def test_by_block_tables(cuda_device, hkv, d, page, packed, dtype, form):
    """Sequences of no token to three, so that a thread's four tokens lie in several; long ones between them; a single
    one.  Entries that name no page, and rows behind the last sequence: zero, or left alone in a caller's tensors."""
    from resinfer_b200.nvfp4.cute_attn import host
    n, extra = _many(cuda_device, hkv * d // 16), 301
    gen = torch.Generator().manual_seed(3)
    if form == "short":
        lens = torch.randint(0, 4, (n,), generator=gen)
    elif form == "one":
        lens = torch.tensor([n])
    else:
        lens = torch.where(torch.rand(400, generator=gen) < 0.5, torch.randint(0, 4, (400,), generator=gen), torch.randint(1, n // 50, (400,), generator=gen))
    lens = lens[:int((torch.cumsum(lens, 0) < n).sum()) + 1]
    lens[-1] -= int(lens.sum()) - n
    cols, pages = (int(lens.max()) + page - 1) // page, 300
    table = torch.randint(-20, pages, (lens.numel(), cols), generator=gen, dtype=torch.int32)
    cu = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(lens, 0)])
    pos = torch.arange(n)
    seq = torch.searchsorted(cu, pos, right=True) - 1
    local = pos - cu[seq]
    entry = table[seq, local // page].long()
    slots = torch.where(entry >= 0, entry * page + local % page, -1).to(cuda_device)
    pool = _filled(cuda_device, pages, hkv, page, d, packed, 4)
    want = _in_small_calls(pool, slots, dtype)
    td, cd = table.to(cuda_device), cu.int().to(cuda_device)
    got = host.gather_paged_kv(pool, td, cd, n + extra, dtype=dtype)
    for a, b in zip(got, want):
        assert torch.equal(a[:n], b) and not a[n:].any()
    mine = tuple(torch.full((n + extra, hkv, d), 3.25, dtype=dtype, device=cuda_device) for _ in range(2))
    host.gather_paged_kv(pool, td, cd, n + extra, out=mine)
    for a, b in zip(mine, want):
        assert torch.equal(a[:n], b) and bool((a[n:] == 3.25).all())
