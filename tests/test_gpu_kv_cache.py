"""Paged NVFP4 KV cache: quantising writes and reads, against the quantiser oracle (bytes) and its dequantisation.

Bytes must be equal: the oracle restates the quantiser operation by operation.  A value read back is code * scale
(exact in FP32) times the global scale, rounded once to FP32 and once to the output type: the oracle's FP32 product
is the same number, so outputs are compared for equality after the same rounding."""
import numpy as np
import pytest
import torch

import oracle as O

pytestmark = pytest.mark.gpu

f32 = np.float32


def _pool(dev, pages, hkv, page, d, packed, fill=0):
    """An NvFp4PagedKVPool on `dev`: dense, or views of an interleaved cache."""
    from resinfer_b200.nvfp4.cute_attn import NvFp4PagedKVPool
    nc, ns = hkv * page * d // 2, hkv * page * d // 16
    if packed:
        buf = torch.full((pages, 2 * (nc + ns)), fill, dtype=torch.uint8, device=dev)
        at, parts = 0, []
        for w, n in ((d // 2, nc), (d // 16, ns), (d // 2, nc), (d // 16, ns)):
            parts.append(buf[:, at:at + n].unflatten(1, (hkv, page, w)))
            at += n
        kd, ks, vd, vs = parts
    else:
        kd, vd = (torch.full((pages, hkv, page, d // 2), fill, dtype=torch.uint8, device=dev) for _ in range(2))
        ks, vs = (torch.full((pages, hkv, page, d // 16), fill, dtype=torch.uint8, device=dev) for _ in range(2))
    return NvFp4PagedKVPool(hkv, d, kd, vd, ks, vs, page_size=page)


def _oracle_rows(x, g, rcp):
    """codes [T, H, D/2] and linear scale bytes [T, H, D/16] of float32 rows x [T, H, D]."""
    t, h, d = x.shape
    dp = (d + 63) // 64 * 64                                  # the oracle's scale layout wants whole groups of 64
    codes, sf = O.nvfp4_quant_plain(np.pad(x.reshape(t * h, d), ((0, 0), (0, dp - d))), f32(1.0) / f32(g), rcp)
    lin = sf[O.sf_offset(np.arange(t * h)[:, None], np.arange(d // 16)[None], dp)]
    return codes[:, :d // 2].reshape(t, h, d // 2), lin.reshape(t, h, d // 16)


def _held(codes, sf, g):
    v = O.e2m1_decode(O.unpack_nibbles(codes))
    v = (v.reshape(*v.shape[:-1], -1, 16) * O.e4m3_decode(sf)[..., None]).reshape(v.shape).astype(f32)
    return v * f32(g)


def _rows(t, h, d, dtype, seed, spread=1.0):
    x = np.random.default_rng(seed).standard_normal((t, h, d)).astype(f32) * f32(spread)
    return torch.from_numpy(x).to(dtype)


@pytest.mark.parametrize("t,hkv,d,page,dtype,packed,bits,g", [
    (1, 8, 128, 16, torch.bfloat16, False, 64, 0.0013),
    (37, 2, 128, 128, torch.bfloat16, False, 32, 0.0021),
    (130, 4, 256, 32, torch.float16, True, 64, 0.00093),
    (65, 1, 64, 48, torch.bfloat16, True, 32, 0.0017),       # page size that is no power of two
    (19, 3, 112, 16, torch.float16, False, 64, 1.0),         # head_dim with an odd number of blocks, global scale 1
    (33, 5, 16, 16, torch.bfloat16, False, 64, 0.0007),      # one block per row
    (9, 40, 256, 16, torch.bfloat16, False, 64, 0.0011),     # a token's row wider than a CTA
])
def test_write_bytes_and_read_back(cuda_device, device_rcp, t, hkv, d, page, dtype, packed, bits, g):
    from resinfer_b200.nvfp4.cute_attn import host
    pages = (t + page - 1) // page + 3
    pool = _pool(cuda_device, pages, hkv, page, d, packed, fill=0x5A)
    pool.k_global_scale, pool.v_global_scale = g, 1.7 * g
    k, v = _rows(t, hkv, d, dtype, 1), _rows(t, hkv, d, dtype, 2, 0.5)
    slots = np.random.default_rng(3).permutation(pages * page)[:t]
    pad = np.random.default_rng(4).random(t) < 0.2
    slots = np.where(pad, np.where(np.arange(t) % 2 == 0, -1, pages * page + np.arange(t)), slots)
    before = [x.clone() for x in (pool.k_data, pool.k_sf, pool.v_data, pool.v_sf)]
    st = torch.from_numpy(slots).to(torch.int64 if bits == 64 else torch.int32).to(cuda_device)
    host.write_paged_kv(k.to(cuda_device), v.to(cuda_device), pool, st)
    torch.cuda.synchronize()
    live = np.nonzero(~pad)[0]
    pg, off = slots[live] // page, slots[live] % page
    got_k, got_v = host.read_paged_kv(pool, st, dtype=dtype)
    got32 = host.read_paged_kv(pool, st, dtype=torch.float32)
    for x, data, sf, gs, was_d, was_s, back, back32 in (
            (k, pool.k_data, pool.k_sf, g, before[0], before[1], got_k, got32[0]),
            (v, pool.v_data, pool.v_sf, 1.7 * g, before[2], before[3], got_v, got32[1])):
        codes, scales = _oracle_rows(x.float().numpy(), gs, O.RecordingRcp(device_rcp))
        want_d, want_s = was_d.cpu().numpy(), was_s.cpu().numpy()
        want_d[pg, :, off], want_s[pg, :, off] = codes[live], scales[live]
        assert np.array_equal(data.cpu().numpy(), want_d)     # the written rows, and nothing else
        assert np.array_equal(sf.cpu().numpy(), want_s)
        held = np.zeros((t, hkv, d), f32)
        held[live] = _held(codes, scales, gs)[live]
        assert np.array_equal(back32.cpu().numpy(), held)
        assert torch.equal(back.cpu(), torch.from_numpy(held).to(dtype))


def test_write_takes_any_strides(cuda_device):
    """Slices of a fused projection (aligned and not), heads before tokens, broadcast heads, more rows than slots."""
    from resinfer_b200.nvfp4.cute_attn import host
    t, hkv, d, page = 21, 2, 128, 16
    base = _rows(t, 5 * hkv + 1, d, torch.bfloat16, 7).to(cuda_device)
    wide = torch.randn(t, 3 * hkv * d + 5, generator=torch.Generator().manual_seed(1)).bfloat16().to(cuda_device)
    forms = [base[:, 2:4], base[:, 3::3][:, :hkv], wide[:, 3:3 + hkv * d].unflatten(1, (hkv, d)),
             base[:, :hkv].transpose(0, 1).contiguous().transpose(0, 1), base[:, :1].expand(t, hkv, d)]
    slots = torch.randperm(3 * page, generator=torch.Generator().manual_seed(2))[:t - 4].to(cuda_device)
    for a in forms:
        for b in forms:
            pool, want = (_pool(cuda_device, 3, hkv, page, d, False, fill=7) for _ in range(2))
            host.write_paged_kv(a, b, pool, slots)
            host.write_paged_kv(a[:t - 4].contiguous(), b[:t - 4].contiguous(), want, slots)
            for x, y in ((pool.k_data, want.k_data), (pool.k_sf, want.k_sf), (pool.v_data, want.v_data), (pool.v_sf, want.v_sf)):
                assert torch.equal(x, y)


def test_write_of_special_values(cuda_device):
    """Zeros, subnormals, saturation, infinities, NaN; tiny blocks whose scale rounds to zero."""
    from resinfer_b200.nvfp4.cute_attn import host
    inf, nan = float("inf"), float("nan")
    rows = torch.zeros(7, 1, 32, dtype=torch.bfloat16)
    rows[1, 0, 0], rows[1, 0, 20] = 1e-4, -1e-30              # scales that round to zero: held as 0
    rows[2, 0, :16] = 1e30                                    # beyond 6 * 448 * g: saturates
    rows[2, 0, 3] = -1e30
    rows[3, 0, 2], rows[3, 0, 5], rows[3, 0, 6] = inf, -inf, 448.0
    rows[4, 0, 4], rows[4, 0, 9], rows[4, 0, 10] = nan, 6.0, -3.0
    rows[5, 0, :] = nan
    rows[6, 0, 17] = -0.0
    pool = _pool(cuda_device, 2, 1, 16, 32, False, fill=0xFF)
    x = rows.to(cuda_device)
    slots = torch.arange(7, device=cuda_device)
    host.write_paged_kv(x, x, pool, slots)
    k, v = host.read_paged_kv(pool, slots, dtype=torch.float32)
    assert torch.equal(k, v)
    want = torch.zeros(7, 32)
    want[2, :16], want[2, 3] = 6 * 448.0, -6 * 448.0
    want[3, 2], want[3, 5], want[3, 6] = 6 * 448.0, -6 * 448.0, 448.0
    want[4, 4], want[4, 9], want[4, 10] = 6.0, 6.0, -3.0       # NaN: the block's largest positive code
    assert torch.equal(k[:, 0].cpu(), want)


@pytest.mark.parametrize("lens,page,d,hkv,packed,dtype", [
    ([5], 16, 128, 2, False, torch.bfloat16), ([0, 17, 0, 1, 33, 0], 16, 128, 3, True, torch.float16),
    ([100, 1, 64, 129], 48, 256, 1, False, torch.float32), (list(range(70)), 32, 64, 2, True, torch.bfloat16)])
def test_gather_by_block_tables(cuda_device, lens, page, d, hkv, packed, dtype):
    """The ragged batch equals the slot form token by token; tail rows, missing table entries and short tables."""
    from resinfer_b200.nvfp4.cute_attn import host
    total, extra = sum(lens), 3
    per = [(n + page - 1) // page for n in lens]
    pages = sum(per) + 2
    pool = _pool(cuda_device, pages, hkv, page, d, packed)
    pool.k_global_scale, pool.v_global_scale = 0.37, 1.9
    g = torch.Generator().manual_seed(5)
    pool.k_data.copy_(torch.randint(0, 256, pool.k_data.shape, generator=g, dtype=torch.uint8))
    pool.v_data.copy_(torch.randint(0, 256, pool.v_data.shape, generator=g, dtype=torch.uint8))
    pool.k_sf.copy_(torch.randint(0, 0x7F, pool.k_sf.shape, generator=g, dtype=torch.uint8))
    pool.v_sf.copy_(torch.randint(0, 0x7F, pool.v_sf.shape, generator=g, dtype=torch.uint8))
    order = torch.randperm(pages, generator=g).int()
    table = torch.full((len(lens), max(max(per), 1) + 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = order[at:at + n]
        at += n
    cu = torch.tensor([0] + np.cumsum(lens).tolist(), dtype=torch.int32)
    slots = torch.tensor([int(table[b, i // page]) * page + i % page for b, n in enumerate(lens) for i in range(n)]
                         + [-1] * extra, dtype=torch.int64)
    want = host.read_paged_kv(pool, slots.to(cuda_device), dtype=dtype)
    td, cd = table.to(cuda_device), cu.to(cuda_device)
    got = host.gather_paged_kv(pool, td, cd, total + extra, dtype=dtype)
    assert all(torch.equal(a, b) for a, b in zip(got, want))   # the rows behind the last sequence are zero
    mine = tuple(torch.full((total + extra, hkv, d), 3.25, dtype=dtype, device=cuda_device) for _ in range(2))
    host.gather_paged_kv(pool, td, cd, total + extra, out=mine)
    for a, b in zip(mine, want):
        assert torch.equal(a[:total], b[:total]) and bool((a[total:] == 3.25).all())
    wide = torch.full((len(lens), 40), -1, dtype=torch.int32, device=cuda_device)
    wide[:, 3:3 + td.shape[1]] = td
    again = host.gather_paged_kv(pool, wide[:, 3:3 + td.shape[1]], cd, total + extra, dtype=dtype)   # strided table rows
    assert all(torch.equal(a, b) for a, b in zip(again, want))
    # a table entry that names no page: that page's tokens are zero, the others are not touched by it
    b = max(range(len(lens)), key=lambda i: lens[i])
    for bad in (-1, pages, 2 ** 31 - 1):
        t2 = td.clone()
        t2[b, 0] = bad
        lo, hi = int(cu[b]), int(cu[b]) + min(page, lens[b])
        k, v = host.gather_paged_kv(pool, t2, cd, total + extra, dtype=dtype)
        for a, w in ((k, want[0]), (v, want[1])):
            assert not a[lo:hi].any() and torch.equal(a[hi:], w[hi:]) and torch.equal(a[:lo], w[:lo])
    # a table with too few columns: what lies beyond them is zero
    k, _ = host.gather_paged_kv(pool, td[:, :1], cd, total + extra, dtype=dtype)
    lo, hi = int(cu[b]) + min(page, lens[b]), int(cu[b + 1])
    assert not k[lo:hi].any()


def test_offsets_beyond_32_bits(cuda_device):
    """A pool of more than 4 GiB of K codes: the last slot's address does not fit 32 bits."""
    from resinfer_b200.nvfp4.cute_attn import NvFp4PagedKVPool, host
    hkv, d, page = 8, 256, 128
    pages = (1 << 32) // (hkv * page * d // 2) + 5
    kd = torch.zeros(pages, hkv, page, d // 2, dtype=torch.uint8, device=cuda_device)
    sf = torch.zeros(pages, hkv, page, d // 16, dtype=torch.uint8, device=cuda_device)
    vd = torch.zeros_like(kd)
    pool = NvFp4PagedKVPool(hkv, d, kd, vd, sf, sf.clone(), page_size=page, k_global_scale=0.01, v_global_scale=0.01)
    x = _rows(3, hkv, d, torch.bfloat16, 4).to(cuda_device)
    slots = torch.tensor([pages * page - 1, 0, pages * page - page - 1], device=cuda_device)
    host.write_paged_kv(x, 2 * x, pool, slots)
    small = _pool(cuda_device, 2, hkv, page, d, False)
    small.k_global_scale = small.v_global_scale = 0.01
    host.write_paged_kv(x, 2 * x, small, torch.arange(3, device=cuda_device))
    want = host.read_paged_kv(small, torch.arange(3, device=cuda_device))
    got = host.read_paged_kv(pool, slots)
    table = torch.tensor([[pages - 1], [0]], dtype=torch.int32, device=cuda_device)
    ends = host.gather_paged_kv(pool, table, torch.tensor([0, page, page + 1], dtype=torch.int32, device=cuda_device), page + 1)
    for a, b, c in zip(got, want, ends):
        assert a.any() and torch.equal(a, b)
        assert torch.equal(c[page - 1], b[0]) and torch.equal(c[page], b[1])


def test_captured_and_replayed(cuda_device):
    """Write and read in one CUDA graph, replayed with new rows and new slots in the same buffers, on another stream."""
    from resinfer_b200.nvfp4.cute_attn import host
    t, hkv, d, page = 12, 2, 128, 16
    pool = _pool(cuda_device, 4, hkv, page, d, True)
    pool.k_global_scale = pool.v_global_scale = 0.002
    k, v = (_rows(t, hkv, d, torch.bfloat16, s).to(cuda_device) for s in (1, 2))
    slots = torch.arange(t, device=cuda_device)
    host.write_paged_kv(k, v, pool, slots)
    host.read_paged_kv(pool, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        host.write_paged_kv(k, v, pool, slots)
        out = host.read_paged_kv(pool, slots)
    side = torch.cuda.Stream()
    for seed in (5, 6):
        k.copy_(_rows(t, hkv, d, torch.bfloat16, seed))
        v.copy_(_rows(t, hkv, d, torch.bfloat16, seed + 10))
        slots.copy_(torch.randperm(4 * page, generator=torch.Generator().manual_seed(seed))[:t])
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            graph.replay()
        torch.cuda.current_stream().wait_stream(side)
        fresh = _pool(cuda_device, 4, hkv, page, d, False)
        fresh.k_global_scale = fresh.v_global_scale = 0.002
        host.write_paged_kv(k, v, fresh, slots)
        want = host.read_paged_kv(fresh, slots)
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_wrapper_refusals(cuda_device):
    from resinfer_b200 import ops
    from resinfer_b200.nvfp4.cute_attn import host
    pool = _pool(cuda_device, 2, 2, 16, 128, False)
    x = torch.zeros(4, 2, 128, dtype=torch.bfloat16, device=cuda_device)
    slots = torch.arange(4, device=cuda_device)
    for k, v, s in ((x.float(), x.float(), slots), (x, x.half(), slots), (x[:, :1], x[:, :1], slots), (x, x[:2], slots),
                    (x.cpu(), x, slots), (x, x, slots.float()), (x, x, slots[None]), (x, x, slots[::2]), (x, x, slots.cpu()),
                    (x.transpose(1, 2).contiguous().transpose(1, 2), x, slots)):
        with pytest.raises(ValueError):
            host.write_paged_kv(k, v, pool, s)
    with pytest.raises(ValueError):
        host.read_paged_kv(pool, slots, out=(x, x[:2]))
    with pytest.raises(RuntimeError):
        host.read_paged_kv(pool, slots, dtype=torch.float64)
    table, cu = torch.zeros(2, 1, dtype=torch.int32, device=cuda_device), torch.zeros(3, dtype=torch.int32, device=cuda_device)
    for t, c in ((table.long(), cu), (table, cu[:2]), (table, cu.long()), (table[:0], cu)):
        with pytest.raises(ValueError):
            host.gather_paged_kv(pool, t, c, 4)
    with pytest.raises(ValueError, match="negative"):
        host.gather_paged_kv(pool, table, cu, -1)
    with pytest.raises(ValueError, match="not both"):
        ops.kv_read(pool.k_data, pool.k_sf, pool.v_data, pool.v_sf, 1.0, 1.0, slots=slots, block_tables=table)
    pool.k_global_scale = 0.0
    with pytest.raises(RuntimeError, match="k_global_scale"):
        host.write_paged_kv(x, x, pool, slots)
    empty = slots[:0]
    pool.k_global_scale = 1.0
    host.write_paged_kv(x, x, pool, empty)
    assert host.read_paged_kv(pool, empty)[0].shape == (0, 2, 128)
    assert not pool.k_data.any()
