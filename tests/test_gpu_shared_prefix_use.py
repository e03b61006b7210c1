"""Shared-prefix decode as it is called: with the cache written by write_paged_kv, through the host entry and its plan, on
streams, in graphs, over interleaved pools and with whatever lies in memory that nobody has written.

Tolerances are those of test_gpu_shared_prefix: 6e-4 in FP32, 3e-3 in BF16, twice the former between two FP32 results, and
between two BF16 results the roundings of both on top (2 * 2.3e-3 + 1.2e-3 < 6e-3); `even` queries beside the plain decode."""
import numpy as np
import pytest
import torch

import oracle as O
from test_gpu_kv_cache import _pool
from test_gpu_shared_prefix import TOL_BF16, TOL_F32, even, make, reference, rel_fro, run

pytestmark = pytest.mark.gpu


def _as_numpy(pool, table, lens):
    return dict(k_data=pool.k_data.cpu().numpy(), v_data=pool.v_data.cpu().numpy(), k_sf=pool.k_sf.cpu().numpy(),
                v_sf=pool.v_sf.cpu().numpy(), block_tables=table.clamp(min=0).cpu().numpy(), seq_lens=np.asarray(lens, np.int32),
                k_global_scale=pool.k_global_scale, v_global_scale=pool.v_global_scale)


def _slots(table, page, seq, lo, hi):
    i = torch.arange(lo, hi)
    return table[seq, i // page].long() * page + i % page


@pytest.mark.parametrize("d,hkv,g,page,prefix,packed,dtype", [
    (128, 2, 8, 16, 150, False, torch.bfloat16), (256, 1, 4, 32, 97, True, torch.float16), (128, 3, 6, 128, 256, True, torch.bfloat16)])
def test_a_generation(cuda_device, d, hkv, g, page, prefix, packed, dtype):
    """A prompt is written once, three sequences append to it token by token, each step decodes; at the end the contexts
    are gathered.  All bytes that were never written are NaN scales."""
    from resinfer_b200 import ops
    from resinfer_b200.nvfp4.cute_attn import host
    gen = torch.Generator().manual_seed(d + page)
    b, steps, hq = 4, 4, hkv * g
    shared = prefix // page
    cols = shared + 3
    pool = _pool(cuda_device, shared + 2 * b + 2, hkv, page, d, packed, fill=0x7F)
    pool.k_global_scale, pool.v_global_scale = 0.0017, 0.0023
    order = torch.randperm(pool.k_data.shape[0], generator=gen).int()
    table = torch.full((b, cols), -1, dtype=torch.int32)
    table[:, :shared] = order[:shared]
    table[:3, shared:shared + 2] = order[shared:shared + 6].view(3, 2)   # row 3 is padding
    table[3] = -1
    prompt_k, prompt_v = (torch.randn(prefix, hkv, d, generator=gen).to(dtype).to(cuda_device) for _ in range(2))
    whole = shared * page
    host.write_paged_kv(prompt_k, prompt_v, pool, _slots(table, page, 0, 0, prefix).to(cuda_device))
    for s in (1, 2):                                              # the page in which the prompt ends belongs to one sequence
        host.write_paged_kv(prompt_k[whole:], prompt_v[whole:], pool, _slots(table, page, s, whole, prefix).to(cuda_device))
    lens = [prefix, prefix, prefix, 0]
    td = table.to(cuda_device)
    rows_k, rows_v = [[] for _ in range(3)], [[] for _ in range(3)]
    for step in range(steps):
        new_k, new_v = (torch.randn(4, hkv, d, generator=gen).to(dtype).to(cuda_device) for _ in range(2))
        slots = torch.tensor([int(_slots(table, page, s, lens[s], lens[s] + 1)) for s in range(3)] + [-1], device=cuda_device)
        host.write_paged_kv(new_k, new_v, pool, slots)
        for s in range(3):
            rows_k[s].append(new_k[s])
            rows_v[s].append(new_v[s])
            lens[s] += 1
        q = torch.randn(b, hq, d, generator=gen).bfloat16().to(cuda_device)
        out = torch.full_like(q, float("nan"))
        host.run_paged_fp4_decode_shared_prefix(q, pool, td, torch.tensor(lens, dtype=torch.int32, device=cuda_device), prefix,
                                                d ** -0.5 * pool.k_global_scale, out, max_seq_len=max(lens), value_scale=pool.v_global_scale,
                                                prefix_row=step % 3)
        torch.cuda.synchronize()
        ops.check_status(q.device)
        want = reference(q.float().cpu().numpy(), _as_numpy(pool, table, lens), d ** -0.5)
        assert not out[3].any()
        for s in range(3):
            assert rel_fro(out[s].float().cpu().numpy(), want[s]) < TOL_BF16, (step, s)
    cu = torch.tensor(np.cumsum([0] + lens[:3] + [0]), dtype=torch.int32, device=cuda_device)
    got_k, got_v = host.gather_paged_kv(pool, td, cu, sum(lens), dtype=torch.float32)
    for got, prompt, rows, gs in ((got_k, prompt_k, rows_k, 0.0017), (got_v, prompt_v, rows_v, 0.0023)):
        for s in range(3):
            held = got[int(cu[s]):int(cu[s + 1])].cpu()
            x = torch.cat([prompt.float(), torch.stack(rows[s]).float()]).cpu()
            # E2M1 spaces its values by at most 2 below 6: half a step is a sixth of the block's amax; the scale's own
            # rounding (2^-4 of itself at most, in blocks whose scale is above 2^-6) moves the amax by 1/16 more, and
            # the scale behind the held codes is up to 17/16 of amax / 6
            amax = x.unflatten(-1, (-1, 16)).abs().amax(-1, keepdim=True)
            err = (held - x).unflatten(-1, (-1, 16)).abs()
            assert bool((err <= amax * (17 / 16 / 6 + 1 / 16) * 1.0001).all())


@pytest.mark.parametrize("d,page", [(128, 16), (256, 64), (128, 128)])
def test_bytes_nobody_wrote(cuda_device, d, page):
    """NaN scales and any codes behind every sequence's end, and in all pages that no table names."""
    lens, prefix = [333, 0, 90, 500, 333, 334], 333
    kv, q, t = make(cuda_device, lens, prefix, 2, 6, d, page)
    used = np.zeros((kv["k_data"].shape[0], page), bool)
    for i, n in enumerate(lens):
        for tok in range(n):
            used[kv["block_tables"][i, tok // page], tok % page] = True
    for tok in range(prefix):
        used[kv["block_tables"][3, tok // page], tok % page] = True
    want = reference(q, kv, d ** -0.5)
    dead = torch.from_numpy(~used).to(cuda_device)[:, None, :, None]
    for x, byte in ((t["k_data"], 0x77), (t["k_sf"], 0x7F), (t["v_data"], 0xF7), (t["v_sf"], 0xFF)):
        x.masked_fill_(dead, byte)
    for ps, sp in ((3, 2), (1, 1), (0, 3)):
        got = run(t, kv, prefix, d ** -0.5, ps, sp, row=3)
        for i, n in enumerate(lens):
            assert (not got[i].any()) if n == 0 else rel_fro(got[i].cpu().numpy(), want[i]) < TOL_F32, (ps, sp, i)


def test_prefix_row_and_entries_that_name_no_page(cuda_device):
    """Padding in row 0, the prefix in row 2; table entries behind a sequence's end may hold anything."""
    lens, prefix, d, page = [0, 400, 290, 261], 256, 128, 16
    kv, q, t = make(cuda_device, lens, prefix, 2, 4, d, page)
    want = reference(q, kv, d ** -0.5)
    t["block_tables"][0] = -7
    for i, n in enumerate(lens):
        t["block_tables"][i, (n + page - 1) // page:] = 2 ** 31 - 1
    got = run(t, kv, prefix, d ** -0.5, 2, 2, row=2)
    assert not got[0].any() and rel_fro(got.cpu().numpy(), want) < TOL_F32
    bad = t["block_tables"].clone()
    bad[2, 3], bad[2, 5] = -1, 2 ** 31 - 1                        # inside the prefix: some page is read, nothing beyond the pool
    assert torch.isfinite(run(dict(t, block_tables=bad), kv, prefix, d ** -0.5, 2, 2, row=2)).all()


@pytest.mark.parametrize("ps,sp", [(256, 1), (1, 256), (256, 256), (40, 3)])
def test_most_pieces(cuda_device, ps, sp):
    """More pieces than there is work for: empty partials, and a merge of up to 512 of them."""
    kv, q, t = make(cuda_device, [6000, 5121, 5200], 5120, 1, 8, 128, 64)
    want = reference(q, kv, 128 ** -0.5)
    got = run(t, kv, 5120, 128 ** -0.5, ps, sp)
    assert rel_fro(got.cpu().numpy(), want) < TOL_F32
    assert torch.equal(run(t, kv, 5120, 128 ** -0.5, ps, sp), got)


@pytest.mark.parametrize("seed", range(6))
def test_drawn_shapes_by_the_host_entry(cuda_device, seed):
    """Drawn batches through the host entry and the plan it chooses, against the plain decode."""
    from resinfer_b200 import ops
    from resinfer_b200.nvfp4.cute_attn import NvFp4PagedKVPool, host
    rng = np.random.default_rng(100 + seed)
    d, page = int(rng.choice([128, 256])), int(rng.choice([16, 32, 48, 64, 128]))
    hkv, g, b = int(rng.integers(1, 5)), int(rng.choice([4, 6, 8])), int(rng.integers(1, 90))
    prefix = int(rng.integers(1, 3000))
    lens = np.where(rng.random(b) < 0.1, rng.integers(0, prefix + 1, b), prefix + rng.integers(0, 200, b)).tolist()
    lens[-1] = prefix + 1
    kv, q, t = make(cuda_device, lens, prefix, hkv, g, d, page, seed=seed, heat=float(rng.choice([0.5, 2.0])))
    pool = NvFp4PagedKVPool(hkv, d, t["k_data"], t["v_data"], t["k_sf"], t["v_sf"], page_size=page)
    sm, vs = d ** -0.5 * kv["k_global_scale"], kv["v_global_scale"]
    t["q"] = even(t["q"])
    got, plain = torch.full_like(t["q"], float("nan")), torch.zeros_like(t["q"])
    host.run_paged_fp4_decode_shared_prefix(t["q"], pool, t["block_tables"], t["seq_lens"], prefix, sm, got, value_scale=vs, prefix_row=b - 1)
    ops.resattn_decode(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"].clamp(min=0), t["seq_lens"], sm, vs, plain, splits=4)
    torch.cuda.synchronize()
    ops.check_status(got.device)
    assert rel_fro(got.float().cpu().numpy(), plain.float().cpu().numpy()) < 6e-3
    again = torch.empty_like(got)
    host.run_paged_fp4_decode_shared_prefix(t["q"], pool, t["block_tables"], t["seq_lens"], prefix, sm, again, value_scale=vs,
                                            prefix_row=b - 1, max_seq_len=max(lens))
    assert torch.equal(again, got)


def test_many_short_sequences(cuda_device):
    """Grid sizes: 1500 sequences, 94 row tiles, against the plain decode."""
    from resinfer_b200 import ops
    n, prefix = 1500, 70
    kv, q, t = make(cuda_device, [prefix + 1 + i % 3 for i in range(n)], prefix, 1, 8, 128, 16)
    t["q"] = even(t["q"])
    got = run(t, kv, prefix, 0.1, 1, 1)
    plain = torch.zeros_like(got)
    ops.resattn_decode(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"].clamp(min=0), t["seq_lens"],
                       0.1 * kv["k_global_scale"], kv["v_global_scale"], plain, splits=1)
    assert rel_fro(got.cpu().numpy(), plain.cpu().numpy()) < 2 * TOL_F32


def test_pool_beyond_32_bit_offsets(cuda_device):
    """Pages in the last megabytes of a pool of more than 4 GiB of codes."""
    from resinfer_b200 import ops
    lens, prefix, hkv, g, d, page = [300, 280], 256, 8, 4, 256, 128
    kv, q, t = make(cuda_device, lens, prefix, hkv, g, d, page)
    n = kv["k_data"].shape[0]
    pages = (1 << 32) // (hkv * page * d // 2) + n + 1
    big = {}
    for name in ("k_data", "k_sf", "v_data", "v_sf"):
        big[name] = torch.zeros((pages,) + t[name].shape[1:], dtype=torch.uint8, device=cuda_device)
        big[name][pages - n:] = t[name]
    far = dict(t, block_tables=torch.where(t["block_tables"] >= 0, t["block_tables"] + (pages - n), t["block_tables"]), **big)
    for ps, sp in ((2, 1), (1, 2)):
        assert torch.equal(run(far, kv, prefix, 0.05, ps, sp), run(t, kv, prefix, 0.05, ps, sp))


def test_interleaved_pool(cuda_device):
    """K, V and scales of a page next to one another: the page stride is larger than a part's page."""
    for d, page in ((128, 16), (256, 128)):
        kv, q, t = make(cuda_device, [400, 311, 290], 290, 2, 8, d, page)
        pool = _pool(cuda_device, kv["k_data"].shape[0], 2, page, d, True)
        parts = {"k_data": pool.k_data, "k_sf": pool.k_sf, "v_data": pool.v_data, "v_sf": pool.v_sf}
        for name, x in parts.items():
            x.copy_(t[name])
        assert torch.equal(run(dict(t, **parts), kv, 290, 0.1, 2, 2), run(t, kv, 290, 0.1, 2, 2))


def test_streams_and_graphs(cuda_device):
    """Calls at once on two streams; two captured graphs replayed in turn and at once, with new queries, lengths and
    tables in the same buffers; a caller's workspace."""
    from resinfer_b200 import ops
    sets = [make(cuda_device, [700, 655, 900, 641], 640, 2, 8, 128, 64, seed=s) for s in (1, 2)]

    def call(t, kv, out, ps=2, sp=2, workspace=None):
        ops.resattn_decode_shared_prefix(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"], t["seq_lens"], 640,
                                         0.1 * kv["k_global_scale"], kv["v_global_scale"], out, prefix_splits=ps, splits=sp,
                                         max_kv_len=1000, workspace=workspace)

    want = [run(t, kv, 640, 0.1, 2, 2, max_len=1000) for kv, q, t in sets]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[torch.zeros_like(w) for _ in range(20)] for w in want]
    torch.cuda.synchronize()
    for i in range(20):
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                call(sets[j][2], sets[j][0], outs[j][i])
    torch.cuda.synchronize()
    for j in range(2):
        assert all(torch.equal(o, want[j]) for o in outs[j])
    graphs, held = [], []
    for j in range(2):
        held.append(torch.zeros_like(want[j]))
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(sets[j][2], sets[j][0], held[j])
            call(sets[j][2], sets[j][0], held[j])
        graphs.append(g)
    for turn in range(3):
        now = []
        for j in range(2):
            kv, q, t = sets[j]
            t["q"].copy_(torch.randn(t["q"].shape, generator=torch.Generator().manual_seed(turn * 2 + j)).bfloat16())
            t["seq_lens"].copy_(torch.tensor([[700, 0, 641, 641], [640, 655, 900, 600], [650, 655, 870, 1]][turn], dtype=torch.int32))
            fresh = torch.zeros_like(want[j])
            call(t, kv, fresh)
            now.append(fresh)
            held[j].fill_(7)
        torch.cuda.synchronize()
        for j in range(2):
            with torch.cuda.stream(streams[j]):
                graphs[j].replay()
        torch.cuda.synchronize()
        assert torch.equal(held[0], now[0]) and torch.equal(held[1], now[1])
    from resinfer_b200 import _cabi
    kv, q, t = sets[0]
    need = _cabi.load().ri_resattn_shared_prefix_workspace_bytes(4, 16, 128, 2, 2)
    own = torch.full((need + 64,), 0xFF, dtype=torch.uint8, device=cuda_device)
    for _ in range(2):                                            # dirty, and used before
        out = torch.zeros_like(want[0])
        call(t, kv, out, workspace=own[:need])
        assert torch.equal(out, now[0]) and bool((own[need:] == 0xFF).all())
    with pytest.raises(RuntimeError, match="workspace"):
        call(t, kv, out, workspace=own[:need - 32])
    with pytest.raises(ValueError, match="workspace"):
        call(t, kv, out, workspace=own.float())
    ops.check_status(cuda_device)


def test_refusals_on_the_device(cuda_device):
    from resinfer_b200 import ops
    kv, q, t = make(cuda_device, [100, 90], 64, 2, 8, 128, 16)
    out = torch.zeros_like(t["q"])

    def call(prefix=64, row=0, ps=1, sp=1, o=out, **kw):
        a = dict(t, **kw)
        return ops.resattn_decode_shared_prefix(a["q"], a["k_data"], a["k_sf"], a["v_data"], a["v_sf"], a["block_tables"], a["seq_lens"],
                                                prefix, 0.1, 1.0, o, prefix_splits=ps, splits=sp, prefix_row=row, max_kv_len=100)

    for kw in (dict(q=t["q"].float()), dict(q=t["q"][:, :, ::2]), dict(q=t["q"][:1]), dict(block_tables=t["block_tables"].long()),
               dict(block_tables=t["block_tables"].t().contiguous().t()), dict(seq_lens=t["seq_lens"].long()), dict(seq_lens=t["seq_lens"][:1]),
               dict(q=t["q"].cpu()), dict(seq_lens=t["seq_lens"].cpu()), dict(row=2), dict(row=-1), dict(o=out.cpu()), dict(o=out[:, :8])):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(prefix=-1), dict(prefix=10 ** 6), dict(ps=300), dict(sp=0), dict(o=out.half())):
        with pytest.raises(RuntimeError):
            call(**kw)
    empty = call(q=t["q"][:0], block_tables=t["block_tables"][:0], seq_lens=t["seq_lens"][:0], o=out[:0])
    assert empty.shape == (0, 16, 128)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("rise,tokens", [(100.0, 2000), (120.0, 600), (-100.0, 2000), (0.0, 600)])
def test_scores_that_grow_or_fall_along_the_prefix(cuda_device, d, rise, tokens):
    """Every step raises every row's maximum (by up to 2^30 a step), or none does after the first.  A score of 120 in
    log2 carries at most 120 * 2^-22 * 4 = 1.2e-4 from the FP32 products, within the bound's margin."""
    from resinfer_b200.nvfp4.cute_attn import host
    hkv, g, page, b = 1, 8, 32, 3
    lens = [tokens + 40, tokens + 1, tokens]
    pool = _pool(cuda_device, (tokens + 40) // page + 1, hkv, page, d, False)
    gen = torch.Generator().manual_seed(3)
    total = tokens + 40
    ramp = torch.linspace(0, 1, total)[:, None, None] * (rise * np.log(2.0) / d ** 0.5)   # q = 1: score = sum over d / sqrt(d)
    k = (ramp + 0.3 * torch.randn(total, hkv, d, generator=gen)).bfloat16().to(cuda_device)
    v = torch.randn(total, hkv, d, generator=gen).bfloat16().to(cuda_device)
    pool.k_global_scale, pool.v_global_scale = 0.004, 0.002
    host.write_paged_kv(k, v, pool, torch.arange(total, device=cuda_device))
    table = torch.arange(total // page + 1, dtype=torch.int32).repeat(b, 1)[:, :pool.k_data.shape[0]].contiguous()
    kv = _as_numpy(pool, table, lens)
    q = torch.ones(b, g * hkv, d) + 0.2 * torch.randn(b, g * hkv, d, generator=gen)
    q = q.bfloat16()
    t = {n: torch.from_numpy(kv[n]).to(cuda_device) for n in ("k_data", "k_sf", "v_data", "v_sf", "seq_lens")}
    t["block_tables"], t["q"] = table.to(cuda_device), q.to(cuda_device)
    want = reference(q.float().numpy(), kv, d ** -0.5)
    for ps, sp in ((1, 1), (3, 2), (0, 1)):
        got = run(t, kv, tokens, d ** -0.5, ps, sp)
        for i in range(b):
            assert rel_fro(got[i].cpu().numpy(), want[i]) < TOL_F32, (ps, sp, i)


def test_a_query_that_is_not_finite_spoils_its_own_head_only(cuda_device):
    kv, q, t = make(cuda_device, [400, 350, 300], 290, 2, 8, 128, 16)
    clean = run(t, kv, 290, 0.1, 2, 2)
    bad = t["q"].clone()
    bad[1, 3], bad[2, 9, 5], bad[0, 15, 64] = float("nan"), float("inf"), float("-inf")
    got = run(dict(t, q=bad), kv, 290, 0.1, 2, 2)
    same = torch.ones(3, 16, dtype=torch.bool, device=cuda_device)
    same[1, 3] = same[2, 9] = same[0, 15] = False
    assert torch.equal(got[same], clean[same])


@pytest.mark.parametrize("d,g", [(128, 8), (128, 4), (256, 6)])
def test_zero_and_tiny_queries(cuda_device, d, g):
    """Blocks of zeros, whole heads of zeros (a plain mean of V), and values whose block scale rounds to zero."""
    lens, prefix = [400, 350, 0, 291], 290
    kv, q, t = make(cuda_device, lens, prefix, 2, g, d, 32)
    q[0, 1] = 0
    q[1, 2, :16] = 0
    q[1, 0, 16:48] = O.bf16_round(np.float32(1e-5))
    q[3] = -0.0
    t["q"].copy_(torch.from_numpy(q))
    want = reference(q, kv, d ** -0.5)
    for ps, sp in ((2, 2), (0, 1)):
        got = run(t, kv, prefix, d ** -0.5, ps, sp)
        for i in (0, 1, 3):
            assert rel_fro(got[i].cpu().numpy(), want[i]) < TOL_F32, (ps, sp, i)
        assert not got[2].any()
