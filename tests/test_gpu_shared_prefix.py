"""Shared-prefix decode against the decode oracle in 64 bits.

Tolerances, relative Frobenius: the FP32 output differs from exact attention over the held cache (query codes included)
by P's rounding to FP16 (half a step: 2^-11, uniform, so 2^-11 / sqrt(3) = 2.8e-4 in the mean square), by 2^x of the
special function unit (2^-22) and FP32 sums over up to 40 K tokens (below 1e-5): together under 3e-4; the bound is 6e-4,
twice that, for the rows where few tokens carry the weight and the errors do not average.  BF16 output adds its own
rounding, 2^-8 at most and 2^-8 / sqrt(3) = 2.3e-3 in the mean square at worst: 2.3e-3 + 3e-4 < 3e-3.  The plain decode
has the same errors, so the two differ by at most the sum, 1.2e-3 in FP32."""
import numpy as np
import pytest
import torch

import oracle as O

pytestmark = pytest.mark.gpu

TOL_F32, TOL_BF16 = 6e-4, 3e-3


def rel_fro(a, b):
    a, b = np.asarray(a, np.float64), np.asarray(b, np.float64)
    return float(np.linalg.norm(a - b) / max(np.linalg.norm(b), 1e-30))


def scale_rcp(x):
    """The reciprocal of a scale, and the scale itself for the reciprocal of one: what the definition divides by."""
    y = 1.0 / np.asarray(x, np.float64)
    grid = O.e4m3_decode(np.arange(1, 0x7F, dtype=np.uint8)).astype(np.float64)
    near = grid[np.abs(grid[None] - y.reshape(-1, 1)).argmin(1)].reshape(y.shape)
    return np.where(np.abs(y / near - 1) < 1e-6, near, y).astype(np.float32)


def even(q):
    """q with every block of 16 scaled so that its largest magnitude is 6 times a power of two."""
    x = q.float().unflatten(-1, (-1, 16))
    amax = x.abs().amax(-1, keepdim=True)
    want = 6 * torch.exp2(torch.round(torch.log2(amax / 6)))
    return torch.where(x.abs() == amax, torch.sign(x) * want, x * (want / amax) * 0.99).flatten(-2).to(q.dtype)


def make(dev, lens, prefix, hkv, g, d, page, seed=1, heat=1.0):
    """A pool in which sequence b's first min(lens[b], prefix) tokens are shared pages (the page in which the prefix ends
    is copied).  numpy oracle inputs and device tensors."""
    b = len(lens)
    kv = O.make_paged_kv([prefix + page] + [max(0, n - prefix // page * page) or 1 for n in lens], hkv, d, page, seed=seed)
    shared, tail = prefix // page, prefix % page
    own = kv["block_tables"]
    cols = max(shared + 1, max((n + page - 1) // page for n in lens), 1) + 1
    bt = np.full((b, cols), -1, np.int32)
    for i, n in enumerate(lens):
        bt[i, :shared] = own[0, :shared]
        k = max(0, (n + page - 1) // page - shared)
        bt[i, shared:shared + k] = own[1 + i, :k]
        if tail:
            if k == 0:
                bt[i, shared] = own[0, shared]                   # a row that ends inside the prefix, or row 0's prefix
            else:
                for part in ("k_data", "k_sf", "v_data", "v_sf"):
                    kv[part][own[1 + i, 0], :, :tail] = kv[part][own[0, shared], :, :tail]
    kv["block_tables"], kv["seq_lens"] = np.maximum(bt, 0), np.asarray(lens, np.int32)
    rng = np.random.default_rng(seed + 7)
    q = O.bf16_round((rng.standard_normal((b, hkv * g, d)) * heat).astype(np.float32))
    t = {k: torch.from_numpy(np.ascontiguousarray(kv[k])).to(dev) for k in ("k_data", "k_sf", "v_data", "v_sf", "seq_lens")}
    t["block_tables"] = torch.from_numpy(np.ascontiguousarray(bt)).to(dev)
    t["q"] = torch.from_numpy(q).to(torch.bfloat16).to(dev)
    return kv, q, t


def reference(q, kv, sm):
    """float64 [B, Hq, D] without output rounding."""
    b, hq, d = q.shape
    hkv, page = kv["k_data"].shape[1:3]
    g = hq // hkv
    qb, qr = O.dequant_grouped_q(*O.nvfp4_quant_grouped_q(q.reshape(b, hkv, g, d), rcp=O.RecordingRcp(scale_rcp)), g)
    qq = qb.astype(np.float64) + qr
    kd, vd = O.dequant_paged(kv["k_data"], kv["k_sf"]), O.dequant_paged(kv["v_data"], kv["v_sf"])
    out = np.zeros((b, hkv, g, d))
    for i, n in enumerate(kv["seq_lens"]):
        if n == 0:
            continue
        pages = kv["block_tables"][i, :(n + page - 1) // page]
        k = kd[pages].transpose(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n].astype(np.float64)
        v = vd[pages].transpose(1, 0, 2, 3).reshape(hkv, -1, d)[:, :n].astype(np.float64)
        s = np.einsum("hgd,htd->hgt", qq[i], k) * (sm * kv["k_global_scale"])
        p = np.exp(s - s.max(-1, keepdims=True))
        out[i] = np.einsum("hgt,htd->hgd", p / p.sum(-1, keepdims=True), v) * kv["v_global_scale"]
    return out.reshape(b, hq, d)


def run(t, kv, prefix, sm, prefix_splits, splits, dtype=torch.float32, row=0, max_len=None):
    from resinfer_b200 import ops
    out = torch.full(t["q"].shape, float("nan"), dtype=dtype, device=t["q"].device)
    ops.resattn_decode_shared_prefix(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"], t["seq_lens"], prefix,
                                     sm * kv["k_global_scale"], kv["v_global_scale"], out, prefix_splits=prefix_splits, splits=splits,
                                     prefix_row=row, max_kv_len=int(kv["seq_lens"].max()) if max_len is None else max_len)
    torch.cuda.synchronize()
    ops.check_status(t["q"].device)
    return out


CASES = [
    # lens, prefix, hkv, g, d, page, prefix_splits, splits, heat
    ([130], 64, 1, 8, 128, 16, 1, 1, 1.0),                       # one step, one row tile
    ([65, 66], 64, 2, 8, 128, 64, 1, 1, 1.0),
    ([1, 2], 1, 1, 4, 128, 16, 1, 1, 1.0),                       # a prefix of one token
    ([300, 257, 290], 256, 2, 8, 128, 128, 2, 2, 1.0),           # pages of 128: the tail's tiles come by TMA
    ([200, 191, 1000], 190, 2, 4, 128, 16, 3, 4, 1.0),           # the prefix ends inside a page and a tile
    ([700] * 20, 555, 1, 8, 128, 48, 4, 1, 2.0),                 # 160 rows: two row tiles, page size no power of two
    ([500, 0, 90, 33, 0, 333], 333, 2, 6, 128, 32, 3, 2, 1.0),   # empty rows, rows inside the prefix, one that ends with it
    ([0, 0, 0], 100, 1, 8, 128, 16, 2, 2, 1.0),                  # nothing to attend to
    ([5000, 4100, 4097], 4096, 2, 8, 128, 128, 16, 4, 3.0),      # peaked rows: maxima move, accumulators are rescaled
    ([130, 77], 64, 1, 8, 256, 16, 1, 1, 1.0),
    ([500, 0, 90, 1333], 333, 2, 6, 256, 64, 3, 3, 1.0),
    ([2600] * 17 + [2555], 2555, 1, 8, 256, 128, 8, 1, 3.0),
    ([300, 400], 0, 2, 8, 128, 16, 0, 3, 1.0),                   # no prefix launch
    ([300, 400], 250, 2, 8, 256, 16, 0, 1, 1.0),
    ([300, 400], 250, 2, 8, 128, 16, 9, 5, 1.0),                 # more pieces than steps
]


@pytest.mark.parametrize("lens,prefix,hkv,g,d,page,ps,splits,heat", CASES)
def test_matches_definition(cuda_device, lens, prefix, hkv, g, d, page, ps, splits, heat):
    from resinfer_b200 import ops
    kv, q, t = make(cuda_device, lens, prefix, hkv, g, d, page, heat=heat)
    sm = d ** -0.5
    want = reference(q, kv, sm)
    got = run(t, kv, prefix, sm, ps, splits)
    assert torch.isfinite(got).all()
    assert rel_fro(got.cpu().numpy(), want) < TOL_F32
    for i, n in enumerate(lens):                                 # each sequence by itself, and zeros for an empty one
        if n == 0:
            assert not got[i].any()
        else:
            assert rel_fro(got[i].cpu().numpy(), want[i]) < TOL_F32, (i, n)
    half = run(t, kv, prefix, sm, ps, splits, dtype=torch.bfloat16)
    assert torch.equal(half, got.to(torch.bfloat16))
    assert rel_fro(half.float().cpu().numpy(), want) < TOL_BF16
    assert torch.equal(run(t, kv, prefix, sm, ps, splits), got)   # no order that changes
    t["q"] = even(t["q"])
    got, plain = run(t, kv, prefix, sm, ps, splits), torch.zeros_like(got)
    ops.resattn_decode(t["q"], t["k_data"], t["k_sf"], t["v_data"], t["v_sf"], t["block_tables"].clamp(min=0), t["seq_lens"],
                       sm * kv["k_global_scale"], kv["v_global_scale"], plain, splits=2)
    assert rel_fro(got.cpu().numpy(), plain.cpu().numpy()) < 2 * TOL_F32
