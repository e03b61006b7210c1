"""Shared-prefix decode without a GPU: the split plan, the refusals of the C entry point and of the Python wrappers."""
import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from resinfer_b200 import _cabi, build
    build.build()
    return _cabi.load()


@pytest.mark.parametrize("head_dim", [128, 256])
@pytest.mark.parametrize("batch,hkv,group", [(1, 1, 4), (2, 8, 8), (17, 3, 6), (64, 8, 8), (1000, 8, 8), (40000, 1, 4)])
@pytest.mark.parametrize("prefix,own", [(0, 1), (0, 5000), (1, 0), (63, 1), (128, 2048), (12345, 17), (1 << 20, 100000)])
def test_plans_are_launchable(head_dim, batch, hkv, group, prefix, own):
    from resinfer_b200.nvfp4.cute_attn.plan import select_shared_prefix_plan
    ps, sp = select_shared_prefix_plan(batch, hkv, group, prefix, prefix + own, 148, head_dim=head_dim)
    steps = -(-prefix // (128 if head_dim == 128 else 64))
    assert (ps == 0) == (prefix == 0) and 0 <= ps <= min(max(steps, 0), 256) and 1 <= sp <= 64
    if ps > 1:
        piece = -(-steps // ps)
        assert (ps - 1) * piece < steps                          # no empty piece
        assert ps * hkv * -(-batch * group // 128) <= 148        # more pieces than one only where they run at once


def _call(lib, *, q=4096, ptr=4096, pages=8, cs=0, ss=0, bt=4096, bt_cols=8, pt=4096, sl=4096, prefix=100, batch=2, hq=16, hkv=2,
          d=128, page=16, max_len=0, scale=0.1, out_scale=1.0, out=4096, dtype=0, ps=2, sp=1, ws=4096, ws_bytes=1 << 30):
    return lib.ri_resattn_decode_shared_prefix(q, ptr, ptr, ptr, ptr, pages, cs, ss, bt, bt_cols, bt_cols, pt, sl, prefix, batch, hq, hkv,
                                               d, page, max_len, scale, out_scale, out, dtype, ps, sp, ws, ws_bytes, None, None)


@pytest.mark.parametrize("kw,text", [
    (dict(d=64), b"head_dim=128 or 256"), (dict(dtype=1), b"bf16 or fp32"), (dict(dtype=3), b"bf16 or fp32"),
    (dict(hkv=0), b"divisible"), (dict(hq=15), b"divisible"), (dict(hq=4), b"GQA"), (dict(hq=10, hkv=2), b"GQA"),
    (dict(page=8), b"page size"), (dict(page=40), b"page size"), (dict(batch=-1), b"bad batch"), (dict(batch=65536), b"bad batch"),
    (dict(pages=0), b"bad batch"), (dict(pages=1 << 31), b"bad batch"), (dict(bt_cols=0), b"bad batch"),
    (dict(bt_cols=1 << 28), b"too long"), (dict(bt_cols=(1 << 27) - 4000), b"too long"), (dict(prefix=-1), b"within the block table"), (dict(prefix=129), b"within the block table"),
    (dict(max_len=-1), b"non-negative"), (dict(scale=0.0), b"positive and finite"), (dict(scale=-0.1), b"positive and finite"),
    (dict(scale=3e38), b"positive and finite"), (dict(scale=float("nan")), b"positive and finite"), (dict(scale=float("inf")), b"positive and finite"),
    (dict(out_scale=float("nan")), b"finite"), (dict(sp=0), b"splits must be"), (dict(sp=257), b"splits must be"),
    (dict(ps=-1), b"splits must be"), (dict(ps=257), b"splits must be"), (dict(batch=65535, hq=64, hkv=8, bt_cols=8, d=256), b"workspace"),
    (dict(batch=65535, hq=8 * 200, hkv=200), b"too many rows"), (dict(cs=1000), b"page strides"), (dict(ss=24), b"page strides"),
    (dict(cs=1 << 31), b"page strides"), (dict(q=None), b"null"), (dict(pt=None), b"null"), (dict(out=None), b"null"),
    (dict(q=4104), b"16-byte aligned"), (dict(out=4104), b"16-byte aligned"), (dict(ptr=4100), b"16-byte aligned"),
    (dict(ws=None), b"workspace"), (dict(ws_bytes=100), b"workspace"), (dict(ws=4112), b"workspace"),
])
def test_entry_refuses(lib, kw, text):
    if kw.get("batch") == 65535 and "hkv" in kw and kw["hkv"] == 8:
        kw = dict(kw, ws_bytes=1000)
    assert _call(lib, **kw) == -1
    assert text in lib.ri_last_error()


def test_empty_batch_is_no_work(lib):
    assert _call(lib, batch=0, q=None, bt=None, sl=None, out=None, ws=None, ptr=4096, pt=None) == 0


def test_workspace_bytes(lib):
    f = lib.ri_resattn_shared_prefix_workspace_bytes
    assert f(3, 16, 128, 4, 2) >= 6 * 3 * 16 * (128 + 2) * 4
    assert f(0, 16, 128, 0, 1) >= 0 and f(1, 16, 128, -1, 1) == -1 and f(1, 16, 128, 1, 0) == -1


def test_host_entry_refuses_without_a_device():
    from resinfer_b200.nvfp4.cute_attn import NvFp4PagedKVPool, host
    kd, ks = torch.zeros(4, 2, 16, 64, dtype=torch.uint8), torch.zeros(4, 2, 16, 8, dtype=torch.uint8)
    pool = NvFp4PagedKVPool(2, 128, kd, kd, ks, ks, page_size=16)
    q, bt, sl = torch.zeros(3, 16, 128, dtype=torch.bfloat16), torch.zeros(3, 4, dtype=torch.int32), torch.ones(3, dtype=torch.int32)
    run = host.run_paged_fp4_decode_shared_prefix
    with pytest.raises(ValueError, match="CUDA"):
        run(q, pool, bt, sl, 16, 0.1, torch.empty_like(q), max_seq_len=20, plan=(1, 1))
    with pytest.raises(ValueError, match="BF16"):
        run(q, pool, bt, sl, 16, 0.1, q.float(), max_seq_len=20)
    for prefix in (-1, 65):
        with pytest.raises(ValueError, match="prefix_len"):
            run(q, pool, bt, sl, prefix, 0.1, torch.empty_like(q), max_seq_len=20)
    with pytest.raises(NotImplementedError):
        run(q[:, :10], pool, bt, sl, 16, 0.1, q[:, :10], max_seq_len=20)
    with pytest.raises(ValueError, match="pool.k_data"):
        run(q, NvFp4PagedKVPool(2, 128, kd, kd, ks, ks, page_size=32), bt, sl, 16, 0.1, torch.empty_like(q), max_seq_len=20)
