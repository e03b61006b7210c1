"""Refusals of the paged KV-cache operators that need no GPU: argument checks of the C entry points and of the Python
wrappers."""
import pytest
import torch

BF16, FP16, F32 = 0, 1, 2


@pytest.fixture(scope="module")
def lib():
    from resinfer_b200 import _cabi, build
    build.build()
    return _cabi.load()


def _write(lib, *, dtype=BF16, slot_bits=64, n=4, ptr=4096, pages=2, cs=0, ss=0, hkv=2, d=128, page=16, kg=1.0, vg=1.0, k=4096, slots=4096):
    return lib.ri_kv_write_nvfp4(k, 4096, dtype, hkv * d, d, hkv * d, d, slots, slot_bits, n, ptr, ptr, ptr, ptr, pages, cs, ss,
                                 hkv, d, page, kg, vg, None)


def _read(lib, *, slots=4096, slot_bits=64, tables=None, cu=None, batch=0, cols=0, n=4, kg=1.0, out=4096, dtype=BF16, hkv=2, d=128, page=16):
    return lib.ri_kv_read_nvfp4(4096, 4096, 4096, 4096, 2, 0, 0, hkv, d, page, slots, slot_bits, tables, cols, cols, cu, batch, n,
                                kg, 1.0, out, out, dtype, 0, None)


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=F32), b"bf16 or fp16"), (dict(slot_bits=16), b"32- or 64-bit"), (dict(n=-1), b"token count"),
    (dict(d=24), b"multiple of 16"), (dict(hkv=0), b"KV head"), (dict(page=8), b"page size"), (dict(page=24), b"page size"),
    (dict(pages=0), b"empty"), (dict(ptr=None), b"empty"), (dict(cs=100), b"page strides"), (dict(ss=16), b"page strides"),
    (dict(ptr=4100), b"16-byte aligned"), (dict(kg=0.0), b"k_global_scale"), (dict(vg=float("nan")), b"v_global_scale"),
    (dict(kg=float("inf")), b"k_global_scale"), (dict(kg=-1.0), b"k_global_scale"), (dict(kg=1e-45), b"k_global_scale"),
    (dict(k=None), b"must not be null"), (dict(slots=None), b"must not be null"), (dict(slots=4100), b"misaligned"),
])
def test_write_refuses(lib, kw, text):
    assert _write(lib, **kw) == -1
    assert text in lib.ri_last_error()


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=3), b"bf16, fp16 or fp32"), (dict(n=-1), b"token count"), (dict(slots=None), b"slots must be given"),
    (dict(slot_bits=8), b"32- or 64-bit"), (dict(slots=None, tables=4096), b"block tables"), (dict(d=8), b"multiple of 16"),
    (dict(slots=None, tables=4096, cu=4096, batch=0, cols=1), b"block tables"), (dict(kg=0.0), b"k_global_scale"),
    (dict(out=None), b"16-byte aligned"), (dict(out=4104), b"16-byte aligned"),
])
def test_read_refuses(lib, kw, text):
    assert _read(lib, **kw) == -1
    assert text in lib.ri_last_error()


def test_no_tokens_is_no_work(lib):
    assert _write(lib, n=0, k=None, slots=None) == 0
    assert _read(lib, n=0, slots=None, out=None) == 0


def test_wrappers_refuse_host_pools():
    from resinfer_b200 import ops
    from resinfer_b200.nvfp4.cute_attn import NvFp4PagedKVPool, host
    kd, ks = torch.zeros(2, 2, 16, 64, dtype=torch.uint8), torch.zeros(2, 2, 16, 8, dtype=torch.uint8)
    pool = NvFp4PagedKVPool(2, 128, kd, kd, ks, ks, page_size=16)
    x, slots = torch.zeros(3, 2, 128, dtype=torch.bfloat16), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="CUDA"):
        host.write_paged_kv(x, x, pool, slots)
    with pytest.raises(ValueError, match="CUDA"):
        host.read_paged_kv(pool, slots)
    with pytest.raises(ValueError, match="pool.k_data"):
        host.gather_paged_kv(NvFp4PagedKVPool(2, 128, kd, kd, ks, ks, page_size=32), slots, slots, 3)
    with pytest.raises(ValueError, match="block scales"):
        ops.kv_write(x, x, kd, kd, kd, kd, slots, 1.0, 1.0)
