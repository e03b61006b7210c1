"""Tensor-level entry points of the GEMM and attention kernels (thin wrappers over the C ABI).

These are the functions the reference-named modules (``nvfp4.cute_fold.host``,
``nvfp4.mxfp4.dense``, ``nvfp4.cute_attn.host``) call.  Workspaces are cached per
(device, size) like the reference caches its reduction workspaces
(ShawRong/ResInfer quant/vllm_integration/attn/decode.py:23-53); nothing is allocated once a
shape has been seen, so the calls stay CUDA-graph capturable after a warm-up.

One rule follows from the sharing: calls that use the same cached workspace (same device, same kind,
same size) must not overlap on the GPU -- issue them on one stream, or order the streams with events.
The split tickets in a workspace are left at zero by every launch that completes.
"""
from __future__ import annotations

import contextlib

import torch

from . import _cabi

_WORKSPACES: dict[tuple, torch.Tensor] = {}
_TICKET_BYTES: dict[tuple, int] = {}
_STATUS: dict[torch.device, torch.Tensor] = {}
_GEMM_PLANS: dict[tuple, tuple] = {}


class _on_device:
    """``torch.cuda.device(dev)`` that costs nothing when ``dev`` is already current (the usual case)."""

    __slots__ = ("ctx",)

    def __init__(self, dev):
        self.ctx = None if dev.index is None or torch.cuda.current_device() == dev.index else torch.cuda.device(dev)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            self.ctx.__exit__(*exc)



def _workspace(device, nbytes: int, tag: str, zero_prefix: int = 0) -> torch.Tensor:
    key = (str(device), tag, nbytes)
    ws = _WORKSPACES.get(key)
    if ws is None:
        ws = torch.empty(max(nbytes, 256), dtype=torch.uint8, device=device)
        if zero_prefix:
            ws[:zero_prefix].zero_()
        _WORKSPACES[key] = ws
        _TICKET_BYTES[key] = int(zero_prefix)
    return ws


def status_word(device) -> torch.Tensor:
    """Device int32 that kernels set non-zero when one of their bounded waits expired."""
    device = torch.device(device)
    st = _STATUS.get(device)
    if st is None:
        st = torch.zeros(1, dtype=torch.int32, device=device)
        _STATUS[device] = st
    return st


def check_status(device) -> None:
    """Synchronising check of the status word.  A non-zero word means that a bounded device-side wait
    expired in some launch since the last check: that launch's output is invalid and it may have left
    split tickets behind, so the ticket areas of the cached workspaces of the device are cleared before
    the error is raised."""
    st = status_word(device)
    v = int(st.item())
    if v:
        st.zero_()
        for key, ws in _WORKSPACES.items():
            if key[0] == str(torch.device(device)) and _TICKET_BYTES.get(key):
                ws[:_TICKET_BYTES[key]].zero_()
        raise RuntimeError(f"a device-side wait expired (status {v})")


_ACTIVE_REDUCER = None
_ACTIVE_REDUCER_EPILOGUE = True
_NO_REDUCER = object()                   # "no reduction for this call" inside a row_parallel_reduction block


@contextlib.contextmanager
def row_parallel_reduction(reducer, epilogue: bool = True):
    """Inside the block every ``fp4_gemm`` call without an explicit ``allreduce`` argument -- in particular the
    ones made by ``residue::nvfp4_linear`` and ``residue::mxfp4_linear``, whose schemas have no room for it --
    returns its output summed over the ranks of ``reducer`` (a ``resinfer_b200.quant.tp.PeerAllReduce``):
    in the GEMM's epilogue (``epilogue=True``), or by the stand-alone kernel with the GEMM writing its partial
    straight into the exported buffer (``epilogue=False``: two launches, no copy in between).  This is where a
    tensor-parallel model wraps the linear of a row-parallel layer; ``None`` switches it off again for a nested
    block.  Process-wide, not per thread."""
    global _ACTIVE_REDUCER, _ACTIVE_REDUCER_EPILOGUE
    prev = (_ACTIVE_REDUCER, _ACTIVE_REDUCER_EPILOGUE)
    _ACTIVE_REDUCER, _ACTIVE_REDUCER_EPILOGUE = reducer, bool(epilogue)
    try:
        yield reducer
    finally:
        _ACTIVE_REDUCER, _ACTIVE_REDUCER_EPILOGUE = prev


def fp4_gemm(act: torch.Tensor, act_sf: torch.Tensor, weight: torch.Tensor, weight_sf: torch.Tensor,
             alpha: torch.Tensor | None, *, m: int, fmt: str = "nvfp4", layout: str = "plain",
             out_dtype: torch.dtype = torch.bfloat16, out: torch.Tensor | None = None,
             splits: int = 0, enable_pdl: bool = True, allreduce=None) -> torch.Tensor:
    """out[m, N] = alpha * act . weight^T with block-scaled FP4 operands.

    act: uint8 codes, [M, K/2] (plain), [2M, K/2] (row_pair) or [M, K] (concat_k); weight uint8
    [N, K/2] (row stride may exceed K/2); scale buffers 128x4-swizzled uint8 (E4M3 for nvfp4, E8M0
    for mxfp4); alpha float32 device tensor with 1 (or, row_pair, 2) elements or None.

    ``allreduce``: a ``resinfer_b200.quant.tp.PeerAllReduce`` makes this the GEMM of a row-parallel
    linear: the kernel stores this rank's BF16 partial into every rank's inbox and sums the partials of
    all ranks itself (``ri_fp4_gemm_allreduce``); ``out`` (BF16) receives the sum.  Every
    rank of the group must make the same calls in the same order."""
    lib = _cabi.load()
    if allreduce is None and _ACTIVE_REDUCER is not None:
        if _ACTIVE_REDUCER_EPILOGUE:
            allreduce = _ACTIVE_REDUCER
        else:
            # the GEMM writes this rank's partial into the exported buffer, the stand-alone kernel sums the ranks
            red, n_out = _ACTIVE_REDUCER, weight.shape[0]
            if out_dtype != torch.bfloat16 or (out is not None and out.dtype != torch.bfloat16):
                raise ValueError("the all-reduce sums BF16 partials")
            part = fp4_gemm(act, act_sf, weight, weight_sf, alpha, m=m, fmt=fmt, layout=layout, out_dtype=out_dtype,
                            out=red.partial((m, n_out)), splits=splits, enable_pdl=enable_pdl, allreduce=_NO_REDUCER)
            return red.reduce(part, out)
    if allreduce is _NO_REDUCER:
        allreduce = None
    fmt_c = {"nvfp4": _cabi.FMT_NVFP4, "mxfp4": _cabi.FMT_MXFP4}[fmt]
    lay_c = {"plain": _cabi.GEMM_PLAIN, "row_pair": _cabi.GEMM_ROW_PAIR, "concat_k": _cabi.GEMM_CONCAT_K}[layout]
    n, kp = weight.shape
    k = kp * 2
    dev = weight.device
    if weight.stride(1) != 1:
        raise ValueError(f"weight must stay K-contiguous within a row; got stride {weight.stride()}")
    if act.dim() != 2 or act.stride(1) != 1:
        raise ValueError(f"activation must be compact rows; got stride {act.stride()}")
    if out is None:
        out = torch.empty((m, n), dtype=out_dtype, device=dev)
    with _on_device(dev):
        ws = None
        plan_key = (dev.index, m, n, k, fmt_c, lay_c, splits)
        plan = _GEMM_PLANS.get(plan_key)
        if plan is None:                                   # workspace size of a shape, asked once per device
            plan = (lib.ri_fp4_gemm_workspace_bytes(m, n, k, fmt_c, lay_c, splits), lib.ri_fp4_gemm_counter_bytes(m, n))
            _GEMM_PLANS[plan_key] = plan
        ws_bytes = plan[0]
        if ws_bytes < 0:
            _cabi.check(_cabi.RI_ERR_ARG, "fp4_gemm plan")
        if ws_bytes > 0:
            ws = _workspace(dev, ws_bytes, "gemm", zero_prefix=plan[1])
        if allreduce is not None:
            if out.dtype != torch.bfloat16 or out.stride(1) != 1:
                raise ValueError("the fused all-reduce writes a BF16 result with contiguous rows")
            inboxes, area = allreduce.next_inbox(m * n)
            st = lib.ri_fp4_gemm_allreduce(
                act.data_ptr(), act.stride(0), act_sf.data_ptr(), act_sf.numel(),
                weight.data_ptr(), weight.stride(0), weight_sf.data_ptr(), weight_sf.numel(),
                _cabi.ptr(alpha), 0 if alpha is None else alpha.numel(), n, m, n, k, fmt_c, lay_c,
                splits, _cabi.ptr(ws), ws_bytes, allreduce.status.data_ptr(), int(enable_pdl),
                _cabi.current_stream(dev), inboxes, area, allreduce.tile_flag_ptrs,
                allreduce.tile_calls.data_ptr(), allreduce.max_tiles, allreduce.rank, allreduce.world,
                out.data_ptr(), out.stride(0))
            _cabi.check(st, "fp4_gemm_allreduce")
            return out
        st = lib.ri_fp4_gemm(
            act.data_ptr(), act.stride(0), act_sf.data_ptr(), act_sf.numel(),
            weight.data_ptr(), weight.stride(0), weight_sf.data_ptr(), weight_sf.numel(),
            _cabi.ptr(alpha), 0 if alpha is None else alpha.numel(),
            out.data_ptr(), _cabi.torch_dtype_code(out.dtype, allow_f32=True), out.stride(0), m, n, k, fmt_c, lay_c,
            splits, _cabi.ptr(ws), ws_bytes, status_word(dev).data_ptr(), int(enable_pdl),
            _cabi.current_stream(dev))
    _cabi.check(st, "fp4_gemm")
    return out


def fp4_gemm_static_scratch(act: torch.Tensor, act_sf: torch.Tensor, weight: torch.Tensor,
                            weight_sf: torch.Tensor, alpha: torch.Tensor | None, *, m: int, out: torch.Tensor,
                            fmt: str = "nvfp4", layout: str = "plain", splits: int = 0,
                            enable_pdl: bool = True) -> torch.Tensor:
    """`fp4_gemm` through the entry point that allocates nothing: `out` is required, the K-split
    scratch is the library's built-in per-device array (shared by all calls on the device, so calls
    must not overlap in time), and sizes that need more than that array raise RuntimeError."""
    lib = _cabi.load()
    fmt_c = {"nvfp4": _cabi.FMT_NVFP4, "mxfp4": _cabi.FMT_MXFP4}[fmt]
    lay_c = {"plain": _cabi.GEMM_PLAIN, "row_pair": _cabi.GEMM_ROW_PAIR, "concat_k": _cabi.GEMM_CONCAT_K}[layout]
    n, kp = weight.shape
    dev = weight.device
    if weight.stride(1) != 1 or act.dim() != 2 or act.stride(1) != 1:
        raise ValueError("operands must be K-contiguous rows")
    with torch.cuda.device(dev):
        st = lib.ri_fp4_gemm_static_scratch(
            act.data_ptr(), act.stride(0), act_sf.data_ptr(), act_sf.numel(),
            weight.data_ptr(), weight.stride(0), weight_sf.data_ptr(), weight_sf.numel(),
            _cabi.ptr(alpha), 0 if alpha is None else alpha.numel(),
            out.data_ptr(), _cabi.torch_dtype_code(out.dtype, allow_f32=True), out.stride(0), m, n, kp * 2,
            fmt_c, lay_c, splits, status_word(dev).data_ptr(), int(enable_pdl), _cabi.current_stream(dev))
    _cabi.check(st, "fp4_gemm_static_scratch")
    return out


@contextlib.contextmanager
def resattn_pv_format(fmt: str):
    """Inside the block ``resattn_decode`` runs its second product in ``fmt``: "fp16" (the default: V exact,
    P with 11 bits) or "e4m3" (V and P rounded to E4M3 like the reference's kernel: faster, about ten times
    further from exact attention).  Process-wide (``ri_resattn_set_pv_format``)."""
    lib = _cabi.load()
    code = {"fp16": 0, "e4m3": 1}[fmt]
    prev = int(lib.ri_resattn_get_pv_format())
    lib.ri_resattn_set_pv_format(code)
    try:
        yield
    finally:
        lib.ri_resattn_set_pv_format(prev)


def kv_page_strides(k_data: torch.Tensor, k_sf: torch.Tensor, v_data: torch.Tensor, v_sf: torch.Tensor):
    """(code bytes, scale bytes) between consecutive pages of a paged NVFP4 KV pool.

    Each of the four tensors is [pages, Hkv, page, D/2 or D/16] with the three inner dimensions dense; the page
    stride is free, so the views vLLM cuts out of its interleaved cache (every page = K codes | K scales |
    V codes | V scales) are taken as they are.  K and V must share their strides."""
    def one(t, name):
        _, h, page, w = t.shape
        want = (page * w, w, 1)
        if t.element_size() != 1 or tuple(t.stride()[1:]) != want or (t.shape[0] > 1 and t.stride(0) < h * page * w):
            raise ValueError(f"{name} must be a byte tensor [pages, Hkv, page, {w}] with dense inner dimensions, got "
                             f"shape {tuple(t.shape)} strides {tuple(t.stride())}")
        return int(t.stride(0)) if t.shape[0] > 1 else h * page * w
    kc, vc = one(k_data, "k_data"), one(v_data, "v_data")
    ks, vs = one(k_sf, "k_sf"), one(v_sf, "v_sf")
    if kc != vc or ks != vs:
        raise ValueError(f"K and V must have the same page strides, got codes {kc} / {vc}, scales {ks} / {vs}")
    return kc, ks


def resattn_decode(q: torch.Tensor, k_data: torch.Tensor, k_sf: torch.Tensor, v_data: torch.Tensor,
                   v_sf: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor,
                   score_scale: float, out_scale: float, out: torch.Tensor, *, splits: int = 1,
                   q_residue: bool = True, q_pack: torch.Tensor | None = None,
                   q_sf: torch.Tensor | None = None, max_kv_len: int = 0,
                   out_global_scale: torch.Tensor | None = None,
                   out_block_scale: torch.Tensor | None = None, reducer: str = "ticket") -> torch.Tensor:
    """Paged NVFP4-KV decode attention.  q bf16 [B,Hq,D]; k_data/v_data uint8 [pages,Hkv,page,D/2];
    k_sf/v_sf uint8 (or float8_e4m3fn) [pages,Hkv,page,D/16] (any page stride: ``kv_page_strides``); out bf16 [B,Hq,D] (written) -- or, with
    ``out_global_scale`` (float32[1]) and ``out_block_scale`` (128x4-swizzled E4M3 bytes), packed NVFP4:
    out uint8 [B, Hq*D/2].  ``reducer``: how the KV splits are combined, "ticket" (through a workspace, the CTA
    that finishes last) or "cluster" (2 to 8 or 16 splits as one thread-block cluster, through shared memory); same bits."""
    lib = _cabi.load()
    b, hq, d = q.shape
    pages, hkv, page, _ = k_data.shape
    dev = q.device
    code_stride, sf_stride = kv_page_strides(k_data, k_sf, v_data, v_sf)
    reducer_c = {"ticket": _cabi.ATTN_REDUCER_TICKET, "cluster": _cabi.ATTN_REDUCER_CLUSTER}[reducer]
    with torch.cuda.device(dev):
        ws = None
        ws_bytes = 0
        if splits > 1 and reducer == "ticket":
            ws_bytes = lib.ri_resattn_workspace_bytes(b, hq, d, splits)
            ws = _workspace(dev, ws_bytes, "attn", zero_prefix=lib.ri_resattn_counter_bytes(b, hq))
        st = lib.ri_resattn_decode_strided(
            q.data_ptr(), k_data.data_ptr(), k_sf.data_ptr(), v_data.data_ptr(), v_sf.data_ptr(), pages,
            code_stride, sf_stride, block_tables.data_ptr(), block_tables.stride(0), seq_lens.data_ptr(), b, hq, hkv, d, page,
            int(max_kv_len), float(score_scale), float(out_scale), out.data_ptr(),
            _cabi.DTYPE_NVFP4 if out_block_scale is not None else _cabi.torch_dtype_code(out.dtype, allow_f32=True),
            _cabi.ptr(q_pack), 0 if q_pack is None else q_pack.numel(),
            _cabi.ptr(q_sf), 0 if q_sf is None else q_sf.numel(),
            _cabi.ptr(out_global_scale), _cabi.ptr(out_block_scale),
            0 if out_block_scale is None else out_block_scale.numel() * out_block_scale.element_size(),
            splits, reducer_c, _cabi.ptr(ws), ws_bytes, int(q_residue), status_word(dev).data_ptr(),
            _cabi.current_stream(dev))
    _cabi.check(st, "resattn_decode")
    return out


def resattn_decode_shared_prefix(q: torch.Tensor, k_data: torch.Tensor, k_sf: torch.Tensor, v_data: torch.Tensor,
                                 v_sf: torch.Tensor, block_tables: torch.Tensor, seq_lens: torch.Tensor, prefix_len: int,
                                 score_scale: float, out_scale: float, out: torch.Tensor, *, prefix_splits: int, splits: int,
                                 prefix_row: int = 0, max_kv_len: int = 0, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention for a batch whose sequences share their first ``prefix_len`` tokens
    (``ri_resattn_decode_shared_prefix``): the result of ``resattn_decode`` on the same tables, the prefix read once.

    q bf16 [B, Hq, D], out bf16 or fp32 [B, Hq, D], both contiguous; ``block_tables`` int32 [B, max pages] cover every sequence
    from its first token and row ``prefix_row`` holds all pages of the prefix; ``seq_lens`` int32 [B] are whole lengths.
    ``prefix_splits`` / ``splits``: pieces of the prefix (0: no launch for it) and of the tokens behind it, see
    ``nvfp4.cute_attn.plan.select_shared_prefix_plan``.  ``workspace``: a uint8 buffer of
    ``ri_resattn_shared_prefix_workspace_bytes``; without one it comes from the caching allocator on the current stream, so
    calls on different streams, and graphs that hold them, do not share it."""
    pages, code_stride, sf_stride, hkv, d, page = _kv_pool_args(k_data, k_sf, v_data, v_sf)
    dev, shape, bt_shape = k_data.get_device(), q.shape, block_tables.shape
    if len(shape) != 3 or shape[2] != d or q.dtype != torch.bfloat16 or not q.is_contiguous() or q.get_device() != dev:
        raise ValueError(f"q must be contiguous BF16 [B, H_q, {d}] on cuda:{dev}")
    b, hq, _ = shape
    if out.shape != shape or out.get_device() != dev or not out.is_contiguous():
        raise ValueError(f"out must be contiguous {tuple(shape)} on cuda:{dev}")
    if (len(bt_shape) != 2 or bt_shape[0] != b or bt_shape[1] < 1 or block_tables.dtype != torch.int32 or block_tables.get_device() != dev
            or block_tables.stride(1) != 1):
        raise ValueError("block_tables must be int32 [batch, max_pages_per_seq] on the Q device with unit column stride")
    if seq_lens.dtype != torch.int32 or seq_lens.get_device() != dev or seq_lens.shape != (b,) or not seq_lens.is_contiguous():
        raise ValueError("seq_lens must be contiguous int32 [batch] on the Q device")
    if b and not 0 <= prefix_row < b:
        raise ValueError(f"prefix_row {prefix_row} is not a row of the block table ({b})")
    if workspace is None:
        need = _cabi.load().ri_resattn_shared_prefix_workspace_bytes(b, hq, d, prefix_splits, splits)
        workspace = torch.empty(max(need, 16), dtype=torch.uint8, device=q.device)
    elif workspace.dtype != torch.uint8 or workspace.get_device() != dev or not workspace.is_contiguous():
        raise ValueError(f"workspace must be contiguous uint8 on cuda:{dev}")
    bt, bt_stride = block_tables.data_ptr(), block_tables.stride(0)
    _call(dev, "ri_resattn_decode_shared_prefix", (
        q.data_ptr(), k_data.data_ptr(), k_sf.data_ptr(), v_data.data_ptr(), v_sf.data_ptr(), pages, code_stride, sf_stride, bt,
        bt_stride, bt_shape[1], bt + 4 * prefix_row * bt_stride, seq_lens.data_ptr(), prefix_len, b, hq, hkv, d, page, max_kv_len,
        score_scale, out_scale, out.data_ptr(),
        _cabi.DTYPE_BF16 if out.dtype == torch.bfloat16 else _cabi.torch_dtype_code(out.dtype, allow_f32=True), prefix_splits,
        splits, workspace.data_ptr(), workspace.numel(), status_word(q.device).data_ptr()))
    return out


def _call(dev: int, name: str, args: tuple) -> None:
    """A C-ABI call whose last argument is the stream, with the tensors' device current; raises on rejection."""
    fn = getattr(_cabi.load(), name)
    if torch._C._cuda_getDevice() == dev:
        st = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            st = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if st:
        _cabi.check(st, name)


_BYTES = (torch.uint8, torch.int8, torch.float8_e4m3fn)


def _kv_pool_args(k_data: torch.Tensor, k_sf: torch.Tensor, v_data: torch.Tensor, v_sf: torch.Tensor):
    """(num_pages, code stride, scale stride, Hkv, D, page_size) of a paged NVFP4 pool, shapes and devices checked.
    The calls that use it take a few microseconds on the device: the usual case is told by a dozen comparisons."""
    shape, cs, ss, dev = k_data.shape, k_data.stride(), k_sf.stride(), k_data.get_device()
    if (len(shape) == 4 and v_data.shape == shape and v_data.stride() == cs and v_sf.stride() == ss and dev >= 0
            and dev == k_sf.get_device() == v_data.get_device() == v_sf.get_device()):
        pages, hkv, page, half = shape
        sf = half // 8
        if (k_sf.shape == (pages, hkv, page, sf) and v_sf.shape == k_sf.shape and half % 8 == 0 and pages > 1
                and cs[3] == 1 and cs[2] == half and cs[1] == page * half and cs[0] >= hkv * page * half
                and ss[3] == 1 and ss[2] == sf and ss[1] == page * sf and ss[0] >= hkv * page * sf
                and k_data.dtype == v_data.dtype == torch.uint8 and (k_sf.dtype == v_sf.dtype) and k_sf.dtype in _BYTES):
            return pages, cs[0], ss[0], hkv, half * 2, page
    if k_data.dim() != 4 or v_data.shape != k_data.shape or k_sf.dim() != 4 or v_sf.shape != k_sf.shape:
        raise ValueError(f"a paged NVFP4 pool is codes [pages, Hkv, page, D/2] and scales [pages, Hkv, page, D/16] for K and V, got "
                         f"{tuple(k_data.shape)} / {tuple(k_sf.shape)} and {tuple(v_data.shape)} / {tuple(v_sf.shape)}")
    pages, hkv, page, half = shape
    if half % 8 or tuple(k_sf.shape) != (pages, hkv, page, half // 8):
        raise ValueError(f"block scales of codes {tuple(k_data.shape)} must be [pages, Hkv, page, D/16] with D a multiple of 16, got {tuple(k_sf.shape)}")
    if not k_data.is_cuda or not (k_data.device == k_sf.device == v_data.device == v_sf.device):
        raise ValueError("the four tensors of a pool must be on one CUDA device")
    code_stride, sf_stride = kv_page_strides(k_data, k_sf, v_data, v_sf)
    return pages, code_stride, sf_stride, hkv, half * 2, page


def _check_slots(slots: torch.Tensor, dev: int) -> int:
    bits = {torch.int64: 64, torch.int32: 32}.get(slots.dtype)
    if bits is None or slots.dim() != 1 or slots.get_device() != dev or not slots.is_contiguous():
        raise ValueError(f"slots must be contiguous 1-D int32 or int64 on cuda:{dev}, got {slots.dtype} {tuple(slots.shape)} on {slots.device}")
    return bits


def _check_rows(name: str, x: torch.Tensor, n: int, hkv: int, d: int, dtype: torch.dtype, dev: int):
    """(token stride, head stride) of K or V rows."""
    shape, st = x.shape, x.stride()
    if (len(shape) != 3 or shape[0] < n or shape[1] != hkv or shape[2] != d or st[2] != 1 or x.dtype != dtype
            or (dtype != torch.bfloat16 and dtype != torch.float16) or x.get_device() != dev):
        raise ValueError(f"{name} must be bf16 or fp16 [>= {n}, {hkv}, {d}] on cuda:{dev} with unit stride along the head dimension, got "
                         f"{x.dtype} {tuple(shape)} strides {tuple(st)} on {x.device}")
    return st[0], st[1]


def kv_write(k: torch.Tensor, v: torch.Tensor, k_data: torch.Tensor, k_sf: torch.Tensor, v_data: torch.Tensor,
             v_sf: torch.Tensor, slots: torch.Tensor, k_global_scale: float, v_global_scale: float) -> None:
    """Quantise K and V rows into a paged NVFP4 cache (``ri_kv_write_nvfp4``).

    k, v: bf16 or fp16 [T, Hkv, D], unit stride along D, any other strides (slices of a fused projection).  ``slots``:
    int32 / int64, one per token: ``page index * page_size + offset``; negative = padding.  Fewer slots than rows: the
    rows behind the last slot are not written.  Slots must be distinct.  Pool tensors as for ``resattn_decode``, head_dim any
    multiple of 16.  The bytes are those of the NVFP4 quantisers with global scale ``1 / *_global_scale``."""
    pages, code_stride, sf_stride, hkv, d, page = _kv_pool_args(k_data, k_sf, v_data, v_sf)
    dev = k_data.get_device()
    bits = _check_slots(slots, dev)
    n, dtype = slots.shape[0], k.dtype
    k_token, k_head = _check_rows("k", k, n, hkv, d, dtype, dev)
    v_token, v_head = _check_rows("v", v, n, hkv, d, dtype, dev)
    _call(dev, "ri_kv_write_nvfp4", (
        k.data_ptr(), v.data_ptr(), _cabi.DTYPE_BF16 if dtype == torch.bfloat16 else _cabi.DTYPE_FP16, k_token, k_head, v_token,
        v_head, slots.data_ptr(), bits, n, k_data.data_ptr(), k_sf.data_ptr(), v_data.data_ptr(), v_sf.data_ptr(), pages,
        code_stride, sf_stride, hkv, d, page, k_global_scale, v_global_scale))


def kv_read(k_data: torch.Tensor, k_sf: torch.Tensor, v_data: torch.Tensor, v_sf: torch.Tensor, k_global_scale: float,
            v_global_scale: float, *, slots: torch.Tensor | None = None, block_tables: torch.Tensor | None = None,
            cu_seqlens: torch.Tensor | None = None, num_tokens: int | None = None, dtype: torch.dtype = torch.bfloat16,
            out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Held values of a paged NVFP4 cache as dense K and V rows [tokens, Hkv, D] (``ri_kv_read_nvfp4``): bf16, fp16 or fp32.

    Either ``slots`` (one per row; rows of negative slots are zero), or ``block_tables`` int32 [B, max pages] with
    ``cu_seqlens`` int32 [B + 1] and ``num_tokens`` rows: the sequences of the batch end to end.  Rows behind the last
    sequence stay as they are in a caller's ``out`` and are zero otherwise; tokens without a table entry are zero."""
    pages, code_stride, sf_stride, hkv, d, page = _kv_pool_args(k_data, k_sf, v_data, v_sf)
    dev = k_data.get_device()
    bits, slots_ptr, bt_ptr, cu_ptr, bt_stride, bt_cols, batch = 64, None, None, None, 0, 0, 0
    if slots is not None:
        if block_tables is not None or cu_seqlens is not None:
            raise ValueError("give slots, or block_tables with cu_seqlens, not both")
        bits = _check_slots(slots, dev)
        n, slots_ptr = slots.shape[0], slots.data_ptr()
        if num_tokens is not None and num_tokens != n:
            raise ValueError(f"num_tokens {num_tokens} does not match {n} slots")
    else:
        if block_tables is None or cu_seqlens is None or num_tokens is None:
            raise ValueError("give slots, or block_tables with cu_seqlens and num_tokens")
        shape = block_tables.shape
        if (len(shape) != 2 or shape[0] < 1 or shape[1] < 1 or block_tables.dtype != torch.int32 or block_tables.get_device() != dev
                or block_tables.stride(1) != 1):
            raise ValueError(f"block_tables must be int32 [batch, max_pages_per_seq] on cuda:{dev} with unit column stride")
        batch, bt_cols = shape
        if cu_seqlens.dtype != torch.int32 or cu_seqlens.get_device() != dev or cu_seqlens.shape != (batch + 1,) or not cu_seqlens.is_contiguous():
            raise ValueError(f"cu_seqlens must be contiguous int32 [{batch + 1}] on cuda:{dev}")
        n, bt_stride, bt_ptr, cu_ptr = int(num_tokens), block_tables.stride(0), block_tables.data_ptr(), cu_seqlens.data_ptr()
        if n < 0:
            raise ValueError(f"num_tokens must not be negative, got {n}")
    if out is None:
        k_out = torch.empty((n, hkv, d), dtype=dtype, device=k_data.device)
        v_out = torch.empty_like(k_out)
    else:
        k_out, v_out = out
        dtype = k_out.dtype
        for x in out:
            if x.shape != (n, hkv, d) or x.dtype != dtype or x.get_device() != dev or not x.is_contiguous():
                raise ValueError(f"out must be two contiguous [{n}, {hkv}, {d}] tensors of one type on cuda:{dev}")
    _call(dev, "ri_kv_read_nvfp4", (
        k_data.data_ptr(), k_sf.data_ptr(), v_data.data_ptr(), v_sf.data_ptr(), pages, code_stride, sf_stride, hkv, d, page,
        slots_ptr, bits, bt_ptr, bt_stride, bt_cols, cu_ptr, batch, n, k_global_scale, v_global_scale, k_out.data_ptr(),
        v_out.data_ptr(), _cabi.DTYPE_BF16 if dtype == torch.bfloat16 else _cabi.torch_dtype_code(dtype, allow_f32=True),
        out is None))
    return k_out, v_out


def rcp_approx(x: torch.Tensor) -> torch.Tensor:
    """rcp.approx.ftz.f32 of a float32 CUDA tensor (test helper)."""
    lib = _cabi.load()
    x = x.contiguous()
    y = torch.empty_like(x)
    with torch.cuda.device(x.device):
        _cabi.check(lib.ri_rcp_approx(x.data_ptr(), y.data_ptr(), x.numel(), _cabi.current_stream(x.device)),
                    "rcp_approx")
    return y
