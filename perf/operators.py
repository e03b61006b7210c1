"""Timed cases of the paged NVFP4 KV-cache operators: quantising K / V into the cache, reading them back, and decode
attention for a batch that shares a long prefix.

The cache is a pool of pages, for K and V each: codes ``[pages, Hkv, page, D/2]`` (E2M1, two to a byte, the even
element in the low nibble) and block scales ``[pages, Hkv, page, D/16]`` (E4M3 bytes); a held value is
``code * block scale * global scale``.  ``slot = page_index * page + offset`` names a token's place, negative slots
are padding.

  append   k, v [T, Hkv, D] are quantised to the slots of T tokens, then read back from them.  Of a block of 16 with
           largest magnitude a:  s = e4m3(a / (6 g)),  code = e2m1(x / (s g)),  0 where s = 0.
  gather   the contexts of a batch, named by block tables, as dense rows [tokens, Hkv, D] in 16 bits.
  prefix   one query token per sequence over the sequence's whole cache; the first ``prefix_len`` tokens are the
           same pages for every sequence.  The query is taken as q^ = NVFP4(q) + NVFP4(q - NVFP4(q)) with global
           scale 1 (the decode kernel's query), out = softmax(sm_scale q^ . K) . V, 0 for an empty sequence.
"""
from __future__ import annotations

import math

import torch

own = False

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0)
_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of a batch of sixteen: sixteen new tokens, latency
        dict(name="append_step", op="append", tokens=16, hkv=8, d=128, page=16, dtype="bf16", packed=False, pad=0),
        # a prefill chunk of the usual size, the pool's default page
        dict(name="append_chunk", op="append", tokens=8192, hkv=8, d=128, page=128, dtype="bf16", packed=False, pad=0),
        # a ragged mixed step of a head_dim 256 model: K and V are slices of the fused QKV output, the cache is the
        # serving engine's interleaved one, and some rows are padding
        dict(name="append_packed_d256", op="append", tokens=1537, hkv=4, d=256, page=32, dtype="fp16", packed=True, pad=77),
        # a long document's prefill, all at once
        dict(name="append_long", op="append", tokens=65536, hkv=8, d=128, page=64, dtype="bf16", packed=True, pad=0),
        # the context of one short conversation
        dict(name="gather_short", op="gather", batch=1, tokens=200, hkv=8, d=128, page=16, dtype="bf16", packed=False),
        # one very long context, for a prefill chunk that attends to all of it
        dict(name="gather_long", op="gather", batch=1, tokens=131072, hkv=8, d=128, page=128, dtype="bf16", packed=False),
        # the contexts of a ragged batch from an interleaved cache of small pages
        dict(name="gather_batch_d256", op="gather", batch=48, tokens=40001, hkv=4, d=256, page=16, dtype="fp16", packed=True),
        # a few requests behind one system prompt: latency
        dict(name="prefix_small", op="prefix", batch=8, prefix=2048, suffix=64, hq=32, hkv=8, d=128, page=16, short=0),
        # a chat service: a long system prompt with tools, short conversations; the prefix ends inside a page
        dict(name="prefix_chat", op="prefix", batch=32, prefix=8190, suffix=1024, hq=64, hkv=8, d=128, page=16, short=0),
        # questions about one long document
        dict(name="prefix_document", op="prefix", batch=64, prefix=32768, suffix=2048, hq=64, hkv=8, d=128, page=128, short=0),
        # head_dim 256 with six query heads to a KV head; two padding rows of length 0 and a row shorter than the prefix
        dict(name="prefix_d256", op="prefix", batch=27, prefix=12001, suffix=512, hq=48, hkv=8, d=256, page=64, short=3),
        # many samples of one prompt (best-of-n, rollouts), a tensor-parallel shard's four KV heads
        dict(name="prefix_samples", op="prefix", batch=256, prefix=16384, suffix=256, hq=32, hkv=4, d=128, page=32, short=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["append", "gather", "prefix"])
    d = rng.choice([128, 128, 256])
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        tokens = _log(rng, 1, 60000)
        hkv = rng.choice([1, 2, 4] if d == 256 else [1, 2, 4, 8])
        return dict(op=op, tokens=tokens, hkv=hkv, d=d, page=page, dtype=rng.choice(["bf16", "fp16"]),
                    packed=rng.random() < 0.5, pad=rng.choice([0, tokens // 9]))
    if op == "gather":
        batch = _log(rng, 1, 64)
        return dict(op=op, batch=batch, tokens=_log(rng, batch, 120000), hkv=rng.choice([1, 2, 4] if d == 256 else [1, 2, 4, 8]),
                    d=d, page=page, dtype=rng.choice(["bf16", "fp16"]), packed=rng.random() < 0.5)
    while True:
        batch, prefix, suffix = _log(rng, 1, 256), _log(rng, 100, 32768), _log(rng, 1, 2048)
        hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([4, 6, 8])
        # no dearer than the largest listed one
        if batch * hkv * group * prefix * d <= 64 * 64 * 32768 * 128 and batch * suffix * hkv * d <= 64 * 2048 * 8 * 128:
            return dict(op=op, batch=batch, prefix=prefix, suffix=suffix, hq=hkv * group, hkv=hkv, d=d, page=page,
                        short=rng.choice([0, min(3, batch - 1)]))


def _context_lens(batch, tokens):
    """A ragged batch: lengths that grow linearly, the first sequences shortest, summing to `tokens`."""
    w = [i + 1 for i in range(batch)]
    ends = [tokens * sum(w[:i + 1]) // sum(w) for i in range(batch)]
    return [e - b for b, e in zip([0] + ends[:-1], ends)]


def _suffix_lens(case):
    """Lengths beyond the prefix, 1 .. suffix evenly."""
    b, n = case["batch"], case["suffix"]
    return [1 + (n - 1) * i // max(1, b - 1) if b > 1 else n for i in range(b)]


def _seq_lens(case):
    lens = [case["prefix"] + s for s in _suffix_lens(case)]
    for i in range(case["short"]):                       # the last rows: half the prefix, then padding rows
        lens[case["batch"] - 1 - i] = case["prefix"] // 2 if i == 0 else 0
    return lens


def work(case):
    hkv, d = case["hkv"], case["d"]
    held = hkv * (d // 2 + d // 16) * 2                  # bytes of one token's K and V in the cache
    dense = hkv * d * 2 * 2                              # ... and as 16-bit rows
    if case["op"] == "append":                           # rows in; codes and scales out and in again; rows out
        live = case["tokens"] - case["pad"]
        return {"bytes": live * (dense + 2 * held) + case["tokens"] * (dense + 8), "flops": 0}
    if case["op"] == "gather":
        return {"bytes": case["tokens"] * (held + dense), "flops": 0}
    lens = _seq_lens(case)
    own_tokens = sum(max(0, n - case["prefix"]) for n in lens)
    rows = 2 * 2 * case["batch"] * case["hq"] * d        # queries in, outputs out
    return {"bytes": (case["prefix"] + own_tokens) * held + rows, "flops": sum(lens) * case["hq"] * d * 4}


# ------------------------------------------------------------------------------------------------ plain pieces
def _e4m3(v):
    """Nearest E4M3 value of v >= 0, ties to the even one, at most 448."""
    _, e = torch.frexp(v)
    q = torch.ldexp(torch.ones_like(v), (e - 1).clamp(min=-6) - 3)
    return (torch.round(v / q) * q).clamp(max=448.0)


def _e2m1(y):
    """Nearest E2M1 magnitude index (0 .. 7) of |y|, ties to the even one, and the sign bit on top."""
    a = y.abs()
    low, mid, high = torch.round(a * 2), torch.round(a) + 2, torch.round(a / 2).clamp(max=3) + 4
    idx = torch.where(a < 2, low, torch.where(a < 4, mid, high)).to(torch.uint8)
    return idx | (torch.signbit(y).to(torch.uint8) << 3)


def _quantise(x, g):
    """x [..., D] -> codes (0 .. 15, one a byte) [..., D] and block scales [..., D/16], global scale g.  In 32 bits
    like the framework's quantisers: the block's multiplier is (1/g) / s."""
    x = x.float()
    inv_g = torch.tensor(1.0, device=x.device) / torch.tensor(g, dtype=torch.float32, device=x.device)
    blocks = x.unflatten(-1, (-1, 16))
    sixth = torch.tensor(1.0, device=x.device) / 6.0
    s = _e4m3(inv_g * (blocks.abs().amax(-1) * sixth))
    mult = torch.where(s > 0, inv_g * (1.0 / torch.where(s > 0, s, 1.0)), 0.0)
    return _e2m1(blocks * mult[..., None]).flatten(-2), s


def _pack(codes):
    return codes[..., 0::2] | (codes[..., 1::2] << 4)


def _held(data, sf):
    """Codes and block scales as stored -> code * scale in 32 bits."""
    table = torch.tensor(_E2M1, device=data.device)
    nibbles = torch.stack([data & 15, data >> 4], dim=-1).flatten(-2)
    return (table[nibbles.long()].unflatten(-1, (-1, 16)) * sf.view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _places(block_tables, positions, page):
    """(page index, offset) of token positions [B, n] of the sequences of a batch."""
    return block_tables.long().gather(1, positions // page), positions % page


# ------------------------------------------------------------------------------------------------ inputs
def _pool_buffers(pages, hkv, page, d, packed, dev):
    """The four tensors of a pool: dense, or as views of an interleaved cache (every page = K codes | K scales |
    V codes | V scales)."""
    n_codes, n_sf = hkv * page * d // 2, hkv * page * d // 16
    if not packed:
        return [torch.zeros(pages, hkv, page, w, dtype=torch.uint8, device=dev) for w in (d // 2, d // 16, d // 2, d // 16)]
    buf = torch.zeros(pages, 2 * (n_codes + n_sf), dtype=torch.uint8, device=dev)
    views, at = [], 0
    for w, n in ((d // 2, n_codes), (d // 16, n_sf), (d // 2, n_codes), (d // 16, n_sf)):
        views.append(buf[:, at:at + n].unflatten(1, (hkv, page, w)))
        at += n
    return views


def _random_rows(gen, dev, rows, hkv, d, dtype):
    """Keys or values: normal, with channels of different spread as trained projections have; and the global scale
    that a calibration over other tokens of the same channels found, a 32-bit number."""
    spread = torch.exp(0.3 * torch.randn(hkv, d, generator=gen, device=dev))
    seen = (torch.randn(512, hkv, d, generator=gen, device=dev) * spread).abs().max()
    return (torch.randn(rows, hkv, d, generator=gen, device=dev) * spread).to(dtype), float(seen / (6.0 * 448.0))


def _fill(gen, dev, pool, page_ids):
    """Random contents for the named pages; returns the K and V global scales."""
    pages, (hkv, page) = len(page_ids), pool[0].shape[1:3]
    d = pool[0].shape[3] * 2
    scales = []
    for data, sf in ((pool[0], pool[1]), (pool[2], pool[3])):
        x, g = _random_rows(gen, dev, pages * page, hkv, d, torch.bfloat16)
        codes, s = _quantise(x, g)
        data[page_ids] = _pack(codes).view(pages, page, hkv, d // 2).transpose(1, 2)
        sf[page_ids] = s.to(torch.float8_e4m3fn).view(torch.uint8).view(pages, page, hkv, d // 16).transpose(1, 2)
        scales.append(g)
    return scales


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    op, hkv, d, page = case["op"], case["hkv"], case["d"], case["page"]
    st = {"case": case}
    if op == "append":
        t = case["tokens"]
        pages = (t + page - 1) // page + 3                   # page 0 holds no sequence
        st["pool"] = _pool_buffers(pages, hkv, page, d, case["packed"], dev)
        (k, gk), (v, gv) = (_random_rows(gen, dev, t, hkv, d, _TYPES[case["dtype"]]) for _ in range(2))
        st["scales"] = [gk, gv]
        if case["packed"]:                                   # slices of the fused projection's output
            fused = torch.zeros(t, 6 * hkv * d, dtype=k.dtype, device=dev)
            fused[:, 4 * hkv * d:] = torch.cat([k.flatten(1), v.flatten(1)], 1)
            k, v = (fused[:, (4 + i) * hkv * d:(5 + i) * hkv * d].unflatten(1, (hkv, d)) for i in range(2))
        st["k"], st["v"] = k, v
        order = 1 + torch.randperm(pages - 1, generator=gen, device=dev)
        pos = torch.arange(t, device=dev)
        slots = order[pos // page] * page + pos % page
        if case["pad"]:
            slots[torch.randperm(t, generator=gen, device=dev)[:case["pad"]]] = -1
        st["slots"] = slots
        return st
    lens = _context_lens(case["batch"], case["tokens"]) if op == "gather" else _seq_lens(case)
    if op == "gather":
        order = torch.randperm(case["batch"], generator=gen, device=dev).tolist()
        lens = [lens[i] for i in order]
    shared = 0 if op == "gather" else case["prefix"] // page  # whole pages that all sequences have in common
    if op == "prefix":                                       # every sequence's table covers the whole prefix
        head = torch.randperm(case["batch"] - case["short"], generator=gen, device=dev).tolist()
        lens = [lens[i] for i in head] + lens[len(head):]
    owned = [max((n + page - 1) // page - shared, 0) for n in lens]
    if op == "prefix":
        owned[0] = max(owned[0], 1)
    total = shared + sum(owned)
    order = 1 + torch.randperm(total + 2, generator=gen, device=dev)[:total]
    st["pool"] = _pool_buffers(total + 3, hkv, page, d, case.get("packed", False), dev)
    st["scales"] = _fill(gen, dev, st["pool"], order)
    table = torch.zeros(case["batch"], shared + max(1, max(owned)), dtype=torch.int32, device=dev)
    table[:, :shared] = order[:shared].int()
    at = shared
    for b, n in enumerate(owned):
        table[b, shared:shared + n] = order[at:at + n].int()
        at += n
    st["block_tables"] = table
    st["seq_lens"] = torch.tensor(lens, dtype=torch.int32, device=dev)
    if op == "gather":
        cu = [0]
        for n in lens:
            cu.append(cu[-1] + n)
        st["cu_seqlens"] = torch.tensor(cu, dtype=torch.int32, device=dev)
        return st
    tail = case["prefix"] % page                             # the page in which the prefix ends: every sequence has a copy
    if tail:
        first = table[:, shared].long()
        for part in st["pool"]:
            part[first, :, :tail] = part[first[0], :, :tail].clone()
    st["prefix_len"], st["max_seq_len"] = case["prefix"], max(lens)
    heat = torch.linspace(0.5, 2.0, case["hq"], device=dev)[:, None]
    st["q"] = (torch.randn(case["batch"], case["hq"], d, generator=gen, device=dev) * heat).bfloat16()
    st["sm_scale"] = d ** -0.5
    return st


# ------------------------------------------------------------------------------------------------ one pass
def run(st):
    return {"append": _append, "gather": _gather, "prefix": _prefix}[st["case"]["op"]](st)


def _own_pool(st):
    from resinfer_b200.nvfp4.cute_attn import NvFp4PagedKVPool
    k_data, k_sf, v_data, v_sf = st["pool"]
    return NvFp4PagedKVPool(num_kv_heads=k_data.shape[1], head_dim=k_data.shape[3] * 2, k_data=k_data, v_data=v_data,
                            k_sf=k_sf, v_sf=v_sf, page_size=k_data.shape[2], k_global_scale=st["scales"][0],
                            v_global_scale=st["scales"][1])


def _append(st):
    if own:
        from resinfer_b200.nvfp4.cute_attn import host
        pool = _own_pool(st)
        host.write_paged_kv(st["k"], st["v"], pool, st["slots"])
        k, v = host.read_paged_kv(pool, st["slots"], dtype=st["k"].dtype)
        return {"k": k, "v": v}
    page = st["pool"][0].shape[2]
    slots = st["slots"]
    at, off = slots.clamp(min=0) // page, slots.clamp(min=0) % page      # padding goes to page 0, which nothing reads
    live = (slots >= 0)[:, None, None]
    out = {}
    for name, x, data, sf, g in (("k", st["k"], *st["pool"][:2], st["scales"][0]), ("v", st["v"], *st["pool"][2:], st["scales"][1])):
        codes, s = _quantise(x, g)
        data[at, :, off] = _pack(codes)
        sf[at, :, off] = s.to(torch.float8_e4m3fn).view(torch.uint8)
        out[name] = torch.where(live, _held(data[at, :, off], sf[at, :, off]) * g, 0.0).to(x.dtype)
    return out


def _gather(st):
    dtype, n = _TYPES[st["case"]["dtype"]], st["case"]["tokens"]
    if own:
        from resinfer_b200.nvfp4.cute_attn import host
        k, v = host.gather_paged_kv(_own_pool(st), st["block_tables"], st["cu_seqlens"], n, dtype=dtype)
        return {"k": k, "v": v}
    page, cu = st["pool"][0].shape[2], st["cu_seqlens"].long()
    pos = torch.arange(n, device=cu.device)
    seq = torch.searchsorted(cu, pos, right=True) - 1
    local = pos - cu[seq]
    at, off = st["block_tables"].long()[seq, local // page], local % page
    out = {}
    for name, data, sf, g in (("k", *st["pool"][:2], st["scales"][0]), ("v", *st["pool"][2:], st["scales"][1])):
        out[name] = (_held(data[at, :, off], sf[at, :, off]) * g).to(dtype)
    return out


def _prefix(st):
    q, tables, lens, n = st["q"], st["block_tables"], st["seq_lens"], st["prefix_len"]
    gk, gv = st["scales"]
    if own:
        from resinfer_b200.nvfp4.cute_attn import host
        out = torch.empty_like(q)
        return host.run_paged_fp4_decode_shared_prefix(q, _own_pool(st), tables, lens, n, st["sm_scale"] * gk, out,
                                                       max_seq_len=st["max_seq_len"], value_scale=gv)
    k_data, k_sf, v_data, v_sf = st["pool"]
    (b, hq, d), hkv, page, dev = q.shape, k_data.shape[1], k_data.shape[2], q.device
    group, rest = hq // hkv, max(1, st["max_seq_len"] - n)
    table = torch.tensor(_E2M1, device=dev)
    codes, s = _quantise(q, 1.0)                             # the query: NVFP4 plus the NVFP4 of what that leaves
    base = (table[codes.long()].unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2)
    codes, s = _quantise(q.float() - base, 1.0)
    qq = (base + (table[codes.long()].unflatten(-1, (-1, 16)) * s[..., None]).flatten(-2)).view(b, hkv, group, d)
    scale = st["sm_scale"] * gk
    # the prefix, once: [Hkv, B G, D] x [Hkv, prefix, D]
    at, off = _places(tables[:1], torch.arange(n, device=dev)[None], page)
    pk, pv = (_held(data[at[0], :, off[0]], sf[at[0], :, off[0]]).transpose(0, 1) for data, sf in ((k_data, k_sf), (v_data, v_sf)))
    s1 = torch.matmul(qq.transpose(0, 1).reshape(hkv, b * group, d), pk.transpose(1, 2)).view(hkv, b, group, n) * scale
    s1 = torch.where(torch.arange(n, device=dev) < lens[None, :, None, None], s1, -math.inf)
    # each sequence's own tokens, padded to the longest: [B, Hkv, G, D] x [B, Hkv, rest, D]
    pos = n + torch.arange(rest, device=dev)[None].expand(b, rest)
    live = pos < lens[:, None]
    at, off = _places(tables, torch.where(live, pos, 0), page)
    sk, sv = (torch.where(live[:, :, None, None], _held(data[at, :, off], sf[at, :, off]), 0.0).transpose(1, 2)
              for data, sf in ((k_data, k_sf), (v_data, v_sf)))
    s2 = torch.where(live[:, None, None], torch.matmul(qq, sk.transpose(2, 3)) * scale, -math.inf)
    m = torch.maximum(s1.amax(-1).transpose(0, 1), s2.amax(-1))
    m = torch.where(m > -math.inf, m, 0.0)
    p1, p2 = torch.exp(s1 - m.transpose(0, 1)[..., None]), torch.exp(s2 - m[..., None])
    total = p1.sum(-1).transpose(0, 1) + p2.sum(-1)
    o = torch.matmul(p1.view(hkv, b * group, n), pv).view(hkv, b, group, d).transpose(0, 1) + torch.matmul(p2, sv)
    o = torch.where(total[..., None] > 0, o / torch.where(total > 0, total, 1.0)[..., None], 0.0) * gv
    return o.reshape(b, hq, d).to(q.dtype)


# ------------------------------------------------------------------------------------------------ in 64 bits
_GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest(x, grid):
    """Nearest value of an ascending grid of non-negative values, the even index on a tie, the last one beyond it."""
    hi = torch.searchsorted(grid, x).clamp(max=grid.numel() - 1)
    lo = (hi - 1).clamp(min=0)
    up = grid[hi] - x
    down = x - grid[lo]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), grid[hi], grid[lo])


def _e4m3_grid(dev):
    vals = [m * 2.0 ** -9 for m in range(8)] + [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)]
    return torch.tensor(vals[:-1], dtype=torch.float64, device=dev)


def _exact_held(x, g, products=torch.float64):
    """What NVFP4 holds for x, without the global scale: x [..., D] in 64 bits.  `products`: the width in which the
    block's multiplier and the products with it are taken."""
    dev = x.device
    blocks = x.double().unflatten(-1, (-1, 16))
    s = _nearest(blocks.abs().amax(-1, keepdim=True) / (6.0 * g), _e4m3_grid(dev))
    safe = torch.where(s > 0, s * g, 1.0)
    y = (blocks.to(products) * (1.0 / safe.to(products))).double() if products != torch.float64 else blocks / safe
    mag = _nearest(y.abs(), torch.tensor(_GRID, dtype=torch.float64, device=dev))
    return (torch.where(s > 0, mag, 0.0) * torch.sign(y) * s).flatten(-2)


def _exact_rows(data, sf, table, count, page):
    """The first `count` tokens of a sequence as [Hkv, count, D] in 64 bits, without the global scale."""
    pages = table[:(count + page - 1) // page].long()
    grid = torch.tensor(_GRID + tuple(-v for v in _GRID), dtype=torch.float64, device=data.device)
    lookup = torch.cat([_e4m3_grid(data.device), torch.full((1,), math.nan, dtype=torch.float64, device=data.device)])
    by, scale = data[pages].int(), lookup[sf[pages].int()]
    x = torch.empty(*by.shape[:-1], 2 * by.shape[-1], dtype=torch.float64, device=data.device)
    x[..., 0::2], x[..., 1::2] = grid[by % 16], grid[by // 16]
    x *= scale.repeat_interleave(16, dim=-1)
    return x.transpose(0, 1).flatten(1, 2)[:, :count]


def exact(case, seed):
    st = prepare(case, seed)
    page, (gk, gv) = case["page"], st["scales"]
    if case["op"] == "append":
        live = (st["slots"] >= 0).double()[:, None, None]
        return {name: _exact_held(x, g) * g * live for name, x, g in (("k", st["k"], gk), ("v", st["v"], gv))}
    k_data, k_sf, v_data, v_sf = st["pool"]
    lens = st["seq_lens"].tolist()
    if case["op"] == "gather":
        out = {}
        for name, data, sf, g in (("k", k_data, k_sf, gk), ("v", v_data, v_sf, gv)):
            out[name] = torch.cat([_exact_rows(data, sf, st["block_tables"][b], n, page).transpose(0, 1) * g
                                   for b, n in enumerate(lens)])
        return out
    q, hkv = st["q"], case["hkv"]
    b, hq, d = q.shape
    # the query's codes are settled on 32-bit products with the block's reciprocal, by the quantiser's definition:
    # with global scale 1 the quotients x / s often lie on a border between two codes
    base = _exact_held(q, 1.0, torch.float32)
    qq = (base + _exact_held(q.double() - base, 1.0, torch.float32)).view(b, hkv, hq // hkv, d)
    out = torch.zeros(b, hkv, hq // hkv, d, dtype=torch.float64, device=q.device)
    for i, n in enumerate(lens):
        if n:
            kk = _exact_rows(k_data, k_sf, st["block_tables"][i], n, page)
            vv = _exact_rows(v_data, v_sf, st["block_tables"][i], n, page)
            p = torch.softmax(torch.einsum("hgd,htd->hgt", qq[i], kk) * (st["sm_scale"] * gk), dim=-1)
            out[i] = torch.einsum("hgt,htd->hgd", p, vv) * gv
    return out.view(b, hq, d)
