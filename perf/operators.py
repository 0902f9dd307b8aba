"""Operators on a paged cache whose tables live on the device, one layer each.

A case is a dict of plain values.  `op` says which operator it times:

  append   K/V rows of new tokens, as they leave a fused projection, quantised
           into their sequences' pages
  read     tokens of sequences read back from the cache into dense rows
  decode   attention of one new token a sequence, sliding window and sinks
  chunk    attention of several new tokens a sequence, the same mask

Sequence b holds ctx + new tokens, spread over ctx_min..ctx_max and
new_min..new_max; token t is in page indices[indptr[b] + t / 16], slot t % 16,
and its last `new` tokens are the rows of the call.  A query at position p sees
tokens t <= p with t > p - window (window 0: all) or t < sinks.  Pages are
shuffled over the pool.  K, V and q are normal; MXFP8 pools carry the 1 %
outliers (20 sigma) that block scaling is there for.  Slots past a sequence's
end hold what an earlier owner of the page left.
"""
import math

import numpy as np
import torch

own = False

PAGE = 16
DEV = "cuda:0"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "fp8": 1, "mxfp8": 1}
CHUNK = 1024    # pages generated at a time
FLOOR = 2.0 ** -64    # least scale of an FP8 block written token by token


def listed():
    return [
        # A decode step's K/V in a large FP8 batch: one token a sequence into
        # partly filled pages, whose block scales may have to grow.  Short
        # contexts: only each last page is touched, whatever comes before it.
        dict(name="append-step-fp8", op="append", hq=32, hkv=8, d=128, q="bf16", kv="fp8", seqs=256, ctx_min=0,
             ctx_max=400, new_min=1, new_max=1),
        # Prompt chunks of odd lengths that begin inside a page, MXFP8.
        dict(name="append-prompt-mxfp8", op="append", hq=64, hkv=8, d=128, q="bf16", kv="mxfp8", seqs=6, ctx_min=0,
             ctx_max=700, new_min=301, new_max=2500),
        # Cached prefixes read back in the model's type, to be moved or re-encoded.
        dict(name="read-prefix-fp8", op="read", hq=32, hkv=8, d=128, q="bf16", kv="fp8", seqs=4, ctx_min=0,
             ctx_max=0, new_min=2000, new_max=9000),
        # The tail of one short sequence of a small model, to look at it.
        dict(name="read-tail-mxfp8", op="read", hq=32, hkv=4, d=64, q="f32", kv="mxfp8", seqs=1, ctx_min=100,
             ctx_max=100, new_min=601, new_max=601),
        # One chat sequence on a small model in full precision: the smallest call.
        dict(name="decode-one-f32", op="decode", hq=32, hkv=4, d=64, q="f32", kv="f32", seqs=1, ctx_min=512,
             ctx_max=512, new_min=1, new_max=1, window=256, sinks=4, tiled=True),
        # Continuous batching under a window of 4096 with four first tokens kept.
        dict(name="decode-batch-bf16", op="decode", hq=32, hkv=8, d=128, q="bf16", kv="bf16", seqs=64, ctx_min=300,
             ctx_max=12000, new_min=1, new_max=1, window=4096, sinks=4, tiled=False),
        # The largest batch: short window, a system prompt that stays visible, FP8.
        dict(name="decode-batch-fp8", op="decode", hq=64, hkv=8, d=128, q="bf16", kv="fp8", seqs=256, ctx_min=60,
             ctx_max=4000, new_min=1, new_max=1, window=1024, sinks=64, tiled=True),
        # One long document, wide heads, no window: the work of a single row
        # has to be split over the whole chip.
        dict(name="decode-long-f16", op="decode", hq=16, hkv=2, d=256, q="f16", kv="f16", seqs=1, ctx_min=100000,
             ctx_max=100000, new_min=1, new_max=1, window=0, sinks=0, tiled=False),
        # A large chunk of a long prompt over its cached context.
        dict(name="chunk-long-bf16", op="chunk", hq=32, hkv=8, d=128, q="bf16", kv="bf16", seqs=1, ctx_min=8192,
             ctx_max=8192, new_min=4096, new_max=4096, window=4096, sinks=16, tiled=False),
        # A batch of short prompts of odd lengths, small heads, short window.
        dict(name="chunk-prompts-f16", op="chunk", hq=32, hkv=4, d=64, q="f16", kv="f16", seqs=12, ctx_min=0,
             ctx_max=0, new_min=37, new_max=1500, window=256, sinks=4, tiled=True),
        # Chunks over a quantised context (prefix reuse).
        dict(name="chunk-ctx-fp8", op="chunk", hq=64, hkv=8, d=128, q="bf16", kv="fp8", seqs=3, ctx_min=3750,
             ctx_max=5000, new_min=300, new_max=900, window=2048, sinks=128, tiled=False),
        # Draft tokens of many sequences verified at once, wide heads, odd window.
        dict(name="verify-mxfp8", op="chunk", hq=16, hkv=2, d=256, q="bf16", kv="mxfp8", seqs=32, ctx_min=200,
             ctx_max=9000, new_min=3, new_max=9, window=2001, sinks=0, tiled=True),
    ]


def _size(rng, lo, hi):
    """Log-uniform whole number in lo..hi."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "decode", "decode", "chunk", "chunk"])
    hq, hkv, d = rng.choice([(32, 4, 64), (32, 8, 128), (64, 8, 128), (16, 2, 256), (8, 8, 128), (16, 4, 64)])
    q, kv = rng.choice([("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("bf16", "mxfp8"), ("f16", "fp8"),
                        ("f16", "mxfp8"), ("f32", "f32")])
    c = dict(op=op, hq=hq, hkv=hkv, d=d, q=q, kv=kv)
    if op in ("append", "read"):
        if rng.random() < 0.4:       # the cache's type apart from the rows'
            c["q"] = rng.choice(["f32", "bf16", "f16"])
        hi = rng.choice([1, _size(rng, 2, 3000)])
        seqs = _size(rng, 1, max(1, min(300, 12000 // hi)))
        lo = _size(rng, 1, hi)
        ctx = rng.choice([0, _size(rng, 1, 500)])
        return dict(c, seqs=seqs, ctx_min=0, ctx_max=ctx, new_min=lo, new_max=hi)
    window, sinks = rng.choice([0, _size(rng, 1, 6000), _size(rng, 16, 6000)]), rng.choice([0, _size(rng, 1, 200)])
    c.update(window=window, sinks=sinks, tiled=rng.random() < 0.5)
    token = 2 * hkv * d * SIZE[kv]
    if op == "decode":
        hi = _size(rng, 5, 100000)
        seen = max(64, min(hi, window + sinks) if window else hi)
        seqs = _size(rng, 1, max(1, min(256, int(9e8 / (seen * token)), 1000000 // hi)))
        return dict(c, seqs=seqs, ctx_min=hi // 3, ctx_max=hi, new_min=1, new_max=1)
    ctx = rng.choice([0, _size(rng, 10, 9000)])
    seen = min(ctx + 2000, window + sinks) if window else ctx + 2000
    most = int(6.5e7 * 1024 / (hq * d * max(seen, 256)))      # rows for the work of the largest listed case
    hi = _size(rng, 2, min(4096, most))
    seqs = _size(rng, 1, max(1, min(48, most // hi, 30000000 // (hi * (hi + seen)))))
    return dict(c, seqs=seqs, ctx_min=ctx * 3 // 4, ctx_max=ctx, new_min=max(1, hi // 3), new_max=hi)


# ------------------------------------------------------------ sizes of a case
def _spread(i, lo, hi):
    """The i-th of a fixed sequence of whole numbers, spread over lo..hi."""
    return int(lo + (hi - lo + 1) * ((0.381966 + i * 0.61803398875) % 1.0)) if hi > lo else lo


def _lens(c):
    """(tokens held, new tokens) of each sequence."""
    new = [_spread(i, c["new_min"], c["new_max"]) for i in range(c["seqs"])]
    ctx = [_spread(3 * i + 1, c["ctx_min"], c["ctx_max"]) for i in range(c["seqs"])]
    return [a + b for a, b in zip(ctx, new)], new


def _pages(c):
    return [(t + PAGE - 1) // PAGE for t in _lens(c)[0]]


# ------------------------------------------------------------------ the inputs
def _gen(seed, k):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + k * 7919 + 29) % (1 << 62))
    return g


def _values(c, shape, seed, k):
    g = _gen(seed, k)
    x = torch.randn(shape, generator=g, device=DEV, dtype=torch.float32)
    if c["kv"] == "mxfp8":
        x = torch.where(torch.rand(shape, generator=g, device=DEV) < 0.01, x * 20, x)
    return x


def _perm(seed, n):
    """Places of the sequences' pages in a pool of n + n // 8 + 3 pages."""
    size = n + n // 8 + 3
    return size, np.random.default_rng(int(seed) + 11).permutation(size)[:n].astype(np.int32)


def _e4m3(y):
    return y.clamp(-448.0, 448.0).to(torch.float8_e4m3fn)


def _mx_codes(x):
    """(E4M3 codes, E8M0 bytes) of rows x [..., d], one scale for 32 values."""
    g = x.unflatten(-1, (-1, 32))
    amax = g.abs().amax(-1, keepdim=True)
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 9, -127).clamp(-127, 127)
    return _e4m3(torch.ldexp(g, -e)).flatten(-2), (e + 127).to(torch.uint8).squeeze(-1)


def _old_pages(c, seed):
    """The pool before the call: (data [P, 2, hkv, 16, d], scales), pages of the
    sequences holding their cached tokens, all in the pool's format."""
    n = sum(_pages(c))
    size, perm = _perm(seed, n)
    hkv, d, kv = c["hkv"], c["d"], c["kv"]
    kind = torch.float8_e4m3fn if kv in ("fp8", "mxfp8") else TYPES[kv]
    data = torch.empty((size, 2, hkv, PAGE, d), dtype=kind, device=DEV)
    scales = None
    if kv == "fp8":
        scales = torch.empty((size, 2, hkv), dtype=torch.float32, device=DEV)
    if kv == "mxfp8":
        scales = torch.empty((size, 2, hkv, PAGE, d // 32), dtype=torch.uint8, device=DEV)
    held = np.full(size, PAGE)       # tokens of a page that count for its block scale
    if c["op"] == "append":
        kv_len, new = _lens(c)
        held[perm] = np.concatenate([np.clip(t - m - PAGE * np.arange((t + PAGE - 1) // PAGE), 0, PAGE)
                                     for t, m in zip(kv_len, new)])
    held = torch.from_numpy(held).to(DEV)
    for k in range(0, size, CHUNK):
        m = min(CHUNK, size - k)
        x = _values(c, (m, 2, hkv, PAGE, d), seed, k // CHUNK)
        if kv == "fp8":
            counts = torch.arange(PAGE, device=DEV)[None, :] < held[k:k + m, None]
            amax = (x.abs() * counts[:, None, None, :, None]).amax((3, 4))
            s = torch.where(amax > 0, amax / 448.0, 1.0)
            data[k:k + m] = _e4m3(x / s[..., None, None])
            scales[k:k + m] = s
        elif kv == "mxfp8":
            data[k:k + m], scales[k:k + m] = _mx_codes(x)
        else:
            data[k:k + m] = x.to(kind)
    return data, scales, perm


class _Memory:
    def __init__(self, ptr, nbytes):
        self.__cuda_array_interface__ = dict(shape=(nbytes,), typestr="|u1", data=(ptr, False), version=2)


def _pool_views(lib, pool, data, scales):
    """The pool's own memory as tensors like data and scales, holding their values."""
    views = []
    for t, ptr in ((data, lib.dh_pool_data(pool._h)), (scales, lib.dh_pool_scales(pool._h))):
        if t is None:
            views.append(None)
            continue
        v = torch.as_tensor(_Memory(ptr, t.numel() * t.element_size()), device=DEV)
        v.copy_(t.view(-1).view(torch.uint8))
        v = v.view(t.dtype).view(t.shape)
        v.pool = pool      # the memory goes with the last reference to the pool
        views.append(v)
    return views


def prepare(c, seed):
    kv_len, new = _lens(c)
    rows, hq, hkv, d = sum(new), c["hq"], c["hkv"], c["d"]
    data, scales, perm = _old_pages(c, seed)
    i32 = dict(dtype=torch.int32, device=DEV)
    s = dict(c, data=data, scales=scales, indices=torch.from_numpy(perm).to(DEV),
             indptr=torch.tensor(np.cumsum([0] + _pages(c)), **i32), kv_len=torch.tensor(kv_len, **i32),
             q_indptr=None if c["op"] == "decode" else torch.tensor(np.cumsum([0] + new), **i32), rows=rows,
             longest=max(kv_len), most_new=max(new))
    if c["op"] == "read":
        s["k"], s["v"] = (torch.empty((rows, hkv, d), dtype=TYPES[c["q"]], device=DEV) for _ in range(2))
    else:      # one fused projection's output: q, k and v are views of its rows
        qkv = _values(c, (rows, (hq + 2 * hkv) * d), seed, -1).to(TYPES[c["q"]])
        s["q_rows"], s["k"], s["v"] = (x.view(rows, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], 1))
    if c["op"] in ("decode", "chunk"):
        s["out"] = torch.empty((rows, hq, d), dtype=TYPES[c["q"]], device=DEV)
    if own:
        from dendrite_amd import _lib, backend as fw
        fmt = {"f32": _lib.KV_F32, "bf16": _lib.KV_BF16, "f16": _lib.KV_F16, "fp8": _lib.KV_FP8_E4M3,
               "mxfp8": _lib.KV_MXFP8}[c["kv"]]
        be = fw.Backend(0)
        pool = fw.Pool(be, data.shape[0], hkv, d, fmt)
        s["data"], s["scales"] = _pool_views(_lib.lib(), pool, data, scales)
        tables = fw.TokenTables(s["indices"], s["indptr"], s["kv_len"], s["q_indptr"], max_kv_len=s["longest"])
        s.update(be=be, pool=pool, tables=tables, status=torch.zeros(1, **i32))
        if "out" in s:
            cfg = fw.AttentionConfig(hq, hkv, d)
            cfg.q_dtype, cfg.kv_format = fw.dtype_code(TYPES[c["q"]]), fmt
            cfg.gqa_mapping = _lib.GQA_TILED if c["tiled"] else _lib.GQA_INTERLEAVED
            cfg.sliding_window = c["window"] or None
            s["cfg"] = cfg
            s["ws"] = torch.empty(max(256, fw.window_workspace_size(cfg, tables, rows, c["sinks"])),
                                  dtype=torch.uint8, device=DEV)
        torch.cuda.synchronize()
    return s


# ---------------------------------------------------------------- plain forms
def _sequences(s):
    """Tokens, new tokens and first row of each sequence."""
    kv = s["kv_len"].long()
    at = s["q_indptr"].long() if s["q_indptr"] is not None else torch.arange(s["seqs"] + 1, device=DEV)
    return kv, at[1:] - at[:-1], at[:-1]


def _places(s):
    """Page and slot of each row's token."""
    kv, n, first = _sequences(s)
    b = torch.repeat_interleave(torch.arange(s["seqs"], device=DEV), n)
    t = (kv - n - first)[b] + torch.arange(s["rows"], device=DEV)
    return s["indices"].long()[s["indptr"].long()[b] + t // PAGE], t % PAGE


def _tokens(s, plane, page, slot):
    """Elements of plane 0 (K) or 1 (V) at (page, slot), in 32 bits: [..., hkv, d]."""
    x = s["data"].view(torch.uint8)[page, plane, :, slot] if s["kv"] in ("fp8", "mxfp8") else \
        s["data"][page, plane, :, slot]
    if s["kv"] == "fp8":
        return x.view(torch.float8_e4m3fn).float() * s["scales"][page, plane][..., None]
    if s["kv"] == "mxfp8":
        e = s["scales"][page, plane, :, slot].int() - 127
        return torch.ldexp(x.view(torch.float8_e4m3fn).float().unflatten(-1, (-1, 32)), e[..., None]).flatten(-2)
    return x.float()


def _plain_append(s):
    page, slot = _places(s)
    data, scales = s["data"], s["scales"]
    x = torch.stack([s["k"], s["v"]], 1).float()          # [rows, 2, hkv, d]
    if s["kv"] == "mxfp8":
        codes, e = _mx_codes(x)
        data.view(torch.uint8)[page, :, :, slot] = codes.view(torch.uint8)
        scales[page, :, :, slot] = e
    elif s["kv"] == "fp8":
        ids, of = torch.unique(page, return_inverse=True)  # the call's pages, and each row's
        amax = torch.zeros((len(ids), 2, s["hkv"]), device=DEV)
        amax.scatter_reduce_(0, of[:, None, None].expand(-1, 2, s["hkv"]), x.abs().amax(-1), "amax")
        begins = torch.zeros(len(ids), dtype=torch.bool, device=DEV)
        begins[of[slot == 0]] = True
        begins = begins[:, None, None]
        old = scales[ids]
        (ma, ea), (mt, et) = torch.frexp(amax), torch.frexp(old * 448.0)
        k = torch.where(~begins & (amax > old * 448.0), ea - et + (ma > mt), 0)
        new = torch.where(begins, (amax / 448.0).clamp(min=FLOOR), torch.ldexp(old, k))
        scales[ids] = new
        block = data.view(torch.uint8)[ids].view(torch.float8_e4m3fn).float()
        shrunk = _e4m3(torch.ldexp(block, -k[..., None, None]))
        below = torch.full((len(ids),), PAGE, device=DEV).scatter_reduce_(0, of, slot, "amin")
        earlier = torch.arange(PAGE, device=DEV)[None, :] < below[:, None]
        data.view(torch.uint8)[ids] = torch.where(earlier[:, None, None, :, None], shrunk.view(torch.uint8),
                                                  data.view(torch.uint8)[ids])
        data.view(torch.uint8)[page, :, :, slot] = _e4m3(x / new[of][..., None]).view(torch.uint8)
    else:
        data[page, :, :, slot] = x.to(data.dtype)
    return [data] if scales is None else [data, scales]


def _plain_read(s):
    page, slot = _places(s)
    s["k"].copy_(_tokens(s, 0, page, slot))
    s["v"].copy_(_tokens(s, 1, page, slot))
    return [s["k"], s["v"]]


def _plain_attend(s):
    kv, n, first = _sequences(s)
    B, hkv, d, W, S, Q = s["seqs"], s["hkv"], s["d"], s["window"], s["sinks"], s["most_new"]
    r = s["hq"] // hkv
    near = min(W + Q - 1 if W else s["longest"], s["longest"])
    S = min(S, s["longest"]) if W else 0
    # the tokens some row of a sequence may see: the sinks, then the window's
    start = (kv - n - W + 1).clamp(min=S) if W else torch.zeros_like(kv)
    t = torch.cat([torch.arange(S, device=DEV).expand(B, S), start[:, None] + torch.arange(near, device=DEV)], 1)
    held = t < kv[:, None]
    t = torch.where(held, t, 0)
    page, slot = s["indices"].long()[s["indptr"].long()[:-1, None] + t // PAGE], t % PAGE
    k = _tokens(s, 0, page, slot).permute(0, 2, 3, 1).contiguous()       # [B, hkv, d, N]
    v = _tokens(s, 1, page, slot).transpose(1, 2).contiguous()           # [B, hkv, N, d]
    i = torch.arange(Q, device=DEV)
    q = s["q_rows"][(first[:, None] + i).clamp(max=s["rows"] - 1)].float()      # [B, Q, hq, d]
    q = q.unflatten(2, (r, hkv) if s["tiled"] else (hkv, r))
    q = q.permute(0, 3, 2, 1, 4) if s["tiled"] else q.permute(0, 2, 3, 1, 4)  # [B, hkv, r, Q, d]
    x = (q.reshape(B, hkv, r * Q, d) @ k).view(B, hkv, r, Q, -1) * float(np.float32(1.0 / math.sqrt(d)))
    p = (kv - n)[:, None] + i
    seen = held[:, None, :] & (t[:, None, :] <= p[:, :, None])
    if W:
        seen &= (t[:, None, :] > p[:, :, None] - W) | (t[:, None, :] < S)
    x.masked_fill_(~seen[:, None, None], -math.inf)
    x -= x.amax(-1, keepdim=True).clamp(min=-3e38)
    x.exp_()
    x /= x.sum(-1, keepdim=True).clamp(min=1e-30)
    o = (x.view(B, hkv, r * Q, -1) @ v).view(B, hkv, r, Q, d)
    o = o.permute(0, 3, 2, 1, 4) if s["tiled"] else o.permute(0, 3, 1, 2, 4)
    s["out"].copy_(o.reshape(B, Q, s["hq"], d)[i < n[:, None]])
    return s["out"]


def run(s):
    if own:
        from dendrite_amd.backend import attend_window
        if s["op"] == "append":
            s["pool"].append_tokens(s["tables"], s["k"], s["v"], s["status"])
            return [s["data"]] if s["scales"] is None else [s["data"], s["scales"]]
        if s["op"] == "read":
            s["pool"].read_tokens(s["tables"], s["k"], s["v"], s["status"])
            return [s["k"], s["v"]]
        attend_window(s["be"], s["pool"], s["cfg"], s["tables"], s["q_rows"], s["out"], s["ws"], s["sinks"],
                      s["status"])
        return s["out"]
    return {"append": _plain_append, "read": _plain_read}.get(s["op"], _plain_attend)(s)


# ------------------------------------------------------------- what it has to be
def work(c):
    kv_len, new = _lens(c)
    hq, hkv, d = c["hq"], c["hkv"], c["d"]
    token = 2 * hkv * d * SIZE[c["kv"]] + (2 * hkv * d // 32 if c["kv"] == "mxfp8" else 0)
    record = 8 * hkv if c["kv"] == "fp8" else 0           # the scales of a page
    if c["op"] in ("append", "read"):
        pages = sum((t + PAGE - 1) // PAGE - (t - m) // PAGE for t, m in zip(kv_len, new))
        return {"bytes": sum(new) * (2 * hkv * d * SIZE[c["q"]] + token) + pages * (record + 4), "flops": 0}
    W, S = c["window"], c["sinks"]
    tokens = pages = pairs = 0
    for t, m in zip(kv_len, new):
        p = np.arange(t - m, t)
        pairs += int((np.minimum(p + 1, W) + np.clip(p + 1 - W, 0, S)).sum() if W else (p + 1).sum())
        lo = max(0, t - m - W + 1) if W else 0
        far = min(S, lo) if W else 0                       # sinks before the window
        tokens += t - lo + far
        pages += (t + PAGE - 1) // PAGE - lo // PAGE + min((far + PAGE - 1) // PAGE, lo // PAGE)
    return {"bytes": tokens * token + pages * (record + 4) + sum(new) * 2 * hq * d * SIZE[c["q"]],
            "flops": 4 * hq * d * pairs}


def exact(c, seed):
    """From the definitions, a sequence at a time, in 64 bits."""
    kv_len, new = _lens(c)
    s = prepare(c, seed)
    hq, hkv, d, kv = c["hq"], c["hkv"], c["d"], c["kv"]
    at, row, outs = 0, 0, []
    whole, scale = s["data"].double(), None
    if kv == "fp8":
        scale = s["scales"].double()
        values = whole * scale[..., None, None] if c["op"] != "append" else None
    elif kv == "mxfp8":
        scale = s["scales"].clone()
        values = (whole.unflatten(-1, (-1, 32)) * torch.exp2(scale.double() - 127)[..., None]).flatten(-2)
    else:
        values = whole
    for t, m in zip(kv_len, new):
        np_ = (t + PAGE - 1) // PAGE
        ids = s["indices"][at:at + np_].long()
        if c["op"] == "append":
            x = torch.stack([s["k"][row:row + m], s["v"][row:row + m]]).double()       # [2, m, hkv, d]
            for j in range((t - m) // PAGE, np_):          # a page at a time
                lo, hi = max(t - m, PAGE * j), min(t, PAGE * (j + 1))
                y = x[:, lo - (t - m):hi - (t - m)].transpose(1, 2)                    # [2, hkv, tokens, d]
                a, b, p = lo - PAGE * j, hi - PAGE * j, ids[j]
                if kv == "fp8":
                    big = y.abs().amax((2, 3))
                    if a == 0:
                        f = torch.clamp(big / 448, min=FLOOR)
                    else:
                        k = torch.ceil(torch.log2(big / (448 * scale[p]))).clamp(min=0)
                        f = scale[p] * torch.exp2(k)
                        whole[p, :, :, :a] = _e4m3(whole[p, :, :, :a] * torch.exp2(-k)[..., None, None]).double()
                    scale[p] = f
                    whole[p, :, :, a:b] = _e4m3(y / f[..., None, None]).double()
                elif kv == "mxfp8":
                    g = y.unflatten(-1, (-1, 32))
                    e = torch.floor(torch.log2(g.abs().amax(-1).clamp(min=1e-300))).clamp(-119, 135) - 8
                    whole[p, :, :, a:b] = _e4m3(g * torch.exp2(-e)[..., None]).double().flatten(-2)
                    scale[p, :, :, a:b] = (e + 127).to(torch.uint8)
                else:
                    whole[p, :, :, a:b] = y.to(TYPES[kv]).double()
        else:
            k, v = (values[ids, i].transpose(1, 2).reshape(-1, hkv, d)[:t] for i in (0, 1))
            if c["op"] == "read":
                outs.append((k[t - m:], v[t - m:]))
            else:
                q = s["q_rows"][row:row + m].double()
                o = torch.empty_like(q)
                p, j = torch.arange(t - m, t, device=DEV)[:, None], torch.arange(t, device=DEV)[None, :]
                see = j <= p
                if c["window"]:
                    see &= (p - j < c["window"]) | (j < c["sinks"])
                for h in range(hq):
                    g = h % hkv if c["tiled"] else h // (hq // hkv)
                    w = (q[:, h] @ k[:, g].t()) * float(np.float32(1.0 / math.sqrt(d)))
                    o[:, h] = torch.softmax(torch.where(see, w, -math.inf), -1) @ v[:, g]
                outs.append(o)
        at, row = at + np_, row + m
    if c["op"] == "append":
        return [whole] if scale is None else [whole, scale if kv == "fp8" else None]
    if c["op"] == "read":
        return [torch.cat([k for k, _ in outs]), torch.cat([v for _, v in outs])]
    return torch.cat(outs)
