"""Plain 64-bit forms of the token operators (dh_pool_append_tokens,
dh_pool_read_tokens, dh_attend_window) on host tensors, and the random caches
their tests run on.

A cache is the pool's memory as tensors: data [P, 2, hkv, 16, d] (float8_e4m3fn
codes or elements) and scales ([P, 2, hkv] float32, or [P, 2, hkv, 16, d / 32]
E8M0 bytes)."""
from __future__ import annotations

import math

import numpy as np
import torch

from dendrite_amd import _lib

PAGE = 16
FORMATS = {"f32": _lib.KV_F32, "bf16": _lib.KV_BF16, "f16": _lib.KV_F16, "fp8": _lib.KV_FP8_E4M3,
           "mxfp8": _lib.KV_MXFP8}
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
PAIRS = [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"), ("f16", "fp8"), ("bf16", "mxfp8"),
         ("f16", "mxfp8")]
FLOOR = 2.0 ** -64


def e4m3(y):
    """Round to nearest even into E4M3, saturated; NaN stays NaN."""
    return torch.where(y.isnan(), y, y.clamp(-448.0, 448.0)).to(torch.float32).to(torch.float8_e4m3fn)


def finite_amax(x, dims):
    a = x.abs()
    return torch.where(a < math.inf, a, 0.0).amax(dims)


def mx_codes(x):
    g = x.unflatten(-1, (-1, 32))
    amax = finite_amax(g, -1)[..., None]
    e = torch.where(amax > 0, torch.frexp(amax).exponent - 9, -127).clamp(-127, 127)
    return e4m3(g.double() * torch.exp2(-e.double())).flatten(-2), (e + 127).to(torch.uint8).squeeze(-1)


def values(data, scales, fmt):
    """What the cache stands for, in 64 bits."""
    x = data.float().double()
    if fmt == "fp8":
        return x * scales.double()[..., None, None]
    if fmt == "mxfp8":
        s = torch.where(scales == 255, math.nan, torch.exp2(scales.double() - 127))
        return (x.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)
    return x


class Case:
    """Sequences of kv_len tokens, the last q_len of them new, on shuffled
    pages.  Slots past a sequence's end, and pages of nobody, are poisoned
    (NaN codes and scales).  `row0` rows come before the first sequence's and
    `pad` after the last one's."""

    def __init__(self, seed, fmt, rows, hq, hkv, d, kv_len, q_len=None, row0=0, pad=0, spare=2, poison=True,
                 amp=1.0):
        self.fmt, self.rows_type, self.hq, self.hkv, self.d = fmt, rows, hq, hkv, d
        self.kv_len = [int(t) for t in kv_len]
        self.single = q_len is None
        self.q_len = [min(1, t) for t in self.kv_len] if self.single else [int(n) for n in q_len]
        g = torch.Generator().manual_seed(seed)
        need = [(t + PAGE - 1) // PAGE for t in self.kv_len]
        size = sum(need) + len(need) * spare + 3
        perm = torch.randperm(size, generator=g).int()
        self.tables, at = [], 0
        for n in need:                       # spare entries after each sequence's pages
            self.tables.append(perm[at:at + n + spare].clone())
            at += n + spare
        x = torch.randn((size, 2, hkv, PAGE, d), generator=g)
        if fmt == "mxfp8":
            x = torch.where(torch.rand(x.shape, generator=g) < 0.01, x * 20, x)
        x[:, 1] *= amp
        if fmt == "fp8":
            self.scales = finite_amax(x, (3, 4)) / 448.0
            self.data = e4m3(x / self.scales[..., None, None])
        elif fmt == "mxfp8":
            self.data, self.scales = mx_codes(x)
        else:
            self.data, self.scales = x.to(TYPES[fmt]), None
        if poison:
            used = torch.zeros(size, dtype=torch.bool)
            for t, table in zip(self.kv_len, self.tables):
                n = (t + PAGE - 1) // PAGE
                used[table[:n].long()] = True
                if t % PAGE:
                    p = int(table[n - 1])
                    self._poison(p, t % PAGE)
            for p in torch.nonzero(~used).flatten().tolist():
                self._poison(p, 0)
                if fmt == "fp8":
                    self.scales[p] = math.nan
        n = row0 + (len(self.kv_len) if self.single else sum(self.q_len)) + pad
        self.row0, self.num_rows = row0, n
        assert not (self.single and row0)
        self.qkv = torch.randn((n, (hq + 2 * hkv) * d + 16), generator=g).to(TYPES[rows])
        self.q_indptr = None if self.single else torch.tensor(np.cumsum([row0] + self.q_len), dtype=torch.int32)
        self.set_tables()

    def _poison(self, p, slot):
        self.data[p, :, :, slot:] = math.nan
        if self.fmt == "mxfp8":
            self.scales[p, :, :, slot:] = 255

    def set_tables(self):
        self.indices = torch.cat(self.tables) if self.tables else torch.zeros(0, dtype=torch.int32)
        self.indptr = torch.tensor(np.cumsum([0] + [len(t) for t in self.tables]), dtype=torch.int32)

    def first_row(self, b):
        return b if self.single else int(self.q_indptr[b])

    # views of the fused rows
    def q(self, x=None):
        x = self.qkv if x is None else x
        return x[:, :self.hq * self.d].view(self.num_rows, self.hq, self.d)

    def k(self, x=None):
        x = self.qkv if x is None else x
        return x[:, self.hq * self.d:(self.hq + self.hkv) * self.d].view(self.num_rows, self.hkv, self.d)

    def v(self, x=None):
        x = self.qkv if x is None else x
        at = (self.hq + self.hkv) * self.d
        return x[:, at:at + self.hkv * self.d].view(self.num_rows, self.hkv, self.d)


def tokens_of(case, b, x):
    """Values x of sequence b's tokens as (K, V) [T, hkv, d], and which of
    them are on pages of the pool."""
    t = case.kv_len[b]
    ids = case.tables[b][:(t + PAGE - 1) // PAGE].long()
    ok = (ids >= 0) & (ids < x.shape[0])
    y = x[ids.clamp(0, x.shape[0] - 1)]
    k, v = (y[:, i].transpose(1, 2).reshape(-1, case.hkv, case.d)[:t] for i in (0, 1))
    return k, v, ok.repeat_interleave(PAGE)[:t]


def append(case):
    """(data, scales) after the call."""
    data, scales = case.data.clone(), None if case.scales is None else case.scales.clone()
    raw = data.view(torch.uint8) if case.fmt in ("fp8", "mxfp8") else data
    for b, (t, m) in enumerate(zip(case.kv_len, case.q_len)):
        if m == 0:
            continue
        r = case.first_row(b)
        x = torch.stack([case.k()[r:r + m], case.v()[r:r + m]]).float()
        for j in range((t - m) // PAGE, (t + PAGE - 1) // PAGE):
            p = int(case.tables[b][j])
            if not 0 <= p < data.shape[0]:
                continue
            lo, hi = max(t - m, PAGE * j), min(t, PAGE * (j + 1))
            y = x[:, lo - (t - m):hi - (t - m)].transpose(1, 2)
            lo, hi = lo - PAGE * j, hi - PAGE * j
            if case.fmt == "fp8":
                amax = finite_amax(y, (2, 3))
                if lo == 0:
                    s = (amax / 448.0).clamp(min=FLOOR)
                else:
                    old = scales[p]
                    # the least k with amax <= 448 old 2^k, by search
                    k = torch.zeros_like(old, dtype=torch.int32)
                    for _ in range(300):
                        k += (amax.double() > (448.0 * old).double() * torch.exp2(k.double())).int()
                    s = torch.ldexp(old, k)
                    grown = e4m3(torch.ldexp(data[p].float(), -k[..., None, None]))
                    raw[p, :, :, :lo] = grown[:, :, :lo].view(torch.uint8)
                scales[p] = s
                raw[p, :, :, lo:hi] = e4m3(y / s[..., None, None]).view(torch.uint8)
            elif case.fmt == "mxfp8":
                codes, e = mx_codes(y)
                raw[p, :, :, lo:hi] = codes.view(torch.uint8)
                scales[p, :, :, lo:hi] = e
            else:
                raw[p, :, :, lo:hi] = y.to(TYPES[case.fmt])
    return data, scales


def attend(case, window, sinks, tiled, scale):
    """(out, bound): the rows' attention in 64 bits (NaN for rows of nobody),
    and how far a kernel may be from it by the roundings it makes.

    With u the half step of the rows' type, a row's exact weights w (sum 1),
    scores s and A = sum w |v|:
      weights rounded once for the products, and in their sum: 2 u A;
      scores accumulated in f32 over d products, scaled, exponentiated:
        |ds| <= (d + 4) 2^-24 (scale sum |q k| + |s| + |reference|) + 2^-22,
        both in the products and in their sum: 2 max|ds| A;
      f16 weights below 2^-14 are off by 2^-25 of the row's reference weight,
        which is at most its sum: 2^-25 sum |v|; in FP8 weights have V's scale
        in them, and so has the reference: 2^-25 sum |v| (largest / own scale);
      the sums of the products, f32: (T + 8) 2^-24 A;
      the result rounded: u |out| + the type's least step."""
    vals = values(case.data, case.scales, case.fmt)
    out = torch.full((case.num_rows, case.hq, case.d), math.nan, dtype=torch.float64)
    bound = torch.zeros_like(out)
    kind = TYPES[case.rows_type]
    u = torch.finfo(kind).eps / 2
    for b, (t, m) in enumerate(zip(case.kv_len, case.q_len)):
        r = case.first_row(b)
        if case.single and t == 0:
            out[r] = 0
            continue
        if m == 0:
            continue
        k, v, ok = tokens_of(case, b, vals)
        q = case.q()[r:r + m].double()
        p, j = torch.arange(t - m, t)[:, None], torch.arange(t)[None, :]
        see = (j <= p) & ok[None, :]
        if window:
            see = see & ((j > p - window) | (j < sinks))
        any_ = see.any(0)
        k, v = torch.where(any_[:, None, None], k, 0.0), torch.where(any_[:, None, None], v, 0.0)
        small = torch.ones(t, case.hkv, dtype=torch.float64)
        if case.fmt == "fp8":
            ids = case.tables[b][:(t + PAGE - 1) // PAGE].long().clamp(0, case.data.shape[0] - 1)
            vs = torch.nan_to_num(case.scales[ids, 1].double(), 0, 0, 0)
            small = (vs.amax(0) / vs.clamp(min=FLOOR)).repeat_interleave(PAGE, 0)[:t]
            log = (vs.clamp(min=FLOOR).log2().abs().amax(0) + 2) * 2.0 ** -23
        for h in range(case.hq):
            g = h % case.hkv if tiled else h // (case.hq // case.hkv)
            s = q[:, h] @ k[:, g].t() * scale
            w = torch.softmax(torch.where(see, s, -math.inf), -1).nan_to_num(0.0)
            o = w @ v[:, g]
            out[r:r + m, h] = o
            A = w @ v[:, g].abs()
            mag = abs(scale) * (q[:, h].abs() @ k[:, g].abs().t())
            ds = ((case.d + 4) * 2.0 ** -24 * (mag + 2 * s.abs().amax(-1, keepdim=True)) * see).amax(-1, keepdim=True)
            f = 2 * u + 2 * (ds + 2.0 ** -22) + (t + 8) * 2.0 ** -24
            if case.rows_type == "f32":
                f = f - 2 * u
            if case.fmt == "fp8":
                f = f + 2 * float(log[g])
            e = f * A + u * o.abs()
            if case.rows_type == "f16":
                e = e + 2.0 ** -25 * (see.double() @ (v[:, g].abs() * small[:, g][:, None]))
            bound[r:r + m, h] = e + float(torch.finfo(kind).smallest_normal) * float(torch.finfo(kind).eps)
    return out, bound


class Memory:
    def __init__(self, ptr, nbytes):
        self.__cuda_array_interface__ = dict(shape=(nbytes,), typestr="|u1", data=(ptr, False), version=2)


def pool_views(pool, data, scales):
    """Uploads a cache into the pool; its memory as tensors like data, scales."""
    L, views = _lib.lib(), []
    for t, ptr in ((data, L.dh_pool_data(pool._h)), (scales, L.dh_pool_scales(pool._h))):
        if t is None:
            views.append(None)
            continue
        v = torch.as_tensor(Memory(ptr, t.numel() * t.element_size()), device="cuda:0")
        v.copy_(t.contiguous().view(-1).view(torch.uint8))
        v = v.view(t.dtype).view(t.shape)
        v.pool = pool
        views.append(v)
    torch.cuda.synchronize()
    return views
