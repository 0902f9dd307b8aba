"""attend_window against its plain 64-bit form (tests/_tokens.py), within the
bound its roundings give."""
import math

import numpy as np
import pytest
import torch

from dendrite_amd import _lib
from dendrite_amd.backend import AttentionConfig, Pool, TokenTables, attend_window, window_workspace_size
from tests import _tokens as T
from tests.test_gpu_tokens import tables, upload

pytestmark = pytest.mark.gpu


def config(case, window, tiled, scale=None):
    cfg = AttentionConfig(case.hq, case.hkv, case.d)
    cfg.q_dtype = {"f32": _lib.DTYPE_F32, "bf16": _lib.DTYPE_BF16, "f16": _lib.DTYPE_F16}[case.rows_type]
    cfg.kv_format = T.FORMATS[case.fmt]
    cfg.gqa_mapping = _lib.GQA_TILED if tiled else _lib.GQA_INTERLEAVED
    cfg.sliding_window = window or None
    if scale is not None:
        cfg.scale = scale
    return cfg


def check(backend, case, window=0, sinks=0, tiled=True, max_kv_len=None, scale=None, status=0, want=None):
    cfg = config(case, window, tiled, scale)
    pool, *_ = upload(backend, case)
    tab = tables(case, max_kv_len)
    n = window_workspace_size(cfg, tab, case.num_rows, sinks)
    ws = torch.full((max(n, 1),), 255, dtype=torch.uint8, device="cuda")      # NaN
    rows = case.qkv.cuda()
    buf = torch.full((case.num_rows, case.hq * case.d + 16), 7.0, dtype=rows.dtype, device="cuda")
    out = buf[:, :case.hq * case.d].view(case.num_rows, case.hq, case.d)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    attend_window(backend, pool, cfg, tab, case.q(rows), out, ws if n else None, sinks, st)
    torch.cuda.synchronize()
    got = out.double().cpu()
    ref, bound = want or T.attend(case, window, sinks, tiled, float(cfg.scale))
    none = ref.isnan().all(-1).all(-1)
    assert (got[none] == 7.0).all(), "a row of nobody was written"
    assert (buf[:, case.hq * case.d:] == 7.0).all()
    err = (got - ref).abs()
    assert not got[~none].isnan().any()
    worst = float((err[~none] / bound[~none].clamp(min=1e-300)).max()) if (~none).any() else 0.0
    assert worst <= 1.0, f"error of {worst:.3g} times the bound, max {float(err[~none].max()):.3g}"
    assert int(st) == status
    return got, n


# (kv_len, q_len or None for single tokens, window, sinks, tiled)
SHAPES = {
    "single": ([1, 0, 15, 16, 17, 33, 100, 257, 600], None, 0, 0, True),
    "single-window": ([1, 5, 16, 17, 0, 64, 65, 300, 601], None, 48, 3, False),
    "single-odd": ([700, 20, 333], None, 101, 37, True),
    "window-1": ([1, 40, 17], None, 1, 0, True),
    "short": ([9, 40, 70, 3, 130], [3, 0, 5, 3, 9], 33, 5, False),
    "short-full": ([20, 75, 16], [4, 7, 2], 0, 0, True),
    "chunk": ([300, 45, 150], [150, 45, 90], 64, 4, True),
    "chunk-full": ([260, 33, 128], [260, 33, 100], 0, 0, False),
    "chunk-odd": ([517, 90], [330, 77], 129, 20, True),
    "chunk-ragged": ([400, 1, 0, 64, 7], [399, 1, 0, 50, 7], 16, 0, False),
}


@pytest.mark.parametrize("rows,fmt", T.PAIRS)
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_attend(backend, rows, fmt, d, shape):
    kv, q, window, sinks, tiled = SHAPES[shape]
    single = q is None
    case = T.Case(21, fmt, rows, 8, 2, d, kv, q, row0=0 if single else 2, pad=3)
    check(backend, case, window, sinks, tiled, max_kv_len=max(kv))


@pytest.mark.parametrize("rows", ["f16", "bf16"])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shape", ["single-window", "short", "chunk"])
@pytest.mark.parametrize("amp", [2.0 ** -12, 2.0 ** 12])
def test_value_scales(backend, rows, d, shape, amp):
    """Weights keep their 16 bits whatever V's block scales are, though a scale
    is multiplied into them."""
    if rows == "f16" and amp > 1:
        amp = 2.0 ** 8          # the result has to stay in f16
    kv, q, window, sinks, tiled = SHAPES[shape]
    case = T.Case(41, "fp8", rows, 8, 2, d, kv, q, row0=0 if q is None else 2, pad=3, amp=amp)
    check(backend, case, window, sinks, tiled, max_kv_len=max(kv))


@pytest.mark.parametrize("shape", ["single-window", "short", "chunk"])
@pytest.mark.parametrize("amp", [2.0 ** -50, 2.0 ** 100])
def test_extreme_value_scales(backend, shape, amp):
    """The row's sum takes V's scales out again: it stays within f32."""
    kv, q, window, sinks, tiled = SHAPES[shape]
    case = T.Case(42, "fp8", "bf16", 8, 2, 128, kv, q, row0=0 if q is None else 2, pad=3, amp=amp)
    check(backend, case, window, sinks, tiled, max_kv_len=max(kv))


@pytest.mark.parametrize("hq,hkv", [(1, 1), (3, 1), (8, 8), (5, 5), (12, 4), (40, 2), (7, 1)])
@pytest.mark.parametrize("rows,fmt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "fp8")])
def test_heads(backend, hq, hkv, rows, fmt):
    """Groups of one to twenty query heads, odd ones, more than a tile's rows."""
    for tiled in (True, False):
        check(backend, T.Case(22, fmt, rows, hq, hkv, 64, [70, 19, 301], None, pad=1), 40, 2, tiled, 301)
        check(backend, T.Case(23, fmt, rows, hq, hkv, 64, [170, 19, 401], [100, 19, 130], row0=1), 40, 2, tiled, 401)


@pytest.mark.parametrize("rows,fmt", T.PAIRS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_split(backend, rows, fmt, d):
    """A bound far above the lengths splits the work over the chip: parts of
    the list that hold pages, a few tokens or nothing, joined."""
    case = T.Case(24, fmt, rows, 4, 1, d, [1500, 3, 0, 77], None, pad=2)
    _, n = check(backend, case, 0, 0, True, _lib.MAX_SEQ_LEN)
    assert n > 0
    check(backend, case, 1200, 20, True, 6000)       # (one part where 16 waves share a list)
    _, n = check(backend, case, 4200, 20, True, 6000)
    assert n > 0
    case = T.Case(25, fmt, rows, 4, 1, d, [1300, 200], [150, 130], row0=1, pad=2)
    _, n = check(backend, case, 0, 0, False, _lib.MAX_SEQ_LEN)
    assert n > 0
    case = T.Case(26, fmt, rows, 4, 1, d, [1300, 40], [6, 3], row0=1, pad=2)
    _, n = check(backend, case, 0, 0, False, _lib.MAX_SEQ_LEN)
    assert n > 0


@pytest.mark.parametrize("rows,fmt,hkv,d,new", [("bf16", "bf16", 2, 128, [515]), ("f16", "fp8", 2, 128, [500, 31]),
                                                ("bf16", "mxfp8", 2, 64, [1030]), ("f16", "f16", 2, 256, [129, 132])])
def test_tail(backend, rows, fmt, hkv, d, new):
    """A few blocks more than the chip holds at once: those are split by
    themselves (64 query heads a KV head make two tokens a block, four at 64
    dims)."""
    kv = [2900 + n if i == 0 else 700 + n for i, n in enumerate(new)]
    case = T.Case(29, fmt, rows, 64 * hkv, hkv, d, kv, new, row0=1, pad=2)
    _, n = check(backend, case, 0, 0, True, max(kv))
    assert n > 0
    case = T.Case(30, fmt, rows, 64 * hkv, hkv, d, kv, new, row0=1, pad=2)
    case.tables[0][90] = -1
    case.set_tables()
    check(backend, case, 2400, 40, False, max(kv))


def test_long_page_lists(backend):
    """Parts of nearly as many pages as a wave's registers and a workgroup's
    list hold: batches that fill the chip, with one very long sequence."""
    case = T.Case(27, "bf16", "bf16", 1, 1, 64, [70001] + [1] * 511, None, spare=0)
    _, n = check(backend, case, 0, 0, True, 70001)
    assert n > 0
    case = T.Case(28, "f16", "f16", 8, 1, 64, [66000] + [8] * 255, [130] + [8] * 255, spare=0)
    _, n = check(backend, case, 0, 0, True, 66000)
    assert n > 0


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp8"])
def test_freed_pages(backend, fmt):
    """Pages between the sinks and the window may be freed: their entries
    INVALID, or stale ids, and nothing of them read."""
    for q in (None, [2, 3], [200, 100]):
        kv = [900, 700]
        case = T.Case(29, fmt, "bf16", 4, 2, 128, kv, q)
        window, sinks = 100, 18
        for b, t in enumerate(kv):
            first = t - (1 if q is None else q[b])
            for j in range((sinks + 15) // 16, (first - window + 1) // 16):
                p = int(case.tables[b][j])
                case._poison(p, 0)
                case.tables[b][j] = -1 if j % 2 else 0x7FFFFFF0
        case.set_tables()
        clean = T.Case(29, fmt, "bf16", 4, 2, 128, kv, q)
        cfg = config(case, window, False)
        check(backend, case, window, sinks, False, 900, want=T.attend(clean, window, sinks, False, float(cfg.scale)))


def test_pages_outside_the_pool(backend):
    """An INVALID page in sight is skipped silently, another id reported; a
    row with no page left is zeros."""
    for q in (None, [40, 90]):
        case = T.Case(30, "bf16", "bf16", 4, 2, 64, [40, 100], q)
        case.tables[0][:] = -1
        case.tables[1][2] = -1
        case.set_tables()
        got, _ = check(backend, case, 0, 0, True, 100)
        assert (got[0] == 0).all()
        case.tables[1][3] = case.data.shape[0]
        case.set_tables()
        check(backend, case, 0, 0, True, 100, status=_lib.DH_EINVAL)


@pytest.mark.parametrize("max_kv_len", [130, _lib.MAX_SEQ_LEN])
def test_refused_sequences(backend, max_kv_len):
    """A sequence whose entries contradict each other gets zeros and a report,
    the others their attention."""
    for q in (None, [100, 100, 100]):
        case = T.Case(31, "bf16", "bf16", 4, 2, 64, [100, 110, 120], q)
        cfg = config(case, 50, True)
        want = T.attend(case, 50, 3, True, float(cfg.scale))
        r = case.first_row(1)
        want[0][r:r + case.q_len[1]] = 0
        for bad in ("len", "negative", "table", "order"):
            kv, indptr = list(case.kv_len), case.indptr.clone()
            if bad == "len":
                kv[1] = 50000000
            elif bad == "negative":
                kv[1] = -5
            elif bad == "table":
                kv[1] = 129 if max_kv_len < 1000 else 1000
                indptr[1:2] = indptr[2:3] - 3          # sequence 0 keeps a longer table
            elif bad == "order":
                indptr[2:3] = int(indptr[3]) + 1000
            other = T.Case.__new__(T.Case)
            other.__dict__ = dict(case.__dict__, kv_len=kv, indptr=indptr)
            w = (want[0].clone(), want[1].clone())
            if bad == "order":                          # sequence 2's table now begins out of bounds
                r2 = case.first_row(2)
                w[0][r2:r2 + case.q_len[2]] = 0
            check(backend, other, 50, 3, True, max_kv_len, status=_lib.DH_EINVAL, want=w)


def test_rows_out_of_order_are_left(backend):
    """q_indptr entries that are not in order: those rows are nobody's."""
    case = T.Case(32, "bf16", "bf16", 4, 2, 64, [100, 110, 120], [90, 90, 90])
    cfg = config(case, 0, True)
    out, bound = T.attend(case, 0, 0, True, float(cfg.scale))
    case.q_indptr = torch.tensor([0, 90, 180, 1 << 20], dtype=torch.int32)
    out[180:] = math.nan
    check(backend, case, 0, 0, True, 120, status=_lib.DH_EINVAL, want=(out, bound))


@pytest.mark.parametrize("rows,fmt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "fp8")])
@pytest.mark.parametrize("scale", [-0.2, 0.0, 3.0])
def test_scales(backend, rows, fmt, scale):
    for kv, q in (([100, 37], None), ([200, 137], [150, 137])):
        check(backend, T.Case(33, fmt, rows, 4, 2, 64, kv, q), 60, 4, True, max(kv), scale=scale)


@pytest.mark.parametrize("rows,fmt", [("bf16", "bf16"), ("f16", "f16")])
def test_large_scores(backend, rows, fmt):
    """Scores that climb through the sequence, so the softmax's reference has
    to move again and again, and ones far below the first."""
    for q in (None, [200, 10]):
        case = T.Case(34, fmt, rows, 4, 2, 64, [600, 10], q)
        for b in range(2):
            for j, p in enumerate(case.tables[b][:(case.kv_len[b] + 15) // 16].tolist()):
                case.data[p, 0] = (case.data[p, 0].float() * (1 + 0.3 * (j if b == 0 else -j))).to(case.data.dtype)
        check(backend, case, 0, 0, True, 600)
        check(backend, case, 256, 16, True, 600)


def test_many_sequences(backend):
    """More sequences than one search round tells apart, some without rows."""
    q = [(5 * b) % 13 if b % 4 else 0 for b in range(200)]
    kv = [n + (11 * b) % 90 for b, n in enumerate(q)]
    check(backend, T.Case(35, "bf16", "bf16", 4, 2, 64, kv, q, row0=4, pad=4), 32, 4, True, max(kv))
    q = [n * 12 for n in q]
    kv = [n + (11 * b) % 90 for b, n in enumerate(q)]
    check(backend, T.Case(36, "bf16", "bf16", 4, 2, 64, kv, q, row0=4, pad=4), 32, 4, True, max(kv))


def test_window_at_least_as_long_as_the_bound(backend):
    """Windows at, above and just below the longest sequence; the largest."""
    case = T.Case(37, "bf16", "bf16", 4, 2, 64, [200, 100], [3, 100])
    for window in (199, 200, 201, (1 << 32) - 1):
        check(backend, case, window, 5, True, 200)
    check(backend, case, (1 << 32) - 1, (1 << 32) - 1, True, 1 << 22)
    check(backend, case, 150, (1 << 32) - 1, True, 1 << 22)


def test_far_pages(backend):
    """Pages past 4 GiB of the pool's data, and past 2^31 of its elements."""
    hkv, d = 8, 128
    pages = (5 << 30) // (2 * hkv * 16 * d * 2)
    pool = Pool(backend, pages, hkv, d, _lib.KV_BF16)
    case = T.Case(38, "bf16", "bf16", 16, hkv, d, [100, 33], [40, 20], spare=0, poison=False)
    n = case.data.shape[0]
    L = _lib.lib()
    view = torch.as_tensor(T.Memory(L.dh_pool_data(pool._h) + (pages - n) * pool.page_bytes, n * pool.page_bytes),
                           device="cuda:0")
    view.copy_(case.data.view(-1).view(torch.uint8))
    tab = TokenTables((case.indices + (pages - n)).cuda(), case.indptr.cuda(),
                      torch.tensor(case.kv_len, dtype=torch.int32).cuda(), case.q_indptr.cuda(), 100)
    rows = case.qkv.cuda()
    out = torch.empty((case.num_rows, 16, d), dtype=torch.bfloat16, device="cuda")
    cfg = config(case, 30, True)
    pool.append_tokens(tab, case.k(rows), case.v(rows))
    attend_window(backend, pool, cfg, tab, case.q(rows), out, sinks=2)
    k, v = torch.empty_like(case.k(rows)), torch.empty_like(case.v(rows))
    pool.read_tokens(tab, k, v)
    torch.cuda.synchronize()
    case.data, _ = T.append(case)
    want, bound = T.attend(case, 30, 2, True, float(cfg.scale))
    assert ((out.double().cpu() - want).abs() <= bound).all()
    assert torch.equal(k, case.k(rows)) and torch.equal(v, case.v(rows))


def _steps(backend, fmt, rows, graph):
    """A prompt in two chunks, then single tokens, of three sequences: append,
    attend, read; each step against the plain forms on the cache as it is."""
    hq, hkv, d, window, sinks = 8, 2, 128, 48, 4
    kv0 = [61, 16, 5]
    case = T.Case(40, fmt, rows, hq, hkv, d, kv0, kv0, spare=6, poison=True)
    pool, data, scales = upload(backend, case)
    cfg = config(case, window, False)
    g = torch.Generator().manual_seed(3)
    tab_idx, tab_ptr = case.indices.cuda(), case.indptr.cuda()
    kv_len = torch.zeros(3, dtype=torch.int32, device="cuda")
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    single = TokenTables(tab_idx, tab_ptr, kv_len, None, 200)
    buf = torch.zeros((3, (hq + 2 * hkv) * d), dtype=T.TYPES[rows], device="cuda")
    out1 = torch.zeros((3, hq, d), dtype=buf.dtype, device="cuda")
    ws = torch.empty(max(256, window_workspace_size(cfg, single, 3, sinks)), dtype=torch.uint8, device="cuda")

    def split(x):
        q, k, v = x.split([hq * d, hkv * d, hkv * d], 1)
        return q.view(-1, hq, d), k.view(-1, hkv, d), v.view(-1, hkv, d)

    def step1():
        q, k, v = split(buf)
        pool.append_tokens(single, k, v, st)
        attend_window(backend, pool, cfg, single, q, out1, ws, sinks, st)

    replay = step1
    held = [0, 0, 0]
    if graph:
        kv_len.zero_()
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            step1()
        torch.cuda.current_stream().wait_stream(s)
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            step1()
        replay = gr.replay
    for new in ([40, 16, 0], [21, 0, 5]) + ([1, 1, 1],) * 20 + ([1, 0, 1],) * 3:
        is1 = max(new) == 1 and held[0] > 0 and new != [21, 0, 5]
        held = [a + n for a, n in zip(held, new)]
        n = 3 if is1 else sum(new)
        x = torch.randn((n, (hq + 2 * hkv) * d), generator=g).to(buf.dtype)
        # the plain side's view of this step
        case.data, case.scales = data.cpu(), None if scales is None else scales.cpu()
        case.single, case.num_rows, case.q_len = is1, n, list(new)
        case.kv_len = [t if m or not is1 else 0 for t, m in zip(held, new)] if is1 else list(held)
        case.q_indptr = None if is1 else torch.tensor(np.cumsum([0] + list(new)), dtype=torch.int32)
        case.qkv = torch.cat([x, x[:, :16]], 1)
        kv_len.copy_(torch.tensor(case.kv_len, dtype=torch.int32))
        if is1:
            buf.copy_(x)
            replay()
            out = out1
        else:
            tab = TokenTables(tab_idx, tab_ptr, kv_len, case.q_indptr.cuda(), 200)
            q, k, v = split(x.cuda())
            out = torch.zeros((n, hq, d), dtype=buf.dtype, device="cuda")
            pool.append_tokens(tab, k, v, st)
            w2 = torch.empty(max(256, window_workspace_size(cfg, tab, n, sinks)), dtype=torch.uint8, device="cuda")
            attend_window(backend, pool, cfg, tab, q, out, w2, sinks, st)
        torch.cuda.synchronize()
        want_data, want_scales = T.append(case)
        nan = want_data.float().isnan()
        assert torch.equal(data.cpu().float()[~nan], want_data.float()[~nan])
        case.data, case.scales = want_data, want_scales
        want, bound = T.attend(case, window, sinks, False, float(cfg.scale))
        assert ((out.double().cpu() - want).abs() <= bound).all()
        assert int(st) == 0
    # all of it read back
    tab = TokenTables(tab_idx, tab_ptr, torch.tensor(held, dtype=torch.int32).cuda(),
                      torch.tensor(np.cumsum([0] + held), dtype=torch.int32).cuda(), 200)
    k = torch.empty((sum(held), hkv, d), dtype=buf.dtype, device="cuda")
    v = torch.empty_like(k)
    pool.read_tokens(tab, k, v, st)
    torch.cuda.synchronize()
    vals = T.values(case.data, case.scales, fmt)
    case.kv_len, at = held, 0
    for b, t in enumerate(held):
        a, c, _ = T.tokens_of(case, b, vals)
        assert torch.equal(k[at:at + t].cpu(), a.float().to(buf.dtype))
        assert torch.equal(v[at:at + t].cpu(), c.float().to(buf.dtype))
        at += t


@pytest.mark.parametrize("rows,fmt", T.PAIRS)
def test_steps_together(backend, rows, fmt):
    _steps(backend, fmt, rows, False)


@pytest.mark.parametrize("rows,fmt", [("bf16", "bf16"), ("bf16", "fp8"), ("f32", "f32")])
def test_steps_captured(backend, rows, fmt):
    """The single-token step as a captured graph, replayed with eager work and
    synchronisations between, following the tables' contents."""
    _steps(backend, fmt, rows, True)


def test_two_streams(backend):
    """Calls on two streams at once, a workspace each."""
    cases = [T.Case(50 + i, "bf16", "bf16", 8, 2, 128, [4000 + i, 900], q) for i, q in enumerate((None, [100, 200]))]
    streams = [torch.cuda.Stream() for _ in cases]
    made = []
    for case in cases:
        cfg = config(case, 0, True)
        tab = tables(case)
        n = window_workspace_size(cfg, tab, case.num_rows)
        made.append((upload(backend, case)[0], cfg, tab, case.q(case.qkv.cuda()),
                     torch.zeros((case.num_rows, 8, 128), dtype=torch.bfloat16, device="cuda"),
                     torch.empty(n, dtype=torch.uint8, device="cuda")))
    torch.cuda.synchronize()
    for _ in range(5):
        for s, (pool, cfg, tab, q, out, ws) in zip(streams, made):
            attend_window(backend, pool, cfg, tab, q, out, ws, stream=s)
    torch.cuda.synchronize()
    for case, (_, cfg, _, _, out, _) in zip(cases, made):
        want, bound = T.attend(case, 0, 0, True, float(cfg.scale))
        assert ((out.double().cpu() - want).abs() <= bound).all()


def test_same_results_every_time(backend):
    """No atomics, fixed parts: the same call gives the same bits."""
    for q in (None, [130, 400]):
        case = T.Case(60, "fp8", "bf16", 8, 2, 128, [3000, 500], q)
        pool, *_ = upload(backend, case)
        cfg, tab = config(case, 0, True), tables(case)
        ws = torch.empty(max(256, window_workspace_size(cfg, tab, case.num_rows)), dtype=torch.uint8, device="cuda")
        outs = []
        for _ in range(3):
            out = torch.empty((case.num_rows, 8, 128), dtype=torch.bfloat16, device="cuda")
            attend_window(backend, pool, cfg, tab, case.q(case.qkv.cuda()), out, ws)
            outs.append(out)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])


def test_refusals(backend):
    """Arguments the host can see."""
    case = T.Case(70, "bf16", "bf16", 8, 2, 64, [100, 50], [10, 20])
    pool, *_ = upload(backend, case)
    cfg, tab = config(case, 0, True), tables(case)
    rows = case.qkv.cuda()
    q, k, v = case.q(rows), case.k(rows), case.v(rows)
    out = torch.empty((30, 8, 64), dtype=torch.bfloat16, device="cuda")

    def refused(call, *a, **kw):
        with pytest.raises(_lib.DhError) as e:
            call(*a, **kw)
        return e.value.status if hasattr(e.value, "status") else None

    n = window_workspace_size(cfg, tab, 30)
    assert n > 0
    ws = torch.empty(n, dtype=torch.uint8, device="cuda")
    attend_window(backend, pool, cfg, tab, q, out, ws)
    refused(attend_window, backend, pool, cfg, tab, q, out)                         # no workspace
    refused(attend_window, backend, pool, cfg, tab, q, out, ws[:-1])
    refused(attend_window, backend, pool, cfg, tab, q, out, torch.empty(n + 16, dtype=torch.uint8, device="cuda")[16:])
    refused(attend_window, backend, pool, cfg, tab, q.cpu(), out, ws)
    refused(attend_window, backend, pool, cfg, tab, q.float(), out, ws)
    refused(attend_window, backend, pool, cfg, tab, q, out[:29], ws)
    refused(attend_window, backend, pool, cfg, tab, q[:, :4], out[:, :4], ws)
    refused(attend_window, backend, pool, cfg, tab, q[:1].expand(30, 8, 64), out, ws)
    refused(attend_window, backend, pool, cfg, tab, q, out.transpose(0, 1).contiguous().transpose(0, 1), ws)
    refused(attend_window, backend, pool, cfg, tab, q, out, ws, -1)
    odd = torch.empty(30 * 513 + 1, dtype=torch.bfloat16, device="cuda")
    refused(attend_window, backend, pool, cfg, tab, odd.as_strided((30, 8, 64), (513, 64, 1)), out, ws)
    refused(attend_window, backend, pool, cfg, tab, odd.as_strided((30, 8, 64), (512, 64, 1), 1), out, ws)
    refused(attend_window, backend, pool, config(T.Case(1, "fp8", "bf16", 8, 2, 64, [1]), 0, True), tab, q, out, ws)
    refused(attend_window, backend, pool, config(T.Case(1, "bf16", "bf16", 8, 4, 64, [1]), 0, True), tab, q, out, ws)
    refused(pool.append_tokens, tab, k, v.float())
    refused(pool.append_tokens, tab, k.double(), v.double())
    refused(pool.append_tokens, tab, k[:, :1], v[:, :1])
    refused(pool.append_tokens, tab, k.cpu(), v.cpu())
    refused(pool.read_tokens, tab, k.cpu(), v.cpu())
    refused(pool.append_tokens, tab, k, v, torch.zeros(1, dtype=torch.int64, device="cuda"))
    refused(pool.append_tokens, tab, k, v, torch.zeros(1, dtype=torch.int32))
    one = TokenTables(tab.indices, tab.indptr, tab.kv_len)
    refused(pool.append_tokens, one, k[:1], v[:1])                                  # fewer rows than sequences
    refused(TokenTables, tab.indices, tab.indptr[:-1], tab.kv_len)
    refused(TokenTables, tab.indices.long(), tab.indptr, tab.kv_len)
    refused(TokenTables, tab.indices, tab.indptr.cpu(), tab.kv_len)
    refused(TokenTables, tab.indices, tab.indptr, tab.kv_len, tab.q_indptr[:2])
    refused(TokenTables, tab.indices, tab.indptr, tab.kv_len, tab.q_indptr, -1)
    refused(TokenTables, tab.indices, tab.indptr, tab.kv_len, tab.q_indptr, 1 << 31)
    # nothing to do is no error
    none = TokenTables(tab.indices, tab.indptr[:1].contiguous(), tab.kv_len[:0])
    attend_window(backend, pool, cfg, none, q[:0], out[:0])
    pool.append_tokens(none, k[:0], v[:0])
