"""Pool.append_tokens and Pool.read_tokens against their plain 64-bit forms
(tests/_tokens.py): bit for bit."""
import math

import pytest
import torch

from tests import _tokens as T
from dendrite_amd import _lib
from dendrite_amd.backend import Pool, TokenTables

pytestmark = pytest.mark.gpu


def tables(case, max_kv_len=None):
    dev = lambda t: None if t is None else t.cuda()  # noqa: E731
    return TokenTables(dev(case.indices), dev(case.indptr), torch.tensor(case.kv_len, dtype=torch.int32).cuda(),
                       dev(case.q_indptr), max_kv_len=_lib.MAX_SEQ_LEN if max_kv_len is None else max_kv_len)


def upload(backend, case):
    pool = Pool(backend, case.data.shape[0], case.hkv, case.d, T.FORMATS[case.fmt])
    return pool, *T.pool_views(pool, case.data, case.scales)


def bits(t):
    t = t.detach().cpu().contiguous()
    return t.view({1: torch.uint8, 2: torch.int16, 4: torch.int32}[t.element_size()])


def same_codes(got, want):
    """Equal bits, any NaN equal to any other."""
    g, w = got.cpu(), want
    nan = w.float().isnan()
    assert torch.equal(g.float().isnan(), nan)
    assert torch.equal(bits(g)[~nan], bits(w)[~nan])


def check_append(backend, case, status=0, want=None):
    pool, data, scales = upload(backend, case)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    rows = case.qkv.cuda()
    for _ in range(2):                 # the second pass finds its own work
        pool.append_tokens(tables(case), case.k(rows), case.v(rows), st)
        torch.cuda.synchronize()
        d, s = want or T.append(case)
        same_codes(data, d)
        if s is not None:
            same_codes(scales, s) if s.dtype == torch.float32 else None
            assert s.dtype == torch.float32 or torch.equal(scales.cpu(), s)
    assert int(st) == status
    return pool, data, scales


SHAPES = {
    "mixed": ([1, 15, 16, 17, 40, 200, 33, 64], [1, 15, 16, 17, 7, 130, 0, 33]),
    "tails": ([21, 48, 5, 1], [1, 2, 5, 1]),
    "one": ([1], [1]),
    "long": ([1000], [999]),
}


@pytest.mark.parametrize("rows,fmt", [("f32", "f32"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "fp8"),
                                      ("f16", "mxfp8"), ("f32", "fp8"), ("f32", "mxfp8"), ("f32", "bf16"),
                                      ("f16", "bf16"), ("bf16", "f32")])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("shape", SHAPES)
def test_append(backend, rows, fmt, d, shape):
    kv, q = SHAPES[shape]
    check_append(backend, T.Case(5, fmt, rows, 2, 3, d, kv, q, row0=2, pad=3))


@pytest.mark.parametrize("fmt", ["bf16", "fp8", "mxfp8"])
def test_append_single_tokens(backend, fmt):
    """q_indptr None: one token a sequence, unused rows among them."""
    check_append(backend, T.Case(6, fmt, "bf16", 4, 2, 128, [1, 0, 16, 17, 31, 0, 100] + list(range(1, 90)), pad=4))


def test_append_many_sequences(backend):
    """More sequences than one search round tells apart (64), some empty."""
    q = [(7 * b) % 40 if b % 5 else 0 for b in range(300)]
    kv = [n + (3 * b) % 50 + 1 for b, n in enumerate(q)]
    check_append(backend, T.Case(7, "fp8", "bf16", 1, 1, 64, kv, q, row0=5, pad=9))


def test_append_block_scale_grows(backend):
    """A block's scale doubles as larger tokens arrive, its earlier codes with
    it, also far enough for them to become subnormal and zero."""
    case = T.Case(8, "fp8", "f32", 1, 4, 64, [20, 20, 20, 3], [1, 1, 1, 2], poison=False)
    x = case.qkv[:, 64:]
    x[0] *= 3.0
    x[1] *= 1000.0
    x[2] *= 1e30
    x[3:] *= 1e-25
    d, s = T.append(case)
    assert (s != case.scales).any()
    check_append(backend, case)


def test_append_zero_then_values(backend):
    """A block begun by zeros keeps full precision for what follows."""
    case = T.Case(9, "fp8", "f32", 1, 2, 64, [1], [1])
    case.qkv[:] = 0
    pool, data, scales = check_append(backend, case)
    p = int(case.tables[0][0])
    assert (scales[p].cpu() == T.FLOOR).all()
    case.data, case.scales = data.cpu(), scales.cpu()
    case.kv_len = [2]
    case.qkv[:] = torch.randn(case.qkv.shape, generator=torch.Generator().manual_seed(1))
    _, data, scales = check_append(backend, case)
    got = T.values(data.cpu(), scales.cpu(), "fp8")[p, 0, :, 1]
    want = case.k()[0].double()
    # normal codes: half a step of E4M3; below, half its least step
    assert ((got - want).abs() <= want.abs() * 2.0 ** -4 + scales[p, 0].cpu().double()[:, None] * 2.0 ** -10).all()


@pytest.mark.parametrize("fmt", ["fp8", "mxfp8", "f16"])
def test_append_nonfinite(backend, fmt):
    """NaN becomes a NaN code, infinities saturate, neither moves a scale."""
    case = T.Case(10, fmt, "f32", 1, 2, 128, [20, 37], [20, 3])
    case.k()[3, 0, 5] = math.nan
    case.k()[7, 1, 9] = math.inf
    case.v()[21, 0, 1] = -math.inf
    check_append(backend, case)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("fmt,rows", [("fp8", "bf16"), ("mxfp8", "f16"), ("bf16", "f32"), ("f32", "f32")])
def test_append_whole_pages_as_write_pages(backend, fmt, rows, d):
    """Whole pages written token by token equal dh_pool_write_pages_device's."""
    case = T.Case(11, fmt, rows, 1, 2, d, [48, 32], [48, 32])
    pool, data, scales = check_append(backend, case)
    other = Pool(backend, case.data.shape[0], 2, d, T.FORMATS[fmt])
    ids = torch.cat([t[:n // 16] for t, n in zip(case.tables, case.kv_len)])
    src = torch.stack([case.k(), case.v()], 1).unflatten(0, (-1, 16)).permute(0, 2, 3, 1, 4).contiguous()
    other.write_pages_device(ids.cuda(), src.cuda())
    torch.cuda.synchronize()
    for p in ids.tolist():
        a, b = pool.read_page(p), other.read_page(p)
        assert (a[0] == b[0]).all() and (a[1] is None or (a[1] == b[1]).all())


def test_append_bad_tables(backend):
    """Refused sequences and pages outside the pool are skipped and reported,
    their neighbours written."""
    case = T.Case(12, "fp8", "bf16", 1, 2, 64, [40, 40, 40, 40], [20, 20, 20, 20])
    case.tables[1][1] = case.data.shape[0]          # an id outside the pool
    case.tables[2][2] = -1                          # INVALID: skipped silently
    case.set_tables()
    check_append(backend, case, status=_lib.DH_EINVAL)
    case.tables[1][1] = -1
    case.set_tables()
    check_append(backend, case, status=0)
    # a sequence whose table is too short for its tokens writes nothing
    want = T.Case.__new__(T.Case)
    want.__dict__ = dict(case.__dict__)
    case.kv_len = [40, 200, 40, 40]
    want.q_len = [20, 0, 20, 20]
    check_append(backend, case, status=_lib.DH_EINVAL, want=T.append(want))


@pytest.mark.parametrize("rows,fmt", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "fp8"), ("f16", "mxfp8"), ("f32", "fp8"),
                                      ("f32", "mxfp8"), ("f16", "f16"), ("bf16", "f32")])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_read(backend, rows, fmt, d):
    """Every token's value, in f32 and then in the rows' type; zeros for INVALID pages; rows of
    nobody left alone."""
    kv, q = SHAPES["mixed"]
    case = T.Case(13, fmt, rows, 1, 3, d, kv, q, row0=2, pad=3)
    case.tables[5][4] = -1
    case.set_tables()
    pool, data, scales = upload(backend, case)
    st = torch.zeros(1, dtype=torch.int32, device="cuda")
    buf = torch.full((case.num_rows, 2, 4 * d), 7.0, dtype=T.TYPES[rows], device="cuda")
    k, v = (buf[:, i, :3 * d].view(case.num_rows, 3, d) for i in (0, 1))
    pool.read_tokens(tables(case), k, v, st)
    torch.cuda.synchronize()
    assert int(st) == 0
    want = torch.full((case.num_rows, 2, 4 * d), 7.0, dtype=T.TYPES[rows])
    vals = T.values(data.cpu(), None if scales is None else scales.cpu(), fmt)
    for b, (t, m) in enumerate(zip(case.kv_len, case.q_len)):
        a, c, ok = T.tokens_of(case, b, vals)
        r = case.first_row(b)
        for i, x in ((0, a), (1, c)):
            x = torch.where(ok[:, None, None], x, 0.0)[t - m:]
            want[r:r + m, i, :3 * d] = x.float().to(T.TYPES[rows]).reshape(m, 3 * d)
    same_codes(buf, want)
    case.tables[5][4] = case.data.shape[0] + 5
    case.set_tables()
    pool.read_tokens(tables(case), k, v, st)
    torch.cuda.synchronize()
    assert int(st) == _lib.DH_EINVAL
    same_codes(buf, want)
