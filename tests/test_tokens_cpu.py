"""The token operators without a GPU: the plain forms the GPU tests compare
with against the decode oracle, workspace sizes, and refusals that need no
device."""
import copy
import ctypes as C

import numpy as np
import pytest
import torch

from dendrite_amd import _lib
from dendrite_amd.backend import AttentionConfig, TokenTables
from tests import _tokens as T


@pytest.mark.parametrize("tiled", [True, False])
def test_plain_attention_is_the_oracles(tiled):
    """No window, whole pages: the plain form agrees with oracle.decode."""
    import oracle
    case = T.Case(1, "f32", "f32", 6, 2, 64, [48, 16, 0, 33], None, spare=0)
    out, bound = T.attend(case, 0, 0, tiled, 0.125)
    n = case.data.shape[0]
    raw = case.data.nan_to_num(0.0).numpy().view(np.uint8).reshape(n, -1)
    pv = oracle.PoolView(np.arange(n, dtype=np.uint32), raw, None, n, _lib.KV_F32, 2, 64)
    last = np.array([(t - 1) % 16 + 1 if t else 16 for t in case.kv_len], np.int32)
    ref = oracle.decode(pv, case.q().contiguous().numpy(), _lib.DTYPE_F32, 6, 0.125,
                        _lib.GQA_TILED if tiled else _lib.GQA_INTERLEAVED, case.indptr.numpy().astype(np.uint32),
                        case.indices.numpy().astype(np.uint32), last)
    assert np.abs(out.numpy() - ref).max() < 1e-5


def test_plain_window_by_hand():
    """Which tokens the window and the sinks leave in sight, from one-hot V."""
    case = T.Case(2, "f32", "f32", 1, 1, 64, [40], [3], spare=0, poison=False)
    case.data[:] = 0
    for t in range(40):
        case.data[case.tables[0][t // 16], 1, 0, t % 16, t] = 1.0
    out, _ = T.attend(case, 7, 2, True, 1.0)
    for i, p in enumerate((37, 38, 39)):
        seen = torch.nonzero(out[i, 0]).flatten().tolist()
        assert seen == [0, 1] + list(range(p - 6, p + 1))


def _tables(rows, batch, max_kv_len, single):
    t = _lib.dh_token_tables()
    t.batch_size, t.rows, t.max_kv_len, t.num_indices = batch, rows, max_kv_len, 1 << 20
    t.q_indptr = None if single else 8
    return t


def test_workspace_size():
    """None where the batch fills the chip; room for every row's parts where
    one sequence has to be split; none for an empty call."""
    L = _lib.lib()
    cfg = AttentionConfig(32, 8, 128).to_c()
    size = lambda *a, sinks=0: L.dh_window_workspace_size(C.byref(cfg), C.byref(_tables(*a)), sinks)  # noqa: E731
    assert size(0, 0, 4096, True) == 0 and size(256, 256, 4096, True) == 0
    one = size(1, 1, 131072, True)
    assert one > 0 and one % 256 == 0
    assert size(1, 1, 64, True) == 0
    assert size(4096, 1, 131072, False) > 0
    small = one
    cfg.sliding_window = 128
    assert size(1, 1, 131072, True) < small
    assert L.dh_window_workspace_size(None, C.byref(_tables(1, 1, 1, True)), 0) == 0
    assert L.dh_window_workspace_size(C.byref(cfg), None, 0) == 0


def test_configs_are_copied_after_use():
    cfg = AttentionConfig(32, 8, 128)
    first = cfg._ref()
    assert cfg._ref() is first
    other = copy.deepcopy(cfg)
    other.sliding_window = 5
    assert other._ref()._obj.sliding_window == 5 and cfg._ref() is first and first._obj.sliding_window == 0
    cfg.scale = 2.0
    assert cfg._ref()._obj.scale == 2.0


def test_null_handles_are_refused():
    L = _lib.lib()
    cfg, t = AttentionConfig(32, 8, 128).to_c(), _tables(1, 1, 64, True)
    assert L.dh_pool_append_tokens(None, C.byref(t), None, None, 0, 0, 1, None, None) == _lib.DH_EINVAL
    assert L.dh_pool_read_tokens(None, C.byref(t), None, None, 0, 0, 1, None, None) == _lib.DH_EINVAL
    assert L.dh_attend_window(None, None, C.byref(cfg), 0, C.byref(t), None, 0, None, 0, None, 0, None,
                              None) == _lib.DH_EINVAL
    assert "NULL" in _lib.last_error()


def test_tables_must_be_on_the_device():
    i = torch.zeros(4, dtype=torch.int32)
    with pytest.raises(_lib.DhError, match="device vector"):
        TokenTables(i, i[:3], i[:2])
