"""Weight accumulation and eviction without a GPU: argument checks, chunk accounting, the allocator's trim (mock driver)."""
import ctypes

import pytest
import torch

from glake_b200 import chunk_manager as CM, ops
from glake_b200._lib import VT_ERR_INVALID, VT_ERR_UNSUPPORTED, VT_KV_BF16, VT_KV_INT4, lib

P = ctypes.c_void_p
BUF = (ctypes.c_ubyte * 4096)()
A16 = ctypes.addressof(BUF) + (-ctypes.addressof(BUF)) % 256
q = lambda x: P(x) if x else None  # noqa: E731


def test_scored_step_checks():
    need = ctypes.c_size_t()
    assert lib.vt_decode_scored_workspace_bytes(2, 8, 128, 64, ctypes.byref(need)) == 0
    plain = ctypes.c_size_t()
    lib.vt_decode_attn_workspace_bytes(2, 8, 128, 64, ctypes.byref(plain))
    assert need.value >= plain.value + 2 * 8 * 64 * 4
    assert lib.vt_decode_scored_workspace_bytes(2, 8, 64, 64, ctypes.byref(need)) == VT_ERR_UNSUPPORTED
    assert lib.vt_decode_scored_workspace_bytes(2, 8, 128, 64, None) == VT_ERR_INVALID
    # batches beyond the schedule's table run in parts on the scratch of one part
    a, b = ctypes.c_size_t(), ctypes.c_size_t()
    lib.vt_decode_scored_workspace_bytes(1024, 8, 128, 64, ctypes.byref(a))
    lib.vt_decode_scored_workspace_bytes(5000, 8, 128, 64, ctypes.byref(b))
    assert a.value == b.value

    def call(scores=A16, key=None, value=None, off=None, rows=64, head=64, slot=512, ws=1 << 30, wsp=A16, d=128, h=8, dt=VT_KV_BF16,
             batch=2, n=64):
        return lib.vt_decode_step_scored(P(A16), 1024, P(A16), 1024, q(key), q(value), 1024, 1024, q(off), P(A16), P(A16), P(A16), P(A16),
                                         batch, h, 8, d, n, 0.1, dt, None, None, None, q(scores), slot, head, rows, q(wsp), ws, None)
    assert call(scores=None) == VT_ERR_INVALID
    assert call(rows=63) == VT_ERR_INVALID                       # a context longer than the scores' rows
    assert call(head=60) == VT_ERR_INVALID and call(slot=60) == VT_ERR_INVALID
    assert call(ws=1000) == VT_ERR_INVALID and call(wsp=None) == VT_ERR_INVALID
    assert call(wsp=A16 + 16) == VT_ERR_INVALID                  # alignment
    assert call(key=A16) == VT_ERR_INVALID                       # key without value
    assert call(key=A16, value=A16) == VT_ERR_INVALID            # and without offsets
    assert call(key=A16 + 2, value=A16, off=A16) == VT_ERR_INVALID
    assert call(d=64) == VT_ERR_UNSUPPORTED and call(h=9) == VT_ERR_UNSUPPORTED
    assert call(dt=VT_KV_INT4) == VT_ERR_INVALID                 # scales missing
    assert call(batch=0) == 0 and call(batch=-1) == VT_ERR_INVALID


def test_prompt_score_checks():
    need = ctypes.c_size_t()
    ok = lambda *a: lib.vt_prompt_scores_workspace_bytes(*a, ctypes.byref(need))  # noqa: E731
    assert ok(2, 8, 2, 128, 100, 16) == 0 and need.value >= 2 * 2 * 16 * 4 * 8
    assert ok(2, 8, 3, 128, 100, 16) == VT_ERR_UNSUPPORTED and ok(2, 8, 2, 64, 100, 16) == VT_ERR_UNSUPPORTED
    assert ok(2, 8, 2, 128, 100, 0) == VT_ERR_INVALID and ok(-1, 8, 2, 128, 100, 1) == VT_ERR_INVALID
    assert ok(1, 16, 1, 128, 100, 1025) == VT_ERR_UNSUPPORTED    # more rows than the kernel keeps

    def call(scores=A16, rows=64, query=A16, stride=1024, ws=1 << 30, wsp=A16, batch=2, n=64, window=4, table=A16):
        return lib.vt_prompt_scores(q(scores), 512, 64, rows, q(query), stride, q(table), P(A16), None, P(A16), P(A16), P(A16), batch, 8, 8,
                                    128, n, window, 0.1, q(wsp), ws, None)
    assert call(scores=None) == VT_ERR_INVALID and call(table=None) == VT_ERR_INVALID
    assert call(rows=32) == VT_ERR_INVALID
    assert call(query=A16 + 2) == VT_ERR_INVALID and call(stride=1023) == VT_ERR_INVALID and call(stride=512) == VT_ERR_INVALID
    assert call(ws=8) == VT_ERR_INVALID and call(wsp=A16 + 8) == VT_ERR_INVALID
    assert call(window=0) == VT_ERR_INVALID
    assert call(batch=0) == 0 and call(n=0) == 0


def test_evict_checks():
    need = ctypes.c_size_t()
    assert lib.vt_evict_workspace_bytes(2, 8, 100, VT_KV_BF16, ctypes.byref(need)) == 0 and need.value == 512 + 2 * 8 * 2 * 4
    assert lib.vt_evict_workspace_bytes(2, 8, 0, VT_KV_BF16, ctypes.byref(need)) == VT_ERR_INVALID
    assert lib.vt_evict_workspace_bytes(2, 8, 10, 9, ctypes.byref(need)) == VT_ERR_UNSUPPORTED

    def call(scores=A16, out=A16, rows=64, budget=10, sink=2, recent=3, kept=A16, ws=1 << 20, wsp=A16, dt=VT_KV_BF16, d=128, batch=2):
        return lib.vt_evict_rows(q(scores), q(out), 512, 64, rows, P(A16), P(A16), P(A16), P(A16), batch, 8, d, 64, budget, sink, recent, dt,
                                 q(kept), q(wsp), ws, None)
    assert call(scores=None) == VT_ERR_INVALID and call(out=None) == VT_ERR_INVALID and call(kept=None) == VT_ERR_INVALID
    assert call(budget=0) == VT_ERR_INVALID and call(sink=-1) == VT_ERR_INVALID and call(recent=-1) == VT_ERR_INVALID
    assert call(sink=6, recent=5) == VT_ERR_INVALID              # more fixed rows than the budget holds
    assert call(sink=2**31 - 1, recent=2**31 - 1) == VT_ERR_INVALID
    assert call(rows=63) == VT_ERR_INVALID
    assert call(ws=100) == VT_ERR_INVALID and call(wsp=A16 + 64) == VT_ERR_INVALID
    assert call(dt=5) == VT_ERR_UNSUPPORTED and call(d=64) == VT_ERR_UNSUPPORTED
    assert call(batch=0) == 0


def test_python_refusals():
    x = torch.zeros(2, 8, 64)
    i = torch.zeros(2, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.evict_rows(x, 0, 0, 8, i, i.int(), 64, 10)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.prompt_scores(x, x.bfloat16(), 0, 8, 0.1, i, i.int(), i.int(), i.int(), 64, 4)


def test_chunk_accounting_of_an_eviction():
    tok = 8 * 256                                       # bytes of a row: 1024 rows per chunk
    m = CM.ChunkSpaceManager(4, 100)
    seq = CM.SequenceChunks(tok)
    seq.append_tokens(5000)
    assert m.allocate(seq) and seq.logical_block_num == 10 and m.num_free == 90
    total = m.sum_all_blocks()
    m.evicted(seq, 1500)
    assert seq.logical_block_num == 4 and m.block_tables[seq.slot] == 4 and m.num_free == 96
    assert seq.reserve_size == 2 * CM.PHY_GRAN and m.sum_all_blocks() == total
    # grows again, one chunk pair at a time, when the reservation is used up
    grown = []
    for _ in range(448 + 1):                             # 2048 - 1500 - 100 rows of headroom are free
        seq.append_tokens(1)
        assert m.append_slots(seq, grown)
    assert grown == [seq.slot] and m.block_tables[seq.slot] == 6
    m.evicted(seq, 5999)                                 # never more than the slot holds
    assert m.block_tables[seq.slot] == 6 and m.sum_all_blocks() == total
    m.free(seq)
    assert m.num_free == 100


def test_chunk_accounting_keeps_the_cached_prefix():
    m = CM.ChunkSpaceManager(2, 40, cache_token=3, cache_seq=1)
    seq = CM.SequenceChunks(8 * 256)
    seq.append_tokens(4500)
    assert m.allocate(seq) and m.block_tables[seq.slot] == 10
    m.evicted(seq, 10)
    assert m.block_tables[seq.slot] == 6 and m.num_free == 34


def test_trim_on_the_mock_driver():
    from glake_b200 import vmmAllocator as A
    chunk = A.granularitySize
    lib.vt_use_mock_driver(1)
    try:
        assert A.init_physical_handle(64, 0)
        seg = A.KVcacheSegment(2, 8 * chunk, chunk, True)          # one chunk of every range is the cached prefix
        seg.ensure_mapped(6 * chunk)
        seg.set_used_size(5 * chunk + 10)
        free = A.showFreeBlocks()
        base = seg.getKeyDevicePtr(1)
        seg.trim(2 * chunk + 1)                                     # whole chunks behind the used bytes
        assert seg.actual_size == 3 * chunk and seg.used_size == 2 * chunk + 1 and A.showFreeBlocks() == free + 3 * 4
        assert seg.getKeyDevicePtr(1) == base
        seg.trim(100, 2 * chunk)                                    # a logical reservation is kept
        assert seg.actual_size == 2 * chunk and seg.used_size == 100
        seg.trim(10)                                                # and so is the cached prefix
        assert seg.actual_size == chunk and seg.used_size == 10
        seq = CM.SequenceChunks(1024)
        seq.append_tokens(5000)
        CM.apply_allocate(seq, seg)
        m = CM.ChunkSpaceManager(1, 30)
        assert m.allocate(seq)
        m.evicted(seq, 3)
        CM.apply_evicted(seq, 3, seg)
        assert seg.actual_size == chunk and seg.used_size == 3 * 1024
        seg.close()
        A.shutdown()
    finally:
        lib.vt_use_mock_driver(0)
