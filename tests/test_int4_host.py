"""The 4-bit cache without a GPU: the format's sizes, argument checks, the engine's accounting, the plain packer."""
import ctypes

import pytest
import torch

from glake_b200 import ops
from glake_b200._lib import VT_ERR_INVALID, VT_ERR_UNSUPPORTED, VT_KV_BF16, VT_KV_FP8_E4M3, VT_KV_INT4, lib
from tests import kv_util as U

P = ctypes.c_void_p
BUF = (ctypes.c_ubyte * 4096)()
A16 = ctypes.addressof(BUF) + (-ctypes.addressof(BUF)) % 256


@pytest.mark.parametrize("kvh,want", [(1, 80), (2, 144), (3, 240), (4, 272), (6, 432), (8, 544), (12, 816), (16, 1088), (32, 2176)])
def test_row_bytes(kvh, want):
    assert ops.kv_row_bytes(kvh, 128, "int4") == want == U.row_bytes(kvh, "int4")
    assert ops.kv_row_bytes(kvh, 128) == kvh * 256 and ops.kv_row_bytes(kvh, 128, "fp8") == kvh * 128


def test_row_bytes_refusals():
    n = ctypes.c_size_t()
    assert lib.vt_kv_row_bytes(8, 64, VT_KV_INT4, ctypes.byref(n)) == VT_ERR_UNSUPPORTED
    assert lib.vt_kv_row_bytes(0, 128, VT_KV_INT4, ctypes.byref(n)) == VT_ERR_INVALID
    assert lib.vt_kv_row_bytes(8, 128, 7, ctypes.byref(n)) == VT_ERR_UNSUPPORTED
    assert lib.vt_kv_row_bytes(8, 128, VT_KV_INT4, None) == VT_ERR_INVALID


def test_plain_packer_round_trip():
    """A value is at most half a step away (inside the calibrated range; the step and the quotient are fp32 roundings: 7.5
    steps x 2 x 2^-24 more), and a second trip changes nothing."""
    g = torch.Generator().manual_seed(1)
    for kvh in (1, 2, 3, 8, 16):
        x = torch.randn(9, kvh, 128, generator=g).bfloat16()
        scale = x.float().abs().amax((0, 2)) / 448.0
        y = U.unpack4(U.pack4(x, scale), kvh, scale)
        _, s8 = U.quantise4(x, scale)
        step = (s8 * scale.double()[:, None]).repeat_interleave(32, -1).view(9, kvh, 128)
        assert bool(((y - x.double()).abs() <= step * (0.5 + 7.5 * 2.0 ** -23)).all())
        assert torch.equal(U.unpack4(U.pack4(y, scale), kvh, scale), U.unpack4(U.pack4(y, scale), kvh, scale))


def test_append_checks():
    def call(kv_dtype=VT_KV_INT4, ks=A16, d=128, max_len=1, stride=1024):
        return lib.vt_append(P(A16), P(A16), stride, stride, P(A16), P(A16), P(A16), P(A16), None, None, max_len, 1, 8, d, kv_dtype,
                             P(ks) if ks else None, P(A16), None)
    assert call(ks=None) == VT_ERR_INVALID
    assert call(kv_dtype=3) == VT_ERR_UNSUPPORTED
    assert call(d=64) == VT_ERR_UNSUPPORTED
    assert call(max_len=4) == VT_ERR_INVALID          # rows without lengths and starts
    assert call(stride=1000) == VT_ERR_INVALID


def test_dequant_checks():
    def call(kt=A16, ks=A16, start=A16, ko=A16, vo=A16, d=128, dt=VT_KV_INT4, batch=1, n=4):
        q = lambda x: P(x) if x else None  # noqa: E731
        return lib.vt_kv_dequant(q(kt), P(A16), P(A16), P(A16), q(start), batch, 8, d, n, dt, q(ks), P(A16), q(ko), q(vo), None)
    assert call(dt=VT_KV_BF16) == VT_ERR_UNSUPPORTED
    assert call(d=64) == VT_ERR_UNSUPPORTED
    assert call(start=None) == VT_ERR_INVALID
    assert call(ko=None, vo=None) == VT_ERR_INVALID
    assert call(ks=None) == VT_ERR_INVALID and call(kt=None) == VT_ERR_INVALID
    assert call(ko=A16 + 2) == VT_ERR_INVALID
    assert call(batch=-1) == VT_ERR_INVALID and call(n=-1) == VT_ERR_INVALID
    assert call(batch=0) == 0 and call(n=0) == 0 and call(dt=VT_KV_FP8_E4M3, batch=0) == 0


def test_decode_checks():
    def call(h=8, kvh=8, ks=A16, out=A16, out_stride=1024, splits=0, ws=1 << 30, q=A16):
        return lib.vt_decode_attn(P(out), out_stride, P(q), 1024, P(A16), P(A16), P(A16), P(A16), 2, h, kvh, 128, 64, 0.1, VT_KV_INT4,
                                  P(ks) if ks else None, P(A16), None, P(A16), ws, splits, None)
    assert call(ks=None) == VT_ERR_INVALID
    assert call(splits=4) == VT_ERR_UNSUPPORTED
    assert call(out=A16 + 4) == VT_ERR_INVALID and call(out_stride=1026) == VT_ERR_INVALID
    assert call(q=A16 + 8) == VT_ERR_INVALID
    assert call(ws=1000) == VT_ERR_INVALID
    assert call(h=3, kvh=1) == VT_ERR_UNSUPPORTED


def test_python_refusals():
    x = torch.zeros(4, 8, 128, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        ops.dequantize_ranges(x, x, 0, 0, 8, x, x, x, 4, "int4", x, x)
    with pytest.raises(RuntimeError, match="no output"):
        ops.dequantize_ranges(None, None, 0, 0, 8, x, x, x, 4, "int4", x, x)
    with pytest.raises(RuntimeError, match="int4"):
        ops.kv_row_bytes(8, 128, "int3")
    assert not ops.decode_tma_supported(32, 8, "int4") and ops.step_is_fused("int4")
