"""CPU checks of the attention-block operators: refusals of the Python
functions and of the C ABI, shapes under fake tensors, the oracle's generator
against its published vectors."""
import ctypes

import numpy as np
import pytest
import torch

from bevfusion_triton_b200 import load_native
from bevfusion_triton_b200._lib import ops
from bevfusion_triton_b200.ops.spconv import (SparseSelfAttention, packed_attention, qk_norm_rotary, residual_dropout,
                                              sample_offsets)
from tests import attention_oracle as oracle
from tests.test_fake_ops import fake_mode

i64, f64, vp = ctypes.c_int64, ctypes.c_double, ctypes.c_void_p
OK, BAD, DTYPE, WORKSPACE, LARGE = 0, -1, -2, -3, -4
P = 1 << 20  # an aligned address that no refused call reads


def test_philox_published_vectors():
    """Known answers of Philox4x32-10 (Random123): counter and key all zeros, all ones."""
    assert [hex(int(v)) for v in oracle.philox(4, 0, 0)] == ['0x6627e8d5', '0xe169c58d', '0xbc57ac4c', '0x9b00dbd8']


def test_oracle_rotary_is_a_rotation():
    g = torch.Generator().manual_seed(0)
    x = torch.randn((7, 2, 32), generator=g, dtype=torch.float64)
    pos = torch.randint(0, 1000, (7, 2), generator=g)
    freq = 10000.0 ** (-torch.arange(16, dtype=torch.float64) / 16)
    for inter in (False, True):
        y = oracle.rotary(x, None, pos, freq, (6, 10), 0.0, inter)
        torch.testing.assert_close(y.norm(dim=-1), x.norm(dim=-1))
        zero = oracle.rotary(x, None, 0 * pos, freq, (6, 10), 0.0, inter)
        torch.testing.assert_close(zero, x)


def test_cpu_tensors_are_refused():
    q = torch.zeros(4, 2, 16, dtype=torch.float16)
    cu = torch.tensor([0, 4], dtype=torch.int32)
    with pytest.raises(RuntimeError):
        packed_attention(q, q, q, cu)
    with pytest.raises(RuntimeError):
        qk_norm_rotary(q, q, torch.zeros(4, 1, dtype=torch.int32), torch.ones(8), (8,))
    with pytest.raises(RuntimeError):
        residual_dropout(q, None, 0.5, torch.zeros(2, dtype=torch.int64))


def _forward(lib, dtype=2, tq=8, tk=8, heads=4, kv=2, dim=64, seqs=1, q=P, out=P, lse=P, cu=P, strides=None,
             scale=1.0):
    s = (i64 * 6)(*(strides or [heads * dim, dim, kv * dim, dim, kv * dim, dim]))
    return lib.bfb_packed_attention(vp(q), vp(P), vp(P), s, dtype, i64(tq), i64(tk), i64(heads), i64(kv), i64(dim),
                                    i64(seqs), vp(cu), vp(cu), vp(0), 0, f64(scale), vp(out), vp(lse), vp(0),
                                    ctypes.c_size_t(0), vp(0))


@pytest.mark.parametrize('kw,code', [
    ({'dtype': 0}, DTYPE), ({'dtype': 7}, DTYPE), ({'heads': 3}, BAD), ({'heads': 0}, BAD), ({'kv': 0}, BAD),
    ({'dim': 136}, BAD), ({'dim': 4}, BAD), ({'dim': 60}, BAD), ({'dim': 0}, BAD), ({'tq': -1}, BAD),
    ({'tk': -1}, BAD), ({'seqs': -1}, BAD), ({'q': 0}, BAD), ({'out': 0}, BAD), ({'lse': 0}, BAD), ({'cu': 0}, BAD),
    ({'q': P + 8}, BAD), ({'out': P + 8}, BAD), ({'strides': [257, 64, 128, 64, 128, 64]}, BAD),
    ({'strides': [256, 64, 128, 60, 128, 64]}, BAD), ({'scale': float('nan')}, BAD), ({'scale': float('inf')}, BAD),
    ({'tq': 1 << 31}, LARGE), ({'tk': 1 << 31}, LARGE), ({'heads': 1 << 20, 'kv': 1 << 20}, LARGE),
    ({'tq': 0}, OK)])
def test_cabi_attention_refusals(kw, code):
    assert _forward(load_native(), **kw) == code


def test_cabi_attention_backward_refusals():
    lib = load_native()
    s = (i64 * 6)(256, 64, 128, 64, 128, 64)

    def call(dout=P, dq=P, dk=P, dv=P, ws=P, ws_bytes=1 << 20, dtype=1):
        return lib.bfb_packed_attention_backward(
            vp(dout), vp(0), vp(P), vp(P), vp(P), s, vp(P), vp(P), dtype, i64(8), i64(8), i64(4), i64(2), i64(64),
            i64(1), vp(P), vp(P), vp(0), 0, f64(1.0), vp(dq), vp(dk), vp(dv), vp(ws), ctypes.c_size_t(ws_bytes), vp(0))

    assert call(dtype=0) == DTYPE
    for name in ('dout', 'dq', 'dk', 'dv'):
        assert call(**{name: 0}) == BAD and call(**{name: P + 4}) == BAD
    assert call(ws=0) == WORKSPACE and call(ws_bytes=16) == WORKSPACE
    n = ctypes.c_size_t()
    assert lib.bfb_packed_attention_workspace_size(i64(8), i64(8), i64(4), i64(2), i64(64), i64(1), 1,
                                                   ctypes.byref(n)) == OK
    assert n.value >= 8 * 4 * 4
    assert lib.bfb_packed_attention_workspace_size(i64(-8), i64(8), i64(4), i64(2), i64(64), i64(1), 1,
                                                   ctypes.byref(n)) == BAD


def _rotary(lib, dtype=2, tokens=4, heads=4, kv=2, dim=64, rotated=64, sections=(16, 16), inter=0, q=P, out=P,
            pos_type=0, row=256, eps=1e-6, qw=0):
    s = (i64 * max(1, len(sections)))(*sections)
    return lib.bfb_qk_norm_rotary(vp(q), vp(P), i64(row), i64(64), i64(128), i64(64), dtype, i64(tokens), i64(heads),
                                  i64(kv), i64(dim), i64(rotated), vp(P), pos_type, i64(2), i64(1), vp(P), 0,
                                  i64(len(sections)), s, vp(qw), vp(0), f64(eps), inter, vp(out), vp(P), vp(0))


@pytest.mark.parametrize('kw,code', [
    ({'dtype': 5}, DTYPE), ({'tokens': -1}, BAD), ({'heads': 0}, BAD), ({'kv': 0}, BAD), ({'dim': 264}, BAD),
    ({'dim': 60}, BAD), ({'rotated': 72}, BAD), ({'rotated': 0, 'sections': (0,)}, BAD),
    ({'rotated': 24, 'sections': (6, 6)}, BAD), ({'sections': (16, 15)}, BAD), ({'sections': (40, -8)}, BAD),
    ({'sections': ()}, BAD), ({'sections': (4,) * 9}, BAD), ({'q': 0}, BAD), ({'q': P + 2}, BAD), ({'out': 0}, BAD),
    ({'pos_type': 3}, DTYPE), ({'row': 257}, BAD), ({'eps': -1.0}, BAD), ({'eps': float('nan')}, BAD),
    ({'qw': P + 4}, BAD), ({'heads': 5000}, LARGE), ({'tokens': 0}, OK)])
def test_cabi_rotary_refusals(kw, code):
    assert _rotary(load_native(), **kw) == code


@pytest.mark.parametrize('kw,code', [({'p': -0.1}, BAD), ({'p': 1.5}, BAD), ({'p': float('nan')}, BAD),
                                     ({'dtype': 3}, DTYPE), ({'n': -1}, BAD), ({'x': 0}, BAD), ({'n': 0}, OK)])
def test_cabi_dropout_refusals(kw, code):
    a = {'x': P, 'dtype': 0, 'n': 8, 'p': 0.5} | kw
    assert load_native().bfb_residual_dropout(vp(a['x']), vp(0), a['dtype'], i64(a['n']), vp(P), f64(a['p']), vp(P),
                                              vp(0)) == code


def test_ops_trace_under_fake_tensors():
    load_native()
    O = ops()
    with fake_mode():
        q = torch.empty(10, 4, 32, dtype=torch.float16, device='cuda')
        k = torch.empty(12, 2, 32, dtype=torch.float16, device='cuda')
        cu = torch.empty(3, dtype=torch.int32, device='cuda')
        out, lse = O.packed_attention(q, k, k, cu, cu, None, True, 0.5)
        assert out.shape == q.shape and out.dtype == q.dtype and lse.shape == (4, 10) and lse.dtype == torch.float32
        dq, dk, dv = O.packed_attention_backward(out, None, q, k, k, out, lse, cu, cu, None, True, 0.5)
        assert dq.shape == q.shape and dk.shape == k.shape and dv.shape == k.shape
        pos, freq, w = torch.empty(10, 3, device='cuda'), torch.empty(16, device='cuda'), torch.empty(32, device='cuda')
        a, b = O.qk_norm_rotary(q, q[:, :2], pos, freq, [4, 6, 6], w, None, 1e-6, False)
        assert a.shape == q.shape and b.shape == (10, 2, 32) and b.is_contiguous()
        g = O.qk_norm_rotary_backward(a, b, q, q[:, :2], pos, freq, [4, 6, 6], w, None, 1e-6, False)
        assert g[2].shape == (32,) and g[3].shape == (0,) and g[2].dtype == torch.float32
        assert O.residual_dropout(q.transpose(0, 1), None, 0.5, cu).is_contiguous()
    for name in ('packed_attention', 'qk_norm_rotary', 'residual_dropout'):
        assert torch._C._dispatch_has_kernel_for_dispatch_key('bfb_b200::' + name, 'Autograd')


def test_sample_offsets():
    rows = torch.tensor([[0, 5], [0, 1], [2, 3], [2, 2], [2, 9]], dtype=torch.int32)
    assert sample_offsets(rows, 4).tolist() == [0, 2, 2, 5, 5] and sample_offsets(rows, 4).dtype == torch.int32
    assert sample_offsets(rows[:0], 2).tolist() == [0, 0, 0]


@pytest.mark.parametrize('args', [(64, 3), (64, 4, 3), (64, 8), (512, 2)])
def test_module_refuses_head_layouts(args):
    with pytest.raises(ValueError):
        SparseSelfAttention(*args)
    with pytest.raises(ValueError):
        SparseSelfAttention(64, 4, dropout=1.5)
