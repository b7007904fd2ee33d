"""The attention-block operators write nothing outside what they are given: every
output and workspace of the C entry points lies inside a larger buffer whose
margins hold a pattern, on small and remainder sizes and on offsets that run
backwards or past the tensors.  The same calls run in the debug build, whose
index checks count none bad, and give the same bits."""
import ctypes
import subprocess
import sys
from pathlib import Path

import numpy as np
import pytest
import torch

from bevfusion_triton_b200 import load_native
from tests.test_attention_block_gpu import BF16, F16, F32, no_wait_gave_up  # noqa: F401

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parent.parent
DEBUG_LIB = ROOT / 'bevfusion_triton_b200' / 'debug' / 'libbfb_b200.so'
i64, f64, vp, size_t = ctypes.c_int64, ctypes.c_double, ctypes.c_void_p, ctypes.c_size_t
CODE = {F32: 0, F16: 1, BF16: 2}
MARGIN, PATTERN = 1 << 16, 0xA5


class Guarded:
    """`n` bytes between two margins."""

    def __init__(self, n):
        self.n = n
        self.raw = torch.full((n + 2 * MARGIN,), PATTERN, dtype=torch.uint8, device='cuda')
        self.inner = self.raw[MARGIN:MARGIN + n]
        self.ptr = vp(self.inner.data_ptr())

    def whole(self):
        return bool((self.raw[:MARGIN] == PATTERN).all()) and bool((self.raw[MARGIN + self.n:] == PATTERN).all())


def ptr(t):
    return vp(0) if t is None else vp(t.data_ptr())


def stream():
    return vp(torch.cuda.current_stream().cuda_stream)


def starts(lens):
    return [0] + [int(x) for x in np.cumsum(lens)]


# name: dtype, heads, kv_heads, dim, query offsets, key offsets, kv_lengths, causal; rows of q and k where the offsets do
# not end at the last
ATTENTION = {
    'one': (F16, 2, 1, 64, [0, 1], [0, 1], None, True),
    'nothing': (BF16, 2, 2, 64, [0, 0], [0, 0], None, False),
    'no keys': (F16, 2, 2, 128, [0, 70], [0, 0], None, True),
    'tiles of 64': (BF16, 3, 3, 40, starts([129, 1, 0, 255]), starts([129, 1, 0, 255]), None, True),
    'tiles of 128': (F16, 4, 2, 120, starts([127, 300, 2]), starts([64, 300, 130]), None, True),
    'many': (BF16, 2, 1, 64, starts([45] * 70), starts([45] * 70), None, False),
    'streams': (BF16, 8, 2, 128, starts([1] * 5), starts([700] * 5), [700, 0, 1, 63, 650], True),
    'streams, odd heads': (F16, 21, 3, 72, starts([2, 0, 1]), starts([100, 5, 2000]), None, False),
    'rows behind': (F16, 2, 2, 64, [0, 100, 150], [0, 100, 150], None, True, 220, 190),
    'rows before': (BF16, 2, 2, 128, [30, 100, 200], [64, 100, 300], None, False, 200, 300),
    'backwards': (F16, 2, 2, 64, [0, 500, 200, 900], [0, 500, 200, 900], [-3, 1 << 30, 9], True, 300, 300),
    'negative': (BF16, 2, 1, 128, [-5, 100, 50, 300], [-5, 100, 50, 300], [-3, 1 << 30, 9], True, 300, 300),
    'down': (F16, 2, 2, 64, [200, 100, 0, 0], [300, 10, 0, -7], None, False, 300, 300),
    'extremes': (BF16, 4, 2, 64, [0, 2 ** 31 - 1, -2 ** 31, 300], [0, 2 ** 31 - 1, -2 ** 31, 300], None, True, 300, 300),
    'backwards, few rows': (F16, 4, 1, 128, [3, 1, 4, 0, 2], [90, 0, 300, 10, 1 << 30], [5, 400, -1, 7], False, 4, 300),
}


def attention(lib, name):
    """Forward and backward of one case; whether every margin is whole, and the outputs."""
    dtype, heads, kv, dim, cu_q, cu_k, lengths, causal, *rows = ATTENTION[name]
    nq, nk = rows or (cu_q[-1], cu_k[-1])
    g = torch.Generator(device='cuda').manual_seed(len(name))
    q, dout = (torch.randn((nq, heads, dim), generator=g, device='cuda').to(dtype) for _ in range(2))
    k, v = (torch.randn((nk, kv, dim), generator=g, device='cuda').to(dtype) for _ in range(2))
    dlse = torch.randn((heads, nq), generator=g, device='cuda')
    ints = lambda x: None if x is None else torch.tensor(x, dtype=torch.int32, device='cuda')  # noqa: E731
    cu_q, cu_k, lengths = ints(cu_q), ints(cu_k), ints(lengths)
    strides = (i64 * 6)(heads * dim, dim, kv * dim, dim, kv * dim, dim)
    sizes = [i64(x) for x in (nq, nk, heads, kv, dim, cu_q.numel() - 1)]
    spaces = []
    for backward in (0, 1):
        n = size_t()
        assert lib.bfb_packed_attention_workspace_size(*sizes, backward, ctypes.byref(n)) == 0
        spaces.append(Guarded(n.value))
    out, lse, dq, dk, dv = (Guarded(n) for n in (2 * q.numel(), 4 * heads * nq, 2 * q.numel(), 2 * k.numel(),
                                                 2 * k.numel()))
    common = [CODE[dtype], *sizes, ptr(cu_q), ptr(cu_k), ptr(lengths), int(causal), f64(dim ** -0.5)]
    assert lib.bfb_packed_attention(ptr(q), ptr(k), ptr(v), strides, *common, out.ptr, lse.ptr, spaces[0].ptr,
                                    size_t(spaces[0].n), stream()) == 0
    assert lib.bfb_packed_attention_backward(
        ptr(dout), ptr(dlse), ptr(q), ptr(k), ptr(v), strides, out.ptr, lse.ptr, *common, dq.ptr, dk.ptr, dv.ptr,
        spaces[1].ptr, size_t(spaces[1].n), stream()) == 0
    torch.cuda.synchronize()
    return all(x.whole() for x in (out, lse, dq, dk, dv, *spaces)), [x.inner for x in (out, lse, dq, dk, dv)]


# dtype, tokens, heads, kv_heads, dim, sections, interleaved
ROTARY = {'one token': (BF16, 1, 1, 1, 64, (32,), 0), 'many tokens': (BF16, 3001, 3, 2, 128, (16, 24, 24), 0),
          'many heads': (F32, 5, 90, 7, 256, (100, 20), 1), 'narrow': (F16, 77, 5, 1, 24, (8,), 0),
          'fp32': (F32, 1000, 4, 4, 80, (0, 16, 16), 0)}


def rotary(lib, name):
    dtype, n, heads, kv, dim, sections, inter = ROTARY[name]
    g = torch.Generator(device='cuda').manual_seed(n)
    q, gq = (torch.randn((n, heads, dim), generator=g, device='cuda').to(dtype) for _ in range(2))
    k, gk = (torch.randn((n, kv, dim), generator=g, device='cuda').to(dtype) for _ in range(2))
    pos = torch.randint(0, 1000, (n, len(sections)), generator=g, device='cuda', dtype=torch.int32)
    freq, w = torch.rand(sum(sections), generator=g, device='cuda'), torch.rand(dim, generator=g, device='cuda')
    size = q.element_size()
    space = size_t()
    assert lib.bfb_qk_norm_rotary_backward_workspace_size(i64(dim), ctypes.byref(space)) == 0
    qo, ko, dq, dk, dqw, dkw, ws = (Guarded(x) for x in (size * q.numel(), size * k.numel(), size * q.numel(),
                                                         size * k.numel(), 4 * dim, 4 * dim, space.value))
    place = [i64(heads * dim), i64(dim), i64(kv * dim), i64(dim), CODE[dtype], i64(n), i64(heads), i64(kv), i64(dim),
             i64(2 * sum(sections)), ptr(pos), 0, i64(pos.stride(0)), i64(pos.stride(1)), ptr(freq), 0,
             i64(len(sections)), (i64 * len(sections))(*sections), ptr(w), ptr(w), f64(1e-6), inter]
    assert lib.bfb_qk_norm_rotary(ptr(q), ptr(k), *place, qo.ptr, ko.ptr, stream()) == 0
    assert lib.bfb_qk_norm_rotary_backward(ptr(gq), ptr(gk), ptr(q), ptr(k), *place, dq.ptr, dk.ptr, dqw.ptr, dkw.ptr,
                                           ws.ptr, space, stream()) == 0
    torch.cuda.synchronize()
    outs = [qo, ko, dq, dk, dqw, dkw]
    return all(x.whole() for x in (*outs, ws)), [x.inner for x in outs]


DROPOUT = {f'{n} {code}': (n, code) for n in (1, 7, 8, 8193) for code in (F32, F16, BF16)}


def dropout(lib, name):
    n, dtype = DROPOUT[name]
    x, seed = torch.ones(n, device='cuda').to(dtype), torch.tensor([5, 6], device='cuda')
    out = Guarded(n * x.element_size())
    assert lib.bfb_residual_dropout(ptr(x), ptr(x), CODE[dtype], i64(n), ptr(seed), f64(0.4), out.ptr, stream()) == 0
    torch.cuda.synchronize()
    return out.whole(), [out.inner]


CALLS = [(f, name) for f, names in ((attention, ATTENTION), (rotary, ROTARY), (dropout, DROPOUT)) for name in names]


@pytest.mark.parametrize('call,name', CALLS, ids=[f'{f.__name__} {n}' for f, n in CALLS])
def test_nothing_outside_is_written(cuda, call, name):
    whole, outs = call(load_native(), name)
    assert whole
    if name not in ('backwards', 'negative', 'down', 'extremes', 'backwards, few rows'):
        # every value of an output was written: none is left as the pattern
        for x in outs:
            width = torch.int32 if x.numel() % 4 == 0 else torch.int16
            left = int.from_bytes([PATTERN] * (4 if x.numel() % 4 == 0 else 2), 'little', signed=True)
            assert not bool((x.view(width) == left).any())


def test_debug_build_agrees(cuda, tmp_path):
    """All of the calls in the debug build: no index out of its range, and the bits of the release build."""
    if not DEBUG_LIB.exists():
        pytest.skip('debug build missing (python -m bevfusion_triton_b200._build --debug-checks)')
    script = ('import sys; sys.path.insert(0, sys.argv[1])\n'
              'from tests.test_attention_bounds_gpu import debug_run\n'
              'debug_run(sys.argv[2], sys.argv[3])')
    r = subprocess.run([sys.executable, '-c', script, str(ROOT), str(DEBUG_LIB), str(tmp_path / 'outs.pt')],
                       capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and r.stdout.strip().endswith('ok'), r.stdout + r.stderr
    theirs = torch.load(tmp_path / 'outs.pt')
    for (call, name), outs in zip(CALLS, theirs):
        if name in ('backwards', 'negative', 'extremes', 'down', 'backwards, few rows'):
            continue  # rows that two sequences claim are written by both
        for a, b in zip(call(load_native(), name)[1], outs):
            assert torch.equal(a.cpu(), b), name


def debug_run(path, to):
    lib, count = ctypes.CDLL(path), ctypes.c_uint64()
    assert lib.bfb_debug_checks_enabled() == 1 and lib.bfb_debug_violations(ctypes.byref(count), 1) == 0
    found = []
    for call, name in CALLS:
        whole, outs = call(lib, name)
        assert whole, name
        assert lib.bfb_debug_violations(ctypes.byref(count), 1) == 0 and count.value == 0, (name, count.value)
        found.append([x.cpu() for x in outs])
    assert lib.bfb_attention_timeouts(ctypes.byref(count), 1) == 0 and count.value == 0
    torch.save(found, to)
    print('ok')
