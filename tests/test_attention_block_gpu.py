"""packed_attention, qk_norm_rotary, residual_dropout and SparseSelfAttention
on the GPU against the 64-bit oracle, within tolerances counted from the
roundings (tests/attention_oracle.py)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from bevfusion_triton_b200 import load_native
from bevfusion_triton_b200.ops.spconv import (SparseConvTensor, SparseSelfAttention, SparseSequential,
                                              packed_attention, qk_norm_rotary, residual_dropout)
from tests import attention_oracle as oracle

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def no_wait_gave_up():
    yield
    if torch.cuda.is_available():
        count = ctypes.c_uint64()
        assert load_native().bfb_attention_timeouts(ctypes.byref(count), 1) == 0 and count.value == 0


F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def offsets(lens):
    return torch.tensor([0] + list(np.cumsum(lens)), dtype=torch.int32, device='cuda')


def make(dtype, heads, kv, dim, lens_q, lens_k, spare_q=0, spare_k=0, seed=0):
    g = torch.Generator(device='cuda').manual_seed(seed)
    new = lambda n, h: torch.randn((n, h, dim), generator=g, device='cuda')  # noqa: E731
    nq, nk = sum(lens_q) + spare_q, sum(lens_k) + spare_k
    return ((1.5 * new(nq, heads)).to(dtype), new(nk, kv).to(dtype), new(nk, kv).to(dtype), new(nq, heads).to(dtype),
            torch.randn((heads, nq), generator=g, device='cuda'))


def both(dtype, heads, kv, dim, lens_q, lens_k=None, causal=False, spare=0, seed=0, scale=None):
    """Forward and backward of one case against the oracle."""
    lens_k = lens_q if lens_k is None else lens_k
    q, k, v, g, gl = make(dtype, heads, kv, dim, lens_q, lens_k, spare, spare, seed)
    if spare:  # rows of no sequence hold whatever they hold
        for t in (q, k, v, g):
            t[-spare:] = math.nan
        gl[:, -spare:] = math.nan
    scale = dim ** -0.5 if scale is None else scale
    for t in (q, k, v):
        t.requires_grad_(True)
    out, lse = packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=causal, scale=scale, return_lse=True)
    # queries that see no key have no log-sum-exp to differentiate
    gl = torch.where(lse.detach() == -math.inf, 0.0, gl)
    got = (out.detach(), lse.detach(), *torch.autograd.grad((out, lse), (q, k, v), (g, gl)))
    value, tol = oracle.attention(q.detach(), k.detach(), v.detach(), lens_q, lens_k, causal, scale, dout=g, dlse=gl)
    for name, x in zip(('out', 'lse', 'dq', 'dk', 'dv'), got):
        oracle.check(x, value[name], tol[name], name)


@pytest.mark.parametrize('lens', [[1], [0], [], [2, 0, 0, 3], [16], [64], [127], [128], [129], [255, 1, 257],
                                  [300, 20, 513], [7] * 40])
@pytest.mark.parametrize('causal', [False, True])
def test_lengths(cuda, lens, causal):
    both(BF16, 2, 2, 64, lens, causal=causal, seed=len(lens))


@pytest.mark.parametrize('dim', [8, 16, 24, 40, 64, 72, 80, 96, 120, 128])
@pytest.mark.parametrize('dtype', [F16, BF16])
def test_dims(cuda, dim, dtype):
    both(dtype, 2, 1, dim, [150, 3, 200], causal=True, seed=dim)


@pytest.mark.parametrize('heads,kv', [(1, 1), (3, 3), (8, 1), (6, 2), (7, 1), (20, 4)])
@pytest.mark.parametrize('causal', [False, True])
def test_heads(cuda, heads, kv, causal):
    both(F16, heads, kv, 32, [140, 9, 260], causal=causal, seed=heads)


@pytest.mark.parametrize('lens_q,lens_k', [([1, 1, 1], [5, 900, 130]), ([4, 0, 2], [0, 7, 2000]), ([200], [50]),
                                           ([130, 1, 300], [129, 300, 1]), ([3], [3000]), ([600, 5], [5, 600]),
                                           ([1], [1]), ([0, 3], [10, 0])])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('dim', [48, 128])
def test_queries_and_keys_of_different_lengths(cuda, lens_q, lens_k, causal, dim):
    """Fewer queries than keys (tokens against a cache) and more (causal: the first see nothing)."""
    both(BF16, 4, 2, dim, lens_q, lens_k, causal=causal, seed=len(lens_q) + dim)


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('lens', [[5], [200, 77], [128], [256, 130]])
def test_rows_of_no_sequence(cuda, causal, lens):
    """Rows behind the last sequence hold NaN: nothing of them shows, and they get zeros."""
    both(F16, 4, 2, 64, lens, causal=causal, spare=70, seed=3)
    both(BF16, 2, 2, 128, lens, causal=causal, spare=1, seed=4)


@pytest.mark.parametrize('lens', [[1, 1, 1, 1], [40, 3, 0, 260]])
@pytest.mark.parametrize('causal', [False, True])
def test_cache_with_room(cuda, lens, causal):
    """kv_lengths below the room of each sequence; the rest of the room holds NaN."""
    used, room, dim = [0, 1, 300, 512], 512, 128
    q, k, v, g, _ = make(BF16, 8, 2, dim, lens, [room] * 4, seed=9)
    for n, used_n in enumerate(used):
        k[n * room + used_n:(n + 1) * room] = math.nan
        v[n * room + used_n:(n + 1) * room] = math.inf
    for t in (q, k, v):
        t.requires_grad_(True)
    for lengths in (torch.tensor(used, device='cuda'), torch.tensor(used, dtype=torch.int32, device='cuda')):
        out, lse = packed_attention(q, k, v, offsets(lens), offsets([room] * 4), kv_lengths=lengths, causal=causal,
                                    return_lse=True)
    got = (out.detach(), lse.detach(), *torch.autograd.grad(out, (q, k, v), g))
    clean = [torch.where(torch.isfinite(t), t, 0.0).detach() for t in (k, v)]
    value, tol = oracle.attention(q.detach(), *clean, lens, used, causal, dim ** -0.5, [room] * 4, dout=g)
    for name, x in zip(('out', 'lse', 'dq', 'dk', 'dv'), got):
        oracle.check(x, value[name], tol[name], name)


def test_large_and_small_scores(cuda):
    """Scores of +-40 about a far mean: the running maximum moves; and a negative and a zero scale."""
    both(BF16, 2, 2, 64, [400], causal=True, scale=1.0)
    both(F16, 2, 2, 64, [400], causal=False, scale=-0.7)
    both(F16, 2, 2, 64, [200, 31], causal=False, scale=0.0)


@pytest.mark.parametrize('dim', [64, 128])
def test_rising_maximum(cuda, dim):
    """Each key scores above the ones before it, by more than any threshold: every block rescales."""
    n = 700
    q, k, v, g, _ = make(BF16, 1, 1, dim, [n], [n], seed=2)
    q = torch.zeros_like(q)
    q[..., 0] = 1
    k[..., 0] = torch.arange(n, device='cuda')[:, None].to(BF16) / 4
    for t in (q, k, v):
        t.requires_grad_(True)
    for causal in (False, True):
        out = packed_attention(q, k, v, offsets([n]), causal=causal, scale=1.0)
        got = (out.detach(), *torch.autograd.grad(out, (q, k, v), g))
        value, tol = oracle.attention(q.detach(), k.detach(), v.detach(), [n], [n], causal, 1.0, dout=g)
        for name, x in zip(('out', 'dq', 'dk', 'dv'), got):
            oracle.check(x, value[name], tol[name], name)


def test_nan_stays_in_its_sequence(cuda):
    """A NaN key, query or value of one sequence leaves the neighbours' results as they are, bit by bit."""
    lens = [100, 60, 190]
    q, k, v, g, _ = make(BF16, 4, 2, 64, lens, lens, seed=5)

    def run(q, k, v):
        q, k, v = (t.detach().clone().requires_grad_(True) for t in (q, k, v))
        out = packed_attention(q, k, v, offsets(lens), causal=True)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), g))

    clean = run(q, k, v)
    for which in range(3):
        dirty = [t.clone() for t in (q, k, v)]
        dirty[which][130] = math.nan
        for a, b in zip(run(*dirty), clean):
            assert torch.equal(a[:100], b[:100]) and torch.equal(a[160:], b[160:])
    dirty = k.clone()
    dirty[130] = math.nan  # seen by the queries from row 130 on
    out = packed_attention(q, dirty, v, offsets(lens), causal=True)
    assert torch.equal(out[:130], clean[0][:130]) and out[130:160].isnan().all()


def test_strided_and_unaligned_inputs(cuda):
    lens = [90, 140]
    n, h, m, d = 230, 4, 2, 64
    g = torch.Generator(device='cuda').manual_seed(1)
    qkv = torch.randn((n, (h + 2 * m) * d), generator=g, device='cuda').half()
    q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split([h * d, m * d, m * d], 1))
    up = torch.randn((n, h, d), generator=g, device='cuda').half()
    cu = offsets(lens)

    def run(q, k, v, up=up):
        q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = packed_attention(q, k, v, cu, causal=True)
        return (out.detach(), *torch.autograd.grad(out, (q, k, v), up))

    want = run(q.contiguous(), k.contiguous(), v.contiguous())

    def shifted(t):  # 2 bytes off a 16-byte boundary
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device='cuda')
        flat[1:] = t.reshape(-1)
        return flat[1:].view(t.shape)

    heads_first = lambda t: t.transpose(0, 1).contiguous().transpose(0, 1)  # noqa: E731
    dims_first = lambda t: t.permute(2, 0, 1).contiguous().permute(1, 2, 0)  # noqa: E731
    for form in (lambda t: t, shifted, heads_first, dims_first):
        for a, b in zip(run(form(q), form(k), form(v), form(up)), want):
            assert torch.equal(a, b)
    one = k[:, :1].contiguous()  # one key head broadcast to four: gradients are summed over the copies
    wide = one.expand(n, h, d)
    for a, b in zip(run(q, wide, wide), run(q, wide.contiguous(), wide.contiguous())):
        assert torch.equal(a, b)


def test_deterministic_and_on_another_stream(cuda):
    lens = [700, 33, 260]
    q, k, v, g, _ = make(BF16, 8, 2, 128, lens, lens, seed=6)
    cu = offsets(lens)

    def run():
        x, y, z = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = packed_attention(x, y, z, cu, causal=True)
        return (out.detach(), *torch.autograd.grad(out, (x, y, z), g))

    want = run()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = run()
    side.synchronize()
    for a, b, c in zip(run(), other, want):
        assert torch.equal(a, c) and torch.equal(b, c)


def test_captured_and_replayed(cuda):
    """Two graphs over the same inputs, replayed in turn with new values, offsets and lengths."""
    room, n = 300, 3
    q, k, v, _, _ = make(F16, 4, 2, 64, [n], [n * room], seed=7)
    cu_q, cu_k = offsets([1] * n), offsets([room] * n)
    lengths = torch.tensor([300, 5, 70], dtype=torch.int32, device='cuda')
    pq, pk, pv, g, _ = make(BF16, 4, 4, 128, [200], [200], seed=8)
    cu = offsets([120, 80])

    def decode():
        return packed_attention(q, k, v, cu_q, cu_k, kv_lengths=lengths, causal=True)

    def prompt():
        x, y, z = (t.detach().requires_grad_(True) for t in (pq, pk, pv))
        out = packed_attention(x, y, z, cu, causal=True)
        return (out.detach(), *torch.autograd.grad(out, (x, y, z), g))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        decode(), prompt()
    torch.cuda.synchronize()
    graphs, outs = [], []
    for f in (decode, prompt):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(f())
    for step in range(3):
        for t in (q, k, v, pq, pk, pv):
            t.add_(0.25)
        lengths.copy_(torch.tensor([10 + step, 300, 0]))
        cu.copy_(torch.tensor([0, 50 * step, 200 - step]))
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        for a, b in zip([outs[0], *outs[1]], [decode(), *prompt()]):
            assert torch.equal(a, b)


def test_wrong_offsets_stay_inside(cuda):
    """Offsets that run backwards or past the tensors give wrong sequences, but nothing outside is touched."""
    guard = torch.full((3, 64, 2, 64), 7.0, dtype=F16, device='cuda')
    q, k, v, g, _ = make(F16, 2, 2, 64, [300], [300], seed=10)
    for bad in ([0, 500, 200, 900], [-5, 100, 50, 300], [200, 100, 0, 0], [0, 2 ** 31 - 1, -2 ** 31, 300]):
        cu = torch.tensor(bad, dtype=torch.int32, device='cuda')
        x, y, z = (t.detach().requires_grad_(True) for t in (q, k, v))
        out = packed_attention(x, y, z, cu, kv_lengths=torch.tensor([-3, 1 << 30, 9], device='cuda'), causal=True)
        torch.autograd.grad(out, (x, y, z), g)
    torch.cuda.synchronize()
    assert bool((guard == 7.0).all())
    both(F16, 2, 2, 64, [300])  # and the next call is right


def test_gradients_against_differences(cuda):
    """Directional derivatives of the oracle's value by central differences in fp64."""
    lens, dim = [37, 90], 32
    q, k, v, g, _ = make(F16, 4, 2, dim, lens, lens, seed=11)
    x, y, z = (t.detach().requires_grad_(True) for t in (q, k, v))
    out = packed_attention(x, y, z, offsets(lens), causal=True)
    grads = torch.autograd.grad(out, (x, y, z), g)
    _, tol = oracle.attention(q, k, v, lens, lens, True, dim ** -0.5, dout=g)
    for n, (grad, name) in enumerate(zip(grads, ('dq', 'dk', 'dv'))):
        way = torch.randn(grad.shape, generator=torch.Generator(device='cuda').manual_seed(n), device='cuda').double()
        h = 2.0 ** -12
        ends = []
        for sign in (1, -1):
            args = [t.double() for t in (q, k, v)]
            args[n] = args[n] + sign * h * way
            ends.append(_loss64(args, lens, dim, g))
        slope = (ends[0] - ends[1]) / (2 * h)
        # h^2 / 6 times a third derivative, with scores' derivatives below 2^3: below 2^-10 of the sum of terms
        slack = float((tol[name] * way.abs()).sum()) + 2.0 ** -10 * float((grad.double() * way).abs().sum())
        assert abs(float((grad.double() * way).sum()) - slope) <= slack


def _loss64(args, lens, dim, g):
    q, k, v = args
    total, a = 0.0, 0
    for n in lens:
        for h in range(q.shape[1]):
            m = h // (q.shape[1] // k.shape[1])
            s = (q[a:a + n, h] @ k[a:a + n, m].t() * dim ** -0.5).masked_fill(
                torch.ones(n, n, dtype=torch.bool, device='cuda').triu(1), -math.inf)
            total += float((torch.softmax(s, 1) @ v[a:a + n, m] * g[a:a + n, h].double()).sum())
        a += n
    return total


def test_attention_refusals(cuda):
    q, k, v, _, _ = make(F16, 4, 2, 64, [10], [10])
    cu = offsets([10])
    for bad in [dict(q=q.float()), dict(k=k.bfloat16()), dict(cu_seqlens_q=cu.float()),
                dict(kv_lengths=torch.ones(1, device='cuda'))]:
        with pytest.raises(TypeError):
            packed_attention(**({'q': q, 'k': k, 'v': v, 'cu_seqlens_q': cu} | bad))
    for bad in [dict(q=q[0]), dict(v=v[:9]), dict(k=k[..., :32], v=v[..., :32]), dict(q=q[:, :3]),
                dict(cu_seqlens_k=offsets([5, 5])), dict(cu_seqlens_q=cu[:0]), dict(cu_seqlens_q=cu[None]),
                dict(kv_lengths=torch.ones(2, dtype=torch.int32, device='cuda')), dict(scale=math.inf),
                dict(q=q[..., :60], k=k[..., :60], v=v[..., :60]), dict(k=k[:, :0], v=v[:, :0])]:
        with pytest.raises(ValueError):
            packed_attention(**({'q': q, 'k': k, 'v': v, 'cu_seqlens_q': cu} | bad))
    with pytest.raises(RuntimeError):
        packed_attention(q, k, v, cu.cpu())


def test_autocast(cuda):
    q, k, v, _, _ = make(F32, 2, 2, 32, [50], [50])
    with torch.autocast('cuda', dtype=BF16):
        out = packed_attention(q, k, v, offsets([50]))
    want = packed_attention(q.bfloat16(), k.bfloat16(), v.bfloat16(), offsets([50]))
    assert out.dtype == F32 and torch.equal(out, want.float())


def test_float_gradients_are_optional(cuda):
    """Only what is asked for: lse alone, out alone, no gradient at all."""
    q, k, v, g, gl = make(F16, 2, 1, 64, [150], [150], seed=13)
    x = q.detach().requires_grad_(True)
    _, lse = packed_attention(x, k, v, offsets([150]), return_lse=True)
    (dq,) = torch.autograd.grad(lse, x, gl)
    value, tol = oracle.attention(q, k, v, [150], [150], False, 64 ** -0.5, dout=torch.zeros_like(g), dlse=gl)
    oracle.check(dq, value['dq'], tol['dq'], 'dq of lse')
    assert not packed_attention(q, k, v, offsets([150])).requires_grad


def test_single_key_has_no_gradient_through_its_score(cuda):
    """One key: P = 1 whatever the score, so q and k get (to fp32's rounding) nothing, although o is rounded."""
    lens = [1] * 50
    q, k, v, g, _ = make(BF16, 2, 2, 128, lens, lens, seed=14)
    x, y, z = (t.requires_grad_(True) for t in (q, k, v))
    out = packed_attention(x, y, z, offsets(lens), causal=True)
    dq, dk, dv = torch.autograd.grad(out, (x, y, z), g)
    # |dP - delta| is below a few fp32 steps of sum |g| |v| < 2^9
    assert float(dq.abs().max()) < 2.0 ** -10 and float(dk.abs().max()) < 2.0 ** -10
    assert torch.equal(dv, g) and torch.equal(out.detach(), v.detach())


@pytest.mark.parametrize('seqs', [31, 64, 100])
@pytest.mark.parametrize('heads,kv', [(4, 4), (24, 2)])
def test_many_streams(cuda, seqs, heads, kv):
    """One to three queries for each of many sequences: cuts through groups, groups of two row tiles, empty caches."""
    rng = np.random.default_rng(seqs)
    lens_k = [int(n) for n in rng.integers(0, 700, seqs)]
    lens_q = [int(n) for n in rng.integers(0, 3, seqs)]
    both(BF16, heads, kv, 64, lens_q, lens_k, causal=True, spare=3, seed=seqs)
    both(F16, heads, kv, 128, [1] * seqs, lens_k, causal=False, seed=seqs + 1)


@pytest.mark.parametrize('heads,kv', [(6, 2), (4, 1)])
@pytest.mark.parametrize('dim', [64, 128])
def test_many_short_sequences_share_heads(cuda, heads, kv, dim):
    """More sequences than one warp looks at in a step, some empty, some of more than one tile, forward and backward."""
    rng = np.random.default_rng(dim + heads)
    lens = [int(n) for n in rng.integers(0, 150, 70)]
    both(BF16, heads, kv, dim, lens, causal=True, spare=5, seed=dim)
    both(F16, heads, kv, dim, lens, [int(n) for n in rng.integers(0, 150, 70)], causal=True, seed=heads)


@pytest.mark.parametrize('queries', [1, 150])
def test_keys_past_two_to_the_31(cuda, queries):
    """The last sequence's keys and their gradients lie past 2 ** 31 elements (and 2 ** 32 bytes)."""
    heads, kv, dim, far, n = 8, 8, 128, 2_150_000, 300
    if torch.cuda.mem_get_info()[0] < 40 * 2 ** 30:
        pytest.skip('needs 40 GB')
    q, ks, vs, g, _ = make(BF16, heads, kv, dim, [queries], [n], seed=queries)
    k, v = (torch.zeros((far + n, kv, dim), dtype=BF16, device='cuda') for _ in range(2))
    k[far:], v[far:] = ks, vs
    assert k.numel() > 2 ** 31
    for t in (q, k, v):
        t.requires_grad_(True)
    out, lse = packed_attention(q, k, v, offsets([0, queries]), offsets([far, n]), causal=True, return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, (q, k, v), g)
    value, tol = oracle.attention(q.detach(), ks, vs, [queries], [n], True, dim ** -0.5, dout=g)
    for name, x in (('out', out), ('lse', lse), ('dq', dq), ('dk', dk[far:]), ('dv', dv[far:])):
        oracle.check(x.detach(), value[name], tol[name], name)
    assert not dk[:far].any() and not dv[:far].any()


def test_two_streams_at_once(cuda):
    """Calls of each kind in flight on two streams give what they give alone."""
    lens, n = [900, 120, 33], 24
    train = make(BF16, 8, 2, 128, lens, lens, seed=1)[:4]
    decode = make(F16, 8, 2, 64, [1] * n, [600] * n, seed=2)[:3]
    cu, cu_q, cu_k = offsets(lens), offsets([1] * n), offsets([600] * n)
    x = torch.randn((1000, 64), device='cuda')
    seed = torch.tensor([3, 4], device='cuda')

    def run():
        a, b, c = (t.detach().requires_grad_(True) for t in train[:3])
        out = packed_attention(a, b, c, cu, causal=True)
        return (out.detach(), *torch.autograd.grad(out, (a, b, c), train[3]),
                packed_attention(*decode, cu_q, cu_k), residual_dropout(x, x, 0.3, seed))

    want = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    found = []
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                found.append(run())
    torch.cuda.synchronize()
    for got in found:
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_second_derivative_is_refused(cuda):
    q, k, v, g, _ = make(F16, 2, 2, 64, [20], [20])
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(packed_attention(q, k, v, offsets([20])), q, g, create_graph=True)
    with pytest.raises(NotImplementedError):
        dq.sum().backward()
    x = torch.randn(4, 2, 16, device='cuda', requires_grad=True)
    pos, freq = torch.zeros(4, 1, device='cuda'), torch.ones(8, device='cuda')
    out, _ = qk_norm_rotary(x, x, pos, freq, (8,))
    (dx,) = torch.autograd.grad(out.sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError):
        dx.sum().backward()
    y = residual_dropout(x, x, 0.5, torch.zeros(2, dtype=torch.int64, device='cuda'))
    (dx,) = torch.autograd.grad(y, x, torch.ones_like(y).requires_grad_(True), create_graph=True)
    assert dx.requires_grad  # linear in the gradient: differentiable again


def test_compiled(cuda):
    """torch.compile traces through the three operators, forward and backward."""
    q, k, v, g, _ = make(F16, 4, 2, 64, [40, 25], [40, 25], seed=15)
    cu, seed = offsets([40, 25]), torch.tensor([3, 4], device='cuda')
    pos, freq = torch.arange(65, device='cuda')[:, None], torch.rand(32, device='cuda')
    w = torch.ones(64, device='cuda', requires_grad=True)

    def block(q, k, v, w):
        a, b = qk_norm_rotary(q, k, pos, freq, (32,), w, w)
        return residual_dropout(packed_attention(a, b, v, cu, causal=True), q, 0.2, seed)

    leaves = [t.requires_grad_(True) for t in (q, k, v)] + [w]
    want = block(*leaves)
    got = torch.compile(block, backend='aot_eager', fullgraph=True)(*leaves)
    assert torch.equal(got, want)
    for a, b in zip(torch.autograd.grad(got, leaves, g), torch.autograd.grad(want, leaves, g)):
        assert torch.equal(a, b)


# ----------------------------------------------------------- norm and rotary
def rotary_case(dtype, tokens, heads, kv, dim, sections, norm, positions, interleaved, reach, seed=0, eps=1e-6):
    g = torch.Generator(device='cuda').manual_seed(seed)
    q = (2 * torch.randn((tokens, heads, dim), generator=g, device='cuda')).to(dtype)
    k = (2 * torch.randn((tokens, kv, dim), generator=g, device='cuda')).to(dtype)
    pos = (torch.rand((tokens, len(sections)), generator=g, device='cuda', dtype=torch.float64) - 0.3) * reach
    pos = pos.to(positions)
    freq = (10000.0 ** (-torch.arange(sum(sections), dtype=torch.float64, device='cuda') / sum(sections))).float()
    w = [(1 + 0.2 * torch.randn(dim, generator=g, device='cuda')) if norm else None for _ in range(2)]
    ups = [torch.randn(t.shape, generator=g, device='cuda').to(dtype) for t in (q, k)]
    leaves = [t.requires_grad_(True) for t in (q, k, *w) if t is not None]
    got = qk_norm_rotary(q, k, pos, freq, sections, *w, eps=eps, interleaved=interleaved)
    grads = torch.autograd.grad(got, leaves, ups)
    u, t = oracle.half_step(dtype), oracle.underflow(dtype)
    exact = [x.detach().double().requires_grad_(True) for x in leaves]
    half = sum(sections)
    for i in range(2):
        wi = exact[2 + i] if norm else None
        y = oracle.rotary(exact[i], wi, pos, freq, sections, eps, interleaved)
        # fp32 inside: the norm's sum (dim / 16 + 12 adds a thread or level), its root, two products, a turn of
        # two products with an angle good to one rounding: below 64 steps of the largest term of the pair
        top = exact[i].detach().abs().amax(-1, keepdim=True)
        n = exact[i].detach().square().mean(-1, keepdim=True)
        if norm:
            top = top * torch.rsqrt(n + eps) * wi.detach().abs().max()
        oracle.check(got[i].detach(), y.detach(), u * y.detach().abs() + t + 64 * 2.0 ** -24 * 2 * top, f'out {i}')
        want = torch.autograd.grad(y, [exact[i]] + ([wi] if norm else []), ups[i].double())
        gtop = ups[i].double().abs().amax(-1, keepdim=True) * 2
        if norm:
            r, wt = torch.rsqrt(n + eps), wi.detach().abs().max()
            # dx = r (w g - xhat mean(w g xhat)): the mean is below the largest |w g| times sqrt(dim) / dim * dim ..
            gtop_x = r * gtop * wt * (1 + (exact[i].detach().abs() * r) * dim ** 0.5)
        else:
            gtop_x = gtop.expand_as(want[0])
        oracle.check(grads[i], want[0], u * want[0].abs() + t + 64 * 2.0 ** -24 * gtop_x, f'gradient {i}')
        if norm:
            # a sum of tokens * heads terms in three levels: at most this many adds in one chain
            h = (heads, kv)[i]
            chain = tokens * h / max(1, min(592 * 16, tokens)) + 700
            terms = (oracle.rotary(ups[i].double(), None, -pos.double(), freq, sections, 0.0, interleaved)
                     * exact[i].detach() * r).abs().sum((0, 1))
            slip = (gtop * (exact[i].detach().abs() * r)).sum((0, 1))
            oracle.check(grads[2 + i], want[1], 2.0 ** -24 * (chain * terms + 64 * slip), f'weight {i}')
    assert all(o.is_contiguous() for o in got) and half > 0


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('dim,sections,inter', [(16, (8,), False), (32, (4, 6, 6), False), (64, (10, 11, 11), False),
                                                (128, (16, 24, 24), False), (256, (128,), False),
                                                (80, (0, 16, 16), False), (24, (8,), False), (136, (30, 34), False),
                                                (8, (3,), True), (24, (5, 7), True), (128, (64,), True),
                                                (200, (1, 2, 3, 4), True), (256, (60, 68), True)])
def test_rotary_dims_and_sections(cuda, dtype, dim, sections, inter):
    rotary_case(dtype, 53, 3, 2, dim, sections, True, torch.int32, inter, 1500, seed=dim)


@pytest.mark.parametrize('tokens,heads,kv', [(1, 1, 1), (0, 2, 2), (3, 32, 8), (700, 5, 1), (4001, 2, 2)])
@pytest.mark.parametrize('norm', [False, True])
def test_rotary_tokens(cuda, tokens, heads, kv, norm):
    rotary_case(BF16, tokens, heads, kv, 64, (8, 12, 12), norm, torch.int64, False, 300, seed=tokens)


@pytest.mark.parametrize('dtype,dim,sections,inter', [(BF16, 128, (16, 24, 24), False), (F32, 256, (128,), False),
                                                      (F16, 24, (5, 7), False), (F16, 24, (5, 7), True)])
@pytest.mark.parametrize('heads,kv', [(48, 48), (64, 1), (1, 33)])
def test_rotary_many_heads(cuda, dtype, dim, sections, inter, heads, kv):
    """More heads than a block has lanes for."""
    if sum(sections) % 8 and not inter:
        with pytest.raises(ValueError, match='a multiple of 8, got 12'):
            rotary_case(dtype, 37, heads, kv, dim, sections, True, torch.int32, inter, 500, seed=heads)
        return
    rotary_case(dtype, 37, heads, kv, dim, sections, True, torch.int32, inter, 500, seed=heads)


@pytest.mark.parametrize('positions', [torch.int32, torch.int64, torch.float32])
@pytest.mark.parametrize('inter', [False, True])
def test_rotary_far_positions(cuda, positions, inter):
    rotary_case(F32, 40, 2, 1, 64, (16, 16), True, positions, inter, 2 ** 30, seed=1)


def test_rotary_one_norm_only_strides_and_zero_rows(cuda):
    g = torch.Generator(device='cuda').manual_seed(3)
    n, h, m, d = 31, 4, 2, 32
    wide = torch.randn((n, (h + 2 * m) * d), generator=g, device='cuda').bfloat16()
    q, k, _ = (t.unflatten(1, (-1, d)) for t in wide.split([h * d, m * d, m * d], 1))
    sites = torch.randint(0, 200, (n, 4), generator=g, device='cuda', dtype=torch.int32)
    freq = torch.rand(16, generator=g, device='cuda', dtype=torch.float64)
    w = torch.rand(d + 1, generator=g, device='cuda')[1:]  # unaligned
    got = qk_norm_rotary(q, k, sites[:, 1:], freq, (4, 6, 6), w)
    want = qk_norm_rotary(q.contiguous(), k.contiguous(), sites[:, 1:].contiguous(), freq, (4, 6, 6), w.clone())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    plain = oracle.rotary(k.double(), None, sites[:, 1:], freq, (4, 6, 6), 0.0, False)
    assert (got[1].double() - plain).abs().max() <= 2.0 ** -8 * plain.abs().max()
    flip = sites[:, 1:].flip(0)
    lanes = qk_norm_rotary(q, k, sites.t().contiguous().t()[:, 1:].flip(0), freq, (4, 6, 6), w)
    assert all(torch.equal(a, b) for a, b in zip(lanes, qk_norm_rotary(q, k, flip.clone(), freq, (4, 6, 6), w)))
    zero = torch.zeros_like(q).requires_grad_(True)
    out, _ = qk_norm_rotary(zero, k, sites[:, 1:], freq, (4, 6, 6), w)
    (grad,) = torch.autograd.grad(out, zero, torch.ones_like(out))
    assert bool((out == 0).all()) and bool(torch.isfinite(grad).all())


def test_rotary_refusals(cuda):
    q = torch.zeros(5, 2, 64, device='cuda')
    pos, freq, w = torch.zeros(5, 2, device='cuda'), torch.ones(16, device='cuda'), torch.ones(64, device='cuda')
    good = dict(q=q, k=q, positions=pos, inv_freq=freq, sections=(8, 8), q_weight=w)
    qk_norm_rotary(**good)
    for bad in [dict(q=q.double()), dict(k=q.half()), dict(positions=pos.half()), dict(inv_freq=freq.half())]:
        with pytest.raises(TypeError):
            qk_norm_rotary(**(good | bad))
    for bad in [dict(sections=(8,)), dict(sections=(8, 9)), dict(sections=(24, -8)), dict(sections=()),
                dict(sections=(4, 8), inv_freq=freq[:12]), dict(positions=pos[:4]), dict(positions=pos[:, 0]),
                dict(q_weight=w[:32]), dict(k=q[:4]), dict(k=q[:, :, :32]), dict(q=q[0]), dict(eps=-1.0),
                dict(q=q[..., :60], k=q[..., :60]), dict(q=q[:, :0])]:
        with pytest.raises(ValueError):
            qk_norm_rotary(**(good | bad))
    with pytest.raises(RuntimeError):
        qk_norm_rotary(**(good | dict(positions=pos.cpu())))


# ------------------------------------------------------------------- dropout
def dropout_expected(x, residual, p, seed):
    words = oracle.philox(x.numel(), *(int(s) for s in seed.tolist()))
    keep = torch.from_numpy(words >= int(p * 2.0 ** 32) if p < 1 else np.zeros(words.shape, bool)).view(x.shape)
    scaled = x.detach().double().cpu() / (1 - p) if p < 1 else x.detach().double().cpu()
    y = torch.where(keep, scaled, 0.0)
    return (y if residual is None else y + residual.detach().double().cpu()), keep


@pytest.mark.parametrize('dtype', [F32, F16, BF16])
@pytest.mark.parametrize('shape', [(1,), (7,), (8,), (3, 1), (129, 33), (1000, 64)])
@pytest.mark.parametrize('p', [0.0, 0.1, 0.5, 0.999, 1.0])
@pytest.mark.parametrize('with_residual', [False, True])
def test_dropout(cuda, dtype, shape, p, with_residual):
    g = torch.Generator(device='cuda').manual_seed(shape[0])
    x = torch.randn(shape, generator=g, device='cuda').to(dtype).requires_grad_(True)
    r = torch.randn(shape, generator=g, device='cuda').to(dtype).requires_grad_(True) if with_residual else None
    up = torch.randn(shape, generator=g, device='cuda').to(dtype)
    seed = torch.randint(-(1 << 63), (1 << 63) - 1, (2,), generator=g, device='cuda')
    y = residual_dropout(x, r, p, seed)
    want, keep = dropout_expected(x, r, p, seed)
    u, t = oracle.half_step(dtype), oracle.underflow(dtype)
    # the scale 1 / (1 - p) rounded to fp32, one fused product and sum in fp32, one rounding
    slip = 2.0 ** -23 * (want.abs() + (x.detach().double().cpu().abs() / max(1 - p, 2.0 ** -10)))
    oracle.check(y.detach().cpu(), want, u * want.abs() + t + slip, 'y')
    grads = torch.autograd.grad(y, [x] + ([r] if with_residual else []), up)
    gwant, _ = dropout_expected(up, None, p, seed)
    oracle.check(grads[0].cpu(), gwant, (u + 2.0 ** -22) * gwant.abs() + t, 'gradient')
    assert bool(((grads[0].cpu() == 0) | keep).all())
    if with_residual:
        assert torch.equal(grads[1], up)


def test_dropout_mask_layouts_and_values(cuda):
    n = 1 << 16
    seed = torch.tensor([123456789, -7], device='cuda')
    x = torch.ones(n, device='cuda')
    y = residual_dropout(x, None, 0.3, seed)
    kept = int((y != 0).sum())
    assert abs(kept - 0.7 * n) < 6 * (0.21 * n) ** 0.5  # six deviations of a binomial
    assert not torch.equal(y, residual_dropout(x, None, 0.3, seed + torch.tensor([1, 0], device='cuda')))
    assert not torch.equal(y, residual_dropout(x, None, 0.3, seed + torch.tensor([0, 1], device='cuda')))
    shifted = torch.ones(n + 1, device='cuda')[1:]  # 4 bytes off: the same values
    assert torch.equal(residual_dropout(shifted, shifted, 0.3, seed), residual_dropout(x, x, 0.3, seed))
    turned = torch.rand(64, 32, device='cuda').t()
    assert torch.equal(residual_dropout(turned, None, 0.3, seed), residual_dropout(turned.contiguous(), None, 0.3, seed))
    bad = x.clone()
    bad[y == 0] = math.nan  # what is dropped shows nowhere
    assert torch.equal(residual_dropout(bad, None, 0.3, seed), y)
    assert residual_dropout(x[:0], x[:0], 0.5, seed).numel() == 0


def test_dropout_replayed_graph_draws_anew(cuda):
    x = torch.rand(4096, device='cuda')
    seed = torch.tensor([1, 0], device='cuda')
    residual_dropout(x, x, 0.5, seed)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = residual_dropout(x, x, 0.5, seed)
    for step in range(3):
        seed[1] = step
        graph.replay()
        assert torch.equal(y, residual_dropout(x, x, 0.5, seed))


def test_dropout_refusals(cuda):
    x, seed = torch.zeros(8, device='cuda'), torch.zeros(2, dtype=torch.int64, device='cuda')
    for bad in [dict(x=x.double()), dict(residual=x.half()), dict(seed=seed.int())]:
        with pytest.raises(TypeError):
            residual_dropout(**(dict(x=x, residual=x, p=0.5, seed=seed) | bad))
    for bad in [dict(p=-0.1), dict(p=1.1), dict(p=math.nan), dict(residual=x[:4]), dict(seed=seed[:1])]:
        with pytest.raises(ValueError):
            residual_dropout(**(dict(x=x, residual=x, p=0.5, seed=seed) | bad))
    with pytest.raises(RuntimeError):
        residual_dropout(x, x, 0.5, seed.cpu())


# -------------------------------------------------------------- the block
def block64(layer, feats, indices, batch, seed):
    """The layer's definition in fp64 from its parameters, differentiable."""
    p = {n: t.detach().double().requires_grad_(True) for n, t in layer.named_parameters()}
    x = feats.detach().double().requires_grad_(True)
    h, m, d = layer.heads, layer.kv_heads, layer.dim
    y = torch.nn.functional.layer_norm(x, x.shape[1:], p['norm.weight'], p['norm.bias'], layer.norm.eps)
    y = y @ p['qkv.weight'].t() + p['qkv.bias']
    q, k, v = y.unflatten(1, (h + 2 * m, d)).split([h, m, m], 1)
    freq = layer.inv_freq.to(x.device)
    q = oracle.rotary(q, p['q_weight'], indices[:, 1:], freq, layer.sections, layer.eps, False)
    k = oracle.rotary(k, p['k_weight'], indices[:, 1:], freq, layer.sections, layer.eps, False)
    outs = []
    for b in range(batch):
        rows = indices[:, 0] == b
        s = torch.einsum('ihd,jhd->hij', q[rows], k[rows].repeat_interleave(h // m, 1)) * d ** -0.5
        if layer.causal:
            s = s.masked_fill(torch.ones_like(s, dtype=torch.bool).triu(1), -math.inf)
        outs.append(torch.einsum('hij,jhd->ihd', torch.softmax(s, -1), v[rows].repeat_interleave(h // m, 1)))
    o = torch.cat(outs).flatten(1) @ p['proj.weight'].t() + p['proj.bias']
    if seed is not None:
        words = oracle.philox(o.numel(), *(int(s) for s in seed.tolist()))
        keep = torch.from_numpy(words >= int(layer.dropout * 2.0 ** 32)).to(o.device).view(o.shape)
        o = torch.where(keep, o / (1 - layer.dropout), 0.0)
    return x + o, x, p


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('train', [False, True])
def test_block_runs_the_operators_together(cuda, causal, train, monkeypatch):
    torch.manual_seed(0)
    batch, channels = 3, 64
    coords = [torch.randperm(12 * 40 * 40)[:n].sort().values for n in (150, 0, 333)]
    indices = torch.cat([torch.stack([torch.full_like(c, b), c // 1600, c // 40 % 40, c % 40], 1)
                         for b, c in enumerate(coords)]).int().cuda()
    feats = torch.randn(len(indices), channels, device='cuda', requires_grad=True)
    layer = SparseSelfAttention(channels, 4, 2, dropout=0.2, causal=causal).cuda().train(train)
    drawn = []
    real = torch.randint
    monkeypatch.setattr(torch, 'randint', lambda *a, **k: drawn.append(real(*a, **k)) or drawn[-1])
    x = SparseConvTensor(feats, indices, [12, 40, 40], batch)
    with torch.autocast('cuda', dtype=F16):
        y = SparseSequential(layer, torch.nn.Identity())(x)
    assert y.indices is indices and y.features.dtype == F32 and len(drawn) == (1 if train else 0)
    want, leaf, params = block64(layer, feats, indices, batch, drawn[0] if train else None)
    # about ten fp16 roundings in a row, each 2^-11 of values whose sums of products are taken over up to 333
    # terms of mixed sign: 2^-5 of the largest value bounds any chain of them
    close = lambda a, b: (a.double() - b).abs().max() <= 2.0 ** -5 * b.abs().max()  # noqa: E731
    assert close(y.features.detach(), want.detach())
    up = torch.randn_like(feats)
    names = [n for n, _ in layer.named_parameters()]
    got = torch.autograd.grad(y.features, [feats] + [t for _, t in layer.named_parameters()], up)
    ref = torch.autograd.grad(want, [leaf] + [params[n] for n in names], up.double())
    for n, a, b in zip(['features'] + names, got, ref):
        assert close(a, b), n


def test_block_half_module_and_refusal(cuda):
    indices = torch.tensor([[0, 1, 2, 3], [0, 1, 2, 9], [1, 0, 0, 0]], dtype=torch.int32, device='cuda')
    layer = SparseSelfAttention(32, 2, dropout=0.1).cuda().half().eval()
    out = layer(SparseConvTensor(torch.randn(3, 32, device='cuda').half(), indices, [4, 4, 16], 2))
    assert out.features.dtype == F16 and bool(torch.isfinite(out.features).all())
    with pytest.raises(TypeError):  # fp32 outside autocast
        SparseSelfAttention(32, 2).cuda()(SparseConvTensor(torch.randn(3, 32, device='cuda'), indices, [4, 4, 16], 2))
