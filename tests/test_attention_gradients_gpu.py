"""Gradients of packed_attention where roundings inside the kernels would show:
rows whose softmax is peaked (dS is then a small difference of large numbers),
small incoming gradients in fp16.

The tolerances are counted for a backward that keeps all but the operands of its
products in fp32.  With u = eps / 2 of the dtype:

* S: fp32 sums of exact products, off by 2^-23 of the sum of absolute terms A at
  each of the dim / 16 + 2 steps; nothing at all where the terms and their sums
  are multiples of 1/16 (`exact`).  The exponent c S - lse is rounded three times,
  the exponential is good to 2^-22, and the sum behind lse takes 40 + keys / 128
  fp32 additions in a chain.  Together E, relative to P.
* dP is off by 2^-20 sum |dO| |v|.  delta = sum P dP - dlse is a sum of fp32
  terms around the first estimate, so it is off by (2^-20 + 2 E + chain) of twice
  W = sum P |dO| |v|, and not by the roundings of the output.
* dS is rounded to the type (u), and only that: a power of two for each row keeps
  it out of fp16's subnormal numbers, down to 2^-38 of the row's bound.
* the first estimate takes delta from the rounded output; what that leaves, e, is
  put right by a product with P rounded to the type: 2 u e P |k|.
"""
import math

import pytest
import torch

from bevfusion_triton_b200.ops.spconv import packed_attention
from tests.test_attention_block_gpu import BF16, F16, make, no_wait_gave_up, offsets  # noqa: F401

pytestmark = pytest.mark.gpu


def gradients(q, k, v, lens_q, lens_k, causal, scale, dout, dlse=None, exact=False):
    """Values and tolerances of dq, dk and dv in fp64."""
    dt = q.dtype
    u = torch.finfo(dt).eps / 2
    least = torch.finfo(dt).smallest_normal * u  # half a step of the subnormal numbers
    group = q.shape[1] // k.shape[1]
    value = {n: torch.zeros(x.shape, dtype=torch.float64, device=q.device) for n, x in
             (('dq', q), ('dk', k), ('dv', v))}
    tol = {n: torch.zeros_like(x) for n, x in value.items()}
    a = b = 0
    for nq, nk in zip(lens_q, lens_k):
        rows, keys = slice(a, a + nq), slice(b, b + nk)
        a, b = a + nq, b + nk
        if nq == 0 or nk == 0:
            continue
        sees = torch.ones(nq, nk, dtype=torch.bool, device=q.device)
        if causal:
            sees = sees.tril(nk - nq)
        for h in range(q.shape[1]):
            m = h // group
            x, y, z, g = (s.double() for s in (q[rows, h], k[keys, m], v[keys, m], dout[rows, h]))
            x, g = (torch.where(sees.any(1)[:, None], s, 0.0) for s in (x, g))
            gl = torch.zeros(nq, dtype=torch.float64, device=q.device) if dlse is None else dlse[h, rows].double()
            gl = torch.where(sees.any(1), gl, 0.0)
            score = (x @ y.t() * scale).masked_fill(~sees, -math.inf)
            lse = torch.logsumexp(score, 1)
            lse = torch.where(lse == -math.inf, 0.0, lse)
            p = torch.exp(score - lse[:, None])
            dp = g @ z.t()
            delta = (p * dp).sum(1) - gl
            ds = p * (dp - delta[:, None]) * scale
            # ------------------------------------------------- what fp32 leaves
            size = abs(scale) * (x.abs() @ y.abs().t())
            steps = q.shape[2] // 16 + 2
            top = torch.where(sees, size, 0.0).amax(1, keepdim=True)
            chain = (40 + nk / 128) * 2.0 ** -24
            e_p = 2.0 ** -22 + chain + 2.0 ** -22 * (torch.where(sees, score, 0.0).abs() + lse.abs()[:, None])
            if not exact:
                e_p = e_p + steps * 2.0 ** -23 * (size + top)
            e_p = torch.where(sees, e_p, 0.0)
            mass = g.abs() @ z.abs().t()
            w = (p * mass).sum(1)
            e_delta = (2.0 ** -20 + 2 * e_p.amax(1) + (70 + nk / 128) * 2.0 ** -24) * (2 * w + gl.abs())
            bound = abs(scale) * (g.norm(dim=1).max() * z.norm(dim=1).max() + gl.abs().max())
            e_ds = (abs(scale) * p * (2.0 ** -20 * mass + e_delta[:, None]) + (e_p + u) * ds.abs() +
                    torch.where(sees, 2.0 ** -36 * bound, 0.0))
            o = p @ z
            slip = abs(scale) * (g.abs() * (2 * u * (p @ z.abs() + o.abs()) + least * z.abs().sum(0))).sum(1)
            value['dq'][rows, h] = ds @ y
            tol['dq'][rows, h] = (e_ds @ y.abs() + (nk / 16 + 8) * 2.0 ** -23 * (ds.abs() @ y.abs()) +
                                  2 * u * slip[:, None] * (p @ y.abs()))
            value['dk'][keys, m] += ds.t() @ x
            tol['dk'][keys, m] += (e_ds.t() @ x.abs() +
                                   (nq * group / 16 + 8) * 2.0 ** -23 * (ds.abs().t() @ x.abs()))
            value['dv'][keys, m] += p.t() @ g
            tol['dv'][keys, m] += ((u + e_p + (nq * group / 16 + 8) * 2.0 ** -23) * p + 2.0 ** -39 * sees).t() @ g.abs()
    for n in tol:
        tol[n] += u * (value[n].abs() + tol[n]) + least + 2.0 ** -126
    return value, tol


def compare(q, k, v, g, gl, lens_q, lens_k, causal, scale, exact=False):
    for t in (q, k, v):
        t.requires_grad_(True)
    out, lse = packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=causal, scale=scale, return_lse=True)
    if gl is not None:
        gl = torch.where(lse.detach() == -math.inf, 0.0, gl)
    got = torch.autograd.grad((out, lse) if gl is not None else out, (q, k, v), (g, gl) if gl is not None else g)
    value, tol = gradients(q.detach(), k.detach(), v.detach(), lens_q, lens_k, causal, scale, g, gl, exact)
    for name, x in zip(('dq', 'dk', 'dv'), got):
        off = (x.double() - value[name]).abs() / tol[name]
        at = int(off.argmax())
        assert off.flatten()[at] <= 1, (
            f'{name}: {x.flatten()[at]} is not {value[name].flatten()[at]} +- {tol[name].flatten()[at]} at {at} '
            f'({float(off.max()):.3g} tolerances; {int((off > 1).sum())} of {off.numel()} are off)')


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('lens', [[129], [700], [2048], [64, 300]])
def test_peaked_rows(cuda, dtype, dim, causal, lens):
    """Queries of size 6 make a softmax with one or two keys in it; a causal prompt's first rows are such in any case.
    Queries and keys are multiples of 1/4, so the scores are exact."""
    q, k, v, g, gl = make(dtype, 4, 2, dim, lens, lens, seed=dim + len(lens))
    q, k = ((4 * x).round().clamp(-60, 60) / 4 for x in (4 * q.float(), k.float()))
    compare(q.to(dtype), k.to(dtype), v, g, gl, lens, lens, causal, dim ** -0.5, exact=True)


@pytest.mark.parametrize('size', [2.0 ** -7, 2.0 ** -10, 2.0 ** -13])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('causal', [False, True])
def test_small_gradients_in_fp16(cuda, size, dim, causal):
    """A mean over many tokens leaves each a small gradient: dS = P (..) would be subnormal."""
    lens = [2100, 37]
    q, k, v, g, _ = make(F16, 2, 1, dim, lens, lens, seed=dim)
    compare(q, k, v, (g.float() * size).half(), None, lens, lens, causal, dim ** -0.5)


@pytest.mark.parametrize('dim', [64, 128])
def test_many_keys_in_fp16(cuda, dim):
    """Even attention over 120 k keys: P near 2^-17 is far below fp16's normal numbers; and a gradient of lse."""
    lens_q, lens_k = [130], [120_000]
    q, k, v, g, gl = make(F16, 1, 1, dim, lens_q, lens_k, seed=dim)
    compare(q, k, v, 16 * g, gl, lens_q, lens_k, False, 2.0 ** -10)


@pytest.mark.parametrize('causal', [False, True])
@pytest.mark.parametrize('dim', [40, 128])
def test_gradients_of_mixed_sizes_in_fp16(cuda, causal, dim):
    """Rows whose gradients differ by up to 2^14, in a batch with a sequence whose gradients are all zero."""
    lens = [300, 700, 5]
    q, k, v, g, gl = make(F16, 4, 2, dim, lens, lens, seed=dim)
    size = 2.0 ** -(torch.arange(sum(lens), device='cuda') * 37 % 15).float()
    size[300:] *= torch.cat([torch.zeros(700), torch.ones(5)]).cuda()
    compare(q, k, v, (g.float() * size[:, None, None]).half(), gl * size, lens, lens, causal, dim ** -0.5)


@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('seqs,queries,keys', [(300, 1, 4096), (1, 1, 120_000), (1, 130, 120_000)])
def test_long_tail_in_fp16(cuda, dim, seqs, queries, keys):
    """One key 2^26 above all others, which alone have values: their part of the output is keys times 2^-26."""
    q, k, v, _, _ = make(F16, 2, 1, dim, [queries * seqs], [keys * seqs])
    q, k, v = torch.zeros_like(q), torch.zeros_like(k), torch.full_like(v, 64)
    q[..., 0], k[::keys, :, 0], v[::keys] = 1, 26, 0
    out = packed_attention(q, k, v, offsets([queries] * seqs), offsets([keys] * seqs), scale=math.log(2))
    tail = (keys - 1) * 2.0 ** -26
    # P and the result are rounded; the exponent is off by 2^-24 of 26 and the exponential by 2^-22; fp32 sums of
    # keys / 16 steps
    tol = 2 * 2.0 ** -11 + 26 * 2.0 ** -23 + 2.0 ** -22 + keys / 16 * 2.0 ** -23
    assert float((out.double() / (64 * tail / (1 + tail)) - 1).abs().max()) <= tol


@pytest.mark.parametrize('dtype', [F16, BF16])
@pytest.mark.parametrize('dim', [64, 128])
@pytest.mark.parametrize('lens_q,lens_k', [([300], [100]), ([129, 40, 260], [1, 40, 259]), ([200], [0]), ([3], [1])])
def test_queries_that_see_nothing_pass_nothing(cuda, dtype, dim, lens_q, lens_k):
    """Causal, more queries than keys: the first see no key, and whatever they and their gradients hold, NaN included,
    nobody else's gradient shows it and theirs is 0."""
    q, k, v, g, gl = make(dtype, 4, 2, dim, lens_q, lens_k, seed=dim + len(lens_q))
    a = 0
    for nq, nk in zip(lens_q, lens_k):
        for t in (q, g):
            t[a:a + max(0, nq - nk)] = math.nan
        gl[:, a:a + max(0, nq - nk)] = math.nan
        a += nq
    for t in (q, k, v):
        t.requires_grad_(True)
    out, lse = packed_attention(q, k, v, offsets(lens_q), offsets(lens_k), causal=True, return_lse=True)
    got = torch.autograd.grad((out, lse), (q, k, v), (g, gl))
    value, tol = gradients(q.detach(), k.detach(), v.detach(), lens_q, lens_k, True, dim ** -0.5, g, gl)
    for name, x in zip(('dq', 'dk', 'dv'), got):
        assert bool(torch.isfinite(x).all()) and bool(((x.double() - value[name]).abs() <= tol[name]).all()), name
