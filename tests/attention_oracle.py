"""64-bit oracle of the attention-block operators, and how far a kernel may be
from it.

The tolerances are counted, element by element, from the roundings a kernel
that computes in fp32 and feeds its products 16-bit operands has to make.
With u = eps / 2 of the dtype (a rounding's largest relative error) and t the
dtype's largest absolute error where it underflows:

* P is rounded before P v: |error of o| <= sum_j p_j |v_j| u (+ t |v_j|: P is
  at least t apart near 0, its largest entry 1), and o itself is rounded.
* lse, delta and the scores are fp32; their error (a few 2^-24 times scores
  below 2^6 here, and exp2's 2^-22) is covered by 2^-14 relative to the sum of
  absolute terms.
* Exponentials below fp32's smallest normal, 2^-126, are flushed to 0 (ex2 with
  ftz): P's absolute error is at least that, whatever the dtype, and reaches dS
  times |dP| + |delta|.
* dS is rounded before dS K and dS^T Q; delta is made of the rounded o, so it
  carries the error of o times |dO|.
"""
import math

import numpy as np
import torch

FP32 = 2.0 ** -14
FLUSH = 2.0 ** -126


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def underflow(dtype):
    return max(torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2, FLUSH)


def attention(q, k, v, lens_q, lens_k, causal, scale, room_k=None, dout=None, dlse=None):
    """Values and tolerances, as dicts of fp64 tensors: out, lse and, with
    ``dout``, dq, dk, dv."""
    dt = q.dtype
    u, t = half_step(dt), underflow(dt)
    group = q.shape[1] // k.shape[1]
    value = {'out': torch.zeros(q.shape, dtype=torch.float64, device=q.device),
             'lse': torch.full((q.shape[1], q.shape[0]), -math.inf, dtype=torch.float64, device=q.device)}
    if dout is not None:
        value |= {n: torch.zeros(x.shape, dtype=torch.float64, device=q.device)
                  for n, x in (('dq', q), ('dk', k), ('dv', v))}
    tol = {n: torch.zeros_like(x) for n, x in value.items()}
    tol['lse'] += 1.0
    a = b = 0
    for nq, nk, room in zip(lens_q, lens_k, lens_k if room_k is None else room_k):
        for h in range(q.shape[1]):
            m = h // group
            x, y, z = (s.double() for s in (q[a:a + nq, h], k[b:b + nk, m], v[b:b + nk, m]))
            if nq == 0 or nk == 0:
                continue
            score = x @ y.t() * scale
            if causal:
                sees = torch.ones(nq, nk, dtype=torch.bool, device=q.device).tril(nk - nq)
                score = score.masked_fill(~sees, -math.inf)
            lse = torch.logsumexp(score, 1)
            p = torch.exp(score - lse.masked_fill(lse == -math.inf, 0.0)[:, None])
            o = p @ z
            mass = p @ z.abs()
            o_tol = u * (mass + o.abs()) + t * (z.abs().sum(0) + 1) + FP32 * mass
            rows, keys = slice(a, a + nq), slice(b, b + nk)
            value['out'][rows, h], tol['out'][rows, h] = o, o_tol
            value['lse'][h, rows] = lse
            tol['lse'][h, rows] = FP32 * (1 + lse.masked_fill(lse == -math.inf, 0.0).abs())
            if dout is None:
                continue
            g = dout[rows, h].double()
            gl = dlse[h, rows].double() if dlse is not None else torch.zeros_like(lse)
            dp = g @ z.t()
            delta = (g * o).sum(1) - gl
            ds = p * (dp - delta[:, None]) * scale
            d_tol = (g.abs() * o_tol).sum(1)
            ds_tol = (u * ds.abs() + p * d_tol[:, None] * abs(scale) + t +
                      (FP32 * p + FLUSH) * (g.abs() @ z.abs().t() + delta.abs()[:, None]) * abs(scale))
            value['dq'][rows, h], tol['dq'][rows, h] = ds @ y, ds_tol @ y.abs()
            value['dk'][keys, m] += ds.t() @ x
            tol['dk'][keys, m] += ds_tol.t() @ x.abs()
            value['dv'][keys, m] += p.t() @ g
            tol['dv'][keys, m] += (u * p + t + FP32 * p).t() @ g.abs()
        a, b = a + nq, b + room
    for n in ('dq', 'dk', 'dv') if dout is not None else ():
        tol[n] += u * (value[n].abs() + tol[n]) + t
    return value, tol


def check(got, value, tol, name=''):
    """Every element within its tolerance; infinities and NaN in the same places."""
    got = got.double()
    fine = torch.isfinite(value)
    assert torch.equal(torch.isfinite(got), fine), f'{name}: finite in other places'
    assert torch.equal(got[~fine], value[~fine]), f'{name}: other infinities'
    off = torch.where(fine, (got - value).abs() - tol, 0.0)
    worst = off.argmax() if off.numel() else None
    assert worst is None or off.flatten()[worst] <= 0, (
        f'{name}: {got.flatten()[worst]} is not {value.flatten()[worst]} +- {tol.flatten()[worst]} at {int(worst)}; '
        f'{int((off > 0).sum())} of {off.numel()} are off')


def rotary(x, w, positions, inv_freq, sections, eps, interleaved):
    """Norm and rotation in fp64, differentiable in x and w (fp64 leaves)."""
    half, dim = sum(sections), x.shape[-1]
    axis = [a for a, n in enumerate(sections) for _ in range(n)]
    angle = (positions.double()[:, axis] * inv_freq.double())[:, None]
    cos, sin = angle.cos(), angle.sin()
    if w is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * w
    if interleaved:
        a, b = x[..., 0:2 * half:2], x[..., 1:2 * half:2]
    else:
        a, b = x[..., :half], x[..., half:2 * half]
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.cat([turned, x[..., 2 * half:dim]], -1)


def philox(n, key, offset):
    """Word i % 4 of Philox4x32-10 at counter (i // 4, offset), i < n (numpy)."""
    low = np.uint64(0xffffffff)
    s32 = np.uint64(32)
    block = np.arange((n + 3) // 4, dtype=np.uint64)
    key, offset = key % 2 ** 64, offset % 2 ** 64
    x = [block & low, block >> s32, np.full_like(block, offset & 0xffffffff), np.full_like(block, offset >> 32)]
    k0, k1 = key & 0xffffffff, key >> 32
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> s32) ^ x[1] ^ np.uint64(k0), b & low, (a >> s32) ^ x[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) % 2 ** 32, (k1 + 0xBB67AE85) % 2 ** 32
    return np.stack(x, 1).reshape(-1)[:n].astype(np.uint32)
