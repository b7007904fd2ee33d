"""Function transforms over the attention-block operators, on the CPU: kernels of
a stand-in library behind the operators' own autograd kernels.  And the module's
own transform, its moves."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

from bevfusion_triton_b200._lib import ops
from bevfusion_triton_b200.ops.spconv import SparseSelfAttention


@pytest.fixture
def stand_in():
    O = ops()
    lib = torch.library.Library('bfb_b200', 'IMPL')
    lib.impl('packed_attention', lambda q, k, v, *a: (q + k + v, q.sum(2).t().float().contiguous()), 'CPU')
    lib.impl('packed_attention_backward', lambda g, gl, q, k, v, *a: (g + 0, g + 0, g + 0), 'CPU')
    lib.impl('qk_norm_rotary', lambda q, k, *a: (2 * q, 2 * k), 'CPU')
    lib.impl('qk_norm_rotary_backward', lambda gq, gk, q, k, *a: (2 * gq, 2 * gk, gq.sum((0, 1)), gk.sum((0, 1))), 'CPU')
    lib.impl('residual_dropout', lambda x, r, p, s: 3 * x if r is None else 3 * x + r, 'CPU')
    yield O
    lib._destroy()


def calls(O):
    """Each operator as a function of its differentiable arguments, and those."""
    q = torch.randn(6, 2, 8)
    cu, seed = torch.tensor([0, 6], dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    pos, freq, w = torch.randn(6, 1), torch.ones(4), torch.ones(8)
    lse = torch.zeros(2, 6)
    return {
        'attention': (lambda q, k, v: O.packed_attention(q, k, v, cu, cu, None, False, 1.0), (q, q + 1, q + 2)),
        'attention backward': (lambda g, gl, q: O.packed_attention_backward(g, gl, q, q, q, q, lse, cu, cu, None, False,
                                                                            1.0), (q, lse, q + 1)),
        'rotary': (lambda q, k, p, f, w: O.qk_norm_rotary(q, k, p, f, [4], w, w, 1e-6, False), (q, q + 1, pos, freq, w)),
        'rotary backward': (lambda g, q, w: O.qk_norm_rotary_backward(g, g, q, q, pos, freq, [4], w, None, 1e-6, False),
                            (q, q + 1, w)),
        'dropout': (lambda x, r: O.residual_dropout(x, r, 0.5, seed), (q, q + 1))}


NAMES = ['attention', 'attention backward', 'rotary', 'rotary backward', 'dropout']


@pytest.mark.parametrize('name', NAMES)
def test_forward_mode_is_refused(stand_in, name):
    """A tangent of any argument, alone, with or without reverse mode beside it: an error, not a tangent of zeros."""
    f, args = calls(stand_in)[name]
    for n, arg in enumerate(args):
        def one(x, n=n):
            return f(*args[:n], x, *args[n + 1:])

        with pytest.raises(NotImplementedError, match='no forward-mode derivative'):
            torch.func.jvp(one, (arg,), (torch.ones_like(arg),))
        for leaf in (False, True):
            with fwd.dual_level(), pytest.raises(NotImplementedError, match='no forward-mode derivative'):
                one(fwd.make_dual(arg.clone().requires_grad_(leaf), torch.ones_like(arg)))
        with fwd.dual_level():
            one(arg)  # no tangent: as ever


@pytest.mark.parametrize('name', ['attention', 'rotary', 'dropout'])
def test_vmap_calls_sample_by_sample(stand_in, name):
    f, args = calls(stand_in)[name]
    many = tuple(torch.stack([a, 2 * a, -a]) for a in args)
    got = torch.vmap(f)(*many)
    want = [f(*(m[i] for m in many)) for i in range(3)]
    for n, t in enumerate(got if isinstance(got, tuple) else (got,)):
        assert torch.equal(t, torch.stack([(w if isinstance(w, tuple) else (w,))[n] for w in want]))
    # reverse mode inside a transform is refused by torch for autograd functions in C++
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: (f(x, *args[1:])[0] if name != 'dropout' else f(x, *args[1:])).sum())(args[0])


def test_reverse_mode_through_the_stand_in(stand_in):
    """The fixture's kernels are those that run: gradients are theirs."""
    f, (x, r) = calls(stand_in)['dropout']
    x = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(f(x, r).sum(), x)
    assert torch.equal(dx, torch.full_like(x, 3.0))


def test_module_moves_its_frequencies():
    """They go where the parameters go, keep their fp32 values under .half(), and do not get lost on meta."""
    layer = SparseSelfAttention(64, 4)
    freq = layer.inv_freq.clone()
    moved = []
    layer.inv_freq = type('Spy', (), {'to': lambda self, device: moved.append(device) or freq})()
    layer.half()
    assert moved == [torch.device('cpu')] and layer.inv_freq is freq and 'inv_freq' not in layer.state_dict()
    layer.to('meta')
    assert layer.inv_freq is freq and torch.equal(layer.to_empty(device='cpu').inv_freq, freq)
