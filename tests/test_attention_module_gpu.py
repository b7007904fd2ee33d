"""SparseSelfAttention on tensors whose rows are not in the order of their samples."""
import pytest
import torch

from bevfusion_triton_b200.ops.spconv import SparseConvTensor, SparseSelfAttention, SparseSequential, SubMConv3d
from tests.test_attention_block_gpu import block64, no_wait_gave_up  # noqa: F401

pytestmark = pytest.mark.gpu


def scan(batch, per, channels, seed):
    g = torch.Generator().manual_seed(seed)
    rows = []
    for b in range(batch):
        cells = torch.randperm(8 * 30 * 30, generator=g)[:per[b]]
        rows.append(torch.stack([torch.full_like(cells, b), cells // 900, cells // 30 % 30, cells % 30], 1))
    indices = torch.cat(rows).int().cuda()
    return indices, torch.randn(len(indices), channels, generator=g).cuda()


@pytest.mark.parametrize('causal', [False, True])
def test_rows_in_any_order(cuda, causal):
    """Shuffled rows against the layer's definition in 64 bits, which picks each sample's rows by their index."""
    torch.manual_seed(1)
    indices, feats = scan(3, (70, 150, 31), 64, 0)
    mixed = torch.randperm(len(indices), generator=torch.Generator().manual_seed(5)).cuda()
    indices, feats = indices[mixed], feats[mixed].requires_grad_(True)
    layer = SparseSelfAttention(64, 4, 2, causal=causal).cuda()
    with torch.autocast('cuda', dtype=torch.float16):
        y = layer(SparseConvTensor(feats, indices, [8, 30, 30], 3))
    assert y.indices is indices
    order = torch.argsort(indices[:, 0], stable=True)  # the definition returns the samples one after another
    want, leaf, params = block64(layer, feats[order], indices[order], 3, None)
    back = torch.argsort(order)
    want = want[back]
    # about ten fp16 roundings in a row, each 2^-11 of values whose sums of products are taken over up to 150 terms
    close = lambda a, b: (a.double() - b).abs().max() <= 2.0 ** -5 * b.abs().max()  # noqa: E731
    assert close(y.features.detach(), want.detach())
    up = torch.randn_like(feats)
    names = [n for n, _ in layer.named_parameters()]
    got = torch.autograd.grad(y.features, [feats] + [t for _, t in layer.named_parameters()], up)
    ref = torch.autograd.grad(want, [leaf] + [params[n] for n in names], up.double())
    for n, a, b in zip(['features'] + names, got, [ref[0][back], *ref[1:]]):
        assert close(a, b), n


def test_order_of_rows_changes_nothing(cuda):
    """Whole samples in another order, and samples dealt out in turn: the same bits, each at its row.  (Within a sample
    the order stays, which the sums follow.)"""
    torch.manual_seed(2)
    indices, feats = scan(2, (90, 90), 32, 1)
    layer = SparseSelfAttention(32, 2, dropout=0.0).cuda().half().eval()
    feats = feats.half()
    want = layer(SparseConvTensor(feats, indices, [8, 30, 30], 2)).features
    n = torch.arange(180, device='cuda')
    for order in (torch.cat([n[90:], n[:90]]), n.view(2, 90).t().flatten()):
        got = layer(SparseConvTensor(feats[order], indices[order], [8, 30, 30], 2)).features
        assert torch.equal(got, want[order])
    layer.grouped = True  # known to be: the same bits without the gathering
    assert torch.equal(layer(SparseConvTensor(feats, indices, [8, 30, 30], 2)).features, want)


def test_after_a_submanifold_convolution(cuda):
    """A submanifold convolution hands rows on as they come; a sample's result does not depend on the other's rows."""
    torch.manual_seed(3)
    indices, feats = scan(2, (120, 40), 32, 2)
    stack = SparseSequential(SubMConv3d(32, 32, 3, indice_key='s'), SparseSelfAttention(32, 2)).cuda().half().eval()
    mixed = torch.randperm(160, generator=torch.Generator().manual_seed(7)).cuda()
    first = mixed[indices[mixed, 0] == 0]  # sample 0's rows in their mixed order
    both = stack(SparseConvTensor(feats[mixed].half(), indices[mixed], [8, 30, 30], 2)).features
    alone = stack(SparseConvTensor(feats[first].half(), indices[first], [8, 30, 30], 1)).features
    # the convolution's sums over 27 sites and the products of the layer may be blocked otherwise: fp16 roundings
    diff = (both[indices[mixed, 0] == 0].double() - alone.double()).abs().max()
    assert diff <= 2.0 ** -6 * alone.double().abs().max()


@pytest.mark.parametrize('train', [False, True])
def test_first_call_captured(cuda, train):
    """The layer's first call may be the captured one (after the library handles of its products are there); replays
    take new features and, training, draw new masks."""
    torch.manual_seed(4)
    indices, feats = scan(2, (60, 45), 32, 3)
    feats = feats.half()
    make = lambda: SparseSelfAttention(32, 2, dropout=0.5).cuda().half().train(train)  # noqa: E731
    side = torch.cuda.Stream()
    with torch.cuda.stream(side), torch.no_grad():  # another layer of the same shape: cuBLAS sets itself up
        make()(SparseConvTensor(feats, indices, [8, 30, 30], 2))
    torch.cuda.synchronize()
    layer, graph = make(), torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        y = layer(SparseConvTensor(feats, indices, [8, 30, 30], 2)).features
    seen = []
    for step in range(2):
        feats.add_(0.25 if step else 0.0)
        graph.replay()
        seen.append(y.clone())
        if not train:
            with torch.no_grad():
                assert torch.equal(y, layer(SparseConvTensor(feats, indices, [8, 30, 30], 2)).features)
    if train:  # a dropped value leaves the feature itself
        kept = [s != f for s, f in zip(seen, (feats - 0.25, feats))]
        assert not torch.equal(kept[0], kept[1])


@pytest.mark.parametrize('rows', [0, 1, 2])
@pytest.mark.parametrize('batch', [1, 3])
def test_hardly_any_sites(cuda, rows, batch):
    """No site, one, and one in each of two samples in descending order: a site that sees itself alone gets its value's
    projection; a training step gives finite gradients."""
    torch.manual_seed(5)
    layer = SparseSelfAttention(32, 2, dropout=0.1).cuda().half()
    indices = torch.tensor([[min(batch - 1, 1 - r), r, 4, 5] for r in range(rows)], dtype=torch.int32,
                           device='cuda').view(rows, 4)
    feats = torch.randn(rows, 32, device='cuda').half().requires_grad_(True)
    y = layer(SparseConvTensor(feats, indices, [8, 30, 30], batch)).features
    y.float().sum().backward()
    grads = [feats.grad] + [p.grad for p in layer.parameters()]
    assert y.shape == feats.shape and all(bool(torch.isfinite(t).all()) for t in [y, *grads])
    if batch > 1:
        with torch.no_grad():
            got = layer.eval()(SparseConvTensor(feats, indices, [8, 30, 30], batch)).features
            value = layer.qkv(layer.norm(feats))[:, 64:]
            want = feats + layer.proj(value)
        assert torch.equal(got, want)
