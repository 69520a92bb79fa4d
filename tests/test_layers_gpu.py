"""Layers of a module that run this package's kernels: what torch's own layers do beside a forward and a backward pass
(forward-mode derivatives, fake tensors, dispatch modes, compilation) still works and gives what torch gives."""
import copy

import pytest
import torch
import torch.autograd.forward_ad as fwAD
import torch.nn as nn
from torch.utils._python_dispatch import TorchDispatchMode

pytestmark = pytest.mark.gpu


class Model(nn.Module):

    def __init__(self, width=40):
        super().__init__()
        self.embed = nn.Embedding(30, width, padding_idx=2)
        self.norm = nn.LayerNorm(width)
        self.plain = nn.LayerNorm((4, width // 4), elementwise_affine=False)
        self.no_bias = nn.LayerNorm(width, bias=False)

    def forward(self, tokens):
        x = self.norm(self.embed(tokens))
        return self.no_bias(self.plain(x.unflatten(-1, (4, -1))).flatten(-2) + torch.tanh(x))


@pytest.fixture
def models(cuda):
    """A model of torch's layers, the same with this package's, and tokens."""
    from elixir_b200 import functional as F
    torch.manual_seed(0)
    theirs = Model().to(cuda)
    ours = copy.deepcopy(theirs)
    assert F.use_kernels(ours) == 4
    return theirs, ours, torch.randint(30, (3, 7), device=cuda)


@pytest.fixture
def launches(monkeypatch):
    """How often the kernels' forward passes were called."""
    from elixir_b200 import kernels as K
    calls = []
    for name in ('layer_norm_forward', 'embedding_forward'):
        def counted(*args, _own=getattr(K, name), **kw):
            calls.append(1)
            return _own(*args, **kw)
        monkeypatch.setattr(K, name, counted)
    return calls


def test_the_kernels_run_where_nothing_watches(models, launches):
    _, ours, tokens = models
    ours(tokens).sum().backward()
    assert len(launches) == 4
    with torch.device('cuda'):    # a default device is no reason
        ours(tokens)
    assert len(launches) == 8


def test_forward_mode_derivatives(models, launches):
    theirs, ours, tokens = models
    tangents = {n: torch.randn_like(p) for n, p in theirs.named_parameters()}
    out = []
    for model in (theirs, ours):
        with fwAD.dual_level():
            dual = {n: fwAD.make_dual(p.detach(), tangents[n]) for n, p in model.named_parameters()}
            out.append(fwAD.unpack_dual(torch.func.functional_call(model, dual, (tokens, ))))
    assert out[1].tangent is not None and not launches
    assert torch.equal(out[0].primal, out[1].primal) and torch.equal(out[0].tangent, out[1].tangent)


def test_fake_tensors_dispatch_modes_and_compilation(models, launches):
    from torch._subclasses.fake_tensor import FakeTensorMode
    theirs, ours, tokens = models
    want = theirs(tokens)

    class Names(TorchDispatchMode):

        def __init__(self):
            super().__init__()
            self.names = []

        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            self.names.append(str(func))
            return func(*args, **(kwargs or {}))

    seen = []
    for model in (theirs, ours):
        with Names() as mode, torch.no_grad():
            assert torch.equal(model(tokens), want)
        seen.append(mode.names)
    assert seen[0] == seen[1] and any('layer_norm' in n for n in seen[1]) and any('embedding' in n for n in seen[1])
    with FakeTensorMode(allow_non_fake_inputs=True):
        assert ours(tokens).shape == want.shape
    assert not launches
    assert torch.equal(torch.compile(ours, backend='eager', fullgraph=True)(tokens), want)
    assert not launches
    # (the check of a trace calls the module itself once more)
    assert torch.equal(torch.jit.trace(ours, (tokens, ), check_trace=False)(tokens), want)
    assert not launches


def test_second_derivatives(models, launches):
    """A penalty on the gradients, its own gradients with respect to every parameter: within the roundings of an fp32
    evaluation of torch's, whose order of sums differs in the first forward pass only."""
    theirs, ours, tokens = models
    weight = torch.randn(3, 7, 40, device=tokens.device)
    grads = []
    for model in (theirs, ours, copy.deepcopy(theirs).double()):
        dtype = model.norm.weight.dtype
        loss = torch.tanh(model(tokens) * weight.to(dtype)).sum()
        first = torch.autograd.grad(loss, list(model.parameters()), create_graph=True)
        second = torch.autograd.grad(sum(g.pow(2).sum() for g in first), list(model.parameters()))
        grads.append((first, second))
    assert len(launches) == 4
    for torchs, mine, exact in zip(*(first + second for first, second in grads)):
        # a few hundred roundings of numbers of the gradients' size lie between the tokens and a second derivative
        assert mine.shape == exact.shape and bool((mine.double() - exact).norm() <= 1000 * 2.0**-24 * exact.norm())
    assert bool((grads[1][0][0][2] == 0).all()) and bool((grads[1][1][0][2] == 0).all())    # the padding token


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16])
def test_second_derivatives_in_16_bits(models, dtype):
    """Those of the same layers in torch, from the same values.  After the forward pass, whose results differ by a rounding
    here and there, both run the same operators."""
    theirs, ours, tokens = models
    theirs, ours = theirs.to(dtype), ours.to(dtype)
    grads = []
    for model in (theirs, ours):
        first = torch.autograd.grad(torch.tanh(model(tokens)).float().sum(), list(model.parameters()), create_graph=True)
        grads.append(first + torch.autograd.grad(sum(g.float().pow(2).sum() for g in first), list(model.parameters())))
    for torchs, mine in zip(*grads):
        # torch's operators leave fp16's range on the way to some second derivatives, for its own layers as well
        assert mine.dtype == dtype and torch.equal(torch.isfinite(mine), torch.isfinite(torchs))
        mine, torchs = (torch.where(torch.isfinite(t), t, 0.0).double() for t in (mine, torchs))
        # some thirty roundings of half a step, on both sides
        assert bool((mine - torchs).norm() <= 60 * torch.finfo(dtype).eps / 2 * torchs.norm())
    if dtype == torch.bfloat16:
        assert all(bool(torch.isfinite(g).all()) for g in grads[1])


def test_second_derivatives_past_a_token_outside_the_table(cuda):
    """Such a token reads as a row of NaN and adds to no row, in a differentiated backward pass as in a plain one."""
    from elixir_b200 import functional as F
    layer = nn.Embedding(10, 8).to(cuda)
    F.use_kernels(layer)
    scale = torch.ones(4, 8, device=cuda, requires_grad=True)
    out = layer(torch.tensor([1, 10, -1, 3], device=cuda)).nan_to_num(0.0)
    g, = torch.autograd.grad((out * scale).sum(), layer.weight, create_graph=True)
    want = torch.zeros(10, 8, device=cuda)
    want[[1, 3]] = 1
    assert torch.equal(g, want)
    twice, = torch.autograd.grad(g.sum(), scale)
    assert torch.equal(twice, torch.tensor([1.0, 0, 0, 1], device=cuda)[:, None].expand(4, 8))
