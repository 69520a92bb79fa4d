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
