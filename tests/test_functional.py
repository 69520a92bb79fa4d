"""Refusals of the model's operators, and which layers of a module they stand in for (CPU)."""
import ctypes

import pytest
import torch
import torch.nn as nn


@pytest.fixture
def native():
    from elixir_b200 import _abi, build, _lib
    build.build()
    lib = ctypes.CDLL(_lib.lib_path())
    _abi.apply_prototypes(lib)
    return lib, _abi


def test_layer_norm_entry_points_reject_bad_arguments(native):
    lib, E = native
    a, odd = ctypes.c_void_p(64), ctypes.c_void_p(65)
    fwd = lambda x=a, w=a, b=a, dt=0, r=4, c=8, eps=1e-5, y=a, m=a, s=a: lib.elx_layer_norm_forward(x, w, b, dt, r, c, eps, y, m, s, None)    # noqa: E731
    assert fwd(x=None) == fwd(y=None) == fwd(m=None) == fwd(s=None) == E.ERR_NULL
    assert fwd(dt=5) == E.ERR_DTYPE
    assert fwd(r=-1) == fwd(c=0) == fwd(c=-3) == E.ERR_SIZE
    assert fwd(c=E.NORM_MAX_COLS + 1) == E.ERR_CAPACITY
    assert fwd(x=odd) == fwd(w=odd) == fwd(b=odd) == fwd(y=odd) == fwd(m=odd) == E.ERR_ALIGN
    assert fwd(eps=-1.0) == fwd(eps=float('nan')) == E.ERR_ARG
    assert fwd(r=0) == E.OK
    need = lib.elx_layer_norm_backward_workspace(4, 8)
    assert need > 0 and lib.elx_layer_norm_backward_workspace(-1, 8) == lib.elx_layer_norm_backward_workspace(1, 0) == E.ERR_SIZE
    bwd = lambda dy=a, x=a, w=a, m=a, s=a, dt=0, r=4, c=8, dx=a, dw=a, db=a, ws=a, n=need: lib.elx_layer_norm_backward(    # noqa: E731
        dy, x, w, m, s, dt, r, c, dx, dw, db, ws, n, None)
    assert bwd(dy=None) == bwd(x=None) == bwd(m=None) == bwd(s=None) == bwd(dx=None) == bwd(ws=None) == E.ERR_NULL
    assert bwd(dt=-1) == E.ERR_DTYPE and bwd(r=-1) == bwd(c=0) == E.ERR_SIZE
    assert bwd(n=need - 1) == bwd(c=E.NORM_MAX_COLS + 1) == E.ERR_CAPACITY
    assert bwd(dw=odd) == bwd(db=odd) == bwd(dx=odd) == bwd(dy=odd) == bwd(ws=ctypes.c_void_p(68)) == E.ERR_ALIGN


def test_embedding_entry_points_reject_bad_arguments(native):
    lib, E = native
    a, odd = ctypes.c_void_p(64), ctypes.c_void_p(65)
    fwd = lambda t=a, ib=8, n=4, w=a, dt=0, v=10, h=8, o=a: lib.elx_embedding_forward(t, ib, n, w, dt, v, h, 1.0, o, None)    # noqa: E731
    assert fwd(t=None) == fwd(w=None) == fwd(o=None) == E.ERR_NULL
    assert fwd(ib=2) == fwd(dt=9) == E.ERR_DTYPE
    assert fwd(n=-1) == fwd(v=0) == fwd(h=0) == E.ERR_SIZE
    assert fwd(n=2**31) == fwd(v=2**31) == fwd(h=2**30) == E.ERR_CAPACITY
    assert fwd(t=ctypes.c_void_p(68)) == fwd(w=odd) == fwd(o=odd) == E.ERR_ALIGN
    assert fwd(n=0, t=None, o=None) == E.OK
    need = lib.elx_embedding_backward_workspace(4, 8)
    assert need > 0 and lib.elx_embedding_backward_workspace(-1, 8) == lib.elx_embedding_backward_workspace(1, 0) == E.ERR_SIZE
    bwd = lambda t=a, ib=4, n=4, d=a, dt=0, v=10, h=8, p=-1, dw=a, ws=a, size=need: lib.elx_embedding_backward(    # noqa: E731
        t, ib, n, d, dt, v, h, 1.0, p, dw, ws, size, None)
    assert bwd(t=None) == bwd(d=None) == bwd(dw=None) == bwd(ws=None) == E.ERR_NULL
    assert bwd(ib=1) == bwd(dt=3) == E.ERR_DTYPE and bwd(n=-1) == bwd(v=0) == bwd(h=0) == E.ERR_SIZE
    assert bwd(p=-2) == bwd(p=10) == E.ERR_ARG
    assert bwd(size=need - 1) == bwd(n=2**31) == E.ERR_CAPACITY
    assert bwd(d=odd) == bwd(dw=odd) == bwd(ws=ctypes.c_void_p(72)) == E.ERR_ALIGN


def test_bindings_refuse_what_the_kernels_do_not_take():
    from elixir_b200 import functional as F, kernels as K
    x, w = torch.zeros(4, 8), torch.zeros(8)
    with pytest.raises(RuntimeError, match='no CPU path'):
        K.layer_norm_forward(x, w, w)
    with pytest.raises(RuntimeError, match='no CPU path'):
        K.layer_norm_backward(x, x, w, torch.zeros(4), torch.zeros(4))
    with pytest.raises(RuntimeError, match='no CPU path'):
        K.embedding_forward(torch.zeros(4, dtype=torch.int64), x)
    with pytest.raises(RuntimeError, match='no CPU path'):
        K.embedding_backward(torch.zeros(4, dtype=torch.int64), x, 10)
    with pytest.raises(RuntimeError, match='no CPU path'):
        K.pack_moments(w, w)
    with pytest.raises(ValueError):
        K.layer_norm_forward(torch.zeros(8, 4).t(), w)
    with pytest.raises(ValueError):
        F.layer_norm(x, (4, ))
    with pytest.raises(ValueError):
        F.layer_norm(x, (8, ), torch.zeros(4))
    with pytest.raises(ValueError):
        F.layer_norm(x, ())
    for bad in (4, -5):
        with pytest.raises(ValueError):
            F.embedding(torch.zeros(2, dtype=torch.int64), x, padding_idx=bad)


class Scaled(nn.Embedding):

    def forward(self, tokens):
        return 2 * super().forward(tokens)


class Named(nn.LayerNorm):
    pass


def test_layers_of_a_module(monkeypatch):
    """Which layers change hands, and that CPU calls of them still are torch's."""
    from elixir_b200 import functional as F
    model = nn.Sequential(nn.Embedding(10, 8, padding_idx=1), nn.LayerNorm(8), Named(8, elementwise_affine=False), nn.Linear(8, 8),
                          Scaled(10, 8), nn.GroupNorm(2, 8))
    before = [dict(m.__dict__) for m in model]
    tokens, x = torch.tensor([[1, 2], [3, 9]]), torch.randn(3, 8)
    want = (model[0](tokens), model[1](x), model[2](x))
    assert F.use_kernels(model) == 3
    assert ['forward' in m.__dict__ for m in model] == [True, True, True, False, False, False]
    assert all(b.keys() <= m.__dict__.keys() for b, m in zip(before, model))
    assert all(torch.equal(a, b) for a, b in zip(want, (model[0](tokens), model[1](x), model[2](x))))
    assert F.use_kernels(model) == 3    # a second time changes nothing
    assert torch.equal(want[1], model[1](x))
    import copy
    twin = copy.deepcopy(model)
    with torch.no_grad():
        twin[1].weight.fill_(3.0)
    assert not torch.equal(twin[1](x), model[1](x)) and torch.equal(want[1], model[1](x))
    assert list(twin.state_dict()) == list(model.state_dict())


def test_a_layer_keeps_a_forward_of_its_own():
    """Set on the layer, before or after the layers change hands, or on the class by a program that patches torch."""
    from elixir_b200 import functional as F
    tokens, x = torch.tensor([[1, 2], [3, 9]]), torch.randn(3, 8)
    model = nn.Sequential(nn.Embedding(10, 8), nn.LayerNorm(8), nn.LayerNorm(8))
    want = [2 * model[0](tokens), 2 * model[1](x), model[2](x)]
    for layer in model[:2]:
        layer.forward = lambda t, own=layer.forward: 2 * own(t)
    own = [layer.__dict__['forward'] for layer in model[:2]]
    for _ in range(2):
        assert F.use_kernels(model) == 1
        assert [layer.__dict__['forward'] for layer in model[:2]] == own
        assert all(torch.equal(w, layer(t)) for w, layer, t in zip(want, model, (tokens, x, x)))
    model[2].forward = lambda t, own=model[2].forward: 3 * own(t)    # around the one that use_kernels put there
    assert F.use_kernels(model) == 0 and torch.equal(model[2](x), 3 * want[2])


@pytest.mark.parametrize('kind,shape', [(nn.LayerNorm, (8, )), (nn.Embedding, (10, 8))])
def test_a_class_keeps_a_forward_that_it_was_given(monkeypatch, kind, shape):
    from elixir_b200 import functional as F
    t = torch.randn(3, 8) if kind is nn.LayerNorm else torch.tensor([[1, 2], [3, 9]])
    early, late = kind(*shape), kind(*shape)
    assert F.use_kernels(early) == 1
    want, torch_forward = 2 * early(t), kind.forward
    monkeypatch.setattr(kind, 'forward', lambda layer, t: 2 * torch_forward(layer, t))
    assert F.use_kernels(late) == 0 and 'forward' not in late.__dict__
    monkeypatch.setattr(F, '_plain_cuda', lambda *a: True)    # as with CUDA tensors: the patch comes first all the same
    assert torch.equal(early(t), want)


@pytest.mark.parametrize('kind,shape', [(nn.LayerNorm, (8, )), (nn.Embedding, (10, 8))])
def test_a_class_keeps_a_forward_that_it_had_before_the_import(monkeypatch, kind, shape):
    import functools
    import importlib.util
    import elixir_b200.functional as F
    torch_forward = kind.forward

    @functools.wraps(torch_forward)
    def patched(layer, t):
        return 2 * torch_forward(layer, t)

    monkeypatch.setattr(kind, 'forward', patched)
    spec = importlib.util.spec_from_file_location('elixir_b200._imported_late', F.__file__)
    late = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(late)
    layer = kind(*shape)
    assert late.use_kernels(layer) == 0 and 'forward' not in layer.__dict__
    monkeypatch.undo()
    assert late._torch_forward(kind) is torch_forward and F._TORCH_FORWARD[kind] is torch_forward


def test_layers_leave_fake_tensors_and_subclasses_to_torch(monkeypatch):
    """A fake CUDA tensor has no memory that a kernel could take."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from elixir_b200 import functional as F, kernels as K

    def never(*args, **kw):
        raise AssertionError('a kernel was called')

    for name in ('layer_norm_forward', 'embedding_forward'):
        monkeypatch.setattr(K, name, never)
    with FakeTensorMode():
        model = nn.Sequential(nn.Embedding(10, 8, device='cuda'), nn.LayerNorm(8, device='cuda'))
        assert F.use_kernels(model) == 2
        out = model(torch.zeros(3, 4, dtype=torch.int64, device='cuda'))
    assert out.shape == (3, 4, 8) and out.is_cuda
    assert model[1](out).is_cuda    # outside the mode as well
