"""The operators together, as a training program runs them: a wrapped model whose embedding and layer norms run this
package's kernels, with the 8-bit optimizer, one rank over NCCL."""
import copy
import math

import pytest
import torch
import torch.distributed as dist
import torch.nn as nn

import _moments8 as ref

pytestmark = pytest.mark.gpu


class Model(nn.Module):
    """Token embedding with a padding token, a tied head, layer norms with and without parameters."""

    def __init__(self, vocab=211, width=64, tied=True):
        super().__init__()
        self.embed = nn.Embedding(vocab, width, padding_idx=3)
        self.norms = nn.ModuleList([nn.LayerNorm(width, elementwise_affine=i != 1) for i in range(6)])
        self.layers = nn.ModuleList([nn.Linear(width, width) for _ in range(6)])
        self.head = nn.Linear(width, vocab, bias=False)
        if tied:
            self.head.weight = self.embed.weight

    def forward(self, tokens):
        x = self.embed(tokens)
        for norm, layer in zip(self.norms, self.layers):
            x = x + torch.tanh(layer(norm(x)))
        return self.head(x)


@pytest.fixture
def one_rank(cuda, tmp_path):
    created = not dist.is_initialized()
    if created:
        dist.init_process_group('nccl', init_method=f'file://{tmp_path}/store', rank=0, world_size=1, device_id=cuda)
    yield dist.GroupMember.WORLD
    if created:
        dist.destroy_process_group()


def _wrap(model, group, dtype, fused, blocks=None, **optim):
    from elixir_b200.optim import HybridAdam
    from elixir_b200.wrapper import ElixirModule, ElixirOptimizer, simple_plan
    plan = simple_plan(model, 1, unified_dtype=dtype, chunk_size=14000, public_block_number=blocks)
    inner = HybridAdam(model.parameters(), **{**dict(lr=1e-2, weight_decay=0.01), **optim})
    emodel = ElixirModule(model, plan, group, dtype=dtype, use_fused_kernels=fused)
    return emodel, ElixirOptimizer(emodel, inner, initial_scale=2.0**10)


def _tokens(step, cuda, n=(4, 37), vocab=211):
    gen = torch.Generator().manual_seed(step)
    return torch.randint(vocab, n, generator=gen).to(cuda)


def _gradients(emodel, eopt):
    """What the step will read: the landed gradients of every parameter, unscaled."""
    out = {}
    for name, param in emodel.grad_state_dict.items():
        chunk = emodel.fetcher.get_one_chunk(param)
        info = chunk.tensors_info[param]
        out[name] = chunk.shard[info.offset:info.end].float().div(eopt.loss_scale).view(param.shape)
    return out


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('tied,blocks', [(True, None), (False, None), (False, 3)])
def test_gradients_and_update_of_a_wrapped_model(cuda, one_rank, dtype, tied, blocks):
    """Gradients of the wrapped model against float64 autograd of the same working copies, then the update of every chunk
    against the restatement given those gradients."""
    torch.manual_seed(0)
    plain = Model(tied=tied)
    model = copy.deepcopy(plain)
    emodel, eopt = _wrap(model, one_rank, dtype, True, blocks, state_bits=8)
    exact = plain.to(cuda).to(dtype).double()
    layers = [m for m in model.modules() if 'forward' in m.__dict__]
    assert len(layers) == 7    # the embedding and six norms
    tokens = _tokens(0, cuda)
    loss_of = lambda logits: nn.functional.cross_entropy(logits.flatten(0, 1), tokens.roll(1).flatten())    # noqa: E731
    eopt.backward(loss_of(emodel(tokens).float()))
    loss_of(exact(tokens)).backward()
    got = _gradients(emodel, eopt)
    want = dict(exact.named_parameters())
    # About 50 roundings of activations and gradients in the type of the model lie between a parameter and the loss; they
    # add up like independent errors in the 2-norm: sqrt(50) * half a step, doubled for their growth along the way.
    bound = 2 * math.sqrt(50) * max(torch.finfo(dtype).eps / 2, 2.0**-20)
    for name, g in got.items():
        if name in want:
            w = want[name].grad
            assert float((g.double() - w).norm()) <= bound * float(w.norm()) + 1e-12, name
    if not tied:
        assert bool((got['embed.weight'][3] == 0).all())    # the padding token
    shards = [[t.clone() for t in s[:4]] for s in eopt.engine.shards]
    eopt.step()
    ctl = eopt.engine.read_control()
    assert ctl.step == 1 and ctl.status == 0
    for c, ((master, sm, sv, grad), now) in enumerate(zip(shards, eopt.engine.shards)):
        p, moved, sm, sv = ref.adam8(master.cpu().numpy(), sm.cpu().numpy(), sv.cpu().numpy(), grad.float().cpu().numpy(),
                                     eopt.engine.table._segs_of(c), eopt.optim.hyper_table(), 1,
                                     None if ctl.div_scale < 0 else ctl.div_scale, index=c)
        off = torch.from_numpy(p).to(cuda) - now[0]
        assert bool((off.abs() <= torch.from_numpy(abs(p) * 2.0**-24 + moved * 2.0**-20).to(cuda)).all())
        assert ref.same_state(now[1].cpu().numpy(), sm, p.size, True) and ref.same_state(now[2].cpu().numpy(), sv, p.size, False)
        assert torch.equal(now[3], now[0].to(dtype))


def test_steps_repeat_bit_for_bit(cuda, one_rank):
    """Nothing on the path adds in an undefined order: two trainings from one start end in the same bits (fp32 matrix
    products of torch included: they are deterministic for one shape on one GPU)."""
    ends = []
    for _ in range(2):
        torch.manual_seed(1)
        emodel, eopt = _wrap(Model(tied=False), one_rank, torch.float16, True, state_bits=8)
        for step in range(4):
            tokens = _tokens(step, cuda)
            logits = emodel(tokens)
            eopt.backward(nn.functional.cross_entropy(logits.float().flatten(0, 1), tokens.roll(1).flatten()))
            eopt.step()
        ends.append([t.clone() for s in eopt.engine.shards for t in s[:4]])
    assert all(torch.equal(a, b) for a, b in zip(*ends))


def test_a_token_outside_the_table_skips_the_step(cuda, one_rank):
    torch.manual_seed(2)
    emodel, eopt = _wrap(Model(tied=False), one_rank, torch.float16, True, state_bits=8)
    before = [[t.clone() for t in s[:3]] for s in eopt.engine.shards]
    tokens = _tokens(0, cuda)
    targets = tokens.roll(1).flatten()
    tokens[1, 4] = 211
    eopt.backward(nn.functional.cross_entropy(emodel(tokens).float().flatten(0, 1), targets))
    eopt.step()
    assert eopt.engine.read_control().skip == 1
    for old, s in zip(before, eopt.engine.shards):
        assert all(torch.equal(a, b) for a, b in zip(old, s))


def test_checkpointed_layers_and_autocast(cuda, one_rank):
    """Recomputed forwards go through the kernels as well; under autocast the layers are torch's."""
    from torch.utils.checkpoint import checkpoint

    class Checkpointed(Model):

        def forward(self, tokens):
            x = self.embed(tokens)
            for norm, layer in zip(self.norms, self.layers):
                x = x + checkpoint(lambda t, n=norm, l=layer: torch.tanh(l(n(t))), x, use_reentrant=False)
            return self.head(x)

    grads = []
    for cls in (Model, Checkpointed):
        torch.manual_seed(3)
        emodel, eopt = _wrap(cls(tied=False), one_rank, torch.float16, True)
        tokens = _tokens(0, cuda)
        eopt.backward(emodel(tokens).float().pow(2).mean())
        grads.append(_gradients(emodel, eopt))
    assert all(torch.equal(grads[0][n], grads[1][n]) for n in grads[0])
    from elixir_b200 import functional as F
    layer = nn.LayerNorm(32).to(cuda)
    x = torch.randn(5, 32, device=cuda)
    F.use_kernels(layer)
    with torch.autocast('cuda', dtype=torch.float16):
        assert torch.equal(layer(x), nn.functional.layer_norm(x, (32, ), layer.weight, layer.bias))


def test_the_8_bit_optimizer_is_refused_where_it_does_not_run(cuda, one_rank):
    """Shards in host memory."""
    from elixir_b200.optim import HybridAdam
    from elixir_b200.wrapper import ElixirModule, ElixirOptimizer, simple_plan
    model = Model()
    plan = simple_plan(model, 1, unified_dtype=torch.float16, chunk_size=14000, shard_device='cpu')
    emodel = ElixirModule(model, plan, one_rank, dtype=torch.float16)
    with pytest.raises(ValueError, match='device-resident'):
        ElixirOptimizer(emodel, HybridAdam(model.parameters(), state_bits=8))
