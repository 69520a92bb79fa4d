"""8-bit moments on the CPU: the form itself against its definition (through the host-memory restatement of the C ABI),
the optimizer that holds its moments in it, checkpoints between both forms, and every refusal."""
import ctypes

import numpy as np
import pytest
import torch
import torch.distributed as dist

import _moments8 as ref


@pytest.fixture(scope='module')
def host_backend(tmp_path_factory):
    from elixir_b200 import _lib
    from _dist_workers import use_host_shim
    before = (_lib._LIB, _lib._HOST_MEMORY)
    use_host_shim()
    created = False
    if not dist.is_initialized():
        store = tmp_path_factory.mktemp('rdzv') / 'store'
        dist.init_process_group('gloo', init_method=f'file://{store}', rank=0, world_size=1)
        created = True
    yield
    if created:
        dist.destroy_process_group()
    _lib._LIB, _lib._HOST_MEMORY = before


def _moments(n, seed):
    rng = np.random.default_rng(seed)
    size = np.exp(4 * rng.standard_normal((n + 63) // 64)).repeat(64)[:n] * 1e-4
    m = (rng.standard_normal(n) * size).astype(np.float32)
    v = (rng.standard_normal(n)**2 * size**2).astype(np.float32)
    m[rng.random(n) < 0.05] = 0
    v[rng.random(n) < 0.05] = 0
    return m, v


@pytest.mark.parametrize('n', [1, 15, 16, 17, 255, 256, 257, 4096, 5003])
def test_pack_and_unpack_follow_the_definition(host_backend, n):
    from elixir_b200 import kernels as K
    m, v = _moments(n, n)
    sm, sv = K.pack_moments(torch.from_numpy(m), torch.from_numpy(v))
    assert sm.numel() == sv.numel() == K.moment_state_bytes(n) == _lib().elx_moment_state_bytes(n)
    assert ref.same_state(sm.numpy(), ref.encode(m.astype(np.float64), True, 0.5), n, True)
    assert ref.same_state(sv.numpy(), ref.encode(v.astype(np.float64), False, 0.5), n, False)
    end = ref.round_up(n, 16) + (n + 255) // 256
    assert not any(s.numpy()[a:b].any() for s in (sm, sv) for a, b in ((n, ref.round_up(n, 16)), (end, s.numel())))
    out = torch.empty(n), torch.empty(n)
    K.unpack_moments(sm, sv, *out)
    assert np.array_equal(out[0].numpy(), ref.decode(sm.numpy(), n, True))
    assert np.array_equal(out[1].numpy(), ref.decode(sv.numpy(), n, False))
    again = torch.empty(n), torch.empty(n)    # what was held is held exactly (under a smaller exponent where the top was rounded down)
    K.unpack_moments(*K.pack_moments(*out), *again)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1])


def _lib():
    from elixir_b200 import _lib as loader
    return loader.get()


def test_extreme_values(host_backend):
    from elixir_b200 import kernels as K
    tiny, big = np.float32(1e-45), np.float32(3.4e38)
    for values in ([0.0], [tiny], [big], [big, tiny], [1.875], [np.nextafter(np.float32(1.875), np.float32(2))], [np.inf, 1.0],
                   [np.nan, 1.0], [-0.0, 1e-30], [2.0**-126], [1.0] + [2.0**-20] * 300):
        x = np.array(values, dtype=np.float32)
        sm, sv = K.pack_moments(torch.from_numpy(x), torch.from_numpy(np.abs(x)))
        assert ref.same_state(sm.numpy(), ref.encode(x.astype(np.float64), True, 0.5), x.size, True), values
        assert ref.same_state(sv.numpy(), ref.encode(np.abs(x).astype(np.float64), False, 0.5), x.size, False), values
        out = torch.empty(x.size), torch.empty(x.size)
        K.unpack_moments(sm, sv, *out)
        finite = np.isfinite(x).reshape(1, -1).all() if x.size <= 256 else True
        assert torch.isfinite(out[0]).all() == bool(finite)
        if finite:
            # rounded to nearest with 3 mantissa bits: half a step is 2^-4 of the value, or 2^-18 of the block's power of
            # two (2^-126 at least: E >= 1) for what falls below the smallest binade; the largest number the form holds
            # is 1.875 * 2^126
            held = np.clip(x.astype(np.float64), -1.875 * 2.0**126, 1.875 * 2.0**126)
            off = np.abs(out[0].numpy().astype(np.float64) - held)
            assert np.all(off <= np.maximum(np.abs(held) * 2.0**-4, max(np.abs(held).max(), 2.0**-126) * 2.0**-18)), values
        assert torch.all((out[1] > 0) | torch.from_numpy(x == 0) | ~torch.isfinite(out[1])), 'a second moment became zero'


def _wrapped(state_bits, seed=0, **kw):
    import torch.nn as nn
    from elixir_b200.optim import HybridAdam
    from elixir_b200.wrapper import ElixirModule, ElixirOptimizer, simple_plan
    torch.manual_seed(seed)
    model = nn.Sequential(nn.Linear(24, 40), nn.LayerNorm(40), nn.Linear(40, 10))
    sr = simple_plan(model, 1, chunk_size=1100, unified_dtype=torch.float16, shard_device='cpu', rcache_device='cpu')
    inner = HybridAdam([dict(params=[model[0].weight, model[2].weight], weight_decay=0.1),
                        dict(params=[p for n, p in model.named_parameters() if p.dim() == 1])], lr=1e-2, state_bits=state_bits)
    emodel = ElixirModule(model, sr, dist.GroupMember.WORLD, dtype=torch.float16)
    return emodel, ElixirOptimizer(emodel, inner, initial_scale=64.0, **kw)


def _grads(emodel, step, scale=64.0, bad=False):
    gen = torch.Generator().manual_seed(100 + step)
    grads = {n: (torch.randn(p.shape, generator=gen) * 0.01 * scale).half() for n, p in emodel.grad_state_dict.items()}
    if bad:
        next(iter(grads.values())).view(-1)[3] = float('inf')
    return grads


def test_optimizer_steps_follow_the_definition(host_backend):
    """Applied and skipped steps, two param groups, chunk padding: masters within the rounding of the restatement, states
    equal code for code."""
    emodel, eopt = _wrapped(8)
    eng = eopt.engine
    hypers = eopt.optim.hyper_table()
    state = [[s[0].numpy().astype(np.float64), s[1].numpy().copy(), s[2].numpy().copy()] for s in eng.shards]
    applied = 0
    for step in range(4):
        bad = step == 2
        emodel.inject_gradients(_grads(emodel, step, bad=bad))
        landed = [s[3].clone().float().numpy() for s in eng.shards]
        before = [s[0].clone() for s in eng.shards]
        eopt.step()
        if bad:
            assert eng.read_control().skip == 1
            assert all(torch.equal(a, s[0]) for a, s in zip(before, eng.shards))
            for st, s in zip(state, eng.shards):
                assert np.array_equal(st[1], s[1].numpy()) and np.array_equal(st[2], s[2].numpy())
            continue
        applied += 1
        for c, s in enumerate(eng.shards):
            p, moved, sm, sv = ref.adam8(before[c].numpy(), state[c][1], state[c][2], landed[c], eng.table._segs_of(c), hypers,
                                         applied, 64.0, index=c)
            # the restatement rounds once, from double: half a unit of fp32
            assert np.all(np.abs(s[0].numpy() - p) <= np.abs(p) * 2.0**-24 + 1e-45)
            assert ref.same_state(s[1].numpy(), sm, p.size, True) and ref.same_state(s[2].numpy(), sv, p.size, False)
            assert torch.equal(s[3], s[0].half())
            state[c] = [p, s[1].numpy().copy(), s[2].numpy().copy()]
    assert eng.read_control().step == applied == 3
    first = next(iter(eopt.param_to_range))
    assert eopt.state[first] == dict(step=3)    # no views of moments that are not numbers
    m, v = eng.moments(0)
    assert np.array_equal(m.numpy(), ref.decode(state[0][1], m.numel(), True)) and float(v.min()) >= 0


@pytest.mark.parametrize('saved_bits,loaded_bits', [(8, 8), (32, 8), (8, 32)])
def test_checkpoints_move_between_both_forms(host_backend, saved_bits, loaded_bits):
    emodel, eopt = _wrapped(saved_bits)
    for step in range(2):
        emodel.inject_gradients(_grads(emodel, step))
        eopt.step()
    saved = eopt.state_dict()
    assert saved['shards'][0]['exp_avg'].dtype == (torch.uint8 if saved_bits == 8 else torch.float32)
    other, oopt = _wrapped(loaded_bits)
    oopt.load_state_dict(saved)
    for c in range(eopt.engine.n_chunks):
        n = eopt.engine.shards[c][0].numel()
        mine, theirs = eopt.engine.moments(c), oopt.engine.moments(c)
        for k, signed in ((0, True), (1, False)):
            want = mine[k].numpy().astype(np.float64)
            if loaded_bits == 8 and saved_bits == 32:
                want = ref.decode(ref.encode(want, signed, 0.5), n, signed)
            assert np.array_equal(theirs[k].numpy(), want)
    assert oopt.engine.read_control().step == 2


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float64])
@pytest.mark.parametrize('loaded_bits', [8, 32])
@pytest.mark.parametrize('strided', [False, True])
def test_checkpoints_hold_moments_of_any_floating_type(host_backend, loaded_bits, dtype, strided):
    """As a checkpoint that was thinned out has them, and as ``engine.moments(i, torch.bfloat16)`` hands them out."""
    emodel, eopt = _wrapped(8)
    for step in range(2):
        emodel.inject_gradients(_grads(emodel, step))
        eopt.step()
    saved = eopt.state_dict()
    for c, entry in enumerate(saved['shards']):
        m, v = eopt.engine.moments(c, torch.bfloat16 if dtype is torch.bfloat16 else torch.float32)
        entry.update(exp_avg=m.to(dtype), exp_avg_sq=v.to(dtype))
        if strided:
            entry.update((k, t.repeat_interleave(2)[::2]) for k, t in list(entry.items()))
    _, oopt = _wrapped(loaded_bits)
    oopt.load_state_dict(saved)
    for c, entry in enumerate(saved['shards']):
        for theirs, key, signed in zip(oopt.engine.moments(c), ('exp_avg', 'exp_avg_sq'), (True, False)):
            want = entry[key].float().numpy().astype(np.float64)
            if loaded_bits == 8:
                want = ref.decode(ref.encode(want, signed, 0.5), want.size, signed)
            assert np.array_equal(theirs.numpy(), want)


def test_engine_step_from_zero_moments_and_sizes_of_one(host_backend):
    from elixir_b200 import kernels as K
    from elixir_b200.engine import ChunkStepEngine
    eng = ChunkStepEngine('cpu', torch.bfloat16, state_bits=8)
    for n in (1, 2, 300):
        eng.add_shard(torch.ones(n), torch.full((n, ), 0.5, dtype=torch.bfloat16), n, [(0, n, 0)])
    eng.finalize()
    eng.set_hyper([K.hyper(lr=0.1)])
    eng.probe()
    eng.step()
    for c in range(3):    # a first step moves by lr towards the gradient's sign
        assert torch.allclose(eng.shards[c][0], torch.tensor(0.9), atol=1e-6)
    assert eng.moments(0)[0].item() in (0.046875, 0.05078125)    # 0.05 is held as one of its neighbours (1 + t/8) 2^-5


def test_a_block_that_is_not_finite_is_reported(host_backend):
    """A finite gradient whose square passes fp32's range, and a block that was lost before."""
    from elixir_b200 import _abi, kernels as K
    from elixir_b200.engine import ChunkStepEngine
    for lost in (False, True):
        eng = ChunkStepEngine('cpu', torch.bfloat16, state_bits=8)
        grad = torch.full((600, ), 0.5, dtype=torch.bfloat16)
        grad[300] = 0.5 if lost else 1e21
        eng.add_shard(torch.ones(600), grad, 600, [(0, 600, 0)])
        if lost:
            eng.shards[0][2][ref.round_up(600, 16) + 1] = 255
        eng.finalize()
        eng.set_hyper([K.hyper()])
        eng.probe()
        eng.step()
        ctl = eng.read_control()
        assert ctl.skip == 0 and ctl.late_inf == 1 and ctl.status == _abi.STAT_LATE_INF
        m, v = eng.moments(0)
        assert torch.equal(torch.isnan(v), (torch.arange(600) // 256) == 1) and bool(torch.isfinite(m).all())
        with pytest.raises(RuntimeError, match='8-bit moments'):
            eng.check_status()


def test_refusals(host_backend):
    from elixir_b200 import _abi, kernels as K
    from elixir_b200.engine import ChunkStepEngine
    from elixir_b200.optim import FusedAdam, HybridAdam
    param = [torch.nn.Parameter(torch.zeros(4))]
    for cls in (HybridAdam, FusedAdam):
        with pytest.raises(ValueError):
            cls(param, state_bits=16)
    with pytest.raises(ValueError):
        ChunkStepEngine('cpu', torch.float16, state_bits=4)
    table = K.ChunkTable('cpu', torch.float16, state_bits=8)
    n = 300
    p, g, s = torch.zeros(n), torch.zeros(n, dtype=torch.float16), torch.zeros(K.moment_state_bytes(n), dtype=torch.uint8)
    with pytest.raises(TypeError):
        table.add_chunk(p, torch.zeros(n), torch.zeros(n), g, n)    # fp32 moments in an 8-bit table
    with pytest.raises(ValueError):
        table.add_chunk(p, s[:-1], s, g, n)
    with pytest.raises(ValueError):
        table.add_chunk(p, s, s, g, n, [(0, n, 0)])    # one array for both
    table.add_chunk(p, s, s.clone(), g, n, [(0, n, 0)])
    table.finalize().set_hyper([K.hyper()])
    with pytest.raises(TypeError):
        K.ChunkTable('cpu', torch.float16).add_chunk(p, s, s, g, n)    # 8-bit state in an fp32 table
    ctl = K.ControlBlock('cpu', 1.0)
    off = torch.zeros(1, dtype=torch.int64)
    for call in (lambda: K.adam_multi_shadow(table, table, ctl), lambda: K.adam_multi_single_pass(table, table, ctl),
                 lambda: K.adam_multi_repair(table, table, ctl), lambda: K.adam_multi_push(table, ctl, None, off),
                 lambda: K.adam_multi_pull_push(table, ctl, None, None, off)):
        with pytest.raises(RuntimeError, match='fp32 moments'):
            call()
    eng = ChunkStepEngine('cpu', torch.float16, state_bits=8)
    eng.add_shard(p, g, n, [(0, n, 0)])
    eng.finalize()
    for call in (eng.enable_single_pass, eng.enable_speculation, eng.enable_streaming, lambda: eng.enable_p2p([n]),
                 lambda: eng.attach_p2p(None, [0]), lambda: eng.enable_multicast([n])):
        with pytest.raises(RuntimeError, match='fp32 moments'):
            call()
    x, y = torch.zeros(n), torch.zeros(n)
    with pytest.raises(ValueError):
        K.pack_moments(x, y[:-1])
    with pytest.raises(TypeError):
        K.pack_moments(x.double(), y)
    with pytest.raises(ValueError):
        K.pack_moments(x, y, s[:-1], s)
    with pytest.raises(ValueError):
        K.pack_moments(torch.zeros(2 * n)[::2], y)    # not contiguous
    with pytest.raises(ValueError):
        K.pack_moments(x, y, s, s)
    with pytest.raises(ValueError):
        K.unpack_moments(s, s, x, x)
    with pytest.raises(TypeError):
        K.unpack_moments(s, s, x.half(), y.half())
    with pytest.raises(TypeError):
        K.unpack_moments(s, s, x, y.bfloat16())
    with pytest.raises(ValueError):
        K.unpack_moments(s[:-1], s, x, y)
    assert K.moment_state_bytes(0) == 0 and _lib().elx_moment_state_bytes(-1) == _abi.ERR_SIZE


def test_the_library_rejects_bad_arguments_before_touching_a_device():
    from elixir_b200 import _abi, build, _lib as loader
    build.build()
    lib = ctypes.CDLL(loader.lib_path())
    _abi.apply_prototypes(lib)
    a, b, odd = ctypes.c_void_p(64), ctypes.c_void_p(128), ctypes.c_void_p(65)
    f16, f32 = _abi.F16, _abi.F32
    E = _abi
    assert lib.elx_moment_state_bytes(257) == 272 + 16
    assert lib.elx_adam8_multi(None, 0, 1, 1, 0, None, None, 1, None, None) == E.ERR_NULL
    assert lib.elx_adam8_multi(a, 0, 1, 1, 0, None, None, 1, a, None) == E.ERR_NULL
    assert lib.elx_adam8_multi(a, 0, 1, 1, 7, a, a, 1, a, None) == E.ERR_DTYPE
    assert lib.elx_adam8_multi(a, 0, -1, 1, 0, a, a, 1, a, None) == E.ERR_SIZE
    assert lib.elx_adam8_multi(a, 0, 1, 1, 0, a, a, 65, a, None) == E.ERR_CAPACITY
    assert lib.elx_adam8_multi(a, 0, 1, 1, 0, a, a, 1, ctypes.c_void_p(72), None) == E.ERR_ALIGN
    assert lib.elx_adam8_multi(a, 0, 0, 0, 0, a, a, 1, a, None) == E.OK
    assert lib.elx_moments_pack(a, None, 4, a, a, None) == E.ERR_NULL
    assert lib.elx_moments_pack(a, b, -1, a, a, None) == E.ERR_SIZE
    assert lib.elx_moments_pack(odd, b, 4, a, a, None) == E.ERR_ALIGN
    assert lib.elx_moments_pack(a, b, 0, a, a, None) == E.OK
    assert lib.elx_moments_unpack(a, b, 4, f16, a, a, None) == E.ERR_DTYPE
    assert lib.elx_moments_unpack(a, b, -4, f32, a, a, None) == E.ERR_SIZE
    assert lib.elx_moments_unpack(a, b, 4, f32, odd, a, None) == E.ERR_ALIGN
