"""The update with 8-bit moments on the GPU against its 64-bit restatement: codes and exponents equal, masters within the
roundings of the kernel's arithmetic, working copies the rounded masters."""
import numpy as np
import pytest
import torch

import _moments8 as ref
from _util import bits_equal

pytestmark = pytest.mark.gpu

# The parameter's step passes through eight roundings of at most one unit (2^-23): the two bias corrections and their
# reciprocals, the approximate root, the sum with eps, the approximate quotient (two units), the decay term.
STEP_ERROR = 8 * 2.0**-23


def _inputs(n, dtype, seed, scale):
    rng = np.random.default_rng(seed)
    size = np.exp(2.5 * rng.standard_normal((n + 63) // 64)).repeat(64)[:n] * 1e-4
    size[rng.random(n) < 0.05] = 0
    master = (rng.standard_normal(n) * 0.02).astype(np.float32)
    grad = torch.from_numpy(np.clip(rng.standard_normal(n) * size * scale, -6e4, 6e4)).to(dtype)
    m = (rng.standard_normal(n) * size * 0.3).astype(np.float32)
    v = ((rng.standard_normal(n)**2 + 0.1) * size**2).astype(np.float32)
    return (torch.from_numpy(master), grad, torch.from_numpy(ref.encode(m.astype(np.float64), True, 0.5)),
            torch.from_numpy(ref.encode(v.astype(np.float64), False, 0.5)))


def _at(t, offset, device):
    """A copy of t on the device whose first element is `offset` elements into its allocation."""
    room = torch.empty(t.numel() + offset, dtype=t.dtype, device=device)
    room[offset:] = t
    return room[offset:]


class Case:
    """Shards on the device and what the restatement says of them."""

    def __init__(self, device, dtype, sizes, segments, hypers, scale=1.0, offset=0, seed=0, step=0, separate=False):
        from elixir_b200.engine import ChunkStepEngine
        from elixir_b200.scaler import ConstantGradScaler
        self.hypers, self.scale, self.step_count = hypers, scale, step
        self.eng = ChunkStepEngine(device, dtype, ConstantGradScaler(scale), state_bits=8)
        self.host, self.dtype = [], dtype
        for i, (n, segs) in enumerate(zip(sizes, segments)):
            master, grad, sm, sv = _inputs(n, dtype, 1000 * seed + i, scale)
            lowp = torch.zeros_like(grad) if separate else grad
            src = _at(grad, offset, device) if separate else None
            dev = [_at(t, offset, device) for t in (master, lowp, sm, sv)]
            self.eng.add_shard(dev[0], dev[1], max([e for _, e, _ in segs], default=0), segs, exp_avg=dev[2], exp_avg_sq=dev[3],
                               grad_src=src)
            self.host.append([master.numpy().copy(), sm.numpy().copy(), sv.numpy().copy(), grad.float().numpy(), segs])
        self.eng.finalize()
        self.eng.set_hyper(hypers)
        if step:
            self.eng.scaler.load_state_dict(dict(scale=scale, step=step))

    def check(self):
        for i, (master, sm, sv, grad, segs) in enumerate(self.host):
            p, moved, sm, sv = ref.adam8(master, sm, sv, grad, segs, self.hypers, self.step_count + 1, self.scale, index=i)
            got, lowp = self.eng.shards[i][0].cpu().numpy(), self.eng.shards[i][3].cpu()
            n = p.size
            # half a unit of the master's own rounding, and the step's error
            assert np.all(np.abs(got - p) <= np.abs(p) * 2.0**-24 + moved * STEP_ERROR + 1e-40), i
            assert ref.same_state(self.eng.shards[i][1].cpu().numpy(), sm, n, True), i
            assert ref.same_state(self.eng.shards[i][2].cpu().numpy(), sv, n, False), i
            assert bits_equal(lowp, torch.from_numpy(got).to(self.dtype)), i
        assert self.eng.read_control().status == 0


def _hyper(**kw):
    from elixir_b200 import kernels as K
    return K.hyper(**{**dict(lr=3e-3, weight_decay=0.1), **kw})


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('n', [1, 7, 255, 256, 257, 4095, 4096, 4097, 12299])
def test_sizes(cuda, dtype, n):
    case = Case(cuda, dtype, [n], [[(0, n, 0)]], [_hyper()], step=9)
    case.eng.step()
    case.check()


@pytest.mark.parametrize('scale', [1.0, 65536.0, 6963.2])
@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
def test_divisors_and_the_separate_gradient(cuda, dtype, scale):
    case = Case(cuda, dtype, [9000, 4096], [[(0, 8000, 0)], [(0, 4096, 0)]], [_hyper()], scale=scale, separate=True, seed=3)
    case.eng.probe()
    case.eng.step()
    case.check()


@pytest.mark.parametrize('segments', [
    [],
    [(0, 1, 0)],
    [(100, 300, 0), (300, 301, 1), (5000, 8191, 1)],
    [(0, 4096, 1), (4096, 8192, 0)],
    [(255, 257, 0)],
    [(9999, 10000, 1)],
])
@pytest.mark.parametrize('offset', [0, 3])
def test_segments_gaps_and_unaligned_shards(cuda, segments, offset):
    """Elements outside every segment keep master and moments, whatever happens to their block's exponent; blocks outside
    keep every byte."""
    n = 10000
    case = Case(cuda, torch.float16, [n], [segments], [_hyper(), _hyper(lr=1e-4, weight_decay=0.0, betas=(0.8, 0.95))], offset=offset,
                seed=4)
    case.eng.step()
    case.check()


@pytest.mark.parametrize('kw', [dict(adamw_mode=False), dict(bias_correction=False), dict(weight_decay=0.0, eps=1e-3),
                                dict(betas=(0.0, 0.0)), dict(betas=(0.95, 0.9999), lr=0.0)])
def test_hyper_parameters(cuda, kw):
    case = Case(cuda, torch.float32, [5000], [[(0, 5000, 0)]], [_hyper(**kw)], step=3, seed=5)
    case.eng.step()
    case.check()


def test_many_groups_and_shards(cuda):
    rng = np.random.default_rng(0)
    sizes = [int(x) for x in rng.integers(1, 9000, 40)]
    segments, hypers = [], [_hyper(lr=1e-3 * (i + 1), weight_decay=0.01 * i) for i in range(64)]
    for n in sizes:
        cuts = sorted(set(rng.integers(0, n + 1, 6).tolist()))
        segments.append([(a, b, int(rng.integers(0, 64))) for a, b in zip(cuts, cuts[1:])])
    case = Case(cuda, torch.bfloat16, sizes, segments, hypers, seed=6)
    case.eng.step()
    case.check()


def test_any_split_into_launches_gives_the_same_bits(cuda):
    sizes, segments = [20000, 100, 8192], [[(0, 19000, 0)], [(0, 100, 0)], [(0, 8192, 0)]]
    one = Case(cuda, torch.float16, sizes, segments, [_hyper()], seed=7)
    two = Case(cuda, torch.float16, sizes, segments, [_hyper()], seed=7)
    one.eng.step()
    two.eng.begin_step()
    for k in (2, 0, 1):
        two.eng.update(first=k, count=1)
    for a, b in zip(one.eng.shards, two.eng.shards):
        assert all(torch.equal(x, y) for x, y in zip(a[:4], b[:4]))
    one.check()


def test_a_skipped_step_changes_nothing_but_the_working_copies(cuda):
    case = Case(cuda, torch.float16, [12299], [[(0, 12000, 0)]], [_hyper()], scale=8.0, seed=8)
    case.eng.shards[0][3][77] = float('inf')
    before = [t.clone() for t in case.eng.shards[0][:3]]
    case.eng.probe()
    case.eng.step()
    assert case.eng.read_control().skip == 1 and case.eng.read_control().step == 0
    assert all(torch.equal(a, b) for a, b in zip(before, case.eng.shards[0]))
    assert bits_equal(case.eng.shards[0][3], before[0].half())


def test_a_non_finite_gradient_nobody_probed_is_reported_and_poisons_its_block_only(cuda):
    from elixir_b200 import _abi
    case = Case(cuda, torch.float32, [4096], [[(0, 4096, 0)]], [_hyper()], seed=9)
    case.eng.shards[0][3][300] = float('nan')
    case.eng.step()    # no probe: applied
    assert case.eng.read_control().status == _abi.STAT_LATE_INF
    m, v = case.eng.moments(0)
    bad = torch.zeros(4096, dtype=torch.bool, device=cuda)
    bad[256:512] = True
    assert torch.equal(torch.isnan(m), bad) and torch.equal(torch.isnan(v), bad)
    nan = torch.isnan(case.eng.shards[0][0])
    assert nan[300] and int(nan.sum()) == 1


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('n', [600, 8192])    # the end of a shard, whole tiles
def test_a_block_that_is_not_finite_is_reported(cuda, dtype, n):
    """A finite gradient whose square passes fp32's range costs the second moments of its block, and the control block says
    so; so it does where the block was lost before."""
    from elixir_b200 import _abi
    bad = torch.arange(n, device=cuda) // 256 == 1
    case = Case(cuda, dtype, [n], [[(0, n, 0)]], [_hyper()], seed=15)
    case.eng.shards[0][3][300] = 1e21
    case.eng.probe()
    case.eng.step()
    ctl = case.eng.read_control()
    assert ctl.skip == 0 and ctl.late_inf == 1 and ctl.status == _abi.STAT_LATE_INF
    m, v = case.eng.moments(0)
    assert torch.equal(torch.isnan(v), bad) and bool(torch.isfinite(m).all())
    assert bool(torch.isfinite(case.eng.shards[0][0]).all())    # as with fp32 moments: the element itself hardly moves
    for which in (1, 2):
        case = Case(cuda, dtype, [n], [[(0, n, 0)]], [_hyper()], seed=16)
        case.eng.shards[0][which][ref.round_up(n, 16) + 1] = 255
        case.eng.probe()
        case.eng.step()
        ctl = case.eng.read_control()
        assert ctl.skip == 0 and ctl.late_inf == 1 and ctl.status == _abi.STAT_LATE_INF
        assert torch.equal(torch.isnan(case.eng.moments(0)[which - 1]), bad) and torch.equal(torch.isnan(case.eng.shards[0][0]), bad)


def test_clipping_divides_by_the_clipped_scale(cuda):
    """With max_norm the divisor is a number the device forms: the restatement takes it from the control block."""
    from elixir_b200.engine import ChunkStepEngine
    from elixir_b200.scaler import ConstantGradScaler
    n = 5000
    eng = ChunkStepEngine(cuda, torch.float16, ConstantGradScaler(64.0), max_norm=1e-3, state_bits=8)
    master, grad, sm, sv = _inputs(n, torch.float16, 11, 64.0)
    eng.add_shard(master.to(cuda), grad.to(cuda), n, [(0, n, 0)], exp_avg=sm.to(cuda), exp_avg_sq=sv.to(cuda))
    eng.finalize()
    eng.set_hyper([_hyper()])
    eng.probe()
    eng.step()
    ctl = eng.read_control()
    assert ctl.clip_coef > 1 and ctl.skip == 0
    p, moved, sm, sv = ref.adam8(master.numpy(), sm.numpy(), sv.numpy(), grad.float().numpy(), [(0, n, 0)], [_hyper()], 1, ctl.div_scale)
    got = eng.shards[0][0].cpu().numpy()
    assert np.all(np.abs(got - p) <= np.abs(p) * 2.0**-24 + moved * STEP_ERROR)
    assert ref.same_state(eng.shards[0][1].cpu().numpy(), sm, n, True) and ref.same_state(eng.shards[0][2].cpu().numpy(), sv, n, False)


def test_stored_moments_are_unbiased(cuda):
    """The mean over many steps' dither of a stored moment is the moment: the average of 4000 roundings lies within six
    standard deviations, and a rounding between neighbours a step apart deviates by at most half that step."""
    from elixir_b200 import kernels as K
    n, steps = 256, 4000
    case = Case(cuda, torch.float32, [n], [[(0, n, 0)]], [_hyper(lr=0.0, betas=(0.0, 0.0))], seed=12)
    grad = case.eng.shards[0][3].clone()
    grad[0] = 10 * grad.abs().max()    # the block's exponent stays
    total_m, total_v = torch.zeros(n, dtype=torch.float64, device=cuda), torch.zeros(n, dtype=torch.float64, device=cuda)
    m, v = torch.empty(n, device=cuda), torch.empty(n, device=cuda)
    for _ in range(steps):
        case.eng.shards[0][3].copy_(grad)
        case.eng.step()
        K.unpack_moments(case.eng.shards[0][1], case.eng.shards[0][2], m, v)
        total_m += m
        total_v += v
    for total, want, fields in ((total_m, grad.double(), 15), (total_v, grad.double()**2, 31)):
        top = 2.0**torch.floor(torch.log2(want.abs().max()) + 1e-9).item()
        step = torch.clamp(2.0**torch.floor(torch.log2(want.abs().clamp(min=1e-300))), min=top * 2.0**(2 - fields)) / 8
        off = (total / steps - want).abs()
        inside = want.abs() > top * 2.0**(-1 - fields)    # below, a second moment is held up to the smallest code
        assert bool((off <= step * (6 * 0.5 / steps**0.5 + 2.0**-16) + 1e-45)[inside].all())


def test_captured_step_equals_the_eager_one_and_two_engines_run_side_by_side(cuda):
    n = 70000
    args = ([n], [[(0, n - 5, 0)]], [_hyper()])
    eager, captured, other = (Case(cuda, torch.float16, *args, scale=8.0, seed=s) for s in (13, 13, 14))
    block = torch.zeros(n, dtype=torch.float16, device=cuda)
    graph = captured.eng.capture_step([block])
    side = torch.cuda.Stream(cuda)
    twin = Case(cuda, torch.float16, *args, scale=8.0, seed=14)
    for step in range(3):
        g = (torch.randn(n, generator=torch.Generator().manual_seed(step)) * 1e-3).half().to(cuda)
        if step == 1:
            g[5] = float('nan')
        block.copy_(g)
        eager.eng.land_all([g], streams=1)
        eager.eng.step()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(side):    # another engine at the same time
            other.eng.land_all([g], streams=1)
            other.eng.step()
        torch.cuda.synchronize()
        twin.eng.land_all([g], streams=1)
        twin.eng.step()
        torch.cuda.synchronize()
    for a, b in ((eager, captured), (other, twin)):
        assert all(bits_equal(x.view(torch.int16) if x.dtype == torch.uint8 else x, y.view(torch.int16) if y.dtype == torch.uint8 else y)
                   for x, y in zip(a.eng.shards[0][:4], b.eng.shards[0][:4]))
        assert a.eng.read_control().step == b.eng.read_control().step == 2


@pytest.mark.parametrize('n', [1, 255, 256, 257, 10007])
@pytest.mark.parametrize('offset', [0, 1])
def test_conversion(cuda, n, offset):
    from elixir_b200 import kernels as K
    rng = np.random.default_rng(n)
    m = (rng.standard_normal(n) * np.exp(6 * rng.standard_normal(n))).astype(np.float32)
    v = (m * m).astype(np.float32)
    room = K.moment_state_bytes(n)
    state = [_at(torch.full((room, ), 7, dtype=torch.uint8), offset, cuda) for _ in range(2)]
    K.pack_moments(_at(torch.from_numpy(m), offset, cuda), _at(torch.from_numpy(v), offset, cuda), *state)
    for s, x, signed in ((state[0], m, True), (state[1], v, False)):
        got = s.cpu().numpy()
        assert ref.same_state(got, ref.encode(x.astype(np.float64), signed, 0.5), n, signed)
        end = ref.round_up(n, 16) + (n + 255) // 256
        assert not got[n:ref.round_up(n, 16)].any() and not got[end:].any()    # the padding: zeros
    for dtype in (torch.float32, torch.bfloat16):
        out = [_at(torch.full((n, ), -1.0, dtype=dtype), offset, cuda) for _ in range(2)]
        K.unpack_moments(*state, *out)
        for o, s, signed in ((out[0], state[0], True), (out[1], state[1], False)):
            assert np.array_equal(o.float().cpu().numpy(), ref.decode(s.cpu().numpy(), n, signed))


def test_a_shard_of_more_than_two_to_the_31_elements(cuda):
    """The last blocks of a shard past 2^31 elements: as the restatement has them (gradients are zero but for the tail)."""
    from elixir_b200.engine import ChunkStepEngine
    n, tail = 2**31 + 5 * 4096 + 77, 3 * 4096 + 77
    eng = ChunkStepEngine(cuda, torch.bfloat16, state_bits=8)
    master, lowp = torch.zeros(n, device=cuda), torch.zeros(n, dtype=torch.bfloat16, device=cuda)
    g = (torch.randn(tail, generator=torch.Generator().manual_seed(1)) * 1e-3).bfloat16()
    lowp[n - tail:] = g.to(cuda)
    eng.add_shard(master, lowp, n, [(0, n, 0)])
    eng.finalize()
    eng.set_hyper([_hyper(weight_decay=0.0)])
    eng.step()
    first = n - tail    # 2^31 + 2 tiles: a multiple of 256
    gd = g.double().numpy()
    f32 = lambda x: np.asarray(x, dtype=np.float64).astype(np.float32).astype(np.float64)    # noqa: E731
    m = f32(f32(1 - float(np.float32(0.9))) * gd)
    v = f32(f32(f32(1 - float(np.float32(0.999))) * gd) * gd)
    up_m, up_v = ref.dither(1, 0, tail, first)
    blocks = (tail + 255) // 256
    at = ref.round_up(n, 16)
    for s, x, signed, up in ((eng.shards[0][1], m, True, up_m), (eng.shards[0][2], v, False, up_v)):
        want = ref.encode(x, signed, up)
        assert np.array_equal(s[first:n].cpu().numpy(), want[:tail])
        assert np.array_equal(s[at + first // 256:at + first // 256 + blocks].cpu().numpy(), want[ref.round_up(tail, 16):][:blocks])
        assert int(s[:first].count_nonzero()) == 0
    moved = eng.shards[0][0][n - tail:].cpu().double().numpy()
    upd = m / (1 - float(np.float32(0.9))) / (np.sqrt(v / (1 - float(np.float32(0.999)))) + 1e-8)
    assert np.all(np.abs(moved + 3e-3 * upd) <= 3e-3 * np.abs(upd) * (STEP_ERROR + 2.0**-24) + 1e-10 * 3e-3)
    assert int(eng.shards[0][0][:first].count_nonzero()) == 0
