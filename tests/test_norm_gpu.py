"""Layer norm, forward and backward, against its definition in 64 bits."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24    # half a unit of fp32


def _half_step(dtype):
    return torch.finfo(dtype).eps / 2


def _check(got, want, bound, dtype):
    """|got - want| within the arithmetic's bound and half a step of the result's own type (fp16: also its subnormals)."""
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    bound = (bound + want.abs() * _half_step(dtype)) * (1 + 2**-10) + tiny
    off = (got.double() - want).abs()
    assert got.dtype == dtype and bool((off <= bound).all()), float((off / bound).max())


def _reference(x, w, b, dy, eps, rows_chain):
    """Values in 64 bits and bounds of an fp32 evaluation.  A sum of C terms passes through at most `chain` additions (those
    of one thread, five steps in a warp, 32 warps): its error is chain * U times the sum of the magnitudes."""
    x64, cols = x.double(), x.shape[1]
    chain = max(32, cols / 1024 + 1) + 5 + 32 + 4
    mean = x64.mean(1, keepdim=True)
    mean_err = chain * U * x64.abs().mean(1, keepdim=True)
    d = x64 - mean
    var = (d * d).mean(1, keepdim=True)
    rstd = (var + eps).rsqrt()
    # d is off by mean_err and a rounding; the sum of squares by that to first order (its linear part cancels but for the
    # rounding) and by chain roundings; half of that in the root, which has three roundings of its own
    d_err = mean_err + 2 * U * (x64.abs() + mean.abs())
    rel = 0.5 * (((2 * d.abs() * d_err + d_err**2).mean(1, keepdim=True)) * rstd**2 + chain * U) + 4 * U
    xhat = d * rstd
    xhat_err = d_err * rstd + xhat.abs() * (rel + 2 * U)
    w64 = torch.ones(cols, dtype=torch.float64, device=x.device) if w is None else w.double()
    y = xhat * w64 + (0 if b is None else b.double())
    y_err = xhat_err * w64.abs() + 2 * U * ((xhat * w64).abs() + y.abs())
    out = dict(mean=(mean[:, 0], mean_err[:, 0] + U * mean[:, 0].abs()), rstd=(rstd[:, 0], (rel * rstd)[:, 0]), y=(y, y_err))
    if dy is None:
        return out
    dy64 = dy.double()
    a = dy64 * w64
    m0, m1 = a.mean(1, keepdim=True), (a * xhat).mean(1, keepdim=True)
    mean_a, mean_ax = a.abs().mean(1, keepdim=True), (a * xhat).abs().mean(1, keepdim=True)
    m0_err = (chain + 2) * U * mean_a
    m1_err = (chain + 4) * U * mean_ax + (a.abs() * xhat_err).mean(1, keepdim=True)
    dx = rstd * (a - m0 - xhat * m1)
    dx_err = rstd * (m0_err + xhat.abs() * m1_err + xhat_err * m1.abs() + 4 * U * (a.abs() + m0.abs() + (xhat * m1).abs())) \
        + dx.abs() * (rel + 2 * U)
    out['dx'] = (dx, dx_err)
    out['dw'] = ((dy64 * xhat).sum(0), (dy64.abs() * xhat_err).sum(0) + rows_chain * U * (dy64 * xhat).abs().sum(0))
    out['db'] = (dy64.sum(0), rows_chain * U * dy64.abs().sum(0))
    return out


def _inputs(rows, cols, dtype, affine, seed=0, device='cuda', offset=0):
    gen = torch.Generator(device=device).manual_seed(seed)
    channel = torch.exp(0.5 * torch.randn(cols, generator=gen, device=device))

    def at(t):    # `offset` elements into an allocation of its own
        if t is None:
            return None
        room = torch.empty(t.numel() + offset, dtype=dtype, device=device)
        room[offset:] = t.reshape(-1)
        return room[offset:].view(t.shape)

    x = at(torch.randn(rows, cols, generator=gen, device=device) * channel + 0.5)
    w = at(1 + 0.2 * torch.randn(cols, generator=gen, device=device)) if affine != 'none' else None
    b = at(0.3 * torch.randn(cols, generator=gen, device=device)) if affine == 'both' else None
    dy = at(torch.randn(rows, cols, generator=gen, device=device))
    return x, w, b, dy


def _run(x, w, b, dy, eps=1e-5):
    from elixir_b200 import kernels as K
    y, mean, rstd = K.layer_norm_forward(x, w, b, eps)
    dx, dw, db = K.layer_norm_backward(dy, x, w, mean, rstd, bias_grad=b is not None)
    want = _reference(x, w, b, dy, eps, rows_chain=x.shape[0] / 64 + 100)
    dtype = x.dtype
    _check(mean, *want['mean'], torch.float32)
    _check(rstd, *want['rstd'], torch.float32)
    _check(y, *want['y'], dtype)
    _check(dx, *want['dx'], dtype)
    for got, key, given in ((dw, 'dw', w), (db, 'db', b)):
        assert (got is None) == (given is None)
        if got is not None:
            _check(got, *want[key], dtype)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('cols', [1, 2, 3, 8, 31, 32, 33, 100, 255, 256, 264, 513, 1000, 1024, 1111, 1600, 2056, 4095, 4096, 4104, 5120,
                                  8192, 8200, 9216, 12288, 12289, 16384, 16392, 20001, 32768, 40000, 66000])
def test_widths(cuda, dtype, cols):
    _run(*_inputs(5, cols, dtype, 'both', seed=cols))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('rows', [1, 2, 63, 64, 591, 593, 4001])
@pytest.mark.parametrize('cols', [40, 777, 1600])
def test_rows(cuda, dtype, rows, cols):
    _run(*_inputs(rows, cols, dtype, 'both', seed=rows))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('lanes,pieces', [(32, p) for p in (1, 2, 3, 4, 5, 6, 7)] + [(64, 4), (96, 3), (1024, 4), (512, 10)])
def test_every_forward_kernel_of_16_byte_pieces(cuda, dtype, lanes, pieces):
    """The widest row of each number of lanes and pieces per lane, and the first row past it."""
    for cols in (lanes * pieces * 16 // dtype.itemsize, (lanes * pieces + 1) * 16 // dtype.itemsize):
        _run(*_inputs(9, cols, dtype, 'both', seed=cols))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('cols', [32, 64, 128, 256, 512, 768, 1024, 1280, 16384, 20480])
def test_every_forward_kernel_of_single_elements(cuda, dtype, cols):
    for past in (0, 1):
        _run(*_inputs(9, cols + past, dtype, 'both', seed=cols, offset=1))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('cols', [5120, 8193, 9216, 9217, 12288, 16384, 16392, 20001])
def test_many_wide_rows(cuda, dtype, cols):
    """Several rows per block where a row takes the whole block: every block comes round four or five times."""
    _run(*_inputs(601, cols, dtype, 'both', seed=cols))


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
@pytest.mark.parametrize('rows', [149, 593, 4001])
def test_many_narrow_rows_and_rows_off_alignment(cuda, dtype, rows):
    """Several groups per block in the kernels that access one element at a time."""
    for cols in (1, 3, 17, 31):
        _run(*_inputs(rows, cols, dtype, 'both', seed=cols))
    for cols in (65, 1601):
        _run(*_inputs(rows, cols, dtype, 'both', seed=cols, offset=1))


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('offset', [1, 3, 7])
@pytest.mark.parametrize('rows,cols', [(1, 33), (5, 65), (601, 1111), (37, 1600), (149, 8201), (7, 16000)])
def test_all_arrays_at_one_distance_from_a_boundary(cuda, dtype, offset, rows, cols):
    """Through the C entry points, which take such arrays: x, y, dy and dx begin at the same odd place, the parameters at
    others.  What lies around the arrays is left as it was."""
    from elixir_b200 import _lib, kernels as K
    lib, n, mark, room = _lib.get(), rows * cols, 123.0, 16

    def at(t):
        buffer = torch.full((room + offset + t.numel() + room, ), mark, dtype=t.dtype, device=cuda)
        inside = buffer[room + offset:room + offset + t.numel()]
        inside.copy_(t.reshape(-1))
        return buffer, inside

    x, w, b, dy = _inputs(rows, cols, dtype, 'both', seed=cols)
    empty = torch.zeros(n, dtype=dtype, device=cuda)
    rooms = {k: at(t) for k, t in dict(x=x, dy=dy, y=empty, dx=empty, dw=w, db=b).items()}
    p = {k: inside.data_ptr() for k, (_, inside) in rooms.items()}
    mean, rstd = torch.empty(rows, device=cuda), torch.empty(rows, device=cuda)
    code, stream = K.dtype_code(dtype), torch.cuda.current_stream(cuda).cuda_stream
    assert lib.elx_layer_norm_forward(p['x'], w.data_ptr(), b.data_ptr(), code, rows, cols, 1e-5, p['y'], mean.data_ptr(),
                                      rstd.data_ptr(), stream) == 0
    size = lib.elx_layer_norm_backward_workspace(rows, cols)
    space = torch.full((size + 64, ), 77, dtype=torch.uint8, device=cuda)
    assert lib.elx_layer_norm_backward(p['dy'], p['x'], w.data_ptr(), mean.data_ptr(), rstd.data_ptr(), code, rows, cols, p['dx'],
                                       p['dw'], p['db'], space.data_ptr(), size, stream) == 0
    want = _reference(x, w, b, dy, 1e-5, rows_chain=rows / 64 + 100)
    _check(mean, *want['mean'], torch.float32)
    _check(rstd, *want['rstd'], torch.float32)
    for key in ('y', 'dx', 'dw', 'db'):
        _check(rooms[key][1].view(want[key][0].shape), *want[key], dtype)
    assert torch.equal(rooms['x'][1], x.view(-1)) and torch.equal(rooms['dy'][1], dy.view(-1))
    for buffer, inside in rooms.values():
        assert bool((buffer[:room + offset] == mark).all()) and bool((buffer[room + offset + inside.numel():] == mark).all())
    assert bool((space[size:] == 77).all())


@pytest.mark.parametrize('affine', ['none', 'weight', 'both'])
@pytest.mark.parametrize('offset', [0, 1, 2, 4])
@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
def test_parameters_and_alignment(cuda, affine, offset, dtype):
    for cols in (1600, 1601, 24, 40000):
        _run(*_inputs(37, cols, dtype, affine, seed=offset, offset=offset))


def test_parameters_alone_off_alignment(cuda):
    """Weights are views into chunks at any element: the rows may be aligned where the parameters are not."""
    x, w, b, dy = _inputs(64, 1600, torch.float16, 'both')
    room = torch.empty(2 * 1600 + 3, dtype=torch.float16, device=cuda)
    room[1:1601], room[1603:] = w, b
    _run(x, room[1:1601], room[1603:], dy)


def test_a_constant_row_and_a_single_column(cuda):
    from elixir_b200 import kernels as K
    x = torch.full((3, 64), 7.0, device=cuda)
    w, b = torch.full((64, ), 2.0, device=cuda), torch.full((64, ), 0.25, device=cuda)
    y, mean, rstd = K.layer_norm_forward(x, w, b, 1e-5)
    assert bool((y == 0.25).all()) and bool((mean == 7).all())
    want = (torch.tensor(1e-5).double())**-0.5
    assert float((rstd.double().cpu() - want).abs().max() / want) <= 2 * 2.0**-23
    one = torch.randn(9, 1, device=cuda)
    y, mean, rstd = K.layer_norm_forward(one, w[:1], b[:1], 1e-5)
    assert bool((y == 0.25).all()) and torch.equal(mean, one[:, 0])
    dx, dw, db = K.layer_norm_backward(torch.randn(9, 1, device=cuda), one, w[:1], mean, rstd)
    assert bool((dx == 0).all()) and bool((dw == 0).all())


def test_a_large_offset_keeps_the_spread(cuda):
    """The variance is that of the differences from the mean: no cancellation of two large sums."""
    gen = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn(16, 1600, generator=gen, device=cuda) + 4096
    w, b = torch.ones(1600, device=cuda), torch.zeros(1600, device=cuda)
    _run(x, w, b, torch.randn(16, 1600, generator=gen, device=cuda))


def test_infinities_and_nan_stay_in_their_row(cuda):
    from elixir_b200 import kernels as K
    x, w, b, dy = _inputs(6, 1600, torch.float32, 'both')
    clean = K.layer_norm_forward(x, w, b)[0]
    x[1, 5], x[4, 1599] = float('inf'), float('nan')
    y, mean, rstd = K.layer_norm_forward(x, w, b)
    assert bool(torch.isnan(y[[1, 4]]).all())
    assert torch.equal(y[[0, 2, 3, 5]], clean[[0, 2, 3, 5]])
    dx, dw, db = K.layer_norm_backward(dy, x, w, mean, rstd)
    assert bool(torch.isnan(dx[[1, 4]]).all()) and bool(torch.isfinite(dx[[0, 2, 3, 5]]).all())
    assert bool(torch.isnan(dw).all()) and bool(torch.isfinite(db).all())


def test_no_rows(cuda):
    from elixir_b200 import kernels as K
    w = torch.ones(16, dtype=torch.float16, device=cuda)
    x = torch.empty(0, 16, dtype=torch.float16, device=cuda)
    y, mean, rstd = K.layer_norm_forward(x, w, w)
    dx, dw, db = K.layer_norm_backward(x, x, w, mean, rstd)
    assert y.shape == dx.shape == x.shape and mean.numel() == 0
    assert bool((dw == 0).all()) and bool((db == 0).all())


def test_same_bits_every_time_and_from_another_stream(cuda):
    from elixir_b200 import kernels as K
    x, w, b, dy = _inputs(3000, 1600, torch.float16, 'both')
    first = None
    side = torch.cuda.Stream(cuda)
    for k in range(4):
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream(cuda)):
            y, mean, rstd = K.layer_norm_forward(x, w, b)
            got = (y, mean, rstd) + K.layer_norm_backward(dy, x, w, mean, rstd)
        torch.cuda.synchronize()
        first = first or got
        assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_two_captured_graphs_replayed_at_once(cuda):
    """Each capture has a workspace of its own: replays that overlap give what each gives alone."""
    from elixir_b200 import kernels as K
    inputs = [_inputs(2000, 1600, torch.float16, 'both', seed=s) for s in (0, 1)]
    graphs, outs, wants = [], [], []
    for x, w, b, dy in inputs:
        y, mean, rstd = K.layer_norm_forward(x, w, b)
        wants.append((y, ) + K.layer_norm_backward(dy, x, w, mean, rstd))
    torch.cuda.synchronize()
    for x, w, b, dy in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y, mean, rstd = K.layer_norm_forward(x, w, b)
            outs.append((y, ) + K.layer_norm_backward(dy, x, w, mean, rstd))
        graphs.append(g)
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for got, want in zip(outs, wants):
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_more_than_two_to_the_31_elements(cuda):
    from elixir_b200 import kernels as K
    rows, cols = 2**31 // 4096 + 3, 4096
    x = torch.zeros(rows, cols, dtype=torch.float16, device=cuda)
    tail, w, b, dy = _inputs(4, cols, torch.float16, 'both')
    x[-4:] = tail
    y, mean, rstd = K.layer_norm_forward(x, w, b)
    small = K.layer_norm_forward(tail.contiguous(), w, b)
    assert torch.equal(y[-4:], small[0]) and torch.equal(mean[-4:], small[1])
    del y
    grad = torch.zeros(rows, cols, dtype=torch.float16, device=cuda)
    grad[-4:] = dy
    dx, dw, db = K.layer_norm_backward(grad, x, w, mean, rstd)
    sx, sw, sb = K.layer_norm_backward(dy, tail.contiguous(), w, small[1], small[2])
    assert torch.equal(dx[-4:], sx)
    want = _reference(tail, w, b, dy, 1e-5, rows_chain=300)
    _check(dw, *want['dw'], torch.float16)
    _check(db, *want['db'], torch.float16)


@pytest.mark.parametrize('shape,norm', [((3, 5, 40), (40, )), ((4, 6, 10), (6, 10)), ((2, 3, 4, 5), (3, 4, 5)), ((16, ), (16, ))])
def test_autograd(cuda, shape, norm):
    """Through the public function: gradients against the definition's (float64 autograd) and against differences."""
    from elixir_b200 import functional as F
    gen = torch.Generator(device=cuda).manual_seed(1)
    x = torch.randn(shape, generator=gen, device=cuda).requires_grad_()
    w = (1 + 0.2 * torch.randn(norm, generator=gen, device=cuda)).requires_grad_()
    b = torch.randn(norm, generator=gen, device=cuda).requires_grad_()
    dy = torch.randn(shape, generator=gen, device=cuda)
    y = F.layer_norm(x, norm, w, b)
    got = torch.autograd.grad(y, (x, w, b), dy)

    def exact(x, w, b):
        flat = x.reshape(*x.shape[:x.dim() - len(norm)], -1)
        d = flat - flat.mean(-1, keepdim=True)
        return (d / (d.pow(2).mean(-1, keepdim=True) + 1e-5).sqrt()).reshape(x.shape) * w + b

    args = [t.detach().double().requires_grad_() for t in (x, w, b)]
    y64 = exact(*args)
    # at most 200 roundings of values of size 10 in these small cases
    assert float((y.double() - y64).abs().max()) <= 2000 * U
    for g, e in zip(got, torch.autograd.grad(y64, args, dy.double())):
        assert g.shape == e.shape and float((g.double() - e).abs().max()) <= 4000 * U
    # differences of the function itself, in a random direction: second order 1e-3^2, rounding 2000 U / 1e-3
    for k, t in enumerate((x, w, b)):
        direction = torch.randn(t.shape, generator=gen, device=cuda)
        ends = []
        for sign in (1, -1):
            moved = [u.detach() for u in (x, w, b)]
            moved[k] = moved[k] + sign * 1e-3 * direction
            ends.append(float((F.layer_norm(moved[0], norm, moved[1], moved[2]).double() * dy).sum()))
        slope, want = (ends[0] - ends[1]) / 2e-3, float((got[k].double() * direction).sum())
        assert abs(slope - want) <= 0.02 * (1 + float((got[k].double() * direction).abs().sum()))


@pytest.mark.parametrize('norm', [(40, ), (5, 8)])
def test_parameters_whose_memory_moves_before_the_backward_pass(cuda, norm):
    """As with the chunks of a small replica cache: the gradient is that of the values in the parameter's new memory."""
    from elixir_b200 import functional as F
    gen = torch.Generator(device=cuda).manual_seed(3)
    x = torch.randn((6, ) + norm, generator=gen, device=cuda).requires_grad_()
    dy = torch.randn((6, ) + norm, generator=gen, device=cuda)
    w, b = (torch.nn.Parameter(torch.randn(norm, generator=gen, device=cuda)) for _ in range(2))
    want = torch.autograd.grad(F.layer_norm(x, norm, w, b), (x, w, b), dy)
    y = F.layer_norm(x, norm, w, b)
    old = w.data
    w.data = old.clone()
    old.fill_(float('nan'))
    got = torch.autograd.grad(y, (x, w, b), dy)
    assert all(torch.equal(g, e) and g.shape == e.shape for g, e in zip(got, want))


def test_autograd_forms(cuda):
    from elixir_b200 import functional as F
    x = torch.randn(6, 32, device=cuda)
    w = torch.ones(32, device=cuda, requires_grad=True)
    F.layer_norm(x, 32, w).sum().backward()    # an expanded gradient, no bias, no gradient of x
    assert w.grad.shape == (32, )
    xt = torch.randn(32, 6, device=cuda).t().requires_grad_()    # not contiguous
    F.layer_norm(xt, 32).pow(2).sum().backward()
    assert xt.grad.shape == (6, 32)
    y = F.layer_norm(x.requires_grad_(), (32, ), w)
    g, = torch.autograd.grad(y.sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()    # first derivatives only
