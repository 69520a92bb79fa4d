"""The embedding lookup with its scale, and its gradient by sorted tokens, against the definition in 64 bits."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0**-24


def _tokens(n, vocab, spread, index, seed):
    gen = torch.Generator().manual_seed(seed)
    if spread == 'one':
        t = torch.full((n, ), int(torch.randint(vocab, (1, ), generator=gen)))
    elif spread == 'few':    # three tokens with long runs
        t = torch.randint(min(3, vocab), (n, ), generator=gen) * max(1, vocab // 3) % vocab
    elif spread == 'zipf':
        t = (2.7 * ((1 + vocab / 2.7)**torch.rand(n, generator=gen, dtype=torch.float64) - 1)).long().clamp(max=vocab - 1)
    else:
        t = torch.randint(vocab, (n, ), generator=gen)
    return t.to(index)


def _want(tokens, dout, vocab, scale, padding):
    """The gradient in 64 bits, and the sum of magnitudes that its error is measured by."""
    keep = (tokens >= 0) & (tokens < vocab)
    if padding is not None:
        keep &= tokens != padding
    t, d = tokens[keep].long().cpu(), dout[keep].double().cpu() * scale
    total = torch.zeros(vocab, dout.shape[-1], dtype=torch.float64).index_add_(0, t, d)
    size = torch.zeros(vocab, dout.shape[-1], dtype=torch.float64).index_add_(0, t, d.abs())
    return total, size


def _check_grad(got, tokens, dout, vocab, scale, padding):
    want, size = _want(tokens, dout, vocab, scale, padding)
    dtype = dout.dtype
    # a sum of up to n terms passes through n additions at most, one product, and the rounding of its own type
    n = max(1, int(torch.bincount(tokens.clamp(0, vocab - 1).long().cpu().reshape(-1), minlength=1).max()) if tokens.numel() else 1)
    eps = torch.finfo(dtype)
    bound = size * (n + 2) * U + want.abs() * (eps.eps / 2) * (1 + 2**-10) + eps.smallest_normal * eps.eps / 2
    off = (got.double().cpu() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert bool((off <= bound).all()), float((off / bound).max())
    assert bool((got.cpu()[size == 0] == 0).all())


def _case(cuda, n, vocab, width, dtype=torch.float16, index=torch.int64, spread='zipf', scale=1.0, padding=None, seed=0, offset=0):
    from elixir_b200 import kernels as K
    gen = torch.Generator(device=cuda).manual_seed(seed)

    def at(shape):
        room = torch.randn(math.prod(shape) + offset, generator=gen, device=cuda).to(dtype)
        return room[offset:].view(shape)

    tokens = _tokens(n, vocab, spread, index, seed).to(cuda)
    weight, dout = at((vocab, width)), at((n, width))
    out = K.embedding_forward(tokens, weight, scale)
    assert torch.equal(out, (weight[tokens.long()].float() * torch.tensor(scale, device=cuda)).to(dtype))
    got = K.embedding_backward(tokens, dout, vocab, scale, padding)
    _check_grad(got, tokens, dout, vocab, torch.tensor(scale).double().item(), padding)
    return tokens, dout, got


@pytest.mark.parametrize('n', [0, 1, 2, 31, 32, 33, 64, 2047, 2048, 2049, 5000, 40000])
@pytest.mark.parametrize('spread', ['zipf', 'one', 'few', 'even'])
def test_numbers_of_tokens(cuda, n, spread):
    _case(cuda, n, 1000, 72, spread=spread, seed=n)


@pytest.mark.parametrize('vocab', [1, 2, 255, 256, 257, 65535, 65536, 70001])
@pytest.mark.parametrize('index', [torch.int32, torch.int64])
def test_vocabularies(cuda, vocab, index):
    _case(cuda, 3000, vocab, 24, index=index, seed=vocab)


def test_a_vocabulary_of_three_digits(cuda):
    _case(cuda, 2500, 17_000_001, 8, spread='even', seed=5)


@pytest.mark.parametrize('n', [65536, 65537, 131072, 200001])    # a cluster sorts 65536 at most
@pytest.mark.parametrize('spread', ['zipf', 'few', 'even'])
@pytest.mark.parametrize('vocab', [1000, 50257, 70001])    # two and three digits
def test_more_tokens_than_a_cluster_sorts(cuda, n, spread, vocab):
    """Padding and tokens outside the table among them.  The sort is stable: tokens that come sorted already, with their rows,
    give the same bits."""
    from elixir_b200 import kernels as K
    tokens = _tokens(n, vocab, spread, torch.int64, n)
    gen = torch.Generator().manual_seed(n)
    tokens[torch.randint(n, (50, ), generator=gen)] = vocab + 3
    tokens[torch.randint(n, (50, ), generator=gen)] = -1
    padding = int(tokens[tokens >= 0][0])
    tokens = tokens.to(cuda)
    dout = torch.randn(n, 24, device=cuda, generator=torch.Generator(device=cuda).manual_seed(n)).half()
    got = K.embedding_backward(tokens, dout, vocab, 1.0, padding)
    _check_grad(got, tokens, dout, vocab, 1.0, padding)
    assert bool((got[padding] == 0).all())
    key = torch.where((tokens < 0) | (tokens >= vocab) | (tokens == padding), vocab, tokens)
    order = torch.sort(key, stable=True).indices
    assert torch.equal(K.embedding_backward(tokens[order], dout[order], vocab, 1.0, padding), got)
    assert torch.equal(K.embedding_backward(tokens.int(), dout, vocab, 1.0, padding), got)


@pytest.mark.parametrize('n', [65537, 70000])
def test_more_tokens_than_a_cluster_sorts_by_four_digits(cuda, n):
    from elixir_b200 import kernels as K
    tokens, dout, got = _case(cuda, n, 2**24 + 51, 4, spread='even', seed=6)
    order = torch.sort(tokens, stable=True).indices
    assert torch.equal(K.embedding_backward(tokens[order], dout[order], 2**24 + 51), got)


@pytest.mark.parametrize('dtype', [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize('width', [1, 2, 3, 4, 7, 8, 12, 64, 100, 257, 1600, 2049, 5120])
def test_widths(cuda, dtype, width):
    _case(cuda, 700, 300, width, dtype=dtype, seed=width, scale=math.sqrt(width))


@pytest.mark.parametrize('offset', [1, 2, 4])
def test_unaligned_tables(cuda, offset):
    for dtype in (torch.float16, torch.float32):
        _case(cuda, 500, 100, 64, dtype=dtype, offset=offset)


@pytest.mark.parametrize('padding', [0, 1, 999])
def test_padding(cuda, padding):
    tokens, dout, got = _case(cuda, 4000, 1000, 40, padding=padding, seed=3)
    assert bool((got[padding] == 0).all())
    from elixir_b200 import kernels as K
    everything = torch.full((100, ), 1, dtype=torch.int64, device=cuda)
    assert bool((K.embedding_backward(everything, dout[:100], 5, padding_idx=1) == 0).all())


def test_tokens_outside_the_table_read_nan_and_add_to_no_row(cuda):
    from elixir_b200 import kernels as K
    for dtype, width in ((torch.float16, 16), (torch.bfloat16, 16), (torch.float32, 16), (torch.float16, 5)):
        for index in (torch.int32, torch.int64):
            tokens = torch.tensor([0, -1, 3, 10, 9, 2**31 - 1, -2**31], dtype=index, device=cuda)
            weight = torch.randn(10, width, device=cuda).to(dtype)
            out = K.embedding_forward(tokens, weight, 2.0)
            bad = torch.tensor([False, True, False, True, False, True, True], device=cuda)
            assert torch.equal(torch.isnan(out).all(1), bad) and bool(torch.isfinite(out[~bad]).all())
            dout = torch.randn(7, width, device=cuda).to(dtype)
            _check_grad(K.embedding_backward(tokens, dout, 10), tokens, dout, 10, 1.0, None)
    far = torch.tensor([2**40, 1], dtype=torch.int64, device=cuda)
    assert bool(torch.isnan(K.embedding_forward(far, weight)[0]).all())


def test_infinities_and_nan_stay_in_their_row(cuda):
    from elixir_b200 import kernels as K
    tokens = _tokens(3000, 200, 'zipf', torch.int64, 1).to(cuda)
    dout = torch.randn(3000, 40, device=cuda)
    clean = K.embedding_backward(tokens, dout, 200)
    dout[17, 3] = float('inf')
    dout[1800, 4] = float('nan')
    got = K.embedding_backward(tokens, dout, 200)
    changed = torch.zeros_like(got, dtype=torch.bool)
    changed[tokens[17], 3] = True
    changed[tokens[1800], 4] = True
    assert torch.equal(~torch.isfinite(got), changed) and torch.equal(got[~changed], clean[~changed])


def test_same_bits_every_time_from_any_stream_and_over_old_workspaces(cuda):
    from elixir_b200 import kernels as K
    tokens = _tokens(20000, 5000, 'zipf', torch.int64, 2).to(cuda)
    dout = torch.randn(20000, 200, device=cuda).half()
    first = K.embedding_backward(tokens, dout, 5000)
    side = torch.cuda.Stream(cuda)
    for k in range(4):
        torch.cuda.synchronize()
        with torch.cuda.stream(side if k % 2 else torch.cuda.current_stream(cuda)):
            junk = torch.full((1 << 22, ), 0xAB, dtype=torch.uint8, device=cuda)
            del junk    # the next workspace may hold it
            got = K.embedding_backward(tokens, dout, 5000)
        torch.cuda.synchronize()
        assert torch.equal(first, got)


def test_two_captured_graphs_replayed_at_once_with_new_tokens(cuda):
    from elixir_b200 import kernels as K
    n, vocab, width = 6000, 3000, 128
    sets = [(_tokens(n, vocab, 'zipf', torch.int64, s).to(cuda), torch.randn(n, width, device=cuda).half(),
             torch.randn(vocab, width, device=cuda).half()) for s in (0, 1)]
    graphs, outs = [], []
    for tokens, dout, weight in sets:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((K.embedding_forward(tokens, weight, 3.0), K.embedding_backward(tokens, dout, vocab, 3.0, 1)))
        graphs.append(g)
    streams = [torch.cuda.Stream(cuda) for _ in range(2)]
    for s, (tokens, _, _) in enumerate(sets):
        tokens.copy_(_tokens(n, vocab, 'few' if s else 'even', torch.int64, 7))
    torch.cuda.synchronize()
    for _ in range(4):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (tokens, dout, weight), got in zip(sets, outs):
        assert torch.equal(got[0], K.embedding_forward(tokens, weight, 3.0))
        assert torch.equal(got[1], K.embedding_backward(tokens, dout, vocab, 3.0, 1))


def test_more_than_two_to_the_31_elements(cuda):
    from elixir_b200 import kernels as K
    n, width, vocab = 2**31 // 4096 + 40, 4096, 50
    tokens = torch.zeros(n, dtype=torch.int32, device=cuda)
    tokens[-3:] = torch.tensor([7, 9, 7], dtype=torch.int32, device=cuda)
    weight = torch.randn(vocab, width, device=cuda).half()
    out = K.embedding_forward(tokens, weight)
    assert torch.equal(out[-3:], weight[[7, 9, 7]]) and torch.equal(out[n // 2], weight[0])
    out[:-3] = 0
    got = K.embedding_backward(tokens, out, vocab)
    want = torch.zeros_like(weight, dtype=torch.float64)
    want[7], want[9] = 2 * weight[7].double(), weight[9].double()
    assert torch.equal(got, want.half())


@pytest.mark.parametrize('dtype', [torch.float16, torch.float32])
def test_autograd(cuda, dtype):
    from elixir_b200 import functional as F
    tokens = torch.randint(30, (4, 9), generator=torch.Generator().manual_seed(0)).to(cuda)
    weight = torch.randn(30, 24, device=cuda).to(dtype).requires_grad_()
    out = F.embedding(tokens, weight, padding_idx=-1, scale=5.0)
    assert out.shape == (4, 9, 24)
    dout = torch.randn(out.shape, device=cuda).to(dtype)
    got, = torch.autograd.grad(out, weight, dout)
    _check_grad(got, tokens.view(-1), dout.view(-1, 24), 30, 5.0, 29)
    out.sum()    # and an expanded gradient, tokens that are not contiguous
    F.embedding(tokens.t(), weight, scale=2.0).sum().backward()
    counts = torch.bincount(tokens.view(-1), minlength=30).to(weight.dtype)
    assert torch.equal(weight.grad, (2 * counts)[:, None].expand(30, 24))
    # the function is linear in the table: a difference over any step is the slope (each of 864 products and the two
    # tables' sums rounds by half a step of the type)
    direction = torch.randn(30, 24, device=cuda).to(dtype)
    end = lambda w: (F.embedding(tokens, w, scale=5.0).double() * dout.double()).sum()    # noqa: E731
    slope = end((weight.detach() + direction)) - end(weight.detach())
    full, size = _want(tokens.view(-1), dout.view(-1, 24), 30, 5.0, None)
    off = 4 * torch.finfo(dtype).eps * float((size.to(cuda) * (weight.detach().double().abs() + direction.double().abs() + 1)).sum())
    assert abs(float(slope - (full.to(cuda) * direction.double()).sum())) <= off
