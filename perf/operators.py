"""Work that the operators of a training step are timed and compared on: AdamW with both moments in 8 bits over many
chunk shards, packing and unpacking of those moments, layer norm with its backward pass, and the scaled embedding
lookup with its gradient.

``listed()`` gives the cases, ``draw()`` more of the same ranges, ``prepare()`` a case's inputs on the GPU, ``run()``
one pass: through the framework where ``own`` is true, in elementary torch operations otherwise.  ``exact()`` is the
operator's definition in 64 bits and ``work()`` what a pass cannot do without.
"""
import math

import torch

own = False

DEVICE = 'cuda'
BLOCK = 256    # elements that share one exponent byte in the 8-bit moment state
# per 8-bit code: the power of two that moves a value's leading bits onto an fp32 exponent of 15 (signed moment,
# 4 exponent bits) or 31 (unsigned moment, 5 exponent bits), and the largest magnitude code
SIGNED, UNSIGNED = (112, 127), (96, 255)
BETAS, EPS, LR, STEP = (0.9, 0.999), 1e-8, (1e-4, 3e-4), 99
WEIGHT_DECAY = (0.01, 0.0)    # the two parameter groups of every shard: weights, then biases and norms
DTYPES = ('float16', 'bfloat16', 'float32')


# ---------------------------------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------------------------------


def listed():
    return [
        # the update of a very small model (three ragged shards of one tile): launch latency
        dict(name='adam8_tiny', op='adam8', dtype='bfloat16', shards=3, elems=4099, scale=1.0),
        # fp32 gradients with a divisor that is not a power of two (a clipped step), odd shard sizes
        dict(name='adam8_fp32_odd', op='adam8', dtype='float32', shards=3, elems=4194301, scale=6963.2),
        # a sixth of the GPT-2-XL chunk set: fp16 chunks of 32 Mi elements under a loss scale
        dict(name='adam8_gpt2xl', op='adam8', dtype='float16', shards=8, elems=33554432, scale=65536.0),
        # one small shard's moments into a checkpoint and back
        dict(name='moments_small', op='moments', elems=100003),
        # a full chunk shard's
        dict(name='moments_chunk', op='moments', elems=67108864),
        # a single token of GPT-2-XL's width
        dict(name='norm_token', op='norm', dtype='bfloat16', rows=1, cols=1600, affine='both', train=False),
        # an evaluation batch of 2048 tokens of the OPT-13B width
        dict(name='norm_eval_5120', op='norm', dtype='float16', rows=2048, cols=5120, affine='both', train=False),
        # a training micro-batch of GPT-2-XL: 8 x 1024 tokens
        dict(name='norm_train_gpt2xl', op='norm', dtype='float16', rows=8192, cols=1600, affine='both', train=True),
        # odd sizes in fp32, no bias
        dict(name='norm_train_odd', op='norm', dtype='float32', rows=1023, cols=1111, affine='weight', train=True),
        # a single token looked up
        dict(name='embed_token', op='embed', dtype='float16', tokens=1, vocab=50257, width=1600, index='int64',
             spread='zipf', padding=-1, scale=1.0, train=False),
        # the GPT-2-XL vocabulary and its micro-batch: lookup and gradient
        dict(name='embed_train_gpt2xl', op='embed', dtype='float16', tokens=8192, vocab=50257, width=1600, index='int64',
             spread='zipf', padding=-1, scale=1.0, train=True),
        # the OPT-13B vocabulary, 8 x 2048 tokens, with a padding token and a scale
        dict(name='embed_train_opt', op='embed', dtype='bfloat16', tokens=16384, vocab=50272, width=5120, index='int32',
             spread='zipf', padding=1, scale=8.0, train=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(('adam8', 'adam8', 'moments', 'norm', 'norm', 'embed', 'embed'))
    if op == 'adam8':
        shards = rng.randint(1, 12)
        return dict(op=op, dtype=rng.choice(DTYPES), shards=shards, elems=_log(rng, 300, 200_000_000 // shards),
                    scale=rng.choice((1.0, 65536.0, 6963.2)))
    if op == 'moments':
        return dict(op=op, elems=_log(rng, 1, 67_000_000))
    if op == 'norm':
        cols = _log(rng, 32, 12288)
        return dict(op=op, dtype=rng.choice(DTYPES), rows=_log(rng, 1, min(16384, 40_000_000 // cols)), cols=cols,
                    affine=rng.choice(('both', 'weight', 'none')), train=rng.random() < 0.6)
    width, vocab = _log(rng, 16, 5120), _log(rng, 100, 50272)
    return dict(op=op, dtype=rng.choice(DTYPES[:2]) if width * vocab > 50_000_000 else rng.choice(DTYPES),
                tokens=_log(rng, 1, min(32768, 80_000_000 // width)), vocab=vocab, width=width,
                index=rng.choice(('int32', 'int64')), spread=rng.choice(('zipf', 'zipf', 'even', 'one')),
                padding=rng.choice((-1, 0, 1)), scale=rng.choice((1.0, math.sqrt(width))), train=rng.random() < 0.7)


def _dtype(case):
    return getattr(torch, case['dtype'])


def _valid(case, i):
    """Used elements of shard i: a few short of its size, the last shard much shorter."""
    n = case['elems']
    return max(1, int(0.6 * n)) if i == case['shards'] - 1 else n - (17 * i) % 61


def _distinct(case):
    """How many different tokens a case is expected to hold."""
    if case['spread'] == 'one':
        return 1
    often = torch.ones(case['vocab'], dtype=torch.float64)
    if case['spread'] == 'zipf':
        often = 1 / (2.7 + torch.arange(case['vocab'], dtype=torch.float64))
    return float((1 - (1 - often / often.sum())**case['tokens']).sum())


def work(case):
    if case['op'] == 'adam8':
        # in: gradient, master, two codes; out: master, two codes, working copy, and the two moments as 16-bit values
        size = 2 if case['dtype'] != 'float32' else 4
        n = case['shards'] * case['elems']
        return dict(bytes=n * (2 * size + 12 + 4 + 4 / BLOCK), flops=25 * n)
    if case['op'] == 'moments':
        # in: two fp32 moments; out: two codes and two fp32 moments
        return dict(bytes=case['elems'] * (8 + 2 + 8 + 2 / BLOCK), flops=10 * case['elems'])
    if case['op'] == 'norm':
        size = 2 if case['dtype'] != 'float32' else 4
        n = case['rows'] * case['cols']
        small = 2 * case['cols'] * size + 8 * case['rows']
        forward = dict(bytes=2 * n * size + small, flops=8 * n)
        if not case['train']:
            return forward
        return dict(bytes=forward['bytes'] + 2 * n * size + small, flops=forward['flops'] + 14 * n)
    size = 2 if case['dtype'] != 'float32' else 4
    n = case['tokens'] * case['width']
    rows = _distinct(case) * case['width']    # rows of the table that are looked at
    index = case['tokens'] * (4 if case['index'] == 'int32' else 8)
    forward = dict(bytes=(rows + n) * size + index, flops=n)
    if not case['train']:
        return forward
    return dict(bytes=forward['bytes'] + (n + case['vocab'] * case['width']) * size, flops=3 * n)


# ---------------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------------


def _inputs(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    if case['op'] == 'adam8':
        n, dtype = case['elems'], _dtype(case)
        shards = []
        for i in range(case['shards']):
            # gradients whose size differs from row to row over several orders, a tenth of the rows without any
            size = torch.exp(1.5 * normal(n // 64 + 1)) * (torch.rand(n // 64 + 1, generator=gen, device=DEVICE) > 0.1)
            size = (1e-4 * size).repeat_interleave(64)[:n]
            grad = normal(n).mul_(size).mul_(case['scale']).clamp_(-6e4, 6e4).to(dtype)
            m, v = normal(n).mul_(size).mul_(0.3), normal(n).square_().add_(0.1).mul_(size).mul_(size)
            valid = _valid(case, i)
            for t in (m, v, grad):
                t[valid:] = 0
            state_m, state_v = _pack(m, SIGNED), _pack(v, UNSIGNED)
            master = normal(n).mul_(0.02)
            shards.append(dict(master=master, lowp=master.to(dtype), grad=grad, m=state_m, v=state_v, valid=valid,
                               split=valid * 2 // 3))
        return dict(shards=shards)
    if case['op'] == 'moments':
        n = case['elems']
        size = (1e-4 * torch.exp(1.5 * normal(n // 64 + 1))).repeat_interleave(64)[:n]
        return dict(m=normal(n).mul_(size), v=normal(n).square_().mul_(size).mul_(size))
    if case['op'] == 'norm':
        rows, cols, dtype = case['rows'], case['cols'], _dtype(case)
        # a residual stream: an offset per row, and channels of different size with a few large ones
        channel = torch.exp(0.5 * normal(cols)) * (1 + 15 * (torch.rand(cols, generator=gen, device=DEVICE) > 0.99))
        x = (normal(rows, cols) * channel + 0.2 + 0.3 * normal(rows, 1)).to(dtype)
        s = dict(x=x, weight=None, bias=None)
        if case['affine'] != 'none':
            s['weight'] = (1 + 0.1 * normal(cols)).to(dtype)
        if case['affine'] == 'both':
            s['bias'] = (0.1 * normal(cols)).to(dtype)
        if case['train']:
            s['dy'] = (normal(rows, cols) * 0.1).to(dtype)
        return s
    tokens, vocab, width, dtype = case['tokens'], case['vocab'], case['width'], _dtype(case)
    if case['spread'] == 'one':
        token = torch.randint(vocab, (1, ), generator=gen, device=DEVICE).expand(tokens)
    elif case['spread'] == 'even':
        token = torch.randint(vocab, (tokens, ), generator=gen, device=DEVICE)
    else:
        # the r-th most frequent token about as often as 1 / (2.7 + r), element by element: no running sum, whose order
        # (and with it a token here and there) could differ between two preparations
        rank = 2.7 * ((1 + vocab / 2.7)**torch.rand(tokens, generator=gen, device=DEVICE, dtype=torch.float64) - 1)
        token = torch.randperm(vocab, generator=gen, device=DEVICE)[rank.long().clamp(max=vocab - 1)]
    s = dict(token=token.to(getattr(torch, case['index'])).contiguous(), weight=(normal(vocab, width) * 0.02).to(dtype))
    if case['train']:
        s['dout'] = (normal(tokens, width) * 0.1).to(dtype)
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    s['case'] = case
    if case['op'] == 'adam8':
        s['step'] = STEP
        s['divisor'] = torch.tensor(case['scale'], device=DEVICE)
        for d in s['shards']:    # where the moments are read out to
            d['m_out'], d['v_out'] = (torch.empty(case['elems'], dtype=torch.bfloat16, device=DEVICE) for _ in range(2))
        if own:    # the tables and the control block that a training program builds once
            from elixir_b200 import kernels
            from elixir_b200.engine import ChunkStepEngine
            from elixir_b200.scaler import ConstantGradScaler
            engine = ChunkStepEngine(torch.device(DEVICE, torch.cuda.current_device()), _dtype(case),
                                     ConstantGradScaler(case['scale']), state_bits=8)
            for d in s['shards']:
                engine.add_shard(d['master'], d['lowp'], d['valid'], [(a, b, g) for a, b, g in
                                                                      ((0, d['split'], 0), (d['split'], d['valid'], 1)) if a < b],
                                 exp_avg=d['m'], exp_avg_sq=d['v'], grad_src=d['grad'])
            engine.finalize()
            engine.set_hyper([kernels.hyper(lr=lr, betas=BETAS, eps=EPS, weight_decay=wd) for lr, wd in zip(LR, WEIGHT_DECAY)])
            engine.scaler.load_state_dict(dict(scale=case['scale'], step=STEP))
            s['engine'] = engine
    return s


# ---------------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------------


def run(state):
    return {'adam8': _run_adam8, 'moments': _run_moments, 'norm': _run_norm, 'embed': _run_embed}[state['case']['op']](state)


def _run_adam8(s):
    if own:
        from elixir_b200 import kernels
        s['engine'].step()
        for d in s['shards']:
            kernels.unpack_moments(d['m'], d['v'], d['m_out'], d['v_out'])
    else:
        s['step'] += 1
        for index, d in enumerate(s['shards']):
            _adam8_plain(d, index, s['step'], s['divisor'])
    return {k: [d[k] for d in s['shards']] for k in ('master', 'lowp', 'm_out', 'v_out')}


def _run_moments(s):
    m, v = s['m'], s['v']
    if own:
        from elixir_b200 import kernels
        state_m, state_v = kernels.pack_moments(m, v)
        m_out, v_out = torch.empty_like(m), torch.empty_like(v)
        kernels.unpack_moments(state_m, state_v, m_out, v_out)
        return dict(m=m_out, v=v_out)
    n = m.numel()
    return dict(m=_unpack(_pack(m, SIGNED), n, SIGNED), v=_unpack(_pack(v, UNSIGNED), n, UNSIGNED))


def _run_norm(s):
    x, weight, bias = s['x'], s['weight'], s['bias']
    if own:
        from elixir_b200 import kernels
        y, mean, rstd = kernels.layer_norm_forward(x, weight, bias, 1e-5)
        out = dict(y=y, mean=mean, rstd=rstd)
        if 'dy' in s:
            dx, dw, db = kernels.layer_norm_backward(s['dy'], x, weight, mean, rstd, bias_grad=bias is not None)
            out.update(dx=dx, dw=dw, db=db)
        return out
    x32 = x.float()
    mean = x32.mean(1)
    d = x32 - mean[:, None]
    rstd = 1 / torch.sqrt(d.square().mean(1) + 1e-5)
    xhat = d * rstd[:, None]
    y = xhat if weight is None else xhat * weight.float()
    y = y if bias is None else y + bias.float()
    out = dict(y=y.to(x.dtype), mean=mean, rstd=rstd)
    if 'dy' in s:
        dy = s['dy'].float()
        a = dy if weight is None else dy * weight.float()
        dx = rstd[:, None] * (a - a.mean(1, keepdim=True) - xhat * (a * xhat).mean(1, keepdim=True))
        out['dx'] = dx.to(x.dtype)
        out['dw'] = None if weight is None else (dy * xhat).sum(0).to(x.dtype)
        out['db'] = None if bias is None else dy.sum(0).to(x.dtype)
    return out


def _run_embed(s):
    case, token, weight = s['case'], s['token'], s['weight']
    padding = case['padding'] if case['padding'] >= 0 else None
    if own:
        from elixir_b200 import kernels
        out = dict(out=kernels.embedding_forward(token, weight, scale=case['scale']))
        if 'dout' in s:
            out['dweight'] = kernels.embedding_backward(token, s['dout'], case['vocab'], scale=case['scale'], padding_idx=padding)
        return out
    out = dict(out=(weight[token].float() * case['scale']).to(weight.dtype))
    if 'dout' in s:
        dout = s['dout'].float() * case['scale']
        if padding is not None:
            dout = dout * (token != padding)[:, None]
        total = torch.zeros(weight.shape, device=DEVICE).index_add_(0, token, dout)
        out['dweight'] = total.to(weight.dtype)
    return out


# ---------------------------------------------------------------------------------------------------
# the 8-bit moment state in elementary operations
#
# A shard of n elements: n codes, then (from the next multiple of 16) one exponent byte E per block of 256 elements.
# A code holds a small float relative to 2^(E - 127): sign, 4 exponent and 3 mantissa bits for the first moment, 5
# exponent and 3 mantissa bits for the second.  E is chosen so that no rounding passes the largest code.
# ---------------------------------------------------------------------------------------------------


def _round_up(n, m):
    return (n + m - 1) // m * m


def _as_blocks(x):
    n = x.numel()
    whole = torch.zeros(_round_up(n, BLOCK), dtype=x.dtype, device=x.device)
    whole[:n] = x
    return whole.view(-1, BLOCK)


def _exponents(x):
    """x: fp32 [blocks, 256] -> int32 [blocks, 1]."""
    top = x.abs().amax(1, keepdim=True).view(torch.int32)
    e = ((top + 0xFFFFF) >> 23).clamp(1, 253)
    e = torch.where(top == 0, torch.zeros_like(e), e)
    return torch.where(top >= 0x7F800000, torch.full_like(e, 255), e)


def _encode(x, kind, dither):
    """x: fp32 [blocks, 256]; dither: what is added below the kept bits -> (codes, exponents), int32."""
    down, largest = kind
    e = _exponents(x)
    y = x.abs() * ((254 - e.clamp(1, 253)) << 23).view(torch.float32)
    c = ((y * 2.0**-down).view(torch.int32) + dither) >> 20
    c = c.clamp(max=largest)
    if kind is SIGNED:
        c = c | ((x.view(torch.int32) >> 24) & 0x80)
    else:
        c = torch.where(x > 0, c.clamp(min=1), c)
    return c, e


def _decode(c, e, kind):
    down, largest = kind
    scale = torch.where(e == 255, torch.full_like(e, 0x7FC00000), e << 23).view(torch.float32)
    x = ((c & largest) << 20).view(torch.float32) * 2.0**down * scale
    return torch.where(c > largest, -x, x)


def _store(c, e, n):
    state = torch.zeros(_round_up(n, 16) + _round_up(e.numel(), 16), dtype=torch.uint8, device=c.device)
    state[:n] = c.view(-1)[:n].to(torch.uint8)
    first = _round_up(n, 16)
    state[first:first + e.numel()] = e.view(-1).to(torch.uint8)
    return state


def _load(state, n):
    blocks, first = (n + BLOCK - 1) // BLOCK, _round_up(n, 16)
    return _as_blocks(state[:n].int()), state[first:first + blocks].int().view(-1, 1)


def _pack(x, kind):
    return _store(*_encode(_as_blocks(x), kind, 0x80000), x.numel())


def _unpack(state, n, kind):
    return _decode(*_load(state, n), kind).view(-1)[:n]


def _mix(x):
    x = x & 0xFFFFFFFF
    x = ((x ^ (x >> 16)) * 0x9E3779B1) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x85157AF5) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dither(step, index, blocks):
    """32 bits for each element of a shard from the step, the shard's index, the block and the place in it."""
    block = torch.arange(blocks, device=DEVICE)[:, None]
    key = _mix(torch.tensor(step * 0x632BE5AB + index * 0x9E3779B1, device=DEVICE) + 0x2545F491)
    key = _mix(_mix(key ^ (block & 0xFFFFFFFF)) ^ (block >> 32))
    return _mix(key + torch.arange(BLOCK, device=DEVICE) * 0x9E3779B1)


def _f32(value):
    return torch.tensor(value, dtype=torch.float32).item()


def _adam8_plain(d, index, step, divisor):
    n, dtype = d['master'].numel(), d['lowp'].dtype
    beta1, beta2 = _f32(BETAS[0]), _f32(BETAS[1])
    rest1, rest2 = _f32(1 - beta1), _f32(1 - beta2)
    (cm, em), (cv, ev) = _load(d['m'], n), _load(d['v'], n)
    m, v = _decode(cm, em, SIGNED), _decode(cv, ev, UNSIGNED)
    g, p = _as_blocks(d['grad'].float() / divisor), _as_blocks(d['master'])
    place = torch.arange(m.numel(), device=DEVICE).view_as(m)
    used, decayed = place < d['valid'], place < d['split']
    # the moments are fp32 numbers, every product and sum rounded once: which code they get hangs on their last bits
    m_new, v_new = m * beta1 + g * rest1, v * beta2 + (g * rest2) * g
    lr = torch.where(decayed, _f32(LR[0]), _f32(LR[1]))
    decay = torch.where(decayed, _f32(WEIGHT_DECAY[0]), _f32(WEIGHT_DECAY[1]))
    move = (m_new / (1 - beta1**step)) / (torch.sqrt(v_new / (1 - beta2**step)) + _f32(EPS)) + decay * p
    p = torch.where(used, p - lr * move, p)
    m, v = torch.where(used, m_new, m), torch.where(used, v_new, v)
    bits = _dither(step, index, m.shape[0])
    cm, em = _encode(m, SIGNED, ((bits & 0xFFFF) << 4).int())
    cv, ev = _encode(v, UNSIGNED, ((bits >> 16) << 4).int())
    d['m'].copy_(_store(cm, em, n))
    d['v'].copy_(_store(cv, ev, n))
    d['master'].copy_(p.view(-1)[:n])
    d['lowp'].copy_(d['master'])
    d['m_out'].copy_(_decode(cm, em, SIGNED).view(-1)[:n])
    d['v_out'].copy_(_decode(cv, ev, UNSIGNED).view(-1)[:n])


# ---------------------------------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------------------------------


def exact(case, seed):
    s = _inputs(case, seed)
    return {'adam8': _exact_adam8, 'moments': _exact_moments, 'norm': _exact_norm, 'embed': _exact_embed}[case['op']](case, s)


def _rounded(x):
    """The 32-bit number next to x, in 64 bits."""
    return x.float().double()


def _held(x, exponent_bits, dither):
    """What the 8-bit state holds for the values x (64 bits) of whole blocks: `exponent_bits` of exponent and 3 of
    mantissa below the block's power of two; `dither` in [0, 1) decides between the two neighbours."""
    size = x.abs()
    top = size.amax(1, keepdim=True)
    power = torch.where(top > 0, torch.floor(torch.log2(top.clamp(min=2.0**-126))), torch.zeros_like(top))
    power = torch.where(top > torch.exp2(power) * 2, power + 1, power)    # log2 may round across a power of two
    power = torch.where(top < torch.exp2(power), power - 1, power).clamp(min=-126)
    power = torch.where(top > 1.875 * torch.exp2(power), power + 1, power)
    lowest = power - (2**exponent_bits - 2)
    mine = torch.maximum(torch.floor(torch.log2(size.clamp(min=1e-300))), lowest)
    mine = torch.where(torch.exp2(mine) > size, torch.maximum(mine - 1, lowest), mine)
    mine = torch.where(torch.exp2(mine + 1) <= size, mine + 1, mine)
    step = torch.exp2(mine - 3)
    held = torch.floor(size / step + dither) * step
    if exponent_bits == 5:
        held = torch.where((size > 0) & (held == 0), torch.exp2(lowest - 3).expand_as(held), held)
    return torch.sign(x) * held


def _values(state, n, exponent_bits):
    """The values that an 8-bit state stands for, in 64 bits."""
    code, at = state[:n].long(), _round_up(n, 16)
    power = state[at:at + (n + BLOCK - 1) // BLOCK].double().repeat_interleave(BLOCK)[:n] - 127
    sign = 1.0
    if exponent_bits == 4:
        sign, code = 1 - 2 * (code >> 7).double(), code & 127
    field, mantissa = (code >> 3).double(), (code & 7).double()
    value = torch.where(field > 0, 1 + mantissa / 8, mantissa / 8) * torch.exp2(torch.clamp(field, min=1) - 2**exponent_bits + 1)
    return torch.where(power > -127, sign * value * torch.exp2(power), torch.zeros_like(value))


def _exact_adam8(case, s):
    out = dict(master=[], lowp=[], m_out=[], v_out=[])
    n, t = case['elems'], STEP + 1
    b1, b2 = _f32(BETAS[0]), _f32(BETAS[1])
    place = torch.arange(n, device=DEVICE)
    for index, d in enumerate(s['shards']):
        used, group = place < d['valid'], (place >= d['split']).long()
        lr, decay = (torch.tensor([_f32(v) for v in pair], dtype=torch.float64, device=DEVICE)[group] for pair in (LR, WEIGHT_DECAY))
        m, v, p = _values(d['m'], n, 4), _values(d['v'], n, 5), d['master'].double()
        # a code is chosen from the moment as an fp32 number, so its roundings belong to the definition
        g = _rounded(d['grad'].double() / _f32(case['scale']))
        m = torch.where(used, _rounded(_rounded(b1 * m) + _rounded(_f32(1 - b1) * g)), m)
        v = torch.where(used, _rounded(_rounded(b2 * v) + _rounded(_rounded(_f32(1 - b2) * g) * g)), v)
        p = torch.where(used, p - lr * ((m / (1 - b1**t)) / (torch.sqrt(v / (1 - b2**t)) + _f32(EPS)) + decay * p), p)
        bits = _dither(t, index, (n + BLOCK - 1) // BLOCK)
        out['master'].append(p)
        out['lowp'].append(p)
        out['m_out'].append(_held(_as_blocks(m), 4, (bits & 0xFFFF) / 65536.0).view(-1)[:n])
        out['v_out'].append(_held(_as_blocks(v), 5, (bits >> 16) / 65536.0).view(-1)[:n])
    return out


def _exact_moments(case, s):
    n = case['elems']
    return dict(m=_held(_as_blocks(s['m'].double()), 4, 0.5).view(-1)[:n], v=_held(_as_blocks(s['v'].double()), 5, 0.5).view(-1)[:n])


def _exact_norm(case, s):
    x, cols = s['x'].double(), case['cols']
    weight = torch.ones(cols, dtype=torch.float64, device=DEVICE) if s['weight'] is None else s['weight'].double()
    mean = x.sum(1) / cols
    var = (x - mean[:, None]).pow(2).sum(1) / cols
    std = (var + 1e-5).sqrt()
    normed = (x - mean[:, None]) / std[:, None]
    y = normed * weight + (0 if s['bias'] is None else s['bias'].double())
    out = dict(y=y, mean=mean, rstd=1 / std)
    if 'dy' in s:
        dy = s['dy'].double()
        a = weight * dy
        along = torch.einsum('rc,rc->r', a, normed)[:, None]
        out['dx'] = (cols * a - a.sum(1, keepdim=True) - normed * along) / (cols * std[:, None])
        out['dw'] = None if s['weight'] is None else torch.einsum('rc,rc->c', dy, normed)
        out['db'] = None if s['bias'] is None else dy.sum(0)
    return out


def _exact_embed(case, s):
    token = s['token'].long()
    out = dict(out=case['scale'] * torch.index_select(s['weight'].double(), 0, token))
    if 'dout' in s:
        kept = torch.nonzero(token != case['padding']).view(-1)
        order = kept[torch.argsort(token[kept], stable=True)]
        total = torch.zeros(case['vocab'], case['width'], dtype=torch.float64, device=DEVICE)
        total.index_add_(0, token[order], s['dout'][order].double())
        out['dweight'] = case['scale'] * total
    return out
