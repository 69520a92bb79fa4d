"""The 8-bit moment form and the update that uses it, restated from the definition in 64 bits (numpy only)."""
import numpy as np

BLOCK = 256


def _f32(x):
    return np.asarray(x, dtype=np.float64).astype(np.float32).astype(np.float64)


def round_up(n, m):
    return (n + m - 1) // m * m


def decode(state, n, signed):
    """Values (float64) of a state array (uint8) for a shard of n elements."""
    state = np.asarray(state, dtype=np.uint8).astype(np.int64)
    code = state[:n]
    exps = np.repeat(state[round_up(n, 16):round_up(n, 16) + (n + BLOCK - 1) // BLOCK], BLOCK)[:n]
    bias, mag = (15, code & 127) if signed else (31, code)
    field, t = mag >> 3, mag & 7
    value = np.where(field > 0, (1 + t / 8) * 2.0**(field - bias), t / 8 * 2.0**(1 - bias))
    value = value * 2.0**(exps - 127.0) * np.where(signed & (code >= 128), -1.0, 1.0)
    value = np.where(exps == 0, 0.0, value)
    return np.where(exps == 255, np.nan, value)


def encode(x, signed, up):
    """State array of the values x (fp32 numbers in float64); `up` in [0, 1): what is added, in units of the last kept
    bit, before the rest is dropped (0.5: to nearest)."""
    n = x.size
    blocks = (n + BLOCK - 1) // BLOCK
    state = np.zeros(round_up(n, 16) + round_up(blocks, 16), dtype=np.uint8)
    up = np.broadcast_to(up, x.shape)
    bias, top = (15, 127) if signed else (31, 255)
    for b in range(blocks):
        part = slice(b * BLOCK, min(n, (b + 1) * BLOCK))
        a, sign = np.abs(x[part]), np.where(np.signbit(x[part]) & signed, 128, 0)
        if not np.all(np.isfinite(a)):
            e, c = 255, None
        elif a.max() == 0:
            e, c = 0, np.zeros(a.size, dtype=np.int64)
        else:
            mant, p = np.frexp(a.max())    # mant in [0.5, 1)
            e = int(np.clip(p - 1 + 127 + (2 * mant > 1.875), 1, 253))
            y = a / 2.0**(e - 127)
            field = np.clip(np.frexp(np.where(y > 0, y, 1e-300))[1] - 1 + bias, 1, bias)
            unit = 2.0**(field - bias - 3.0)
            held = np.floor(y / unit * 2**20) / 2**20    # 23 bits of a binade are kept before the rounding
            c = np.floor(held + up[part]).astype(np.int64) + (field - 1) * 8
            c = np.minimum(c, top)
            if not signed:
                c = np.where(a > 0, np.maximum(c, 1), c)
        state[round_up(n, 16) + b] = e
        if c is not None:
            state[part] = c | sign
    return state


def _mix(x):
    x = x.astype(np.uint64) & 0xFFFFFFFF
    x = ((x ^ (x >> np.uint64(16))) * np.uint64(0x9E3779B1)) & np.uint64(0xFFFFFFFF)
    x = ((x ^ (x >> np.uint64(15))) * np.uint64(0x85157AF5)) & np.uint64(0xFFFFFFFF)
    return x ^ (x >> np.uint64(16))


def dither(step, index, n, first=0):
    """(first, second moment): what is added before dropping, in [0, 1), for elements [first, first + n)."""
    block, place = np.divmod(np.arange(first, first + n, dtype=np.uint64), np.uint64(BLOCK))
    key = np.array([(step * 0x632BE5AB + index * 0x9E3779B1 + 0x2545F491) & 0xFFFFFFFF], dtype=np.uint64)
    key = _mix(_mix(_mix(key) ^ (block & np.uint64(0xFFFFFFFF))) ^ (block >> np.uint64(32)))
    bits = _mix(key + place * np.uint64(0x9E3779B1))
    return (bits & np.uint64(0xFFFF)) / 65536.0, (bits >> np.uint64(16)) / 65536.0


def adam8(master, state_m, state_v, grad, segments, hypers, step, div, index=0):
    """One applied update of a shard.  segments: (begin, end, group).  Returns (master in float64, how far it moved,
    state_m, state_v); moments are fp32 numbers, each product and sum rounded."""
    n = master.size
    p = np.asarray(master, dtype=np.float64).copy()
    moved = np.zeros(n)
    m, v = decode(state_m, n, True), decode(state_v, n, False)
    touched = np.zeros((n + BLOCK - 1) // BLOCK, dtype=bool)
    with np.errstate(all='ignore'):
        for b, e, group in segments:
            h = hypers[group]
            s = slice(b, e)
            b1, b2, lr, eps, wd = (float(np.float32(x)) for x in (h.beta1, h.beta2, h.lr, h.eps, h.weight_decay))
            g = np.asarray(grad[s], dtype=np.float64)
            if div is not None and div != 1:
                g = _f32(g / float(np.float32(div)))
            if not h.adamw_mode:
                g = _f32(g + wd * p[s])
            m[s] = _f32(_f32(b1 * m[s]) + _f32(_f32(1 - b1) * g))
            v[s] = _f32(_f32(b2 * v[s]) + _f32(_f32(_f32(1 - b2) * g) * g))
            c1, c2 = (1 - b1**step, 1 - b2**step) if h.bias_correction else (1.0, 1.0)
            upd = m[s] / c1 / (np.sqrt(v[s] / c2) + eps) + (wd * p[s] if h.adamw_mode else 0.0)
            p[s] = p[s] - lr * upd
            moved[s] = np.abs(lr * upd) + np.abs(lr * wd * p[s])
            touched[b // BLOCK:(e + BLOCK - 1) // BLOCK] = True
    up_m, up_v = dither(step, index, n)
    new_m, new_v = encode(m, True, up_m), encode(v, False, up_v)
    keep = ~np.repeat(touched, BLOCK)[:n]
    first = round_up(n, 16)
    for new, old in ((new_m, state_m), (new_v, state_v)):
        old = np.asarray(old)
        new[:n][keep] = old[:n][keep]
        new[first:first + touched.size][~touched] = old[first:first + touched.size][~touched]
    return p, moved, new_m, new_v


def same_state(got, want, n, signed):
    """Codes and exponents equal; the codes of a block that is not finite do not matter, nor does the sign of a zero."""
    got, want = np.asarray(got), np.asarray(want)
    first, blocks = round_up(n, 16), (n + BLOCK - 1) // BLOCK
    if not np.array_equal(got[first:first + blocks], want[first:first + blocks]):
        return False
    free = np.repeat(want[first:first + blocks] == 255, BLOCK)[:n]
    if signed:
        free |= (got[:n] & 127 == 0) & (want[:n] & 127 == 0)
    return bool(np.all((got[:n] == want[:n]) | free))
