"""Plain 64-bit forms of the operators beside the projections (rotary positions, 8-bit key/value cache, attention, low-rank
adapters) on numpy arrays, and the error that each kernel may have, derived from its roundings."""
import numpy as np

HALF16 = 2.0 ** -11  # half a step of binary16, relative
TINY16 = 2.0 ** -25  # half a step of its smallest numbers
STEP32 = 2.0 ** -24
BLOCK = 64


def rotate(t, positions, frequencies, factor, layout, sign=1):
    """t [tokens, heads, dim] -> (turned in 64 bits, allowed error of one rounding to binary16 behind binary32 arithmetic)."""
    t = t.astype(np.float64)
    half = len(frequencies)
    one = np.arange(half) * (2 if layout == "interleaved" else 1)
    two = one + (1 if layout == "interleaved" else half)
    angle = np.outer(np.asarray(positions, np.float64), frequencies)[:, None]
    c, s = np.cos(angle) * factor, sign * np.sin(angle) * factor
    out, room = t.copy(), np.zeros_like(t)
    out[..., one] = t[..., one] * c - t[..., two] * s
    out[..., two] = t[..., one] * s + t[..., two] * c
    # sine and cosine to 2 units in the last place of an angle of 2^-25 turns, two products and a sum: 8 half steps in all
    room[..., one] = room[..., two] = 2 * np.pi * 8 * STEP32 * factor * (np.abs(t[..., one]) + np.abs(t[..., two]))
    return out, HALF16 * np.abs(out) + room * 1.001 + TINY16


class PlainCache:
    """Codes and scales of one cache, stored token by token as the definition says (binary32 arithmetic, correctly rounded)."""

    def __init__(self, n_blocks, heads, dim):
        self.codes = [np.zeros((n_blocks, heads, BLOCK, dim), np.int32) for _ in range(2)]
        self.scale = [np.zeros((n_blocks, heads), np.float32) for _ in range(2)]

    def append(self, k, v, offsets, lengths, table):
        for b, length in enumerate(lengths):
            count = offsets[b + 1] - offsets[b]
            first = length - count
            p = max(first, 0)
            while p < length:
                end = min(length, (p // BLOCK + 1) * BLOCK)
                block = table[b][p // BLOCK]
                rows = slice(offsets[b] + p - first, offsets[b] + end - first)
                if 0 <= block < len(self.scale[0]):
                    for i, x in enumerate((k, v)):
                        self._store(i, block, p % BLOCK, x[rows].astype(np.float32))
                p = end

    def _store(self, i, block, slot, x):
        for h in range(x.shape[1]):
            codes, t = self.codes[i][block, h], x[:, h]
            need = np.float32(np.abs(t).max() / np.float32(127))
            old = self.scale[i][block, h] if slot else np.float32(0)
            scale = old
            if need > old:
                scale = need
                if old > 0:
                    e = 0
                    while np.ldexp(old, e) < need:
                        e += 1
                    scale = np.ldexp(old, e)
                    codes[:slot] = np.rint(codes[:slot] * 2.0 ** -e)
            self.scale[i][block, h] = scale
            q = np.rint(t / scale) if scale > 0 else np.zeros_like(t)
            codes[slot:slot + len(t)] = np.clip(q, -127, 127)

    def values(self, i, b, length, table):
        """[length, heads, dim] in 64 bits."""
        rows = [self.codes[i][table[b][p]] * self.scale[i][table[b][p]].astype(np.float64)[:, None, None]
                for p in range(-(-length // BLOCK))]
        heads, dim = self.codes[i].shape[1], self.codes[i].shape[3]
        return np.concatenate(rows, 1).transpose(1, 0, 2)[:length] if rows else np.zeros((0, heads, dim))


def attend(q, k, v, first, scale, there=None):
    """q [rows, q_heads, dim], k and v [tokens, kv_heads, dim] -> (out, allowed error).  Row i is at position first + i."""
    q, out = q.astype(np.float64), np.zeros(q.shape)
    room = np.full(q.shape, TINY16)
    group, dim = q.shape[1] // k.shape[1], q.shape[2]
    there = np.ones(len(k), bool) if there is None else there
    for i in range(len(q)):
        seen = np.flatnonzero((np.arange(len(k)) <= first + i) & there)
        if not len(seen):
            continue
        for h in range(q.shape[1]):
            kk, vv = k[seen, h // group], v[seen, h // group]
            s = scale * (kk @ q[i, h])
            p = np.exp(s - s.max())
            p /= p.sum()
            out[i, h] = p @ vv
            # scores: products summed in binary32 (no chain longer than dim + 8), times a factor that is rounded twice
            wrong = (dim + 12) * STEP32 * scale * (np.abs(kk) @ np.abs(q[i, h])).max() + 4 * STEP32
            # a probability: its score's error in numerator and sum, binary16 (also of the smallest), binary32 sums
            each = np.expm1(2 * wrong) + HALF16 + (len(seen) + 16) * STEP32
            room[i, h] += HALF16 * np.abs(out[i, h]) + each * (p @ np.abs(vv)) + len(seen) * TINY16 * np.abs(vv).max(0)
    return out, room * 1.001


def adapt(x, y, down, up, scaling, ids, activation=None):
    """(act(y + scaling (x down^T) up^T), allowed error)."""
    x, out = x.astype(np.float64), y.astype(np.float64).copy()
    down, up = down.astype(np.float64), up.astype(np.float64)
    size = np.zeros_like(out)
    for a in range(len(down)):
        r = ids == a
        out[r] += scaling[a] * ((x[r] @ down[a].T) @ up[a].T)
        size[r] = np.abs(scaling[a]) * ((np.abs(x[r]) @ np.abs(down[a]).T) @ np.abs(up[a]).T)
    room = size * product_error(down.shape[2], down.shape[1]) + 2 * STEP32 * np.abs(out)
    if activation == "relu":
        out = np.maximum(out, 0)
    elif activation == "gelu_tanh":
        # slope at most 1.13; binary32 evaluation: a few units of 1 + tanh, which may cancel against |v| up to 5.6
        room = 1.13 * room + 16 * STEP32 * np.minimum(np.abs(out), 6) + 4 * STEP32 * np.abs(out)
        out = 0.5 * out * (1 + np.tanh(np.sqrt(2 / np.pi) * (out + 0.044715 * out ** 3)))
    return out, (room + HALF16 * np.abs(out)) * 1.001 + TINY16


def product_error(*lengths):
    """Relative to the sum of magnitudes: binary32 sums of chained products of these lengths (32 products at a time, then the
    chain of those, partial sums of at most 64), and 2^-20 for the intermediate in two binary16 numbers."""
    return sum(32 + n / 32 + 64 for n in lengths) * STEP32 + 2.0 ** -20


def adapt_grad(x, dy, dx, down, up, scaling, ids):
    """((dx, d_down, d_up), allowed errors)."""
    x, dy = x.astype(np.float64), dy.astype(np.float64)
    down, up = down.astype(np.float64), up.astype(np.float64)
    dx, d_down, d_up = dx.astype(np.float64).copy(), np.zeros_like(down), np.zeros_like(up)
    rooms = [np.zeros_like(t) for t in (dx, d_down, d_up)]
    for a in range(len(down)):
        r = ids == a
        if not r.any():
            continue
        s, n = scaling[a], r.sum()
        dv, v = dy[r] @ up[a], x[r] @ down[a].T
        big_dv, big_v = np.abs(dy[r]) @ np.abs(up[a]), np.abs(x[r]) @ np.abs(down[a]).T
        dx[r] += s * dv @ down[a]
        d_down[a], d_up[a] = s * dv.T @ x[r], s * dy[r].T @ v
        k, m, rank = down.shape[2], up.shape[1], down.shape[1]
        rooms[0][r] = np.abs(s) * (big_dv @ np.abs(down[a])) * product_error(m, rank)
        # (what the two binary16 numbers lose is relative to the largest of the 512 rows that are scaled together)
        top_dv, top_v = np.broadcast_to(big_dv.max(), dv.shape), np.broadcast_to(big_v.max(), v.shape)
        rooms[1][a] = np.abs(s) * (big_dv.T @ np.abs(x[r]) * product_error(m, n) + top_dv.T @ np.abs(x[r]) * 2.0 ** -22)
        rooms[2][a] = np.abs(s) * (np.abs(dy[r]).T @ big_v * product_error(k, n) + np.abs(dy[r]).T @ top_v * 2.0 ** -22)
    rooms[0] = (rooms[0] + (HALF16 + 2 * STEP32) * np.abs(dx)) * 1.001 + TINY16
    return (dx, d_down, d_up), [rooms[0], rooms[1] * 1.001 + 1e-30, rooms[2] * 1.001 + 1e-30]


def assert_within(got, want, room, what=""):
    got = np.asarray(got, dtype=np.float64)
    assert got.shape == want.shape, f"{what}: shape {got.shape} != {want.shape}"
    assert np.isfinite(got).all(), f"{what}: {int((~np.isfinite(got)).sum())} values are not finite"
    over = np.abs(got - want) - room
    assert (over <= 0).all(), (f"{what}: {int((over > 0).sum())} of {got.size} values outside, worst at "
                               f"{np.unravel_index(over.argmax(), over.shape)}: {np.abs(got - want).flat[over.argmax()]:.3g} of {room.flat[over.argmax()]:.3g}")
